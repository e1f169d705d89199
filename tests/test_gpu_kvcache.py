"""The paged key/value cache (kvcache.PagedKV) on the GPU against plain 64-bit restatements of each operator (kv_reference.py).

Tolerances count roundings, u = eps / 2 of a type (bf16 2^-8, fp32 2^-24):
  append  the head norm's sum (14 additions deep), mean, root, quotient, weight and the rotation's three operations are under 32
          fp32 roundings of numbers no larger than |a| + |b| of the rotated pair; storing rounds once more.
  attend  bf16: one rounding of the output, one of each probability (averaged by the weights they are: u times the weighted mean of
          |v|); 4 bits: the probability times its step is what is rounded.  fp32: a score is off by at most (D + 4) u sum |q k| scale, and a
          relative error of e^score follows; sums of N terms add N u.  4 bits also subtracts 136 times a sum: 144 u per value."""
import math

import pytest
import torch

from kv_reference import Pages, attention, norm_rotate

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
ACT = {"f32": torch.float32, "bf16": torch.bfloat16, "int4": torch.bfloat16}


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=DEV).to(dtype)


def _cache(dtype, G, D, ps, lens, rows=None, spare=3, layers=1, seed=0, width=None):
    """A cache whose rows hold `lens` tokens on shuffled pages, every place filled with NaN."""
    from qwen3_tts_amd.kvcache import PagedKV
    n = [-(-x // ps) for x in lens]
    width = max(n) + 2 if width is None else width
    kv = PagedKV(layers, G, D, sum(n) + spare, ps, rows or len(lens), width, dtype, DEV)
    order = torch.randperm(kv.pages, generator=torch.Generator().manual_seed(seed)).tolist()
    for r, c in enumerate(n):
        ids = [order.pop() for _ in range(c)]
        kv.table[r, :c] = torch.tensor(ids, dtype=torch.int32)
        kv.refs[torch.tensor(ids, dtype=torch.long, device=DEV)] += 1
        kv.lens[r] = lens[r]
    if dtype == "int4":
        for t in (kv.k, kv.v):
            t.fill_(0x11)
        for t in (kv.k_scale, kv.v_scale):
            t.fill_(float("nan"))
    else:
        for t in (kv.k, kv.v):
            t.fill_(float("nan"))
    return kv


def _fill(kv, layer, lens, g, spread=1.0):
    """Random K and V for all tokens of all rows, through append without norm and rotation.  -> per row (k, v) float64, as stored"""
    off = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0).to(torch.int32).to(DEV)
    T = sum(lens)
    k, v = (_randn(g, T, kv.kv_heads, kv.head_dim).mul_(spread).to(kv.activations) for _ in range(2))
    rows = torch.arange(len(lens), dtype=torch.int32, device=DEV)
    kv.append(layer, k, k, v, rows, off)
    kk, vv = kv.gather(layer, rows, off, tokens=T, dtype="f32")
    if kv.dtype != "int4":
        assert torch.equal(kk, k.float()) and torch.equal(vv, v.float())
    return list(zip(kk.double().split(lens), vv.double().split(lens)))


def _offsets(counts):
    return torch.tensor([0] + list(counts), dtype=torch.int32).cumsum(0).to(torch.int32).to(DEV)


def _check_attend(got, want, mag, dot, kv, N, scale, q=None, prompt=False):
    """`prompt`: many tokens of a request at once, whose 4-bit keys and values n * step the kernel rounds to bf16 as operands: a product q_d k_d is
    off by u of itself, which moves the output by u mag.rounded_keys (1.05: the second order, e^x - 1 - x for x <= 0.1), and the mean of the values
    by u of the mean of |v|."""
    u = U[got.dtype]
    score = (kv.head_dim + 4) * 2.0 ** -24 * dot * scale
    if kv.dtype == "int4":                          # 136 sum q of each group is taken out again, in fp32
        top = float(kv.k_scale.float().nan_to_num(0.0).max())
        score += 8 * 144 * 2.0 ** -24 * float(q.abs().sum(-1).max()) * top * scale
    rel = 2 * score + 2.0 ** -20 + N * 2.0 ** -24
    if got.dtype == torch.float32:
        bound = rel * mag + u * want.abs()
    else:
        bound = u * mag * 1.01 + rel * mag + u * want.abs() * 1.01
    if kv.dtype == "int4" and prompt:
        bound = bound + u * 1.05 * mag.rounded_keys + u * 1.05 * mag
    if kv.dtype == "int4":
        bound = bound + 144 * 16 * 2.0 ** -24 * float(kv.v_scale.float().nan_to_num(0.0).max())
    off = (got.double() - want).abs()
    assert bool((off <= bound + 1e-30).all()), f"max excess {float((off - bound).max()):.3e}, max error {float(off.max()):.3e}"


@pytest.mark.parametrize("dtype", ["bf16", "f32", "int4"])
def test_attend_cuts_rows_of_any_length(dtype):
    """Long rows are cut into shares that a second kernel joins; how long rows can be is known from the table or said by max_len, which
    only steers that: a bound that is too low changes nothing.  Rows of one share, of several, and the last one ragged."""
    g = _gen(23)
    G, group, D, ps, lens = 1, 2, 64, 32, [40, 5000, 2048, 513, 9001]
    kv = _cache(dtype, G, D, ps, lens)
    store = _fill(kv, 0, lens, g)
    q = _randn(g, 5, G * group, D).mul_(2).to(kv.activations)
    rows = torch.arange(5, dtype=torch.int32, device=DEV)
    for window, sinks in ((0, 0), (4000, 40), (10, 3000)):
        for max_len in (0, 100, 2000, 9001):
            out = kv.attend(0, q, rows, window=window, sinks=sinks, max_len=max_len)
            for r, L in enumerate(lens):
                want, mag, dot = attention(q[r:r + 1], *store[r], [L - 1], window, sinks, D ** -0.5)
                _check_attend(out[r:r + 1], want, mag, dot, kv, L, D ** -0.5, q[r:r + 1].double())


# ---- append ----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,D,rot,G,H,ps,norm", [
    ("bf16", 128, 128, 8, 16, 32, True), ("bf16", 128, 64, 2, 14, 8, True), ("bf16", 64, 64, 16, 16, 16, False),
    ("bf16", 16, 16, 1, 3, 256, True), ("bf16", 80, 40, 3, 3, 16, True), ("bf16", 256, 0, 1, 8, 64, True), ("bf16", 112, 8, 5, 10, 32, False),
    ("f32", 64, 64, 16, 16, 16, True), ("f32", 128, 128, 2, 6, 128, True), ("f32", 80, 80, 3, 12, 8, False), ("f32", 256, 256, 1, 1, 16, True),
])
@pytest.mark.parametrize("counts", [None, [5, 0, 1, 70]])
def test_append_norms_rotates_and_stores(dtype, D, rot, G, H, ps, norm, counts):
    from qwen3_tts_amd.kvcache import rope_tables
    g = _gen(D + H)
    new = [1] * 4 if counts is None else counts
    lens = [n + p for n, p in zip(new, (0, 9, 300, 31))]
    kv = _cache(dtype, G, D, ps, lens, rows=6, layers=2)
    before_k, before_v = kv.k.clone(), kv.v.clone()
    T, extra = sum(new), 3                                        # three tokens behind the last request
    if counts is None:
        extra = 0
    qkv = _randn(g, T + extra, (H + 2 * G) * D).mul_(4).to(kv.activations)
    q, k, v = (x.view(T + extra, -1, D) for x in qkv.split([H * D, G * D, G * D], 1))
    wq, wk = ((torch.rand(D, generator=g, device=DEV) + 0.5) for _ in range(2)) if norm else (None, None)
    cos, sin = rope_tables(kv.max_tokens, rot, device=DEV) if rot else (None, None)
    rows = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=DEV)
    off = None if counts is None else _offsets(new)
    out = torch.full((T + extra, H, D), 7.0, dtype=kv.activations, device=DEV)
    got = kv.append(1, q, k, v, rows, off, q_weight=wq, k_weight=wk, rope=None if not rot else (cos, sin), eps=1e-6, out=out)
    assert got is out and bool((out[T:] == 7.0).all())
    kv.check()
    pos = torch.cat([torch.arange(L - n, L) for L, n in zip(lens, new)]).to(DEV)
    u = U[kv.activations]
    at = [(r, int(p)) for r, (L, n) in enumerate(zip(lens, new)) for p in range(L - n, L)]
    pages = torch.tensor([int(kv.table[r, p // ps]) for r, p in at], device=DEV, dtype=torch.long)
    slots = torch.tensor([p % ps for _, p in at], device=DEV, dtype=torch.long)
    for what, x, w, stored in (("q", q, wq, out[:T]), ("k", k, wk, kv.k[1, pages, :, slots])):
        want = norm_rotate(x[:T], w, cos, sin, pos, 1e-6)
        plain = norm_rotate(x[:T], w, None, None, pos, 1e-6).abs()
        pair = plain.clone()
        if rot:
            h = rot // 2
            pair[..., :h] = pair[..., h:rot] = plain[..., :h] + plain[..., h:rot]
        bound = (u * want.abs() if dtype == "bf16" else 0) + 32 * 2.0 ** -24 * pair + 1e-37
        off_by = (stored.double() - want).abs()
        assert bool((off_by <= bound * 1.01).all()), f"{what}: {float((off_by - bound).max())}"
    assert torch.equal(kv.v[1, pages, :, slots], v[:T])
    back_k, back_v = kv.gather(1, rows, off, tokens=T)
    assert torch.equal(back_k, kv.k[1, pages, :, slots]) and torch.equal(back_v, v[:T])
    for new_t, old_t in ((kv.k, before_k), (kv.v, before_v)):     # and nothing else was touched
        rest = new_t.clone()
        rest[1, pages, :, slots] = old_t[1, pages, :, slots]
        bits = torch.int16 if dtype == "bf16" else torch.int32
        assert torch.equal(rest.view(bits), old_t.view(bits))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rot", [True, False])
def test_append_int4_holds_each_group_to_half_a_step(D, rot):
    from qwen3_tts_amd.kvcache import rope_tables
    g = _gen(D)
    new, lens, G, H, ps = [3, 1, 40], [3, 77, 40], 3, 6, 16
    kv = _cache("int4", G, D, ps, lens)
    T = sum(new)
    q, k, v = (_randn(g, T, n, D).mul_(3).to(torch.bfloat16) for n in (H, G, G))
    k[2] = 0.0                                                    # a row of zeros
    v[1, 0, :32] = 0.0
    v[0, 1, 5] = float("inf")
    v[0, 2, 40] = float("nan")
    wq, wk = ((torch.rand(D, generator=g, device=DEV) + 0.5) for _ in range(2))
    rope = rope_tables(kv.max_tokens, D, device=DEV) if rot else None
    rows = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    out = kv.append(0, q, k, v, rows, _offsets(new), q_weight=wq, k_weight=wk, rope=rope)
    kv.check()
    pos = torch.cat([torch.arange(L - n, L) for L, n in zip(lens, new)]).to(DEV)
    cos, sin = rope or (None, None)
    wq64 = norm_rotate(q, wq, cos, sin, pos, 1e-6)
    assert bool(((out.double() - wq64).abs() <= 2.0 ** -8 * wq64.abs() + 64 * 2.0 ** -24 * wq64.abs().amax(-1, keepdim=True)).all())
    got_k, got_v = kv.gather(0, rows, _offsets(new), tokens=T, dtype="f32")
    for got, want in ((got_k, norm_rotate(k, wk, cos, sin, pos, 1e-6)), (got_v, v.double())):
        w, x = want.view(T, G, D // 32, 32), got.double().view(T, G, D // 32, 32)
        top = w.abs().amax(-1, keepdim=True)
        good = torch.isfinite(w).all(-1, keepdim=True).expand_as(w)
        # step = top / 7 rounded to bf16 (1 + 2^-8), a value to half a step, and top itself is at most 7.5 steps: clamping costs nothing more
        bound = top / 7 * (1 + 2.0 ** -8) / 2 * (1 + 2.0 ** -10) + 64 * 2.0 ** -24 * top
        assert bool(((x - w).abs() <= bound)[good].all())
        assert bool((x[good] == 0)[(top.expand_as(w) == 0)[good]].all())
        assert bool(torch.isnan(x[~good]).all())                  # a group with an infinity or a NaN reads back as NaN
    assert torch.isfinite(got_v).sum() == T * G * D - 64


def test_append_and_attend_read_any_strides():
    g = _gen(3)
    lens = [40, 7]
    kv = _cache("bf16", 2, 64, 16, lens)
    store = _fill(kv, 0, lens, g)
    rows = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    base = _randn(g, 2, 4, 64, dtype=torch.bfloat16)
    want = kv.attend(0, base, rows)
    heads_first = base.transpose(0, 1).contiguous().transpose(0, 1)         # [token][head] over a [head][token] tensor
    wide = torch.zeros(2, 4, 80, dtype=torch.bfloat16, device=DEV)
    wide[..., 4:68] = base
    odd = torch.zeros(2 * 4 * 64 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(2, 4, 64)     # not aligned to four values
    odd.copy_(base)
    spaced = torch.zeros(2, 4, 64, 2, dtype=torch.bfloat16, device=DEV)[..., 0]                  # dim not contiguous
    spaced.copy_(base)
    for x in (heads_first, wide[..., 4:68], odd, spaced, base[:1].expand(2, 4, 64)):
        ref = want if x.stride(0) else kv.attend(0, base[:1].repeat(2, 1, 1), rows)
        assert torch.equal(kv.attend(0, x, rows), ref)
    kn = _randn(g, 2, 2, 64, dtype=torch.bfloat16)
    ref_q = kv.append(0, base, kn, kn, rows)
    ref = kv.gather(0, rows)
    for x in (heads_first, wide[..., 4:68], odd, spaced):
        kv.k.zero_()
        assert torch.equal(kv.append(0, x, kn.transpose(0, 1).contiguous().transpose(0, 1), kn, rows), ref_q)
        assert all(torch.equal(a, b) for a, b in zip(kv.gather(0, rows), ref))
    assert store


# ---- attend ----------------------------------------------------------------------------------------------------------------------
SHAPES = [("bf16", 128, 2, 2, 32), ("bf16", 64, 1, 1, 8), ("bf16", 128, 1, 7, 16), ("bf16", 256, 2, 4, 64), ("bf16", 80, 3, 1, 16), ("bf16", 16, 1, 20, 128),
          ("f32", 64, 2, 1, 16), ("f32", 128, 1, 4, 8), ("f32", 256, 1, 2, 256), ("f32", 48, 2, 3, 32),
          ("int4", 64, 2, 2, 8), ("int4", 128, 2, 4, 32), ("int4", 256, 1, 1, 16)]


@pytest.mark.parametrize("dtype,D,G,group,ps", SHAPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (40, 0), (33, 5), (64, 100)])
def test_attend_prompts_and_pieces(dtype, D, G, group, ps, window, sinks):
    """Whole prompts (new == length), a piece behind a past, one token, none at all, and a row of nothing."""
    g = _gen(D + group + window)
    lens, new = [67, 130, 1, 55, 0, 18], [67, 19, 1, 0, 0, 17]
    kv = _cache(dtype, G, D, ps, lens)
    store = _fill(kv, 0, lens, g)
    T = sum(new)
    q = _randn(g, T + 2, G * group, D).mul_(2).to(kv.activations)
    out = torch.full_like(q, 5.0)
    rows = torch.arange(6, dtype=torch.int32, device=DEV)
    kv.attend(0, q, rows, _offsets(new), window=window, sinks=sinks, out=out)
    kv.check()
    assert bool((out[T:] == 5.0).all())
    scale, at = D ** -0.5, 0
    for r, (L, n) in enumerate(zip(lens, new)):
        want, mag, dot = attention(q[at:at + n], *store[r], list(range(L - n, L)), window, sinks, scale) if n else (None, None, 0)
        if n:
            _check_attend(out[at:at + n], want, mag, dot, kv, L, scale, q[at:at + n].double(), prompt=True)
        at += n


@pytest.mark.parametrize("dtype,D,G,group,ps", SHAPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 3)])
def test_attend_single_tokens(dtype, D, G, group, ps, window, sinks):
    """One new token per row, from the first token on; long rows are split over workgroups."""
    g = _gen(D * 3 + group + window)
    lens = [1, 2, 15, 16, 17, 31, 33, 64, 250, 1030]
    kv = _cache(dtype, G, D, ps, lens)
    store = _fill(kv, 0, lens, g, 1.5)
    q = _randn(g, len(lens), G * group, D).mul_(2).to(kv.activations)
    rows = torch.tensor([9, 0, 1, 2, 3, 4, 5, 6, 7, 8], dtype=torch.int32, device=DEV)
    scale = 0.7 * D ** -0.5
    for max_len in (0, 1030):
        out = kv.attend(0, q, rows, window=window, sinks=sinks, scale=scale, max_len=max_len)
        for i, r in enumerate(rows.tolist()):
            want, mag, dot = attention(q[i:i + 1], *store[r], [lens[r] - 1], window, sinks, scale)
            _check_attend(out[i:i + 1], want, mag, dot, kv, lens[r], scale, q[i:i + 1].double())


@pytest.mark.parametrize("dtype", ["bf16", "f32", "int4"])
def test_attend_long_prompt_agrees_with_its_tokens_one_by_one(dtype):
    """A prompt of many tiles, ragged against the tile and page sizes, and each of its tokens asked for alone."""
    g = _gen(17)
    G, group, D, ps, lens, new = 2, 3, 128, 32, [701, 333], [523, 333]
    kv = _cache(dtype, G, D, ps, lens)
    _fill(kv, 0, lens, g)
    q = _randn(g, sum(new), G * group, D).mul_(2).to(kv.activations)
    rows = torch.arange(2, dtype=torch.int32, device=DEV)
    for window, sinks in ((0, 0), (150, 4)):
        out = kv.attend(0, q, rows, _offsets(new), window=window, sinks=sinks)
        for r, i in ((0, 0), (0, 31), (0, 522), (1, 0), (1, 200), (1, 332)):
            kv.lens[r] = lens[r] - new[r] + i + 1
            t = (0 if r == 0 else new[0]) + i
            alone = kv.attend(0, q[t:t + 1], rows[r:r + 1], window=window, sinks=sinks)
            kv.lens[r] = lens[r]
            u = U[kv.activations]
            tol = 4 * u * (6.0 if dtype != "f32" else 64.0)       # both are within the bounds above; |v| <= 6 here
            assert float((alone.float() - out[t:t + 1].float()).abs().max()) <= tol


@pytest.mark.parametrize("dtype", ["bf16", "f32", "int4"])
def test_attend_leaves_out_what_is_not_seen(dtype):
    """Infinities and NaN in keys and values: a token's output depends on the rows it sees alone (others of its tile may see them)."""
    g = _gen(5)
    G, group, D, ps, lens = 1, 2, 64, 8, [60, 45]
    kv = _cache(dtype, G, D, ps, lens)
    store = _fill(kv, 0, lens, g)
    q = _randn(g, sum(lens), G * group, D).to(kv.activations)
    rows = torch.arange(2, dtype=torch.int32, device=DEV)
    clean = kv.attend(0, q, rows, _offsets(lens), window=20, sinks=2)

    def poison(row, pos, which, value):
        page, slot = int(kv.table[row, pos // ps]), pos % ps
        if dtype == "int4":
            getattr(kv, which + "_scale")[0, page, 0, slot, 0] = value
        else:
            getattr(kv, which)[0, page, 0, slot, 3] = value
    poison(0, 25, "v", float("inf"))
    poison(0, 40, "v", float("nan"))
    poison(1, 30, "k", float("nan"))
    got = kv.attend(0, q, rows, _offsets(lens), window=20, sinks=2)
    for row, start, bad in ((0, 0, set(range(25, 60))), (1, 60, set(range(30, 45)))):
        for p in range(lens[row]):
            sees = p in bad and any(b <= p < b + 20 for b in ((25, 40) if row == 0 else (30,)))
            if sees:
                assert not bool(torch.isfinite(got[start + p]).all()), (row, p)
            else:
                assert torch.equal(got[start + p], clean[start + p]), (row, p)
    assert store


@pytest.mark.parametrize("dtype", ["bf16", "int4"])
def test_attend_missing_pages_and_bad_rows(dtype):
    g = _gen(6)
    G, group, D, ps, lens = 2, 2, 64, 16, [100, 50, 20]
    kv = _cache(dtype, G, D, ps, lens, rows=3)
    store = _fill(kv, 0, lens, g)
    kv.table[0, 2] = -1                                            # positions 32 .. 47
    kv.table[0, 4] = kv.pages + 7                                  # 64 .. 79: outside the pool
    kv.table[1, :] = -1
    q = _randn(g, 5, G * group, D).mul_(2).to(kv.activations)
    out = kv.attend(0, q, torch.tensor([0, 1, 2, -1, 3], dtype=torch.int32, device=DEV))
    there = torch.ones(100, dtype=torch.bool, device=DEV)
    there[32:48] = there[64:80] = False
    scale = D ** -0.5
    want, mag, dot = attention(q[:1], *store[0], [99], 0, 0, scale, there)
    _check_attend(out[:1], want, mag, dot, kv, 100, scale, q[:1].double())
    want, mag, dot = attention(q[2:3], *store[2], [19], 0, 0, scale)
    _check_attend(out[2:3], want, mag, dot, kv, 20, scale, q[2:3].double())
    assert bool((out[[1, 3, 4]] == 0).all())
    # more new tokens than the row holds: those before its beginning see nothing
    kv.lens[2] = 3
    out = kv.attend(0, q, torch.tensor([2], dtype=torch.int32, device=DEV), _offsets([5]))
    assert bool((out[:2] == 0).all())
    want, mag, dot = attention(q[2:], store[2][0][:3], store[2][1][:3], [0, 1, 2], 0, 0, scale)
    _check_attend(out[2:], want, mag, dot, kv, 3, scale, q[2:].double())


def test_append_bad_rows_and_missing_pages_are_flagged_not_written():
    from qwen3_tts_amd import _lib
    g = _gen(8)
    kv = _cache("bf16", 1, 64, 8, [5, 9])
    before = kv.k.clone()
    q, k = _randn(g, 4, 2, 64, dtype=torch.bfloat16), _randn(g, 4, 1, 64, dtype=torch.bfloat16)
    kv.table[1, 1] = -1
    out = kv.append(0, q, k, k, torch.tensor([-1, 1, 7, 0], dtype=torch.int32, device=DEV))
    assert bool((out[[0, 2]] == 0).all()) and torch.equal(out[[1, 3]], q[[1, 3]])
    with pytest.raises(_lib.Q3cError, match="row id.*no free page"):
        kv.check()
    kv.check()                                                     # cleared
    page, slot = int(kv.table[0, 0]), 4
    assert torch.equal(kv.k[0, page, :, slot], k[3])
    kv.k[0, page, :, slot] = before[0, page, :, slot]
    assert torch.equal(kv.k.view(torch.int16), before.view(torch.int16))
    kv.append(0, q[:2], k[:2], k[:2], torch.tensor([0, 0], dtype=torch.int32, device=DEV))       # a row named twice: the first counts
    assert torch.equal(kv.k[0, page, :, slot], k[0])
    with pytest.raises(_lib.Q3cError, match="row id"):
        kv.check()
    kv.append(0, q, k, k, torch.tensor([0], dtype=torch.int32, device=DEV), _offsets([4]))       # fits
    kv.lens[0] = 2
    out = kv.append(0, q, k, k, torch.tensor([0], dtype=torch.int32, device=DEV), _offsets([4])) # two tokens before the row's beginning
    assert bool((out[:2] == 0).all()) and torch.equal(out[2:], q[2:])
    with pytest.raises(_lib.Q3cError, match="row id"):
        kv.check()


def test_places_past_two_to_the_31():
    """Element offsets beyond 32 bits: the last page of the last layer of a pool of 2.2e9 values."""
    from qwen3_tts_amd.kvcache import PagedKV
    g = _gen(9)
    G, D, ps, P = 8, 128, 128, 8400
    kv = PagedKV(2, G, D, P, ps, rows=3, pages_per_row=4, dtype="bf16", device=DEV)
    assert kv.k.numel() > 2 ** 31
    kv.table[0, :2] = torch.tensor([P - 1, P - 2], dtype=torch.int32)
    kv.refs[-2:] = 1
    kv.lens[0] = 200
    k, v, q = (_randn(g, 200, n, D, dtype=torch.bfloat16) for n in (G, G, 16))
    rows = torch.zeros(1, dtype=torch.int32, device=DEV)
    kv.append(1, q, k, v, rows, _offsets([200]))
    assert torch.equal(kv.k[1, P - 1].transpose(0, 1), k[:128]) and torch.equal(kv.v[1, P - 2].transpose(0, 1)[:72], v[128:])
    out = kv.attend(1, q[-1:].contiguous(), rows)
    want, mag, dot = attention(q[-1:], k, v, [199], 0, 0, D ** -0.5)
    _check_attend(out, want, mag, dot, kv, 200, D ** -0.5)
    kv.fork([0], [1])
    kv.copy_pages([P - 1], [P - 3])
    kv.check()
    assert kv.table[1, :3].tolist() == [P - 1, 0, -1] and kv.refs[P - 1] == 2
    assert torch.equal(kv.k[:, 0], kv.k[:, P - 2]) and torch.equal(kv.v[:, P - 3], kv.v[:, P - 1])
    assert int(kv.compact()) == 3
    kv.check()
    assert kv.table[:2, :2].tolist() == [[2, 1], [2, 0]]
    assert torch.equal(kv.attend(1, q[-1:].contiguous(), rows), out)


# ---- pages -----------------------------------------------------------------------------------------------------------------------
def _same(kv, ref):
    assert kv.table.tolist() == ref.table and kv.lens.tolist() == ref.lens and kv.refs.tolist() == ref.refs
    assert int(kv.status) == ref.status


@pytest.mark.parametrize("dtype,pages,rows,width,seed", [("bf16", 40, 7, 9, 0), ("int4", 23, 5, 6, 1), ("f32", 20000, 40, 30, 2), ("bf16", 9, 3, 4, 3)])
def test_page_operations_follow_the_rules(dtype, pages, rows, width, seed):
    """A random life of a pool, checked after every operation against lists; pools that run out and rows that fill up among it."""
    import random

    from qwen3_tts_amd.kvcache import PagedKV
    rng, ps = random.Random(seed), 8
    kv = PagedKV(2, 1, 64 if dtype == "int4" else 16, pages, ps, rows, width, dtype, DEV)
    tensors = [t for t in (kv.k, kv.v, kv.k_scale, kv.v_scale) if t is not None]
    g = _gen(seed)
    for t in tensors:
        t.copy_(torch.randint(0, 200, t.shape, generator=g, device=DEV).to(t.dtype))
    ref = Pages(pages, ps, rows, width)
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    for step in range(60):
        want = [t.clone() for t in tensors]
        op = rng.choice(["reserve", "reserve", "tokens", "fork", "release", "trim", "copy", "compact"])
        some = [rng.randrange(rows) for _ in range(rng.randint(1, rows))]
        if op == "reserve":
            if step % 7 == 0:
                some += [-1, rows]
            counts = [rng.choice([0, 1, 7, 8, 30]) for _ in some]
            kv.reserve(dev(some), _offsets(counts), tokens=sum(counts))
            ref.reserve(some, counts)
        elif op == "tokens":
            some = sorted(set(some))
            kv.reserve(some)
            ref.reserve(some, [1] * len(some))
        elif op == "fork":
            up = [rng.randrange(-1, rows) for _ in some]
            kv.fork(dev(up), dev(some))
            for s, d in ref.fork(up, some):
                for t in want:
                    t[:, d] = t[:, s].clone()
        elif op == "release":
            kv.release(dev(some))
            ref.release(some)
        elif op == "trim":
            w, s = rng.randint(1, 40), rng.choice([0, 3, 8, 9])
            kv.trim(dev(some), w, s)
            ref.trim(some, w, s)
        elif op == "copy":
            n = rng.randint(0, 6)
            src, dst = [rng.randrange(-1, pages) for _ in range(n)], [rng.randrange(pages + 1) for _ in range(n)]
            kv.copy_pages(dev(src), dev(dst))
            old = [t.clone() for t in want]
            for s, d in ref.copy(src, dst):
                for t, o in zip(want, old):
                    t[:, d] = o[:, s]
        else:
            live = kv.compact()
            old = [t.clone() for t in want]
            pairs, n = ref.compact()
            assert int(live) == n
            for s, d in pairs:
                for t, o in zip(want, old):
                    t[:, d] = o[:, s]
        _same(kv, ref)
        assert all(torch.equal(a, b) for a, b in zip(tensors, want)), op
        if ref.status:
            with pytest.raises(Exception):
                kv.check()
            ref.status = 0


def test_reserve_and_fork_of_more_rows_than_a_workgroup():
    from qwen3_tts_amd.kvcache import PagedKV
    rows, ps = 2300, 8
    kv = PagedKV(1, 1, 16, 9000, ps, 2 * rows, 3, "bf16", DEV)
    ref = Pages(9000, ps, 2 * rows, 3)
    order = torch.randperm(rows, generator=torch.Generator().manual_seed(1)).tolist()
    counts = [(7 * i) % 19 for i in range(rows)]
    kv.reserve(torch.tensor(order, dtype=torch.int32, device=DEV), _offsets(counts), tokens=sum(counts))
    ref.reserve(order, counts)
    _same(kv, ref)
    up, ch = list(range(rows)), list(range(rows, 2 * rows))
    kv.fork(up, ch)
    ref.fork(up, ch)
    _same(kv, ref)
    twice = order + order[:5]
    kv.reserve(torch.tensor(twice, dtype=torch.int32, device=DEV))
    ref.reserve(twice, [1] * len(twice))
    _same(kv, ref)


def test_empty_calls_do_nothing():
    g = _gen(1)
    kv = _cache("bf16", 1, 64, 16, [20])
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    q = _randn(g, 0, 2, 64, dtype=torch.bfloat16)
    kv.reserve(none)
    kv.release(none)
    kv.trim(none, 5)
    kv.fork(none, none)
    kv.copy_pages(none, none)
    assert kv.append(0, q, q[:, :1], q[:, :1], none).shape == (0, 2, 64) and kv.attend(0, q, none).shape == (0, 2, 64)
    assert kv.gather(0, none)[0].shape == (0, 1, 64)
    one = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert kv.attend(0, q, one, _offsets([0])).shape == (0, 2, 64)
    kv.check()
    assert kv.lens.tolist() == [20]


# ---- together --------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f32", "int4"])
def test_a_generation_with_forks_trims_and_a_compaction(dtype):
    """Two layers, a prompt, three requests forked from it, steps of one token under a window with sinks, pages given back and the pool
    compacted on the way: every output against 64-bit attention over all keys the row ever had."""
    from qwen3_tts_amd.kvcache import PagedKV, rope_tables
    g = _gen(21)
    G, H, D, ps, window, sinks = 2, 4, 64, 8, 24, 4
    kv = PagedKV(2, G, D, 40, ps, rows=5, pages_per_row=12, dtype=dtype, device=DEV)
    rope = rope_tables(kv.max_tokens, D, device=DEV)
    wq, wk = ((torch.rand(D, generator=g, device=DEV) + 0.5) for _ in range(2))
    history = {}                                                    # (layer, row) -> [k, v] as stored

    def tokens(rows, counts):
        off, T = (None, len(rows)) if counts is None else (_offsets(counts), sum(counts))
        counts = counts or [1] * len(rows)
        ids = torch.tensor(rows, dtype=torch.int32, device=DEV)
        kv.reserve(ids, off, tokens=T)
        for layer in range(2):
            qkv = _randn(g, T, (H + 2 * G) * D).mul_(2).to(kv.activations)
            q, k, v = (x.view(T, -1, D) for x in qkv.split([H * D, G * D, G * D], 1))
            q = kv.append(layer, q, k, v, ids, off, q_weight=wq, k_weight=wk, rope=rope)
            out = kv.attend(layer, q, ids, off, window=window, sinks=sinks)
            kk, vv = kv.gather(layer, ids, off, tokens=T, dtype="f32")
            at = 0
            for r, n in zip(rows, counts):
                h = history.setdefault((layer, r), [torch.empty(0, G, D, device=DEV, dtype=torch.float64)] * 2)
                h[0], h[1] = torch.cat([h[0], kk[at:at + n].double()]), torch.cat([h[1], vv[at:at + n].double()])
                L = h[0].shape[0]
                want, mag, dot = attention(q[at:at + n], h[0], h[1], list(range(L - n, L)), window, sinks, D ** -0.5)
                _check_attend(out[at:at + n], want, mag, dot, kv, L, D ** -0.5, q[at:at + n].double(), prompt=counts[0] > 1)
                at += n

    tokens([0, 4], [21, 6])
    kv.fork([0, 0, 0], [1, 2, 3])
    for layer in range(2):
        for r in (1, 2, 3):
            history[layer, r] = list(history[layer, 0])
    for step in range(40):
        tokens([3, 0, 1, 2] if step < 20 else [3, 1], None if step % 5 else [2] * (4 if step < 20 else 2))
        kv.trim([0, 1, 2, 3], window, sinks)
        if step == 19:
            kv.release([0, 2])
            kv.compact()
    kv.check()
    kv.release([1, 3, 4])
    assert kv.free_pages() == kv.pages and int(kv.lens.sum()) == 0 and bool((kv.table == -1).all())


@pytest.mark.parametrize("dtype", ["bf16", "int4"])
def test_captured_steps_replay_beside_each_other(dtype):
    """A step (reserve, append, attend, trim) captured once and replayed token by token, beside a second graph of another cache on
    another stream and eager work between: every replay equals the same step run eagerly."""
    from qwen3_tts_amd.kvcache import PagedKV, rope_tables
    G, H, D, ps = 2, 4, 128, 8
    sides = []
    for seed in (1, 2):
        g = _gen(seed)
        pair = [PagedKV(1, G, D, 200, ps, rows=3, pages_per_row=60, dtype=dtype, device=DEV) for _ in range(2)]
        rope = rope_tables(pair[0].max_tokens, D, device=DEV)
        rows = torch.tensor([2, 0, 1], dtype=torch.int32, device=DEV)
        qkv = [torch.empty(3, n, D, dtype=torch.bfloat16, device=DEV) for n in (H, G, G)]
        for kv in pair:
            kv.reserve(rows, _offsets([100, 201, 5]), tokens=306)
            gg = _gen(seed + 10)
            x = [_randn(gg, 306, n, D, dtype=torch.bfloat16) for n in (H, G, G)]
            kv.append(0, *x, rows, _offsets([100, 201, 5]), rope=rope)

        def step(kv, qkv=qkv, rows=rows, rope=rope):
            kv.reserve(rows)
            out = kv.attend(0, kv.append(0, *qkv, rows, rope=rope), rows, window=64, sinks=3)
            kv.trim(rows, 64, 3)
            return out
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        for t in qkv:
            t.copy_(_randn(g, *t.shape))
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            out = step(pair[0])
        sides.append((pair, qkv, step, graph, out, stream, g))
    torch.cuda.synchronize()
    for i in range(6):
        for pair, qkv, step, graph, out, stream, g in sides:
            for t in qkv:
                t.copy_(_randn(g, *t.shape))
        torch.cuda.synchronize()
        for pair, qkv, step, graph, out, stream, g in sides:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for pair, qkv, step, graph, out, stream, g in sides:
            assert torch.equal(out, step(pair[1])), i
            assert torch.equal(pair[0].table, pair[1].table) and torch.equal(pair[0].lens, pair[1].lens)
            for kv in pair:
                kv.check()


def test_another_stream_and_the_torch_ops():
    from qwen3_tts_amd import torch_ops
    g = _gen(4)
    kv = _cache("bf16", 2, 64, 16, [33, 90])
    _fill(kv, 0, [33, 90], g)
    rows = torch.tensor([1, 0], dtype=torch.int32, device=DEV)
    q = _randn(g, 2, 4, 64, dtype=torch.bfloat16)
    want = kv.attend(0, q, rows, window=50, sinks=1)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = kv.attend(0, q, rows, window=50, sinks=1)
    s.synchronize()
    assert torch.equal(got, want)
    h = torch_ops.register_kv(kv)
    assert torch.equal(torch.ops.q3tts.kv_attend(q, rows, None, 50, 1, h, 0), want)
    k = _randn(g, 2, 2, 64, dtype=torch.bfloat16)
    w = torch.rand(64, generator=g, device=DEV)
    a = torch.ops.q3tts.kv_append(q, k, k, rows, None, w, w, None, None, 1e-6, h, 0)
    assert torch.equal(a, kv.append(0, q, k, k, rows, q_weight=w, k_weight=w))
    torch_ops.unregister_kv(h)
    with pytest.raises(KeyError):
        torch.ops.q3tts.kv_attend(q, rows, None, 50, 1, h, 0)


def test_refusals_with_tensors_on_the_gpu():
    kv = _cache("bf16", 2, 64, 16, [33, 90])
    rows = torch.tensor([1, 0], dtype=torch.int32, device=DEV)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=DEV)
    k = q[:, :2]
    cos = torch.zeros(kv.max_tokens, 32, device=DEV)
    for bad in (dict(q=q.float()), dict(q=q[..., :32]), dict(k=q), dict(rows=rows.long()), dict(rows=rows.cpu()), dict(rows=rows[:1]),
                dict(q=q[:1]), dict(q_weight=torch.ones(64, dtype=torch.bfloat16, device=DEV)), dict(q_weight=torch.ones(32, device=DEV)),
                dict(rope=(cos[:-1], cos[:-1])), dict(rope=(cos, cos[:, :16])), dict(rope=(cos[:, :3].contiguous(),) * 2), dict(out=q.float()),
                dict(offsets=torch.tensor([0, 2], dtype=torch.int32, device=DEV)), dict(rows=[0, 0]), dict(q=q.cpu())):
        a = dict(q=q, k=k, v=k, rows=rows, offsets=None, q_weight=None, k_weight=None, rope=None, out=None)
        a.update(bad)
        with pytest.raises(ValueError):
            kv.append(0, a["q"], a["k"], a["v"], a["rows"], a["offsets"], q_weight=a["q_weight"], k_weight=a["k_weight"], rope=a["rope"], out=a["out"])
    for kw in (dict(window=-1), dict(sinks=-1), dict(scale=0.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(max_len=-2)):
        with pytest.raises(ValueError):
            kv.attend(0, q, rows, **kw)
    with pytest.raises(ValueError):
        kv.attend(0, q[:, :3], rows)                                # three heads on two kv heads
    for layer in (-1, 1):
        with pytest.raises(IndexError):
            kv.attend(layer, q, rows)
    for ids in ([2], [-1]):
        with pytest.raises(IndexError):
            kv.release(ids)
    with pytest.raises(ValueError):
        kv.trim(rows, 0)
    with pytest.raises(ValueError):
        kv.fork([0], [1, 0])
    with pytest.raises(ValueError):
        kv.gather(0, rows, _offsets([1, 1]))                        # how many tokens is not said
    kv.check()
    assert math.isnan(float(kv.k.float().sum()))                    # and nothing was written


@pytest.mark.parametrize("dtype,D,G,group,ps", SHAPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (72, 0), (90, 10)])
def test_attend_prompts_of_many_tiles(dtype, D, G, group, ps, window, sinks):
    """Prompts long enough for the kernel that shares key tiles between waves: ragged ends, a past, a row of one token, an empty one."""
    g = _gen(D * 5 + group + window)
    lens, new = [300, 211, 1, 0], [300, 150, 1, 0]
    kv = _cache(dtype, G, D, ps, lens)
    store = _fill(kv, 0, lens, g)
    T = sum(new)
    q = _randn(g, T + 1, G * group, D).mul_(2).to(kv.activations)
    out = torch.full_like(q, 5.0)
    rows = torch.arange(4, dtype=torch.int32, device=DEV)
    kv.attend(0, q, rows, _offsets(new), window=window, sinks=sinks, out=out)
    kv.check()
    assert bool((out[T:] == 5.0).all())
    scale = D ** -0.5
    for r, start, some in ((0, 0, [0, 1, 31, 32, 63, 64, 127, 128, 200, 299]), (1, 300, [0, 5, 63, 100, 149]), (2, 450, [0])):
        i = torch.tensor(some, device=DEV)
        pos = [lens[r] - new[r] + p for p in some]
        want, mag, dot = attention(q[start + i], *store[r], pos, window, sinks, scale)
        _check_attend(out[start + i], want, mag, dot, kv, lens[r], scale, q[start + i].double(), prompt=True)


# ---- calls of unusual shape ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f32", "int4"])
def test_tokens_before_the_first_request_are_left_alone(dtype):
    """A batch padded in front: offsets that begin at 3.  Nothing of the padding reaches the cache, nothing is written to its outputs."""
    g = _gen(31)
    G, group, D, ps, lens, new = 2, 2, 64, 8, [30, 21], [4, 9]
    kv = _cache(dtype, G, D, ps, lens)
    _fill(kv, 0, lens, g)
    rows = torch.tensor([1, 0], dtype=torch.int32, device=DEV)
    q, k, v = (_randn(g, 16 + 2, n, D, dtype=kv.activations) for n in (G * group, G, G))
    off = _offsets(new)
    held = [t.clone() for t in (kv.k, kv.v)]
    want = kv.append(0, q[3:16], k[3:16], v[3:16], rows, off)
    seen = kv.attend(0, q[3:16], rows, off, window=10, sinks=2)
    after = [t.clone() for t in (kv.k, kv.v)]
    kk, vv = kv.gather(0, rows, off, tokens=13)
    for t, h in zip((kv.k, kv.v), held):
        t.copy_(h)
    out = torch.full_like(q, 5.0)
    kv.append(0, q, k, v, rows, off + 3, out=out)
    assert torch.equal(out[3:16], want) and bool((out[:3] == 5.0).all()) and bool((out[16:] == 5.0).all())
    for t, a in zip((kv.k, kv.v), after):
        assert torch.equal(t.view(torch.uint8), a.view(torch.uint8))
    out.fill_(5.0)
    kv.attend(0, q, rows, off + 3, window=10, sinks=2, out=out)
    assert torch.equal(out[3:16], seen) and bool((out[:3] == 5.0).all()) and bool((out[16:] == 5.0).all())
    k3, v3 = kv.gather(0, rows, off + 3, tokens=18)
    assert torch.equal(k3[3:16], kk) and torch.equal(v3[3:16], vv)
    lens0 = kv.lens.tolist()
    kv.reserve(rows, off + 3, tokens=18)
    assert kv.lens.tolist() == [lens0[0] + 9, lens0[1] + 4]
    kv.check()


@pytest.mark.parametrize("dtype,D,G,H", [("bf16", 80, 3, 5 * 3), ("bf16", 128, 8, 16), ("f32", 48, 5, 5), ("int4", 64, 9, 9), ("int4", 128, 3, 21), ("int4", 256, 10, 10)])
def test_many_tokens_at_once_are_the_same_as_a_few(dtype, D, G, H):
    """append and gather give a wave more of a token's heads when tokens are many: the same values, bit for bit, as in small calls."""
    g = _gen(D + G)
    lens, ps = [2500, 901], 16
    kv = _cache(dtype, G, D, ps, lens)
    T = sum(lens)
    x = _randn(g, T, H + 2 * G, D).mul_(3).to(kv.activations)
    q, k, v = x.split([H, G, G], 1)
    wq, wk = (torch.rand(D, generator=g, device=DEV) + 0.5 for _ in range(2))
    from qwen3_tts_amd.kvcache import rope_tables
    rope = rope_tables(kv.max_tokens, D, device=DEV)
    rows = torch.arange(2, dtype=torch.int32, device=DEV)
    out = kv.append(0, q, k, v, rows, _offsets(lens), q_weight=wq, k_weight=wk, rope=rope)
    got = {t: kv.gather(0, rows, _offsets(lens), tokens=T, dtype=t) for t in ("f32", "bf16")}
    whole = [t.clone() for t in (kv.k, kv.v)]
    some, at = torch.empty_like(out), 0
    for r, L in enumerate(lens):
        for i in range(0, L, 100):
            n = min(100, L - i)
            kv.lens[r] = i + n
            s = slice(at + i, at + i + n)
            one = rows[r:r + 1]
            some[s] = kv.append(0, q[s], k[s], v[s], one, _offsets([n]), q_weight=wq, k_weight=wk, rope=rope)
            for t in ("f32", "bf16"):
                kk, vv = kv.gather(0, one, _offsets([n]), tokens=n, dtype=t)
                assert torch.equal(kk, got[t][0][s]) and torch.equal(vv, got[t][1][s])
        at += L
    assert torch.equal(some, out)
    for t, w in zip((kv.k, kv.v), whole):
        assert torch.equal(t.view(torch.uint8), w.view(torch.uint8))
    if dtype != "int4":
        assert torch.equal(got["f32"][1], v.float()) and torch.equal(got["bf16"][1], v.to(torch.bfloat16))
    kv.check()


def _some_rows(kv, out, q, store, lens, rows, some, window, sinks, scale):
    for i in some:
        r = rows[i]
        if 0 <= r < kv.rows and lens[r]:
            want, mag, dot = attention(q[i:i + 1], *store[r], [lens[r] - 1], window, sinks, scale)
            _check_attend(out[i:i + 1], want, mag, dot, kv, lens[r], scale, q[i:i + 1].double())
        else:
            assert bool((out[i] == 0).all()), i


@pytest.mark.parametrize("dtype,D,G,group,ps,S", [("bf16", 128, 8, 2, 32, 300), ("bf16", 64, 1, 20, 8, 400), ("f32", 64, 4, 1, 16, 1024), ("int4", 128, 8, 2, 32, 200),
                                                  ("int4", 64, 2, 3, 8, 1000), ("bf16", 256, 2, 1, 64, 700), ("int4", 256, 1, 4, 128, 1024), ("f32", 256, 1, 1, 256, 1023),
                                                  ("bf16", 128, 8, 2, 32, 1030), ("f32", 48, 8, 2, 16, 1100), ("int4", 64, 8, 1, 8, 1025)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 5)])
def test_attend_single_tokens_of_many_rows(dtype, D, G, group, ps, S, window, sinks):
    """Hundreds of rows of all lengths, empty ones and bad ids among them: one line of runs up to a thousand rows, a wave for each beyond."""
    g = _gen(S + D)
    r = torch.Generator().manual_seed(S)
    lens = torch.randint(1, 60, (S,), generator=r).tolist()
    lens[0], lens[1], lens[2], lens[S // 2], lens[-1] = 1, 0, 1900, 700, 0
    for i in range(3, S, 17):
        lens[i] = 0
    kv = _cache(dtype, G, D, ps, lens, width=-(-6000 // ps))
    store = _fill(kv, 0, lens, g)
    rows = torch.randperm(S, generator=r).tolist()
    rows[5], rows[6] = -1, S + 4
    q = _randn(g, S, G * group, D).mul_(2).to(kv.activations)
    out = torch.full_like(q, 7.0)
    kv.attend(0, q, torch.tensor(rows, dtype=torch.int32, device=DEV), window=window, sinks=sinks, out=out)
    where = {x: i for i, x in enumerate(rows)}
    some = [where[x] for x in (0, 1, 2, 3, S // 2, S - 1, S - 2, S - 3) if x in where] + [0, 5, 6, S - 1, S // 3]
    _some_rows(kv, out, q, store, lens, rows, some, window, sinks, D ** -0.5)
    nothing = torch.tensor([i for i, x in enumerate(rows) if not 0 <= x < S or not lens[x]], device=DEV)
    assert bool((out[nothing] == 0).all()) and bool(torch.isfinite(out).all())
    kv.lens.zero_()                                                # and rows that see nothing, all of them
    assert bool((kv.attend(0, q, torch.tensor(rows, dtype=torch.int32, device=DEV), window=window, sinks=sinks) == 0).all())


@pytest.mark.parametrize("dtype,D,G,group,ps", [("bf16", 128, 8, 2, 32), ("f32", 64, 8, 1, 16), ("int4", 128, 8, 2, 8), ("f32", 256, 16, 1, 32), ("bf16", 48, 16, 3, 16)])
def test_attend_many_short_pieces(dtype, D, G, group, ps):
    """Many short rows with a few new tokens each: a wave for each tile.  Rows that no token of a tile but its neighbours sees hold NaN."""
    g = _gen(D + G + 1)
    S = 140
    r = torch.Generator().manual_seed(3)
    new = torch.randint(0, 8, (S,), generator=r).tolist()
    lens = [n + p for n, p in zip(new, torch.randint(0, 90, (S,), generator=r).tolist())]
    kv = _cache(dtype, G, D, ps, lens, width=-(-200 // ps))
    store = _fill(kv, 0, lens, g)
    T = sum(new)
    q = _randn(g, T + 3, G * group, D).mul_(2).to(kv.activations)
    rows = torch.arange(S, dtype=torch.int32, device=DEV)
    out = torch.full_like(q, 7.0)
    kv.attend(0, q, rows, _offsets(new), window=30, sinks=3, out=out)
    assert bool((out[T:] == 7.0).all())
    start = [sum(new[:i]) for i in range(S)]
    for i in (0, 1, 2, 50, 77, 138, 139):
        if new[i]:
            s = slice(start[i], start[i] + new[i])
            want, mag, dot = attention(q[s], *store[i], list(range(lens[i] - new[i], lens[i])), 30, 3, D ** -0.5)
            _check_attend(out[s], want, mag, dot, kv, lens[i], D ** -0.5, q[s].double(), prompt=True)
    i = next(i for i in range(S) if new[i] >= 5 and lens[i] - new[i] > 40)
    bad = lens[i] - 2                                               # seen by the last two of the row's tokens
    page, slot = int(kv.table[i, bad // ps]), bad % ps
    if dtype == "int4":
        kv.v_scale[0, page, 0, slot, 0] = float("nan")
    else:
        kv.v[0, page, 0, slot, 3] = float("nan")
    again = kv.attend(0, q, rows, _offsets(new), window=30, sinks=3)
    end = start[i] + new[i]
    assert not bool(torch.isfinite(again[end - 2:end]).all(-1).all(-1).any())
    assert torch.equal(again[:end - 2], out[:end - 2]) and torch.equal(again[end:T], out[end:T])


@pytest.mark.parametrize("dtype", ["bf16", "int4"])
def test_captured_calls_of_long_rows_follow_their_lengths(dtype):
    """A call in one line of runs and a whole prompt, captured; lengths, tables and queries change between replays, with eager work of the
    same cache between them.  Every replay equals the eager call."""
    g = _gen(41)
    G, H, D, ps, S = 8, 16, 128, 32, 40
    lens = [1000 - 20 * i for i in range(S)]
    kv = _cache(dtype, G, D, ps, lens, width=60)
    _fill(kv, 0, lens, g)
    rows = torch.arange(S, dtype=torch.int32, device=DEV)
    q = _randn(g, S, H, D, dtype=torch.bfloat16)
    qp = _randn(g, 300, H, D, dtype=torch.bfloat16)
    off = _offsets([200, 100])
    s = torch.cuda.Stream()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=s):
            graphs.append((graph, kv.attend(0, q, rows, window=1000, sinks=4), kv.attend(0, qp, rows[:2], off)))
    for i in range(4):
        q.copy_(_randn(g, S, H, D))
        qp.copy_(_randn(g, 300, H, D))
        kv.lens.copy_(torch.tensor([max(0, n - 231 * i * (j % 3)) for j, n in enumerate(lens)], dtype=torch.int32))
        kv.table[2:4] = kv.table[2:4].flip(0).clone()
        a, b = kv.attend(0, q, rows, window=1000, sinks=4), kv.attend(0, qp, rows[:2], off)
        torch.cuda.synchronize()
        streams = (torch.cuda.current_stream(), s)
        for st, (graph, _, _) in zip(streams, graphs):              # both at once
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for _, c, d in graphs:
            # bits: a row that took over a table whose last places nobody wrote sees their NaN
            assert torch.equal(a.view(torch.int16), c.view(torch.int16)) and torch.equal(b.view(torch.int16), d.view(torch.int16)), i


def test_rows_of_a_very_wide_table():
    """A table of 2^25 entries a row: release, trim, reserve, fork and attend reach the last of them."""
    from qwen3_tts_amd.kvcache import PagedKV
    g = _gen(51)
    W, ps, D = 1 << 25, 8, 64
    kv = PagedKV(1, 1, D, 12, ps, rows=2, pages_per_row=W, dtype="f32", device=DEV)
    kv.lens[0] = W * ps - 9                                          # as after a long stream whose pages were trimmed
    kv.table[0, 0], kv.table[0, W - 2] = 0, 1
    kv.refs[:2] = 1
    kv.reserve([0], _offsets([8]), tokens=8)
    assert int(kv.table[0, W - 1]) == 2 and int(kv.lens[0]) == W * ps - 1
    x = _randn(g, 8, 1, D)
    rows = torch.zeros(1, dtype=torch.int32, device=DEV)
    kv.append(0, x, x, x, rows, _offsets([8]))
    out = kv.attend(0, x[-1:], rows, window=2 ** 31 - 1, sinks=2 ** 31 - 1)
    near = kv.attend(0, x[-1:], rows, window=8)
    want, mag, dot = attention(x[-1:], x, x, [7], 0, 0, D ** -0.5)
    _check_attend(near, want, mag, dot, kv, 8, D ** -0.5)
    kk = torch.cat([x.new_zeros(8 + 7, 1, D), x])                    # the first page, what the last but one held before
    want, mag, dot = attention(x[-1:], kk, kk, [22], 0, 0, D ** -0.5)
    _check_attend(out, want, mag, dot, kv, 23, D ** -0.5)
    kv.fork([0], [1])
    assert int(kv.table[1, W - 2]) == 1 and int(kv.table[1, W - 1]) == 3
    kv.trim([1], window=7, sinks=0)
    assert kv.table[1, :1].tolist() == [-1] and int(kv.table[1, W - 2]) == -1 and int(kv.table[1, W - 1]) == 3
    kv.check()
    kv.release([0, 1])
    assert kv.free_pages() == 12 and bool((kv.table == -1).all())
    kv.check()


def test_tensors_that_ask_for_gradients_are_refused():
    kv = _cache("f32", 1, 64, 16, [20])
    rows = torch.zeros(1, dtype=torch.int32, device=DEV)
    q, k = (torch.zeros(1, 1, 64, device=DEV, requires_grad=r) for r in (True, False))
    for call in (lambda: kv.attend(0, q, rows), lambda: kv.append(0, q, k, k, rows), lambda: kv.append(0, k, k, q, rows)):
        with pytest.raises(ValueError, match="gradient"):
            call()
    with torch.no_grad():
        kv.append(0, q, q, q, rows)
    kv.check()


@pytest.mark.parametrize("dtype,D,G,group,ps", [("bf16", 128, 2, 8, 32), ("bf16", 64, 1, 20, 8), ("bf16", 256, 4, 3, 64), ("bf16", 80, 3, 5, 16), ("bf16", 16, 12, 1, 256),
                                                ("int4", 64, 8, 17, 16), ("int4", 128, 17, 8, 8), ("int4", 128, 8, 17, 32), ("int4", 256, 4, 9, 128), ("int4", 256, 12, 3, 8)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (72, 0), (90, 10)])
def test_attend_prompts_with_many_heads(dtype, D, G, group, ps, window, sinks):
    """Enough columns for the kernel that shares key tiles between waves, in each type and head size: a whole prompt, a piece behind a past,
    a row of one token, an empty one; a missing page and one outside the pool; NaN where no query of a token looks; captured."""
    g = _gen(D * 7 + group + window)
    lens, new = [400, 333, 1, 0, 170], [400, 200, 1, 0, 160]
    kv = _cache(dtype, G, D, ps, lens)
    store = _fill(kv, 0, lens, g)
    T = sum(new)
    q = _randn(g, T + 2, G * group, D).mul_(2).to(kv.activations)
    out = torch.full_like(q, 5.0)
    rows = torch.arange(5, dtype=torch.int32, device=DEV)
    kv.attend(0, q, rows, _offsets(new), window=window, sinks=sinks, out=out)
    kv.check()
    assert bool((out[T:] == 5.0).all())
    scale = D ** -0.5
    for r, start, some in ((0, 0, [0, 31, 64, 127, 257, 399]), (1, 400, [0, 63, 199]), (2, 600, [0]), (4, 601, [0, 159])):
        i = torch.tensor(some, device=DEV)
        pos = [lens[r] - new[r] + p for p in some]
        want, mag, dot = attention(q[start + i], *store[r], pos, window, sinks, scale)
        _check_attend(out[start + i], want, mag, dot, kv, lens[r], scale, q[start + i].double(), prompt=True)
    graph, off = torch.cuda.CUDAGraph(), _offsets(new)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        again = kv.attend(0, q, rows, off, window=window, sinks=sinks)
    for _ in range(3):
        again.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(again[:T], out[:T])

    page, slot = int(kv.table[1, 250 // ps]), 250 % ps              # position 250 of the second row: token 117 of its piece
    where = kv.v_scale[0, page, G - 1, slot, 1:2] if dtype == "int4" else kv.v[0, page, G - 1, slot, 3:4]
    was = where.clone()
    where.fill_(float("inf") if dtype == "int4" else float("nan"))
    got = kv.attend(0, q, rows, _offsets(new), window=window, sinks=sinks)
    where.copy_(was)
    sees = torch.zeros(T, dtype=torch.bool, device=DEV)
    sees[400 + 117:600 if not window else min(600, 400 + 117 + window)] = True
    # Not bit for bit what it was: such a tile is computed again position by position, and the maximum that its probabilities are rounded against
    # moves for a whole wave at a time.  Each result by itself is within the bound of the formula, in which the bad row has no part.
    assert bool(torch.isfinite(got[:T][~sees]).all())
    for tok in (0, 63, 110, 116, 189, 199):
        if not bool(sees[400 + tok]):
            want, mag, dot = attention(q[400 + tok:401 + tok], *store[1], [133 + tok], window, sinks, scale)
            _check_attend(got[400 + tok:401 + tok], want, mag, dot, kv, 333, scale, q[400 + tok:401 + tok].double(), prompt=True)
    assert not bool(torch.isfinite(got[:T][sees][:, (G - 1) * group:]).all(-1).any())

    kv.table[0, 32 // ps] = -1
    kv.table[0, 300 // ps] = kv.pages + 1
    there = torch.ones(400, dtype=torch.bool, device=DEV)
    for p in (32, 300):
        there[p // ps * ps:p // ps * ps + ps] = False
    got = kv.attend(0, q, rows, _offsets(new), window=window, sinks=sinks)
    i = torch.tensor([0, 31, 64, 127, 257, 330, 399], device=DEV)
    want, mag, dot = attention(q[i], *store[0], i.tolist(), window, sinks, scale, there)
    _check_attend(got[i], want, mag, dot, kv, 400, scale, q[i].double(), prompt=True)


def test_numbers_that_32_bits_do_not_hold_are_refused():
    kv = _cache("bf16", 1, 64, 16, [20])
    rows = torch.zeros(1, dtype=torch.int32, device=DEV)
    q = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device=DEV)
    for kw in (dict(window=2 ** 32 + 5), dict(window=4, sinks=2 ** 31), dict(max_len=2 ** 33 + 1)):
        with pytest.raises(ValueError):
            kv.attend(0, q, rows, **kw)
    for window, sinks in ((2 ** 32 + 1, 0), (1, 2 ** 32)):
        with pytest.raises(ValueError):
            kv.trim(rows, window, sinks)
    for call in (lambda: kv.reserve(rows, _offsets([1]), tokens=2 ** 32), lambda: kv.gather(0, rows, _offsets([1]), tokens=2 ** 32 + 1),
                 lambda: kv.reserve(rows, _offsets([1]), tokens=-1)):
        with pytest.raises(ValueError):
            call()
    assert int(kv.lens[0]) == 20 and kv.table[0, :2].tolist().count(-1) == 0
    kv.check()


@pytest.mark.parametrize("dtype", ["bf16", "f32", "int4"])
def test_one_token_of_a_projection_of_odd_width(dtype):
    """q, k and v as views of one row of a wider matrix: its row stride, 3 past a multiple of four, belongs to a dimension of one element."""
    g = _gen(61)
    G, H, D = 1, 2, 64
    kv = _cache(dtype, G, D, 16, [20, 7])
    _fill(kv, 0, [20, 7], g)
    for T in (1, 2):
        x = _randn(g, 3, (H + 2 * G) * D + 3, dtype=kv.activations)
        q, k, v = (t.unflatten(1, (-1, D))[:T] for t in x[:, :(H + 2 * G) * D].split([H * D, G * D, G * D], 1))
        rows = torch.arange(T, dtype=torch.int32, device=DEV)
        assert q.stride(0) % 4
        a = kv.append(0, q, k, v, rows)
        assert torch.equal(a, q)
        kk, vv = kv.gather(0, rows)
        out = kv.attend(0, q, rows)
        copies = [t.clone(memory_format=torch.contiguous_format) for t in (q, k, v)]
        kv.append(0, *copies, rows)
        k2, v2 = kv.gather(0, rows)
        assert torch.equal(kk, k2) and torch.equal(vv, v2) and torch.equal(kv.attend(0, copies[0], rows), out)
    kv.check()


@pytest.mark.parametrize("dtype", ["bf16", "int4"])
def test_captured_page_operations_replay(dtype):
    """fork, append, gather, copy, trim, release and compact captured in one graph and replayed four times, each time equal to the same calls
    run eagerly on a twin, with eager work of both between."""
    from qwen3_tts_amd.kvcache import PagedKV
    G, D, ps = 2, 64, 8
    pair = [PagedKV(2, G, D, 90, ps, rows=6, pages_per_row=20, dtype=dtype, device=DEV) for _ in range(2)]
    rows = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    children = torch.tensor([3, 2, 5], dtype=torch.int32, device=DEV)
    parents = torch.tensor([0, 1, 0], dtype=torch.int32, device=DEV)
    src, dst = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([1, 3, 3], [80, 81, 80]))
    x = torch.zeros(3, G, D, dtype=torch.bfloat16, device=DEV)
    g = _gen(71)
    for kv in pair:
        kv.reserve(rows, _offsets([45, 70]), tokens=115)
        y = _randn(_gen(72), 115, G, D, dtype=torch.bfloat16)
        for layer in (0, 1):
            kv.append(layer, y, y, -y, rows, _offsets([45, 70]))

    def calls(kv):
        kv.fork(parents, children)
        kv.reserve(children)
        kv.append(1, x, x, x, children)
        kv.copy_pages(src, dst)
        kv.trim(children, 20, 3)
        live = kv.compact()
        k, v = kv.gather(1, children)
        out = kv.attend(1, x, children, window=20, sinks=3)
        kv.release(children)
        return live, k, v, out
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = calls(pair[0])
    for i in range(4):
        x.copy_(_randn(g, 3, G, D))
        graph.replay()
        want = calls(pair[1])
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), i
        for n in ("table", "lens", "refs"):
            assert torch.equal(getattr(pair[0], n), getattr(pair[1], n)), (i, n)
        assert torch.equal(pair[0].k, pair[1].k) and torch.equal(pair[0].v, pair[1].v)
        for kv in pair:                                            # the parents grow between
            kv.check()
            kv.reserve(rows)
            for layer in (0, 1):
                kv.append(layer, x[:2], x[:2], x[1:], rows)


@pytest.mark.parametrize("dtype", ["bf16", "int4"])
def test_a_traced_step_is_the_eager_one(dtype):
    """Two layers whose first append's queries nobody takes, and attends before and behind an append: compiled, where functionalization gives
    the ops copies of the cache, the outputs and the cache are bit for bit those of the calls made eagerly on a twin."""
    from qwen3_tts_amd import torch_ops
    from qwen3_tts_amd.kvcache import PagedKV
    g = _gen(81)
    G, H, D = 2, 4, 64
    pair = [PagedKV(2, G, D, 30, 16, rows=3, pages_per_row=8, dtype=dtype, device=DEV) for _ in range(2)]
    rows, off = torch.tensor([2, 0], dtype=torch.int32, device=DEV), _offsets([40, 33])
    x = [_randn(g, 73, n, D, dtype=torch.bfloat16) for n in (H, G, G)]
    y = [_randn(g, 2, n, D, dtype=torch.bfloat16) for n in (H, G, G)]
    handles = [torch_ops.register_kv(kv) for kv in pair]

    def prefill(kv, h, q, k, v):
        for layer in (0, 1):
            torch.ops.q3tts.kv_append(q, k, v, rows, off, None, None, None, None, 1e-6, h, layer, *kv.state)

    def step(kv, h, q, k, v):
        a = torch.ops.q3tts.kv_attend(q, rows, None, 20, 2, h, 1, *kv.state)
        torch.ops.q3tts.kv_append(q, k, v, rows, None, None, None, None, None, 1e-6, h, 1, *kv.state)
        return a, torch.ops.q3tts.kv_attend(q, rows, None, 20, 2, h, 1, *kv.state)
    results = []
    for kv, h, wrap in zip(pair, handles, (lambda f: f, lambda f: torch.compile(f, backend="aot_eager", fullgraph=True))):
        kv.reserve(rows, off, tokens=73)
        wrap(lambda *a, kv=kv, h=h: prefill(kv, h, *a))(*x)
        kv.reserve(rows)
        results.append(wrap(lambda *a, kv=kv, h=h: step(kv, h, *a))(*y))
        kv.check()
    (a0, b0), (a1, b1) = results
    assert torch.equal(a0, a1) and torch.equal(b0, b1) and not torch.equal(a0, b0)
    for s, t in zip(pair[0].state, pair[1].state):
        assert s is None and t is None or torch.equal(s, t)
    for h in handles:
        torch_ops.unregister_kv(h)
    torch._dynamo.reset()


@pytest.mark.parametrize("dtype", ["bf16", "f32", "int4"])
def test_offsets_that_end_behind_the_tokens_mean_one_thing(dtype):
    """Offsets [0, 3, 9] in a call of 5 tokens: every call takes the second row's tokens to be the two that are there, and reports it."""
    from qwen3_tts_amd import _lib
    g = _gen(91)
    G, H, D = 2, 4, 64
    kv = _cache(dtype, G, D, 16, [20, 30])
    store = _fill(kv, 0, [20, 30], g)
    kv.check()
    rows, off, fits = torch.tensor([0, 1], dtype=torch.int32, device=DEV), _offsets([3, 6]), _offsets([3, 2])
    x = [_randn(g, 5, n, D, dtype=kv.activations) for n in (H, G, G)]
    kv.reserve(rows, off, tokens=5)
    assert kv.lens.tolist() == [23, 32]
    with pytest.raises(_lib.Q3cError, match="the call's tokens"):
        kv.check()
    q = kv.append(0, *x, rows, off)
    with pytest.raises(_lib.Q3cError, match="the call's tokens"):
        kv.check()
    assert torch.equal(q, x[0])
    back = kv.gather(0, rows, off, tokens=5, dtype="f32")
    with pytest.raises(_lib.Q3cError, match="the call's tokens"):
        kv.check()
    kk, vv = kv.gather(0, rows, fits, tokens=5, dtype="f32")
    assert torch.equal(back[0], kk) and torch.equal(back[1], vv)
    if dtype != "int4":
        assert torch.equal(kk, x[1].float()) and torch.equal(vv, x[2].float())
    out = kv.attend(0, q, rows, off)
    kv.check()
    for r, s, L in ((0, slice(0, 3), 23), (1, slice(3, 5), 32)):
        k, v = (torch.cat([a, b[s].double()]) for a, b in zip(store[r], (kk, vv)))
        n = s.stop - s.start
        want, mag, dot = attention(q[s], k, v, list(range(L - n, L)), 0, 0, D ** -0.5)
        _check_attend(out[s], want, mag, dot, kv, L, D ** -0.5, q[s].double())


def test_attend_leaves_the_status_alone():
    """Bad rows, missing pages and pages outside the pool give zeros and unseen keys; what says so is the append before."""
    from qwen3_tts_amd import _lib
    g = _gen(92)
    kv = _cache("bf16", 1, 64, 16, [40, 20])
    _fill(kv, 0, [40, 20], g)
    kv.check()
    kv.table[0, 0], kv.table[1, 1] = kv.pages + 3, -1
    rows = torch.tensor([0, 1, 7], dtype=torch.int32, device=DEV)
    q, k = _randn(g, 3, 2, 64, dtype=torch.bfloat16), _randn(g, 3, 1, 64, dtype=torch.bfloat16)
    out = kv.attend(0, q, rows)
    kv.check()
    assert bool((out[2] == 0).all()) and bool(torch.isfinite(out).all())
    kv.append(0, q, k, k, rows)
    with pytest.raises(_lib.Q3cError, match="row id.*has no page"):
        kv.check()


@pytest.mark.parametrize("dtype,D,G,group,ps", [("bf16", 80, 4, 8, 16), ("bf16", 16, 8, 4, 8), ("bf16", 208, 4, 8, 32), ("f32", 80, 2, 2, 16), ("f32", 48, 2, 2, 8),
                                                ("f32", 208, 1, 2, 32), ("bf16", 128, 4, 8, 16), ("f32", 64, 2, 2, 16)])
def test_a_key_of_minus_infinity_has_no_weight_in_any_head_size(dtype, D, G, group, ps):
    """A key whose product with every query is -inf counts as little as one that is not there, also where the head is padded to the matrix
    instructions' size: through single tokens (short, long and many rows), pieces and prompts."""
    g = _gen(D + G)
    lens = [260, 410, 33]
    kv = _cache(dtype, G, D, ps, lens, width=1024)
    store = _fill(kv, 0, lens, g)
    there = [torch.ones(L, dtype=torch.bool, device=DEV) for L in lens]
    for r, pos, dim in ((0, 7, 3), (0, 100, 0), (1, 200, 1), (1, 31, 7), (2, 9, D - 1)):
        kv.k[0, int(kv.table[r, pos // ps]), :, pos % ps, dim] = -float("inf")
        there[r][pos] = False

    def queries(n):
        q = _randn(g, n, G * group, D).to(kv.activations)
        for d in (0, 1, 3, 7, D - 1):
            q[..., d] = q[..., d].abs() + 0.5
        return q

    def look(out, q, rows, pos):
        assert bool(torch.isfinite(out).all())
        for i, (r, p) in enumerate(zip(rows, pos)):
            want, mag, dot = attention(q[i:i + 1], *store[r], [p], 0, 0, D ** -0.5, there[r])
            _check_attend(out[i:i + 1], want, mag, dot, kv, lens[r], D ** -0.5, q[i:i + 1].double())
    rows = torch.arange(3, dtype=torch.int32, device=DEV)
    q = queries(3)
    for max_len in (410, 0):                                        # whole rows, and (a table of 1 024 pages) rows that are cut
        look(kv.attend(0, q, rows, max_len=max_len), q, range(3), [L - 1 for L in lens])
    many = torch.arange(600, dtype=torch.int32, device=DEV) % 3
    q = queries(600)
    for max_len in (410, 0):
        out = kv.attend(0, q, many, max_len=max_len)
        look(out[:3], q[:3], range(3), [L - 1 for L in lens])
        look(out[-3:], q[-3:], range(3), [L - 1 for L in lens])
    for new in ([5, 3, 2], lens):
        q = queries(sum(new))
        out = kv.attend(0, q, rows, _offsets(new))
        at = 0
        for r, (L, n) in enumerate(zip(lens, new)):
            some = sorted({0, n // 2, n - 1})
            i = torch.tensor([at + x for x in some], device=DEV)
            look(out[i], q[i], [r] * len(some), [L - n + x for x in some])
            at += n
    out = kv.attend(0, q, rows, _offsets(lens), window=50, sinks=10)
    assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("D,G,group,ps", [(64, 8, 8, 8), (64, 16, 4, 32), (128, 8, 8, 16), (128, 16, 4, 32), (256, 8, 2, 64), (256, 4, 8, 8)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (500, 7)])
def test_prompts_over_four_bits_take_keys_as_they_are(D, G, group, ps, window, sinks):
    """A prompt on the kernel of 128 columns is held to the bound of single tokens, and one rounding of the values to bf16 (u of the mean of |v|):
    nothing is rounded in front of the scores.  Steps and queries of very unlike sizes among it, and a key whose step is NaN."""
    g = _gen(D + G + window)
    lens, new = [900, 777], [850, 777]
    kv = _cache("int4", G, D, ps, lens)
    off = _offsets(lens)
    k, v = (_randn(g, sum(lens), G, D).mul_(2) for _ in range(2))
    k[::7] *= 2.0 ** -30                                            # whole keys
    k[:, :, :32] *= 2.0 ** -12                                      # a group of every key
    k[3::11] *= 2.0 ** 5
    rows = torch.arange(2, dtype=torch.int32, device=DEV)
    kv.append(0, k.bfloat16(), k.bfloat16(), v.bfloat16(), rows, off)
    kk, vv = kv.gather(0, rows, off, tokens=sum(lens), dtype="f32")
    store = list(zip(kk.double().split(lens), vv.double().split(lens)))
    kv.k_scale[0, int(kv.table[1, 600 // ps]), 0, 600 % ps, 1] = float("nan")
    q = _randn(g, sum(new), G * group, D).mul_(2)
    q[::3] *= 2.0 ** -40
    q[1::5, :, : D // 2] *= 2.0 ** -9
    q = q.bfloat16()
    out = kv.attend(0, q, rows, _offsets(new), window=window, sinks=sinks)
    scale = D ** -0.5
    for r, start, some in ((0, 0, [0, 127, 128, 400, 849]), (1, 850, [0, 31, 64, 300, 599])):
        i = torch.tensor([start + x for x in some], device=DEV)
        pos = [lens[r] - new[r] + x for x in some]
        want, mag, dot = attention(q[i], *store[r], pos, window, sinks, scale)
        score = (D + 4) * 2.0 ** -24 * dot * scale + 8 * 144 * 2.0 ** -24 * float(q[i].double().abs().sum(-1).max()) * float(kv.k_scale.float().nan_to_num(0.0).max()) * scale
        u = 2.0 ** -8
        bound = (2 * u * 1.05 + 2 * score + 2.0 ** -20 + lens[r] * 2.0 ** -24) * mag + u * want.abs() * 1.01
        off_by = (out[i].double() - want).abs()
        assert bool((off_by <= bound + 1e-30).all()), (r, float((off_by - bound).max()))
    after = [850 + x for x in (600, 601, 776)]
    assert not bool(torch.isfinite(out[after][:, :group]).any()) if not window else not bool(torch.isfinite(out[after[:2]][:, :group]).any())
    assert bool(torch.isfinite(out[after][:, group:]).all())


def _time(call):
    """The least of some runs, in ms."""
    for _ in range(3):
        call()
    best = math.inf
    for _ in range(7):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        for _ in range(3):
            call()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b) / 3)
    return best


SECOND = [("bf16", 128, 4, 4, 16), ("bf16", 64, 1, 2, 32), ("bf16", 80, 4, 8, 16), ("int4", 128, 8, 8, 32), ("int4", 64, 1, 3, 8), ("int4", 256, 4, 4, 16), ("f32", 64, 2, 2, 16)]


@pytest.mark.parametrize("dtype,D,G,group,ps", SECOND)
def test_one_bad_row_or_token_does_not_multiply_the_time(dtype, D, G, group, ps):
    """A value that is not finite, seen by every later token (the first position, a sink), and a query that is not: neither is worth a second
    look at every tile, one for each of its positions.  Four times are left for the tile that holds the row."""
    g = _gen(D + G + 5)
    lens = [1700]
    kv = _cache(dtype, G, D, ps, lens)
    _fill(kv, 0, lens, g)
    rows, off = torch.zeros(1, dtype=torch.int32, device=DEV), _offsets([1500])
    q = _randn(g, 1500, G * group, D).to(kv.activations)
    out = torch.empty_like(q)

    def run():
        return kv.attend(0, q, rows, off, window=0, out=out)
    clean = _time(run)
    keep = out.clone()
    q[777] = float("nan")
    query = _time(run)
    assert bool(torch.isnan(out[777]).all()) and bool(torch.isfinite(out[:777]).all()) and bool(torch.isfinite(out[778:]).all())
    q[777] = 0.0
    page = int(kv.table[0, 0])
    (kv.v_scale if dtype == "int4" else kv.v)[0, page, G - 1, 2, 1] = float("inf")
    value = _time(run)
    assert torch.equal(out[:777, :(G - 1) * group], keep[:777, :(G - 1) * group]) and not bool(torch.isfinite(out[:, (G - 1) * group:]).all(-1).any())
    assert query < 4 * clean and value < 4 * clean, (clean, query, value)


@pytest.mark.parametrize("dtype,D,G,group,ps", SECOND)
@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 3)])
def test_bad_values_stay_with_the_tokens_that_see_them(dtype, D, G, group, ps, window, sinks):
    """Infinities and NaN in values of other dimensions: one at the first position (a sink of all), one between, one that enters and leaves the
    window inside tiles.  Every output element is finite or not as the rows that its token sees say, and the finite ones are right."""
    g = _gen(D + G + 6)
    lens, new = [1000, 60], [900, 60]
    kv = _cache(dtype, G, D, ps, lens)
    store = [[k.clone(), v.clone()] for k, v in _fill(kv, 0, lens, g)]
    bad = {0: (1, float("inf")), 333: (40, float("nan")), 650: (D - 1, -float("inf")), 651: (D - 1, float("inf"))}
    for pos, (dim, x) in bad.items():
        page, slot = int(kv.table[0, pos // ps]), pos % ps
        if dtype == "int4":
            kv.v_scale[0, page, :, slot, dim // 32] = x
            store[0][1][pos, :, dim // 32 * 32:dim // 32 * 32 + 32] = float("nan")      # n times an infinite step: of either sign, or NaN
        else:
            kv.v[0, page, :, slot, dim] = x
            store[0][1][pos, :, dim] = x
    q = _randn(g, sum(new), G * group, D).to(kv.activations)
    rows = torch.arange(2, dtype=torch.int32, device=DEV)
    out = kv.attend(0, q, rows, _offsets(new), window=window, sinks=sinks)
    some = [0, 1, 127, 128, 230, 232, 233, 240, 255, 256, 400, 530, 532, 533, 534, 548, 549, 550, 551, 560, 700, 830, 845, 849, 850, 851, 852, 899]
    for i in some:
        p = 100 + i
        see = [x for x in range(p + 1) if not window or x > p - window or x < sinks]
        v, finite = store[0][1][see], torch.isfinite(store[0][1][see]).all(0)                        # [G, D]
        finite = finite.repeat_interleave(group, 0)
        assert torch.equal(torch.isfinite(out[i]), finite), i
        want, mag, dot = attention(q[i:i + 1], store[0][0], store[0][1].nan_to_num(0.0, 0.0, 0.0), [p], window, sinks, D ** -0.5)
        got = torch.where(finite, out[i], want[0].to(out.dtype))
        _check_attend(got[None], want, mag, dot, kv, p + 1, D ** -0.5, q[i:i + 1].double(), prompt=True)
    assert bool(torch.isfinite(out[900:]).all())


def test_weights_tables_and_outputs_that_ask_for_gradients_are_refused():
    """A module's parameters, as they are, outside torch.no_grad(): their gradients would be cut off without a word."""
    kv = _cache("bf16", 1, 64, 16, [20])
    rows = torch.zeros(1, dtype=torch.int32, device=DEV)
    q = torch.ones(1, 1, 64, dtype=torch.bfloat16, device=DEV)
    w = torch.nn.Parameter(torch.ones(64, device=DEV))
    cos, sin = (torch.ones(kv.max_tokens, 32, device=DEV, requires_grad=r) for r in (True, False))
    out = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    calls = [lambda: kv.append(0, q, q, q, rows, q_weight=w), lambda: kv.append(0, q, q, q, rows, k_weight=w), lambda: kv.append(0, q, q, q, rows, rope=(cos, sin)),
             lambda: kv.append(0, q, q, q, rows, rope=(sin, cos)), lambda: kv.append(0, q, q, q, rows, out=out), lambda: kv.attend(0, q, rows, out=out)]
    for call in calls:
        with pytest.raises(ValueError, match="gradient"):
            call()
    assert bool(torch.isnan(kv.k[0, int(kv.table[0, 1]), 0, 3]).all())      # nothing was written
    with torch.no_grad():
        for call in calls:
            call()
    kv.check()


def test_ids_that_are_no_whole_numbers_are_refused():
    import numpy as np
    kv = _cache("bf16", 1, 64, 16, [20, 7])
    for call in (lambda: kv.release([0.9]), lambda: kv.trim([1.0], 4), lambda: kv.copy_pages([0.5], [1]), lambda: kv.fork([0], ["1"]), lambda: kv.reserve([None])):
        with pytest.raises(TypeError):
            call()
    assert kv.lens.tolist() == [20, 7]
    kv.reserve(np.array([1, 0]))
    assert kv.lens.tolist() == [21, 8]
    kv.check()


# ---- which kernel a call takes, and what only long rows reach ------------------------------------------------------------------------
def _kernels(call):
    """Names of the cache's kernels that a call launches."""
    import re
    from torch.profiler import ProfilerActivity, profile
    call()
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        call()
        torch.cuda.synchronize()
    return {m.group(1) for e in p.key_averages() for m in [re.search(r"(kv_[a-z_]+?_kernel)", e.key)] if m}


def _check_tight(got, q, k, v, pos, window, sinks, kv, N, there=None, prompt=False):
    """As _check_attend, but keys count as unrounded everywhere; `prompt`: values over 4 bits are rounded to bf16 once (u of the mean of |v|)."""
    scale = kv.head_dim ** -0.5
    want, mag, dot = attention(q, k, v, pos, window, sinks, scale, there)
    if not (prompt and kv.dtype == "int4"):
        return _check_attend(got, want, mag, dot, kv, N, scale, q.double())
    u = 2.0 ** -8
    top = float(kv.k_scale.float().nan_to_num(0.0).max())
    score = (kv.head_dim + 4) * 2.0 ** -24 * dot * scale + 8 * 144 * 2.0 ** -24 * float(q.double().abs().sum(-1).max()) * top * scale
    bound = (2 * u * 1.05 + 2 * score + 2.0 ** -20 + N * 2.0 ** -24) * mag + u * want.abs() * 1.01
    off_by = (got.double() - want).abs()
    assert bool((off_by <= bound + 1e-30).all()), f"max excess {float((off_by - bound).max()):.3e}"


@pytest.mark.parametrize("dtype,D,G,group,ps,L", [("bf16", 128, 2, 8, 8, 1600), ("bf16", 64, 4, 4, 32, 3100), ("bf16", 256, 2, 8, 16, 1300), ("bf16", 80, 4, 4, 8, 1500),
                                                  ("int4", 64, 8, 8, 8, 1600), ("int4", 128, 8, 8, 32, 3100), ("int4", 256, 4, 8, 8, 1500)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (700, 5), (130, 1000)])
def test_prompts_over_more_pages_than_a_wave_has_lanes(dtype, D, G, group, ps, L, window, sinks):
    """The prompt kernel holds 64 entries of the table at a time: rows of 81 to 200 pages, read from front to back, and from the sinks to the window's
    start; whole prompts and a piece behind a past; a missing page and one outside the pool among the later ones."""
    g = _gen(D + L + window)
    lens, new = [L, L - 77], [L, 500]
    kv = _cache(dtype, G, D, ps, lens)
    store = _fill(kv, 0, lens, g)
    there = [torch.ones(n, dtype=torch.bool, device=DEV) for n in lens]
    for r, pos, value in ((0, L - 300, -1), (1, L - 400, kv.pages + 5), (1, 65 * ps, -1)):
        j = pos // ps
        kv.table[r, j] = value
        there[r][j * ps:(j + 1) * ps] = False
    q = _randn(g, sum(new), G * group, D).mul_(2).to(kv.activations)
    rows = torch.arange(2, dtype=torch.int32, device=DEV)
    out = torch.empty_like(q)
    assert _kernels(lambda: kv.attend(0, q, rows, _offsets(new), window=window, sinks=sinks, out=out)) == {"kv_prompt_kernel"}
    for r, start, some in ((0, 0, [0, 63, 64 * ps - 1, 64 * ps, 65 * ps + 3, L - 301, L - 150, L - 1]), (1, L, [0, 5, 130, 499])):
        i = torch.tensor([start + x for x in some], device=DEV)
        _check_tight(out[i], q[i], *store[r], [lens[r] - new[r] + x for x in some], window, sinks, kv, L, there[r], prompt=True)


@pytest.mark.parametrize("dtype,D,G,group,ps", [("bf16", 128, 2, 2, 16), ("bf16", 64, 1, 5, 8), ("bf16", 256, 1, 4, 32), ("bf16", 80, 2, 3, 8), ("int4", 128, 2, 2, 16), ("int4", 64, 1, 7, 8),
                                                ("int4", 256, 2, 1, 64), ("f32", 64, 2, 2, 16), ("f32", 128, 1, 3, 8)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (3000, 40)])
def test_pieces_behind_a_long_past_are_cut_and_joined(dtype, D, G, group, ps, window, sinks):
    """A few tokens of each request behind thousands: tiles of several positions whose keys are cut into shares."""
    g = _gen(D + G + window)
    lens, new = [6001, 4096, 70, 5333], [5, 19, 2, 40]
    kv = _cache(dtype, G, D, ps, lens)
    store = _fill(kv, 0, lens, g)
    q = _randn(g, sum(new), G * group, D).mul_(2).to(kv.activations)
    rows = torch.arange(4, dtype=torch.int32, device=DEV)
    out = torch.empty_like(q)
    assert _kernels(lambda: kv.attend(0, q, rows, _offsets(new), window=window, sinks=sinks, out=out)) == {"kv_attend_kernel", "kv_join_kernel"}
    at = 0
    for r, n in enumerate(new):
        some = sorted({0, n // 2, n - 1})
        i = torch.tensor([at + x for x in some], device=DEV)
        _check_tight(out[i], q[i], *store[r], [lens[r] - n + x for x in some], window, sinks, kv, lens[r])
        at += n


@pytest.mark.parametrize("dtype", ["bf16", "f32", "int4"])
def test_which_kernel_a_call_takes(dtype):
    """The rule for each kernel, by a call on either side of it: many columns a request, one token of long rows, short rows, and the rest."""
    G, group, D, ps = 8, 4, 128, 32
    kv = _cache(dtype, G, D, ps, [1] * 600, width=300)
    rows = torch.arange(600, dtype=torch.int32, device=DEV)

    def names(new, n, **kw):
        q = torch.zeros(new * n, G * group, D, dtype=kv.activations, device=DEV)
        off = None if new == 1 else torch.arange(0, new * n + 1, new, dtype=torch.int32, device=DEV)
        return _kernels(lambda: kv.attend(0, q, rows[:n], off, **kw))
    flat, cut, whole, short, prompt = {"kv_flat_kernel", "kv_flat_join_kernel"}, {"kv_attend_kernel", "kv_join_kernel"}, {"kv_attend_kernel"}, {"kv_short_kernel"}, {"kv_prompt_kernel"}
    assert names(1, 64) == flat and names(1, 64, max_len=200) == whole
    assert names(1, 2) == (flat if dtype == "f32" else cut) and names(1, 2, max_len=500) == whole       # (fp32 chunks are half as long)
    assert names(1, 600, max_len=200) == flat and names(1, 600, max_len=15) == short
    assert names(4, 300, window=60) == short and names(4, 20, window=60) == whole
    assert names(800, 4) == (whole if dtype == "f32" else prompt)
    assert names(10, 4) == cut


@pytest.mark.parametrize("dtype,D", [("bf16", 64), ("bf16", 80), ("f32", 64), ("f32", 256)])
def test_scores_that_are_all_minus_infinity_give_zeros(dtype, D):
    """Rows whose every visible key is -inf against the query: as if nothing were seen, in single tokens, cut rows, pieces and prompts."""
    g = _gen(D)
    G, group, lens = 4, 8, [3000, 500]
    kv = _cache(dtype, G, D, 16, lens, width=1024)
    _fill(kv, 0, lens, g)
    kv.k[0, :, :, :, 5] = -float("inf")
    rows = torch.arange(2, dtype=torch.int32, device=DEV)
    for new in (None, [3, 2], [700, 500]):
        T = 2 if new is None else sum(new)
        q = _randn(g, T, G * group, D).to(kv.activations)
        q[..., 5] = q[..., 5].abs() + 0.5
        for max_len in (0, 500):
            out = kv.attend(0, q, rows, None if new is None else _offsets(new), max_len=max_len)
            assert bool((out == 0).all()), (new, max_len)


def test_part_of_the_state_is_refused():
    from qwen3_tts_amd import torch_ops
    kv = _cache("bf16", 1, 64, 16, [20])
    _fill(kv, 0, [20], _gen(1))
    rows, q = torch.zeros(1, dtype=torch.int32, device=DEV), torch.ones(1, 2, 64, dtype=torch.bfloat16, device=DEV)
    h = torch_ops.register_kv(kv)
    want = kv.attend(0, q, rows)
    assert torch.equal(torch.ops.q3tts.kv_attend(q, rows, None, 0, 0, h, 0, *kv.state), want)
    for some in (kv.state[:2], (None,) + kv.state[1:]):
        with pytest.raises(ValueError, match="all of the cache's tensors"):
            torch.ops.q3tts.kv_attend(q, rows, None, 0, 0, h, 0, *some)
    other = tuple(None if t is None else t.clone() for t in kv.state)
    other[0].zero_()                                                # uniform weights: the mean of the values
    out = torch.ops.q3tts.kv_attend(q, rows, None, 0, 0, h, 0, *other)
    mean = kv.gather(0, rows, _offsets([20]), tokens=20, dtype="f32")[1].double().mean(0)
    assert float((out[0].double() - mean).abs().max()) <= 2.0 ** -8 * 2 * float(kv.v.float().nan_to_num(0.0).abs().max())
    torch_ops.unregister_kv(h)


@pytest.mark.parametrize("dtype,D,G,group,ps", SECOND)
@pytest.mark.parametrize("window", [0, 700])
def test_a_bad_token_amid_a_prompt_costs_its_tile_a_look_or_two(dtype, D, G, group, ps, window):
    """A token whose key and value are NaN, as a bad hidden state makes them, in the middle of a prompt: the positions of its tile before and
    behind it are looked at as two runs, not one by one (which took up to 33 looks), and so where it leaves the window."""
    g = _gen(D + G + 8)
    lens, pos = [1700], 200 + 901
    kv = _cache(dtype, G, D, ps, lens)
    _fill(kv, 0, lens, g)
    rows, off = torch.zeros(1, dtype=torch.int32, device=DEV), _offsets([1500])
    q = _randn(g, 1500, G * group, D).to(kv.activations)
    out = torch.empty_like(q)

    def run():
        return kv.attend(0, q, rows, off, window=window, out=out)
    clean = _time(run)
    keep = out.clone()
    for t in (kv.k_scale, kv.v_scale) if dtype == "int4" else (kv.k, kv.v):
        t[0, int(kv.table[0, pos // ps]), :, pos % ps] = float("nan")
    bad = _time(run)
    sees = torch.zeros(1500, dtype=torch.bool, device=DEV)
    sees[901:min(1500, 901 + window) if window else 1500] = True
    assert bool(torch.isnan(out[sees]).all()) and bool(torch.isfinite(out[~sees]).all())
    assert torch.equal(out[:700], keep[:700])                       # (tiles that the token is in may round their probabilities otherwise)
    assert bad < 4 * clean, (clean, bad)
