"""What the paged key/value cache refuses on the host, without a GPU: sizes and layouts through the class, pointers, sizes and
workspaces through the C entry points (each refusal comes before any launch), and the fixed points of the plain restatement."""
import ctypes as C

import pytest
import torch

import qwen3_tts_amd  # noqa: F401
from kv_reference import Pages, attention, norm_rotate
from qwen3_tts_amd import _lib
from qwen3_tts_amd.kvcache import PagedKV, rope_tables

OK, INVALID, WORKSPACE, UNSUPPORTED = 0, -1, -4, -7
PTR = 1 << 20                     # an aligned address that no refused call touches


def _tensors(L=1, P=4, G=2, ps=16, D=64, dtype=torch.bfloat16, rows=3, width=2):
    i = dict(dtype=torch.int32)
    k = torch.zeros(L, P, G, ps, D, dtype=dtype)
    return dict(k=k, v=k.clone(), table=torch.zeros(rows, width, **i), lens=torch.zeros(rows, **i), refs=torch.zeros(P, **i))


@pytest.mark.parametrize("change", [
    dict(ps=12), dict(ps=4), dict(ps=512), dict(D=24), dict(D=272), dict(dtype=torch.float16), dict(dtype=torch.uint8), dict(P=0), dict(rows=0)])
def test_layouts_that_are_refused(change):
    with pytest.raises(ValueError):
        PagedKV.from_tensors(**_tensors(**change))


def test_tensors_that_are_refused():
    good = _tensors()
    for name, t in (("v", good["v"][..., :32]), ("v", good["v"].float()), ("table", good["table"].long()), ("table", good["table"][0]),
                    ("lens", good["lens"][:2]), ("refs", torch.zeros(5, dtype=torch.int32)), ("status", torch.zeros(2, dtype=torch.int32)),
                    ("k_scale", torch.zeros(1)), ("k", torch.zeros(1, 4, 16, 2, 64, dtype=torch.bfloat16).transpose(2, 3)),
                    ("k", good["k"][0])):
        with pytest.raises(ValueError):
            PagedKV.from_tensors(**{**good, name: t})
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        PagedKV.from_tensors(**good)
    for kw in (dict(dtype="fp16"), dict(layers=0), dict(pages_per_row=0), dict(dtype="int4", head_dim=80)):
        with pytest.raises(ValueError):
            PagedKV(**{**dict(layers=1, kv_heads=1, head_dim=64, pages=2, device="cpu"), **kw})


def test_cache_tensors_that_ask_for_gradients_are_refused():
    good = _tensors()
    for n in ("k", "v"):
        with pytest.raises(ValueError, match=f"{n} requires a gradient"):
            PagedKV.from_tensors(**{**good, n: good[n].clone().requires_grad_()})
        with pytest.raises(RuntimeError, match="no CPU fallback"), torch.no_grad():
            PagedKV.from_tensors(**{**good, n: good[n].clone().requires_grad_()})


def _kv(**change):
    c = _lib.Q3cKv()
    c.struct_size = C.sizeof(_lib.Q3cKv)
    c.dtype, c.layers, c.pages, c.kv_heads, c.page_size, c.head_dim, c.rows, c.pages_per_row = 1, 2, 8, 2, 16, 64, 4, 3
    for n in ("k", "v", "table", "lens", "refs", "status"):
        setattr(c, n, PTR)
    for n, v in change.items():
        setattr(c, n, v)
    return C.byref(c)


def test_c_entry_points_refuse_bad_descriptions():
    lib = _lib.load()
    for change, rc in ((dict(struct_size=8), INVALID), (dict(dtype=3), INVALID), (dict(dtype=-1), INVALID), (dict(layers=0), INVALID), (dict(pages=0), INVALID),
                       (dict(rows=0), INVALID), (dict(pages_per_row=0), INVALID), (dict(k=None), INVALID), (dict(k=PTR + 8), INVALID), (dict(status=None), INVALID),
                       (dict(page_size=24), UNSUPPORTED), (dict(page_size=512), UNSUPPORTED), (dict(page_size=4), UNSUPPORTED), (dict(head_dim=72), UNSUPPORTED),
                       (dict(head_dim=512), UNSUPPORTED), (dict(dtype=2), INVALID), (dict(dtype=2, head_dim=80, k_scale=PTR, v_scale=PTR), UNSUPPORTED),
                       (dict(pages_per_row=1 << 27), UNSUPPORTED), (dict(kv_heads=1 << 17), UNSUPPORTED)):
        kv = _kv(**change)
        n = C.c_size_t()
        assert lib.q3c_kv_reserve(kv, PTR, None, 1, 1, None) == rc, change
        assert lib.q3c_kv_append(kv, 0, PTR, 64, 64, PTR, 64, 64, PTR, 64, 64, 2, PTR, None, 1, 1, None, None, None, None, 0, 0, 1e-6, PTR, None) == rc, change
        assert lib.q3c_kv_gather(kv, 0, PTR, None, 1, 1, PTR, PTR, 1, None) == rc, change
        assert lib.q3c_kv_attend_workspace_bytes(kv, 1 << 17 if "kv_heads" in change else 2, 1, 1, 0, 0, 0, C.byref(n)) == rc, change
        assert lib.q3c_kv_attend(kv, 0, PTR, 64, 64, 2, PTR, None, 1, 1, 0, 0, 1.0, 0, PTR, PTR, 1 << 30, None) == rc, change
        assert lib.q3c_kv_fork(kv, PTR, PTR, 1, PTR, 12, None) == rc, change
        assert lib.q3c_kv_release(kv, PTR, 1, None) == rc and lib.q3c_kv_trim(kv, PTR, 1, 4, 0, None) == rc, change
        assert lib.q3c_kv_copy_pages(kv, PTR, PTR, 1, PTR, 4, None) == rc and lib.q3c_kv_compact(kv, PTR, PTR, 1 << 20, None) == rc, change
    assert lib.q3c_kv_reserve(None, PTR, None, 1, 1, None) == INVALID


def test_c_entry_points_refuse_bad_calls():
    lib, kv = _lib.load(), _kv()

    def append(layer=0, q=PTR, q_ts=256, q_hs=64, k_hs=64, heads=2, rows=PTR, offsets=None, seqs=1, tokens=1, w=None, cos=None, positions=0, rot=0, out=PTR, kv=kv):
        return lib.q3c_kv_append(kv, layer, q, q_ts, q_hs, PTR, 128, k_hs, PTR, 128, 64, heads, rows, offsets, seqs, tokens, w, None, cos, cos, positions, rot, 1e-6, out, None)
    for kw, rc in ((dict(layer=2), INVALID), (dict(layer=-1), INVALID), (dict(q=None), INVALID), (dict(q=PTR + 2), INVALID), (dict(q_ts=66), INVALID), (dict(k_hs=-64), INVALID),
                   (dict(heads=0), INVALID), (dict(rows=None), INVALID), (dict(seqs=2), INVALID), (dict(seqs=0, offsets=PTR), INVALID), (dict(tokens=-1), INVALID),
                   (dict(w=PTR + 4), INVALID), (dict(rot=64), INVALID), (dict(rot=64, cos=PTR, positions=47), INVALID), (dict(rot=12, cos=PTR, positions=48), UNSUPPORTED),
                   (dict(rot=72, cos=PTR, positions=48), UNSUPPORTED), (dict(out=None), INVALID), (dict(out=PTR + 4), INVALID),
                   (dict(rot=32, cos=PTR, positions=48, kv=_kv(dtype=2, k_scale=PTR, v_scale=PTR)), UNSUPPORTED), (dict(seqs=1 << 25, tokens=1 << 25), UNSUPPORTED)):
        assert append(**kw) == rc, kw

    def attend(layer=0, q=PTR, heads=4, rows=PTR, offsets=None, seqs=1, tokens=1, window=0, sinks=0, scale=1.0, max_len=0, out=PTR, ws=PTR, size=1 << 30):
        return lib.q3c_kv_attend(kv, layer, q, 256, 64, heads, rows, offsets, seqs, tokens, window, sinks, scale, max_len, out, ws, size, None)
    for kw, rc in ((dict(layer=2), INVALID), (dict(q=None), INVALID), (dict(heads=3), INVALID), (dict(heads=0), INVALID), (dict(window=-1), INVALID), (dict(sinks=-1), INVALID),
                   (dict(scale=0.0), INVALID), (dict(scale=float("nan")), INVALID), (dict(scale=float("inf")), INVALID), (dict(max_len=-1), INVALID), (dict(out=None), INVALID),
                   (dict(tokens=3), INVALID), (dict(rows=None), INVALID)):
        assert attend(**kw) == rc, kw
    long = _kv(pages_per_row=4096)
    n = C.c_size_t()
    assert lib.q3c_kv_attend_workspace_bytes(long, 4, 1, 1, 0, 0, 0, C.byref(n)) == OK and n.value > 0
    assert lib.q3c_kv_attend(long, 0, PTR, 256, 64, 4, PTR, None, 1, 1, 0, 0, 1.0, 0, PTR, PTR, n.value - 1, None) == WORKSPACE
    assert lib.q3c_kv_attend(long, 0, PTR, 256, 64, 4, PTR, None, 1, 1, 0, 0, 1.0, 0, PTR, None, n.value, None) == INVALID
    assert lib.q3c_kv_attend_workspace_bytes(long, 4, 1, 1, 0, 0, 0, None) == INVALID
    assert lib.q3c_kv_fork(kv, PTR, PTR, 2, PTR, 23, None) == WORKSPACE and lib.q3c_kv_fork(kv, None, PTR, 2, PTR, 24, None) == INVALID
    assert lib.q3c_kv_fork(_kv(layers=1 << 16, page_size=256), PTR, PTR, 1 << 20, PTR, 1 << 40, None) == UNSUPPORTED
    assert lib.q3c_kv_copy_pages(kv, PTR, PTR, 2, PTR, 7, None) == WORKSPACE and lib.q3c_kv_copy_pages(kv, PTR, PTR, -1, PTR, 7, None) == INVALID
    assert lib.q3c_kv_compact(kv, PTR, PTR, 79, None) == WORKSPACE and lib.q3c_kv_compact(kv, None, PTR, 80, None) == INVALID
    assert lib.q3c_kv_trim(kv, PTR, 1, 0, 0, None) == INVALID and lib.q3c_kv_trim(kv, PTR, 1, 1, -1, None) == INVALID
    assert lib.q3c_kv_release(kv, None, 1, None) == INVALID and lib.q3c_kv_release(kv, PTR, -1, None) == INVALID
    assert lib.q3c_kv_gather(kv, 0, PTR, None, 1, 1, PTR, PTR, 2, None) == INVALID and lib.q3c_kv_gather(kv, 0, PTR, None, 1, 1, None, PTR, 1, None) == INVALID


def test_calls_larger_than_a_launch_are_refused():
    """A launch has fewer than 2^32 threads along its first axis: calls whose grid would pass that are refused before anything runs."""
    lib, kv, n = _lib.load(), _kv(), C.c_size_t()
    for heads, seqs, tokens, rc in ((2, 1, 1 << 20, OK), (256, 1, 1 << 21, UNSUPPORTED), (2, 1 << 23, 1 << 23, UNSUPPORTED), (2, 1 << 22, 1 << 22, OK)):
        assert lib.q3c_kv_attend_workspace_bytes(kv, heads, seqs, tokens, 0, 0, 0, C.byref(n)) == rc, (heads, seqs, tokens)
        if rc:
            assert lib.q3c_kv_attend(kv, 0, PTR, 256, 64, heads, PTR, PTR, seqs, tokens, 0, 0, 1.0, 0, PTR, PTR, 1 << 40, None) == rc
    assert lib.q3c_kv_append(kv, 0, PTR, 256, 64, PTR, 128, 64, PTR, 128, 64, 60, PTR, PTR, 1, 1 << 21, None, None, None, None, 0, 0, 1e-6, PTR, None) == UNSUPPORTED
    assert lib.q3c_kv_gather(_kv(kv_heads=64), 0, PTR, PTR, 1, 1 << 20, PTR, PTR, 1, None) == UNSUPPORTED
    assert lib.q3c_kv_release(kv, PTR, 1 << 24, None) == UNSUPPORTED and lib.q3c_kv_trim(kv, PTR, 1 << 24, 4, 0, None) == UNSUPPORTED
    assert lib.q3c_kv_copy_pages(_kv(layers=64), PTR, PTR, 1 << 17, PTR, 1 << 40, None) == UNSUPPORTED
    assert lib.q3c_kv_fork(_kv(layers=64), PTR, PTR, 1 << 17, PTR, 1 << 40, None) == UNSUPPORTED


@pytest.mark.parametrize("dtype,tb", [(0, 16), (1, 32)])
def test_shares_cover_the_chunks_that_a_window_can_touch(dtype, tb):
    """How a long row is cut follows from the most chunks of 16 or 32 tokens that a tile can see under the window: a bound, held here against all
    places of a window of one position and of 16 (the workspace says how many shares of 8 chunks there are; none: at most 32 chunks, uncut)."""
    lib, kv, n = _lib.load(), _kv(dtype=dtype, pages=4096, pages_per_row=4096), C.c_size_t()
    for window in list(range(1, 5)) + list(range(tb * 31 - 20, tb * 33 + 20, 3)) + list(range(1200, 1300, 5)) + list(range(1210, 1222)):
        for sinks in (0, 1, 5, tb, tb + 1):
            assert lib.q3c_kv_attend_workspace_bytes(kv, 2, 1, 1, window, sinks, 0, C.byref(n)) == OK
            shares = (n.value // (4 * 2) - 1) // (16 * 66)            # of each of the two heads: shares of [16][64 + 2], one count
            for positions in (1, 16):
                first = 10 * tb + sinks + window                       # far behind the sinks: the most there is
                most = max(-(-sinks // tb) + (p + positions - 1) // tb - (p - window + 1) // tb + 1 for p in range(first, first + tb))
                assert most <= (8 * shares if n.value else 32), (window, sinks, positions)


def test_a_scale_that_overflows_is_refused():
    """The scale is held times log2(e), and times 16 where keys are: 1e37 is the last decade whose products fp32 holds."""
    lib, kv = _lib.load(), _kv()
    for scale in (1e37, 3e38, 0.0, -1.0):
        assert lib.q3c_kv_attend(kv, 0, PTR, 256, 64, 4, PTR, None, 1, 1, 0, 0, scale, 0, PTR, PTR, 1 << 30, None) == INVALID, scale


def test_rope_tables_of_far_positions():
    cos, sin = rope_tables(200001, 8, theta=1e6, device="cpu")
    import math
    for p in (0, 1, 199999, 200000):
        for i in range(4):
            a = p * 1e6 ** (-i / 4)
            assert abs(float(cos[p, i]) - math.cos(a)) < 1e-7 and abs(float(sin[p, i]) - math.sin(a)) < 1e-7


def test_rope_tables_of_odd_sizes_are_refused():
    """15 dimensions would make 8 angles of theta^(-2 i / 15), which append takes for 16 dimensions'."""
    for positions, rot in ((10, 15), (10, 0), (10, -2), (0, 16)):
        with pytest.raises(ValueError):
            rope_tables(positions, rot, device="cpu")


def test_the_plain_restatement_itself():
    """Fixed points that need no second implementation: uniform weights, a window of one token, rotation keeps lengths."""
    g = torch.Generator().manual_seed(0)
    v = torch.randn(6, 1, 4, generator=g, dtype=torch.float64)
    out, _, _ = attention(torch.zeros(1, 2, 4), torch.randn(6, 1, 4, generator=g), v, [5], 3, 1, 1.0)
    assert torch.allclose(out[0, 0], v[[0, 3, 4, 5], 0].mean(0)) and torch.equal(out[0, 0], out[0, 1])
    out, _, _ = attention(torch.randn(6, 1, 4, generator=g), v, v, list(range(6)), 1, 0, 1.0)
    assert torch.allclose(out[:, 0], v[:, 0])
    x = torch.randn(5, 2, 16, generator=g)
    cos, sin = rope_tables(9, 16, device="cpu")
    y = norm_rotate(x, None, cos, sin, torch.arange(5) + 2, 0.0)
    assert torch.allclose(y.norm(dim=-1), x.double().norm(dim=-1), rtol=1e-6) and not torch.allclose(y, x.double())
    p = Pages(6, 8, 3, 4)
    p.reserve([0], [20])
    assert p.fork([0], [1]) == [(2, 3)] and p.refs == [2, 2, 1, 1, 0, 0]
    p.release([0])
    assert p.refs == [1, 1, 0, 1, 0, 0] and p.compact() == ([(3, 2)], 3) and p.table[1] == [0, 1, 2, -1]


class _Stub:
    """Stands for a cache where only the order of calls and what they write counts: append adds to the tensors that it is given."""

    def __init__(self, state, calls):
        self.state, self.calls = state, calls

    def over(self, state):
        return _Stub(state, self.calls)

    def append(self, layer, q, k, v, rows, offsets, **kw):
        self.calls.append(("append", layer))
        self.state[0][layer] += k.sum()
        self.state[1][layer] += 1
        return q * 2

    def attend(self, layer, q, rows, offsets, **kw):
        self.calls.append(("attend", layer))
        return q + self.state[0][layer] + self.state[5][0]


@pytest.fixture
def traced_ops():
    """The two ops with CPU kernels, over a stub of a cache -> (handle, stub, its state)."""
    from qwen3_tts_amd import torch_ops
    state = [torch.zeros(3), torch.zeros(3), None, None, torch.zeros(2, 2, dtype=torch.int32), torch.full((2,), 7, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)]
    lib = torch.library.Library("q3tts", "FRAGMENT")
    lib.impl("kv_append", torch_ops._plain(torch_ops._kv_append), "CPU")
    lib.impl("kv_attend", torch_ops._plain(torch_ops._kv_attend), "CPU")
    stub = _Stub(state, [])
    h = torch_ops.register_kv(stub)
    yield h, stub, state
    torch_ops.unregister_kv(h)
    lib._destroy()
    torch._dynamo.reset()


def _programs(h, state):
    ops = torch.ops.q3tts

    def append(q, rows, layer):
        return ops.kv_append(q, q, q, rows, None, None, None, None, None, 1e-6, h, layer, *state)

    def attend(q, rows, layer):
        return ops.kv_attend(q, rows, None, 0, 0, h, layer, *state)

    def prefill(q, rows):                      # a cached prompt: nobody takes the hidden states
        for layer in range(3):
            append(q, rows, layer)
        return q + 1

    def between(q, rows):
        a = attend(q, rows, 1)
        append(q, rows, 1)
        return a, attend(q, rows, 1)

    def step(q, rows):
        for layer in range(3):
            q = attend(append(q, rows, layer), rows, layer)
        return q
    return {"prefill": (prefill, ["append"] * 3), "between": (between, ["attend", "append", "attend"]), "step": (step, ["append", "attend"] * 3)}


@pytest.mark.parametrize("name", ["prefill", "between", "step"])
@pytest.mark.parametrize("backend", ["aot_eager", "inductor"])
def test_a_traced_program_keeps_its_cache_calls(traced_ops, name, backend):
    """An append whose queries are not wanted is no dead code, and attends on either side of one are not one call: compiled programs make
    the calls that eager ones make, in their order, with the same results and the same cache."""
    h, stub, state = traced_ops
    fn, calls = _programs(h, state)[name]
    q, rows = torch.tensor([1.0, 2.0]), torch.zeros(1, dtype=torch.int32)
    want, k, v = fn(q, rows), state[0].clone(), state[1].clone()
    assert [c for c, _ in stub.calls] == calls
    for t in state[:2]:
        t.zero_()
    stub.calls.clear()
    got = torch.compile(fn, backend=backend, fullgraph=True)(q, rows)
    assert [c for c, _ in stub.calls] == calls
    for a, b in zip(*((x if isinstance(x, tuple) else (x,)) for x in (got, want))):
        assert torch.equal(a, b)
    assert torch.equal(state[0], k) and torch.equal(state[1], v)


def test_dead_code_elimination_leaves_appends(traced_ops):
    from torch.fx.experimental.proxy_tensor import make_fx
    h, stub, state = traced_ops
    prefill, _ = _programs(h, state)["prefill"]
    graph = make_fx(prefill)(torch.ones(2), torch.zeros(1, dtype=torch.int32))
    graph.graph.eliminate_dead_code()
    assert sum(n.target is torch.ops.q3tts.kv_append.default for n in graph.graph.nodes) == 3
    schema = torch.ops.q3tts.kv_append.default._schema
    assert [a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write] == ["k_pages", "v_pages", "k_steps", "v_steps", "status"]


def test_a_program_traced_without_the_caches_tensors_is_refused(traced_ops):
    h, stub, state = traced_ops
    q, rows = torch.ones(2), torch.zeros(1, dtype=torch.int32)
    for fn in (lambda q, r: torch.ops.q3tts.kv_append(q, q, q, r, None, None, None, None, None, 1e-6, h, 0),
               lambda q, r: torch.ops.q3tts.kv_attend(q, r, None, 0, 0, h, 0)):
        assert fn(q, rows).shape == q.shape                         # eagerly the handle's own tensors are meant
        with pytest.raises(Exception, match="has to pass the cache's tensors"):
            torch.compile(fn, backend="aot_eager", fullgraph=True)(q, rows)
