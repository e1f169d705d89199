"""Paged key/value cache for the autoregressive model that produces the codes, and the operators on it.

The reference leaves this to its dependency: the codes come out of `Qwen3TTSModel.generate_*` (reference server.py:245-251,
models.py:86-101), whose attention is a library chosen by name (models.py:22).  Here they are kernels of libq3c.so, one per step of a
generation, and nothing in them reads device values on the host: a whole step can be captured into a HIP graph.

    kv = PagedKV(layers=28, kv_heads=8, head_dim=128, pages=4096, page_size=32, rows=64, dtype="bf16")
    rope = rope_tables(kv.max_tokens, 128, device=kv.device)
    kv.reserve(rows)                                             # a place for one new token of each row (or `offsets` of each)
    for layer in range(28):
        q = kv.append(layer, q, k, v, rows, q_weight=wq, k_weight=wk, rope=rope)      # head norms, rotation, K and V into their pages
        out = kv.attend(layer, q, rows, window=4096, sinks=4)
    kv.trim(rows, window=4096, sinks=4)                          # pages that the window has left behind go back to the pool
    kv.fork(prompt_rows, new_rows)                               # requests that start from a cached voice prompt share its pages
    kv.release(ended_rows)

`rows` are table rows, one per request: an int32 tensor on the device (distinct; checked there) or a sequence of ints (checked here).
`offsets` (int32 [len(rows) + 1] on the device) gives each row's new tokens in a ragged call; without it every row has one; tokens
before offsets[0] and from offsets[-1] on belong to no row and are left alone.  Offsets that end behind the call's tokens count as ending there
(`check` says so).  `dtype` "f32" and "bf16" hold what the activations are;
"int4" holds bf16 activations in 4 bits with a step per 32 dimensions.  There is no backward pass: a cache is state, this package trains
nothing, and tensors that ask for gradients are refused where autograd is on.

Every call runs on the current stream of the cache's device.  attend and gather calls may run beside each other on any streams; a call
that changes the cache (the others) must be ordered with those around it, as writes to a tensor are.  Calls that are captured into a
graph take `rows` as a tensor: a sequence is copied to the device by the call.
"""
from __future__ import annotations

import ctypes as C
import operator
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib

Rows = Union[torch.Tensor, Sequence[int]]

GROUP = 32                                     # dimensions that share a step in a 4-bit cache
_HELD = {torch.float32: 0, torch.bfloat16: 1, torch.uint8: 2}
_ACT = (torch.float32, torch.bfloat16, torch.bfloat16)
_MOST = 2 ** 31 - 1
# the current device and its stream's handle, without the objects that torch.cuda wraps them in (a call of a generation step is host-bound)
_device, _stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
_STATUS = ((1, "a row id outside the table, named twice in a call, or offsets that do not fit a row's length or the call's tokens"),
           (2, "no free page was left (or a token was appended that has no page)"),
           (4, "a page id outside the pool, or a copy whose source is another copy's destination"),
           (8, "a row grew past page_size * pages_per_row tokens"))


def _no_gradient(t: torch.Tensor, what: str) -> None:
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what} requires a gradient, and the cache's operators have none: call them under torch.no_grad()")


def rope_tables(positions: int, rot_dim: int, theta: float = 10000.0, device: Union[str, torch.device] = "cuda:0") -> Tuple[torch.Tensor, torch.Tensor]:
    """(cos, sin), float32 [positions, rot_dim / 2] each, of position * theta^(-2 i / rot_dim): angles in float64, so that far positions
    are as exact as near ones."""
    if positions < 1 or rot_dim < 2 or rot_dim % 2:
        raise ValueError(f"rope tables need a position and an even number of rotated dimensions, got {positions} and {rot_dim}")
    inv = theta ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64) / rot_dim)
    ang = torch.arange(positions, dtype=torch.float64)[:, None] * inv
    return ang.cos().float().to(device), ang.sin().float().to(device)


class PagedKV:
    """`pages` pages of `page_size` tokens for every layer, and a table of `rows` rows that name them (see the module's text and
    include/q3c.h, q3c_kv, for the layout).  The tensors are attributes: k, v, k_scale, v_scale, table, lens, refs, status."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, pages: int, page_size: int = 32, rows: int = 64,
                 pages_per_row: Optional[int] = None, dtype: str = "bf16", device: Union[str, torch.device] = "cuda:0"):
        if dtype != "int4" and dtype not in _lib.PRECISION:
            raise ValueError(f"dtype must be 'int4' or one of {sorted(_lib.PRECISION)}, got {dtype!r}")
        if min(layers, kv_heads, head_dim, pages, page_size, rows) < 1 or (pages_per_row is not None and pages_per_row < 1):
            raise ValueError("layers, kv_heads, head_dim, pages, page_size, rows and pages_per_row must be positive")
        if dtype == "int4" and head_dim % GROUP:
            raise ValueError(f"a 4-bit cache needs head_dim 64, 128 or 256, got {head_dim}")
        dev = torch.device(device)
        held = torch.uint8 if dtype == "int4" else (torch.float32, torch.bfloat16)[_lib.PRECISION[dtype]]
        shape = (layers, pages, kv_heads, page_size)
        k, v = (torch.zeros(shape + (head_dim // 2 if dtype == "int4" else head_dim,), dtype=held, device=dev) for _ in range(2))
        ks = vs = None
        if dtype == "int4":
            ks, vs = (torch.zeros(shape + (head_dim // GROUP,), dtype=torch.bfloat16, device=dev) for _ in range(2))
        table = torch.full((rows, pages if pages_per_row is None else pages_per_row), -1, dtype=torch.int32, device=dev)
        self._adopt(k, v, table, torch.zeros(rows, dtype=torch.int32, device=dev), torch.zeros(pages, dtype=torch.int32, device=dev), ks, vs, None)

    @classmethod
    def from_tensors(cls, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor,
                     k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
                     status: Optional[torch.Tensor] = None) -> "PagedKV":
        """A cache over tensors that the caller has: k, v [layers, pages, kv_heads, page_size, head_dim] float32 or bfloat16 (uint8 with
        head_dim / 2 bytes for 4 bits, beside bfloat16 steps k_scale, v_scale [.., head_dim / 32]), table [rows, pages_per_row], lens [rows],
        refs [pages] and status [1] int32, contiguous, on one GPU."""
        self = cls.__new__(cls)
        self._adopt(k, v, table, lens, refs, k_scale, v_scale, status)
        return self

    def _adopt(self, k, v, table, lens, refs, k_scale, v_scale, status) -> None:
        if k.dim() != 5 or k.dtype not in _HELD:
            raise ValueError("k must be a float32, bfloat16 or (4 bits) uint8 tensor [layers, pages, kv_heads, page_size, head_dim]")
        L, P, G, ps, D = k.shape
        code = _HELD[k.dtype]
        four = code == 2
        if four:
            D *= 2
        if min(L, P, G, ps, D) < 1:
            raise ValueError(f"empty cache: {tuple(k.shape)}")
        if ps & (ps - 1) or not 8 <= ps <= 256:
            raise ValueError(f"page_size must be a power of two from 8 to 256, got {ps}")
        if D % 16 or D > 256 or (four and D not in (64, 128, 256)):
            raise ValueError(f"head_dim must be a multiple of 16 up to 256 (4 bits: 64, 128 or 256), got {D}")
        if v.shape != k.shape or v.dtype != k.dtype:
            raise ValueError("v must be like k")
        if four:
            for n, t in (("k_scale", k_scale), ("v_scale", v_scale)):
                if t is None or t.dtype != torch.bfloat16 or tuple(t.shape) != (L, P, G, ps, D // GROUP):
                    raise ValueError(f"a 4-bit cache needs {n}, bfloat16 {(L, P, G, ps, D // GROUP)}")
        elif k_scale is not None or v_scale is not None:
            raise ValueError("k_scale and v_scale belong to a 4-bit cache")
        if status is None:
            status = torch.zeros(1, dtype=torch.int32, device=k.device)
        if table.dim() != 2 or table.shape[0] < 1 or table.shape[1] < 1:
            raise ValueError("table must be [rows, pages_per_row]")
        for n, t, shape in (("table", table, tuple(table.shape)), ("lens", lens, (table.shape[0],)), ("refs", refs, (P,)), ("status", status, (1,))):
            if t.dtype != torch.int32 or tuple(t.shape) != shape:
                raise ValueError(f"{n} must be int32 {shape}, got {t.dtype} {tuple(t.shape)}")
        if table.shape[1] * ps > 1 << 30:
            raise ValueError("a row may hold at most 2^30 tokens")
        for n, t in (("k", k), ("v", v), ("k_scale", k_scale), ("v_scale", v_scale), ("table", table), ("lens", lens), ("refs", refs), ("status", status)):
            if t is None:
                continue
            if not t.is_contiguous() or t.device != k.device:
                raise ValueError(f"{n} must be contiguous and on {k.device}")
            if n in ("k", "v", "k_scale", "v_scale") and t.data_ptr() % 16:
                raise ValueError(f"{n} must be 16-byte aligned")
            _no_gradient(t, n)
        if k.device.type != "cuda":
            raise RuntimeError("qwen3_tts_amd.kvcache needs a ROCm GPU (MI355X); there is no CPU fallback")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.table, self.lens, self.refs, self.status = table, lens, refs, status
        self.layers, self.pages, self.kv_heads, self.page_size, self.head_dim = L, P, G, ps, D
        self.rows, self.pages_per_row = int(table.shape[0]), int(table.shape[1])
        self.dtype = ("f32", "bf16", "int4")[code]
        self.activations = _ACT[code]
        self._act_bytes = 4 if code == 0 else 2
        self._max_tokens = ps * self.pages_per_row
        self.device = k.device
        self._index = k.device.index if k.device.index is not None else torch.cuda.current_device()
        self._lib = _lib.load()
        c = _lib.Q3cKv()
        c.struct_size = C.sizeof(_lib.Q3cKv)
        c.dtype, c.layers, c.pages, c.kv_heads, c.page_size, c.head_dim = code, L, P, G, ps, D
        c.rows, c.pages_per_row = self.rows, self.pages_per_row
        c.k, c.v = k.data_ptr(), v.data_ptr()
        c.k_scale, c.v_scale = (k_scale.data_ptr(), v_scale.data_ptr()) if four else (None, None)
        c.table, c.lens, c.refs, c.status = table.data_ptr(), lens.data_ptr(), refs.data_ptr(), status.data_ptr()
        self._c = c
        self._ref = C.byref(c)
        self._need = {}                        # attend: workspace bytes by the sizes of the call

    @property
    def state(self) -> Tuple[Optional[torch.Tensor], ...]:
        """k, v, k_scale, v_scale, table, lens, status: what `torch.ops.q3tts.kv_append` and `kv_attend` take last, so that a traced program
        knows what they write and read."""
        return self.k, self.v, self.k_scale, self.v_scale, self.table, self.lens, self.status

    def over(self, state: Sequence[Optional[torch.Tensor]]) -> "PagedKV":
        """This cache, or one over `state` (tensors like self.state) where those are others than its own."""
        if all(a is b or (a is not None and b is not None and a.data_ptr() == b.data_ptr()) for a, b in zip(state, self.state)):
            return self
        if any((a is None) != (b is None) for a, b in zip(state, self.state)):
            raise ValueError("all of the cache's tensors are wanted, in the order of `state`")
        k, v, k_scale, v_scale, table, lens, status = state
        return PagedKV.from_tensors(k, v, table, lens, self.refs, k_scale, v_scale, status)

    # ---- what every call does ------------------------------------------------------------------------------------------------
    @property
    def max_tokens(self) -> int:
        """Tokens that one row can hold."""
        return self._max_tokens

    def _call(self, fn, *args) -> None:
        i = self._index
        if _device() == i:
            rc = fn(self._ref, *args, _stream(i))
        else:
            with torch.cuda.device(i):
                rc = fn(self._ref, *args, _stream(i))
        if rc:
            raise _lib.Q3cError(rc, f"{fn.__name__} failed")

    def _ids(self, ids, what: str, most: int, distinct: bool = True) -> torch.Tensor:
        if isinstance(ids, torch.Tensor):
            if ids.dtype != torch.int32 or ids.dim() != 1 or not ids.is_contiguous() or ids.get_device() != self._index:
                raise ValueError(f"{what} must be a contiguous int32 tensor [n] on {self.device} (or a sequence of ints)")
            return ids
        ids = [operator.index(i) for i in ids]                  # whole numbers only: 1.9 is no row
        for i in ids:
            if not 0 <= i < most:
                raise IndexError(f"{what}: {i} is not in [0, {most})")
        if distinct and len(set(ids)) != len(ids):
            raise ValueError(f"{what} must be distinct")
        return torch.tensor(ids, dtype=torch.int32, device=self.device)

    def _batch(self, rows: Rows, offsets: Optional[torch.Tensor], tokens: Optional[int]):
        rows = self._ids(rows, "rows", self.rows)
        n = rows.shape[0]
        if offsets is None:
            if tokens is not None and tokens != n:
                raise ValueError(f"{tokens} tokens for {n} rows: without offsets every row has one")
            return rows, n, None, n
        if offsets.dtype != torch.int32 or offsets.dim() != 1 or offsets.shape[0] != n + 1 or not offsets.is_contiguous() or offsets.get_device() != self._index:
            raise ValueError(f"offsets must be a contiguous int32 tensor [{n + 1}] on {self.device}")
        if tokens is not None and not 0 <= tokens <= 1 << 24:
            raise ValueError(f"a call takes at most 2^24 tokens, got {tokens}")
        return rows, n, offsets, tokens

    def _heads(self, x: torch.Tensor, what: str, heads: Optional[int]):
        """[tokens, heads, head_dim] in the cache's activation type -> (tensor, shape, pointer, token stride, head stride); copied only
        where its strides are not what the kernels read: multiples of four (the stride of a dimension of one element may be anything, and is
        passed on rounded down)."""
        shape = x.shape
        if len(shape) != 3 or shape[2] != self.head_dim or (heads is not None and shape[1] != heads) or shape[1] < 1:
            raise ValueError(f"{what} must be [tokens, {'heads' if heads is None else heads}, {self.head_dim}], got {tuple(shape)}")
        if x.dtype != self.activations or x.get_device() != self._index:
            raise ValueError(f"{what} must be {self.activations} on {self.device}, got {x.dtype} on {x.device}")
        if x.requires_grad:
            _no_gradient(x, what)
        ts, hs, ds = x.stride()
        p, quad = x.data_ptr(), 4 * self._act_bytes
        if ds != 1 or (ts % 4 and shape[0] != 1) or (hs % 4 and shape[1] != 1) or p % quad:
            x = x.contiguous()
            if x.data_ptr() % quad:                            # a contiguous view that starts between two quads
                x = x.clone()
            ts, hs, ds = x.stride()
            p = x.data_ptr()
        return x, shape, p, ts & -4, hs & -4

    def _table(self, t: torch.Tensor, dims: int, what: str, shape: str) -> int:
        p = t.data_ptr()
        if t.dtype != torch.float32 or t.dim() != dims or not t.is_contiguous() or t.get_device() != self._index or p % 16:
            raise ValueError(f"{what} must be a contiguous, 16-byte aligned float32 tensor {shape} on {self.device}")
        if t.requires_grad:
            _no_gradient(t, what)
        return p

    def _layer(self, layer: int) -> int:
        if not 0 <= layer < self.layers:
            raise IndexError(f"layer {layer} is not in [0, {self.layers})")
        return layer

    def _out(self, out: Optional[torch.Tensor], shape, dtype, what: str = "out") -> torch.Tensor:
        if out is None:
            return torch.empty(shape, dtype=dtype, device=self.device)
        if out.dtype != dtype or tuple(out.shape) != tuple(shape) or not out.is_contiguous() or out.get_device() != self._index or out.data_ptr() % 16:
            raise ValueError(f"{what} must be a contiguous, 16-byte aligned {dtype} tensor {tuple(shape)} on {self.device}")
        _no_gradient(out, what)
        return out

    def check(self) -> None:
        """Waits for the stream; raises what calls found wrong on the device since the last check (and clears it)."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            raise _lib.Q3cError(-1, "; ".join(text for b, text in _STATUS if bits & b))

    # ---- tokens ----------------------------------------------------------------------------------------------------------------
    def reserve(self, rows: Rows, offsets: Optional[torch.Tensor] = None, tokens: Optional[int] = None) -> None:
        """Make room for the rows' new tokens (one each, or as `offsets` say): lens grows, free pages are taken lowest first, in the order
        of `rows`.  Pages that the pool cannot give are missing (`check` says so): their tokens are dropped by append, and seen by nobody."""
        rows, n, offsets, tokens = self._batch(rows, offsets, tokens)
        self._call(self._lib.q3c_kv_reserve, rows.data_ptr(), None if offsets is None else offsets.data_ptr(), n, 1 << 24 if tokens is None else tokens)

    def append(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, rows: Rows, offsets: Optional[torch.Tensor] = None, *,
               q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
               rope: Optional[Tuple[torch.Tensor, torch.Tensor]] = None, eps: float = 1e-6, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The rows' newest tokens (those that `reserve` made room for) into one layer: RMS norm of each head of q and k with `q_weight`,
        `k_weight` (float32 [head_dim]; None: no norm), rotation by position with `rope` = (cos, sin) (see rope_tables; half the rotated
        dimensions wide; None: none), k and v stored, q returned (`out`, or a new tensor) [tokens, heads, head_dim].  q, k, v: [tokens,
        heads, head_dim], any strides - views of one projection's output are read in place.  q tokens behind offsets[-1] are left as
        they are in `out` (undefined in a new tensor)."""
        q, (T, H, D), qp, qt, qh = self._heads(q, "q", None)
        k, ks, kp, kt, kh = self._heads(k, "k", self.kv_heads)
        v, vs, vp, vt, vh = self._heads(v, "v", self.kv_heads)
        if ks[0] != T or vs[0] != T:
            raise ValueError(f"q, k and v hold {T}, {ks[0]} and {vs[0]} tokens")
        rows, n, offsets, _ = self._batch(rows, offsets, T)
        if not n and T:
            raise ValueError(f"{T} tokens without a row")
        wq = None if q_weight is None else self._table(q_weight, 1, "q_weight", f"[{D}]")
        wk = None if k_weight is None else self._table(k_weight, 1, "k_weight", f"[{D}]")
        if wq is not None or wk is not None:
            for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
                if w is not None and w.shape[0] != D:
                    raise ValueError(f"{name} must be a contiguous, 16-byte aligned float32 tensor [{D}] on {self.device}")
            if not eps > 0:
                raise ValueError(f"eps must be positive, got {eps}")
        rot = positions = 0
        cp = sp = None
        if rope is not None:
            cos, sin = rope
            cp, sp = self._table(cos, 2, "rope's cos", "[positions, rotated / 2]"), self._table(sin, 2, "rope's sin", "[positions, rotated / 2]")
            positions, half = cos.shape
            if sin.shape != cos.shape:
                raise ValueError(f"rope's cos and sin must have one shape, got {tuple(cos.shape)} and {tuple(sin.shape)}")
            rot = 2 * half
            if rot % 8 or not 0 < rot <= D or (self.dtype == "int4" and rot != D):
                raise ValueError(f"rope rotates {rot} of {D} dimensions: a multiple of 8 is wanted (all of them in a 4-bit cache)")
            if positions < self.max_tokens:
                raise ValueError(f"rope covers {positions} positions, a row can hold {self.max_tokens}")
        out = self._out(out, (T, H, D), self.activations)
        self._call(self._lib.q3c_kv_append, self._layer(layer), qp, qt, qh, kp, kt, kh, vp, vt, vh, H, rows.data_ptr(),
                   None if offsets is None else offsets.data_ptr(), n, T, wq, wk, cp, sp, positions, rot, eps, out.data_ptr())
        return out

    def gather(self, layer: int, rows: Rows, offsets: Optional[torch.Tensor] = None, tokens: Optional[int] = None,
               dtype: Optional[str] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """What the cache holds of the rows' newest tokens, in one piece: (k, v) [tokens, kv_heads, head_dim] in `dtype` ("f32" or "bf16";
        default: the activations').  With `offsets`, `tokens` = offsets[-1], which is not read here.  Zeros where a token has no page."""
        rows, n, offsets, tokens = self._batch(rows, offsets, tokens)
        if tokens is None:
            raise ValueError("gather with offsets needs `tokens`")
        if tokens < 0 or (not n and tokens):
            raise ValueError(f"{tokens} tokens for {n} rows")
        code = _HELD[self.activations] if dtype is None else _lib.PRECISION.get(dtype)
        if code is None:
            raise ValueError(f"dtype must be one of {sorted(_lib.PRECISION)}, got {dtype!r}")
        shape = (tokens, self.kv_heads, self.head_dim)
        k, v = (torch.empty(shape, dtype=_ACT[code], device=self.device) for _ in range(2))
        self._call(self._lib.q3c_kv_gather, self._layer(layer), rows.data_ptr(), None if offsets is None else offsets.data_ptr(), n, tokens,
                   k.data_ptr(), v.data_ptr(), code)
        return k, v

    def attend(self, layer: int, q: torch.Tensor, rows: Rows, offsets: Optional[torch.Tensor] = None, *, window: int = 0, sinks: int = 0,
               scale: Optional[float] = None, max_len: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of the rows' newest tokens over the cache: the token at position p sees the keys j <= p, with `window` > 0 only
        those with j > p - window or j < `sinks`.  q [tokens, heads, head_dim] (heads a multiple of kv_heads; head h reads kv head
        h // (heads / kv_heads)) -> the same shape; a token that sees nothing, or whose scores are all -inf, gives zeros; tokens behind
        offsets[-1] are left as they are in `out` (undefined in a new tensor).  fp32 inside, but that probabilities (and over a 4-bit cache, in
        calls of many tokens, values) are rounded to bf16 where they are operands of bf16 products.  `scale`: head_dim ** -0.5 unless given.
        `max_len`: no row is longer than this (0: not known); a good bound helps to cut the work of long rows.  What is wrong with rows, offsets
        or pages is not reported here but by the append before it: attend leaves `status` alone.
        The rows of a call are treated alike: one token behind a very long past, in a call with prompts, is not spread over the card as in a call
        of its own (100 000 tokens beside a prompt of 2 000: 2.0 ms against 54 + 123 us apart).  Make two calls of such a batch."""
        q, (T, H, D), qp, qt, qh = self._heads(q, "q", None)
        if H % self.kv_heads:
            raise ValueError(f"{H} query heads do not share {self.kv_heads} kv heads evenly")
        if window < 0 or sinks < 0 or max_len < 0 or window > _MOST or sinks > _MOST or max_len > _MOST:
            raise ValueError("window, sinks and max_len must be from 0 to 2^31 - 1")
        scale = D ** -0.5 if scale is None else float(scale)
        if not 0.0 < scale < 1e37:
            raise ValueError(f"scale must be positive and below 1e37, got {scale}")
        rows, n, offsets, _ = self._batch(rows, offsets, T)
        if not n and T:
            raise ValueError(f"{T} tokens without a row")
        out = self._out(out, (T, H, D), self.activations)
        key = (H, n, T, window, sinks, max_len)
        need = self._need.get(key)
        if need is None:
            size = C.c_size_t()
            rc = self._lib.q3c_kv_attend_workspace_bytes(self._ref, H, n, T, window, sinks, max_len, C.byref(size))
            if rc:
                raise _lib.Q3cError(rc, "q3c_kv_attend_workspace_bytes failed")
            if len(self._need) >= 1024:
                self._need.clear()
            need = self._need[key] = int(size.value)
        # a workspace of its own for each call: calls on two streams, or two captured graphs, share none
        ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        self._call(self._lib.q3c_kv_attend, self._layer(layer), qp, qt, qh, H, rows.data_ptr(),
                   None if offsets is None else offsets.data_ptr(), n, T, window, sinks, scale, max_len, out.data_ptr(),
                   None if ws is None else ws.data_ptr(), need)
        return out

    # ---- pages -----------------------------------------------------------------------------------------------------------------
    def fork(self, parents: Rows, children: Rows) -> None:
        """Every child (an empty row) becomes a copy of its parent: full pages are shared, a partly filled last one is copied."""
        parents = self._ids(parents, "parents", self.rows, distinct=False)
        children = self._ids(children, "children", self.rows)
        n = children.shape[0]
        if parents.shape[0] != n:
            raise ValueError(f"{parents.shape[0]} parents for {n} children")
        ws = torch.empty(max(3 * n, 1), dtype=torch.int32, device=self.device)
        self._call(self._lib.q3c_kv_fork, parents.data_ptr(), children.data_ptr(), n, ws.data_ptr(), 12 * n)

    def release(self, rows: Rows) -> None:
        """The rows end: their pages go back to the pool (a shared one when its last row lets go), their lengths become 0."""
        rows = self._ids(rows, "rows", self.rows)
        self._call(self._lib.q3c_kv_release, rows.data_ptr(), rows.shape[0])

    def trim(self, rows: Rows, window: int, sinks: int = 0) -> None:
        """Pages that no later `attend` with this window and these sinks sees go back to the pool."""
        if not 1 <= window <= _MOST or not 0 <= sinks <= _MOST:
            raise ValueError("trim needs window >= 1 and sinks >= 0 (below 2^31)")
        rows = self._ids(rows, "rows", self.rows)
        self._call(self._lib.q3c_kv_trim, rows.data_ptr(), rows.shape[0], window, sinks)

    def copy_pages(self, src, dst) -> None:
        """Page dst[i] = page src[i] in every layer (ids as an int32 device tensor or a sequence of ints).  The pairs are simultaneous: of
        those with one destination the last counts, one whose source is another's destination is refused (`check` says so)."""
        src, dst = self._ids(src, "src", self.pages, distinct=False), self._ids(dst, "dst", self.pages, distinct=False)
        n = dst.shape[0]
        if src.shape[0] != n:
            raise ValueError(f"{src.shape[0]} sources for {n} destinations")
        ws = torch.empty(max(n, 1), dtype=torch.int32, device=self.device)
        self._call(self._lib.q3c_kv_copy_pages, src.data_ptr(), dst.data_ptr(), n, ws.data_ptr(), 4 * n)

    def compact(self) -> torch.Tensor:
        """Move the live pages to the front of the pool (the fewest moves that do it; table and counts follow).  -> their number, an int32
        device tensor [1]; the pages from there on are free."""
        live = torch.empty(1, dtype=torch.int32, device=self.device)
        ws = torch.empty(2 * self.pages + 4, dtype=torch.int32, device=self.device)
        self._call(self._lib.q3c_kv_compact, live.data_ptr(), ws.data_ptr(), 4 * ws.numel())
        return live

    def free_pages(self) -> int:
        """How many pages are free now (waits for the stream)."""
        return int((self.refs == 0).sum().item())
