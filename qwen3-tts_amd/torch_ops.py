"""PyTorch custom ops (`torch.ops.q3tts.*`) over the C-ABI library.

The ops are thin: each looks up a `Decoder` by integer handle (contexts own device memory and cannot travel through
an op schema) and calls the same ctypes entry point the `Decoder` methods use, on torch's current stream.  Shape
functions are registered so the ops can be traced with fake tensors; there is no CPU kernel - calling an op on CPU
tensors raises NotImplementedError from the dispatcher.

    h = torch_ops.register_decoder(dec)
    wav = torch.ops.q3tts.decode_forward(codes, h)          # [B,1,T*1920-555]
    sums = torch.ops.q3tts.rvq_dequant(codes, h)            # [B,T,G,codebook_dim], bit-exact fp32
    y = torch.ops.q3tts.causal_conv1d(x, w, b, 1, "f32")    # operator level, channels-last
"""
from __future__ import annotations

import re
from typing import Dict, Optional

import torch

_decoders: Dict[int, object] = {}
_next = [1]


def register_decoder(decoder) -> int:
    h = _next[0]
    _next[0] += 1
    _decoders[h] = decoder
    return h


def unregister_decoder(handle: int) -> None:
    _decoders.pop(handle, None)


def _dec(handle: int):
    try:
        return _decoders[handle]
    except KeyError:
        raise KeyError(f"no decoder registered under handle {handle}") from None


@torch.library.custom_op("q3tts::decode_forward", mutates_args=(), device_types="cuda")
def decode_forward(codes: torch.Tensor, handle: int) -> torch.Tensor:
    return _dec(handle).forward(codes)


@decode_forward.register_fake
def _(codes, handle):
    cfg = _dec(handle).cfg
    return codes.new_empty((codes.shape[0], 1, cfg.output_length(codes.shape[2])), dtype=torch.float32)


@torch.library.custom_op("q3tts::chunked_decode", mutates_args=(), device_types="cuda")
def chunked_decode(codes: torch.Tensor, handle: int, chunk_size: int, left_context_size: int) -> torch.Tensor:
    return _dec(handle).chunked_decode(codes, chunk_size, left_context_size)


@chunked_decode.register_fake
def _(codes, handle, chunk_size, left_context_size):
    cfg = _dec(handle).cfg
    n = cfg.chunked_output_length(codes.shape[2], chunk_size, left_context_size)
    return codes.new_empty((codes.shape[0], 1, n), dtype=torch.float32)


@torch.library.custom_op("q3tts::rvq_dequant", mutates_args=(), device_types="cuda")
def rvq_dequant(codes: torch.Tensor, handle: int) -> torch.Tensor:
    return _dec(handle).rvq_dequant(codes)


@rvq_dequant.register_fake
def _(codes, handle):
    cfg = _dec(handle).cfg
    groups = 2 if cfg.num_quantizers > cfg.num_semantic_quantizers else 1
    return codes.new_empty((codes.shape[0], codes.shape[2], groups, cfg.codebook_dim), dtype=torch.float32)


@torch.library.custom_op("q3tts::causal_conv1d", mutates_args=(), device_types="cuda")
def causal_conv1d(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], dilation: int,
                  precision: str) -> torch.Tensor:
    from . import decoder
    return decoder.causal_conv1d(x, weight, bias, dilation, precision)


@causal_conv1d.register_fake
def _(x, weight, bias, dilation, precision):
    return x.new_empty((x.shape[0], x.shape[1], weight.shape[0]), dtype=torch.float32)


@torch.library.custom_op("q3tts::causal_trans_conv1d", mutates_args=(), device_types="cuda")
def causal_trans_conv1d(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], stride: int,
                        precision: str) -> torch.Tensor:
    from . import decoder
    return decoder.causal_trans_conv1d(x, weight, bias, stride, precision)


@causal_trans_conv1d.register_fake
def _(x, weight, bias, stride, precision):
    lout = (x.shape[1] - 1) * stride - weight.shape[2] + 2 * stride
    return x.new_empty((x.shape[0], max(lout, 0), weight.shape[1]), dtype=torch.float32)


@torch.library.custom_op("q3tts::snake_beta", mutates_args=(), device_types="cuda")
def snake_beta(x: torch.Tensor, alpha: torch.Tensor, beta: torch.Tensor, eps: float) -> torch.Tensor:
    from . import decoder
    return decoder.snake_beta(x, alpha, beta, eps)


@snake_beta.register_fake
def _(x, alpha, beta, eps):
    return torch.empty_like(x, dtype=torch.float32)


# ---- paged key/value cache (kvcache.PagedKV, registered under a handle like a decoder) ---------------------------------------------
#     h = torch_ops.register_kv(kv)
#     q = torch.ops.q3tts.kv_append(q, k, v, rows, None, wq, wk, cos, sin, 1e-6, h, layer, *kv.state)
#     o = torch.ops.q3tts.kv_attend(q, rows, None, 4096, 4, h, layer, *kv.state)
# The cache's tensors are arguments, and the schema names those that kv_append writes: a traced program then keeps an append whose queries
# nobody takes, and its order against the attends around it.  Eager calls may leave them out (the handle's own are meant); a program that is
# traced without them is refused, since nothing in it would say that one call writes what the next one reads.
_caches: Dict[int, object] = {}


def register_kv(cache) -> int:
    h = _next[0]
    _next[0] += 1
    _caches[h] = cache
    return h


def unregister_kv(handle: int) -> None:
    _caches.pop(handle, None)


def _kv(handle: int):
    try:
        return _caches[handle]
    except KeyError:
        raise KeyError(f"no cache registered under handle {handle}") from None


def _kv_over(handle: int, state):
    """The handle's cache; over other tensors where a compiler has put copies in the place of its own."""
    kv = _kv(handle)
    return kv if all(t is None for t in state) else kv.over(state)


def _traced(state) -> None:
    if state[0] is None:
        raise RuntimeError("a traced program has to pass the cache's tensors to kv_append and kv_attend (*kv.state, the last arguments)")


def _kv_append(q, k, v, rows, offsets, q_weight, k_weight, cos, sin, eps, handle, layer, *state):
    return _kv_over(handle, state).append(layer, q, k, v, rows, offsets, q_weight=q_weight, k_weight=k_weight,
                                          rope=None if cos is None else (cos, sin), eps=eps)


def _kv_append_fake(q, k, v, rows, offsets, q_weight, k_weight, cos, sin, eps, handle, layer, *state):
    _traced(state)
    return q.new_empty(q.shape)


def _kv_attend(q, rows, offsets, window, sinks, handle, layer, *state):
    return _kv_over(handle, state).attend(layer, q, rows, offsets, window=window, sinks=sinks)


def _kv_attend_fake(q, rows, offsets, window, sinks, handle, layer, *state):
    _traced(state)
    return q.new_empty(q.shape)


def _plain(fn):
    """The kernel with all arguments by position, left out ones as None (the dispatcher drops trailing defaults)."""
    return lambda *a: fn(*(a + (None,) * (fn.__code__.co_argcount + 7 - len(a))))


_KV_STATE = ("Tensor(a!)? k_pages=None, Tensor(b!)? v_pages=None, Tensor(c!)? k_steps=None, Tensor(d!)? v_steps=None, "
             "Tensor? table=None, Tensor? lens=None, Tensor(e!)? status=None")
torch.library.define("q3tts::kv_append", "(Tensor q, Tensor k, Tensor v, Tensor rows, Tensor? offsets, Tensor? q_weight, Tensor? k_weight, "
                     "Tensor? cos, Tensor? sin, float eps, int handle, int layer, " + _KV_STATE + ") -> Tensor")
torch.library.define("q3tts::kv_attend", "(Tensor q, Tensor rows, Tensor? offsets, int window, int sinks, int handle, int layer, "
                     + re.sub(r"\(.!\)", "", _KV_STATE) + ") -> Tensor")
for _name, _fn, _fake in (("kv_append", _kv_append, _kv_append_fake), ("kv_attend", _kv_attend, _kv_attend_fake)):
    torch.library.impl("q3tts::" + _name, "cuda")(_plain(_fn))
    torch.library.register_fake("q3tts::" + _name)(_plain(_fake))
kv_append, kv_attend = torch.ops.q3tts.kv_append, torch.ops.q3tts.kv_attend
