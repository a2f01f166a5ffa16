"""Kernel-level entry points on torch CUDA tensors (device memory and streams come from torch).

These call the C ABI directly with device pointers; they are the unit-level surface used by the
selector microbenchmark and the kernel parity tests, and the operators of a server that batches
requests: the paged 8-bit K/V cache (plan_cache, append_cache_q8, read_cache_q8, attend_cache_q8) and
the token scorer (select_logprobs).
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import torch

from . import _lib


def _stream_ptr(stream: torch.cuda.Stream | None) -> int:
    s = stream if stream is not None else torch.cuda.current_stream()
    return int(s.cuda_stream)


def selector_scratch(n_rows: int, vocab: int, device) -> torch.Tensor:
    nbytes = int(_lib.load().drt_selector_scratch_bytes(int(n_rows), int(vocab)))
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def select_rows(logits: torch.Tensor, *, mode: int = _lib.SELECT_MAX_PROB, temperature: float = 0.0,
                scratch: torch.Tensor | None = None, conf: torch.Tensor | None = None,
                token: torch.Tensor | None = None, stream: torch.cuda.Stream | None = None):
    """Per-row (confidence f64, token i32) of f32 logits [rows, vocab] (row stride may exceed vocab)."""
    if logits.dtype != torch.float32 or not logits.is_cuda or logits.dim() != 2 or logits.stride(1) != 1:
        raise ValueError("logits must be a row-major CUDA float32 [rows, vocab] tensor")
    rows, vocab = logits.shape
    dev = logits.device
    if scratch is None:
        scratch = selector_scratch(rows, vocab, dev)
    if conf is None:
        conf = torch.empty(rows, dtype=torch.float64, device=dev)
    if token is None:
        token = torch.empty(rows, dtype=torch.int32, device=dev)
    _lib.check(_lib.load().drt_selector_rows(logits.data_ptr(), logits.stride(0), rows, vocab, int(mode),
                                             float(temperature), scratch.data_ptr(), conf.data_ptr(),
                                             token.data_ptr(), _stream_ptr(stream)))
    return conf, token


def select_sample(logits: torch.Tensor, positions: torch.Tensor, *, temperature: float, seed: int, forward: int,
                  row_index: torch.Tensor | None = None, stream: torch.cuda.Stream | None = None):
    """Temperature-sampled (confidence f64, token i32, tie i32) per row of f32 logits [rows, vocab]
    (or of the rows row_index), keyed by (seed, forward, positions[r]) as drt_selector_sample."""
    if logits.dtype != torch.float32 or not logits.is_cuda or logits.dim() != 2 or logits.stride(1) != 1:
        raise ValueError("logits must be a row-major CUDA float32 [rows, vocab] tensor")
    if positions.dtype != torch.int32 or not positions.is_cuda or not positions.is_contiguous():
        raise ValueError("positions must be a contiguous CUDA int32 tensor")
    n = positions.numel() if row_index is None else row_index.numel()
    if row_index is None and n != logits.shape[0]:
        raise ValueError("one position per logits row")
    vocab = logits.shape[1]
    dev = logits.device
    scratch = selector_scratch(n, vocab, dev)
    conf = torch.empty(n, dtype=torch.float64, device=dev)
    token = torch.empty(n, dtype=torch.int32, device=dev)
    tie = torch.empty(n, dtype=torch.int32, device=dev)
    _lib.check(_lib.load().drt_selector_sample(logits.data_ptr(), logits.stride(0),
                                               0 if row_index is None else row_index.data_ptr(), n, vocab,
                                               float(temperature), int(seed) & (2**64 - 1), int(forward),
                                               positions.data_ptr(), scratch.data_ptr(), conf.data_ptr(),
                                               token.data_ptr(), tie.data_ptr(), _stream_ptr(stream)))
    return conf, token, tie


CHOICE_TOPK = 0
CHOICE_THRESHOLD = 1


def select_gather(logits: torch.Tensor, row_index: torch.Tensor, *, mode: int = _lib.SELECT_MAX_PROB,
                  temperature: float = 0.0, scratch: torch.Tensor | None = None, conf: torch.Tensor | None = None,
                  token: torch.Tensor | None = None, stream: torch.cuda.Stream | None = None):
    """(confidence f64, token i32) for the rows row_index (int32 CUDA) of f32 logits [rows, vocab]."""
    if logits.dtype != torch.float32 or not logits.is_cuda or logits.dim() != 2 or logits.stride(1) != 1:
        raise ValueError("logits must be a row-major CUDA float32 [rows, vocab] tensor")
    if row_index.dtype != torch.int32 or not row_index.is_cuda or not row_index.is_contiguous():
        raise ValueError("row_index must be a contiguous CUDA int32 tensor")
    n = row_index.numel()
    vocab = logits.shape[1]
    dev = logits.device
    if scratch is None:
        scratch = selector_scratch(n, vocab, dev)
    if conf is None:
        conf = torch.empty(n, dtype=torch.float64, device=dev)
    if token is None:
        token = torch.empty(n, dtype=torch.int32, device=dev)
    _lib.check(_lib.load().drt_selector_gather(logits.data_ptr(), logits.stride(0), row_index.data_ptr(), n, vocab,
                                               int(mode), float(temperature), scratch.data_ptr(), conf.data_ptr(),
                                               token.data_ptr(), _stream_ptr(stream)))
    return conf, token


def select_topp_entropy(logits: torch.Tensor, row_index: torch.Tensor | None = None, *, temperature: float = 0.2,
                        top_p: float = 0.95, exclude_token: int = -1, tie_rel: float = 2.0 ** -30,
                        stream: torch.cuda.Stream | None = None):
    """NegEntropy with a top-p nucleus over rows (row_index, int32 CUDA, or every row) of f32 logits:
    (confidence f64 holding the f32 value, token i32, tie bits i32)."""
    if logits.dtype != torch.float32 or not logits.is_cuda or logits.dim() != 2 or logits.stride(1) != 1:
        raise ValueError("logits must be a row-major CUDA float32 [rows, vocab] tensor")
    if row_index is not None and (row_index.dtype != torch.int32 or not row_index.is_contiguous()):
        raise ValueError("row_index must be a contiguous CUDA int32 tensor")
    n = row_index.numel() if row_index is not None else logits.shape[0]
    dev = logits.device
    conf = torch.empty(n, dtype=torch.float64, device=dev)
    token = torch.empty(n, dtype=torch.int32, device=dev)
    tie = torch.empty(max(1, n), dtype=torch.int32, device=dev)
    _lib.check(_lib.load().drt_selector_topp(logits.data_ptr(), logits.stride(0),
                                             row_index.data_ptr() if row_index is not None else None, n,
                                             logits.shape[1], float(temperature), float(top_p), int(exclude_token),
                                             float(tie_rel), conf.data_ptr(), token.data_ptr(), tie.data_ptr(),
                                             _stream_ptr(stream)))
    return conf, token, tie[:n]


def select_choices(conf: torch.Tensor, offsets: torch.Tensor, *, mode: int, k: int = 1, tau: float = 0.9,
                   tie_rel: float = 2.0 ** -40, chosen: torch.Tensor | None = None, tie: torch.Tensor | None = None,
                   stream: torch.cuda.Stream | None = None):
    """Top-k (mode CHOICE_TOPK) or threshold (CHOICE_THRESHOLD) choices per confidence run
    offsets[b] .. offsets[b + 1]: chosen[row] in {0, 1} (int32) and tie[b] certification bits."""
    if conf.dtype != torch.float64 or offsets.dtype != torch.int32:
        raise ValueError("conf must be float64 and offsets int32 CUDA tensors")
    n_items = offsets.numel() - 1
    if chosen is None:
        chosen = torch.empty(conf.numel(), dtype=torch.int32, device=conf.device)
    if tie is None:
        tie = torch.empty(max(1, n_items), dtype=torch.int32, device=conf.device)
    _lib.check(_lib.load().drt_select_choices(conf.data_ptr(), offsets.data_ptr(), n_items, int(mode), int(k),
                                              float(tau), float(tie_rel), chosen.data_ptr(), tie.data_ptr(),
                                              _stream_ptr(stream)))
    return chosen, tie


def linear_bf16(x: torch.Tensor, w: torch.Tensor, *, splits: int = 1, round_bf16: bool = True,
                out: torch.Tensor | None = None, scratch: torch.Tensor | None = None,
                stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """y = x @ w^T on the tcgen05 path: x [rows, K] bf16, w [n, K] bf16 -> y [rows, n] f32."""
    if x.dtype != torch.bfloat16 or w.dtype != torch.bfloat16 or not x.is_contiguous() or not w.is_contiguous():
        raise ValueError("x and w must be contiguous bf16 CUDA tensors")
    rows, K = x.shape
    n = w.shape[0]
    if out is None:
        out = torch.empty(rows, n, dtype=torch.float32, device=x.device)
    lib = _lib.load()
    if scratch is None:
        scratch = torch.empty(int(lib.drt_linear_scratch_bytes(rows, n, K, splits)), dtype=torch.uint8, device=x.device)
    _lib.check(lib.drt_linear_bf16(x.data_ptr(), w.data_ptr(), out.data_ptr(), rows, n, K, int(splits),
                                   int(bool(round_bf16)), scratch.data_ptr(), _stream_ptr(stream)))
    return out


def quantize_q4(w: torch.Tensor, *, stream: torch.cuda.Stream | None = None):
    """4-bit affine quantization of a bf16 [rows, K] weight: (packed uint8 [rows, K/2],
    scale bf16 [rows, K/64], bias bf16 [rows, K/64])."""
    if w.dtype != torch.bfloat16 or not w.is_contiguous() or w.dim() != 2:
        raise ValueError("w must be a contiguous bf16 CUDA matrix")
    rows, K = w.shape
    q = torch.empty(rows, K // 2, dtype=torch.uint8, device=w.device)
    scale = torch.empty(rows, K // 64, dtype=torch.bfloat16, device=w.device)
    bias = torch.empty(rows, K // 64, dtype=torch.bfloat16, device=w.device)
    _lib.check(_lib.load().drt_quantize_q4(w.data_ptr(), rows, K, q.data_ptr(), scale.data_ptr(), bias.data_ptr(),
                                           _stream_ptr(stream)))
    return q, scale, bias


def quantize_q8(w: torch.Tensor, *, stream: torch.cuda.Stream | None = None):
    """int8 weight-only quantization of a bf16 [rows, K] weight: (bytes uint8 [rows, K] = q + 128,
    scale bf16 [rows, K/64], bias = -128 * scale bf16 [rows, K/64])."""
    if w.dtype != torch.bfloat16 or not w.is_contiguous() or w.dim() != 2:
        raise ValueError("w must be a contiguous bf16 CUDA matrix")
    rows, K = w.shape
    q = torch.empty(rows, K, dtype=torch.uint8, device=w.device)
    scale = torch.empty(rows, K // 64, dtype=torch.bfloat16, device=w.device)
    bias = torch.empty(rows, K // 64, dtype=torch.bfloat16, device=w.device)
    _lib.check(_lib.load().drt_quantize_q8(w.data_ptr(), rows, K, q.data_ptr(), scale.data_ptr(), bias.data_ptr(),
                                           _stream_ptr(stream)))
    return q, scale, bias


def linear_q8(x: torch.Tensor, q: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor, *, splits: int = 1,
              out: torch.Tensor | None = None, stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """y = bf16(x @ dequant(q, scale, bias)^T) widened to f32 (int8 weight-only): x [rows <= 64, K] bf16."""
    rows, K = x.shape
    n = q.shape[0]
    if out is None:
        out = torch.empty(rows, n, dtype=torch.float32, device=x.device)
    _lib.check(_lib.load().drt_linear_q8(x.data_ptr(), q.data_ptr(), scale.data_ptr(), bias.data_ptr(), out.data_ptr(),
                                         rows, n, K, int(splits), _stream_ptr(stream)))
    return out


def linear_q4(x: torch.Tensor, q: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor, *, splits: int = 1,
              out: torch.Tensor | None = None, stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """y = x @ dequant(q, scale, bias)^T (f32, no output rounding): x [rows <= 64, K] bf16."""
    rows, K = x.shape
    n = q.shape[0]
    if out is None:
        out = torch.empty(rows, n, dtype=torch.float32, device=x.device)
    _lib.check(_lib.load().drt_linear_q4(x.data_ptr(), q.data_ptr(), scale.data_ptr(), bias.data_ptr(), out.data_ptr(),
                                         rows, n, K, int(splits), _stream_ptr(stream)))
    return out


# ------------------------------------------------------------------ batch serving: paged 8-bit cache, token scores
_TYPES = {torch.float32: _lib.TYPE_F32, torch.bfloat16: _lib.TYPE_BF16, torch.float16: _lib.TYPE_F16}
_CODES = {torch.int8: _lib.CODE_INT8, torch.float8_e4m3fn: _lib.CODE_E4M3}


def _need(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def _ints(t: torch.Tensor, name: str, device, shape: tuple[int, ...] | None = None) -> torch.Tensor:
    _need(isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.device == device and t.is_contiguous()
          and (t.dim() == 1 if shape is None else tuple(t.shape) == shape),
          f"{name} must be a contiguous int32 tensor{'' if shape is None else f' of shape {shape}'} on {device}")
    return t


def _launch(device, stream: torch.cuda.Stream | None, made: list, call) -> None:
    """call(stream pointer) with `device` current. Tensors made here are allocated on the current stream;
    the allocator is told when the work runs on another one."""
    with torch.cuda.device(device):
        current = torch.cuda.current_stream(device)
        use = stream if stream is not None else current
        _need(use.device == device, f"the stream belongs to {use.device}, the tensors to {device}")
        if use != current and made:
            use.wait_stream(current)  # memory that the allocator hands out may still be in use there
            for t in made:
                t.record_stream(use)
        _lib.check(call(int(use.cuda_stream)))


class CachePlan(NamedTuple):
    """A step's slot maps (all int32): row r of the batch is rows row_start[r] .. row_start[r + 1]."""

    row_start: torch.Tensor   # [requests + 1]
    slots: torch.Tensor       # [max_rows], -1 behind the last row
    positions: torch.Tensor   # [max_rows], -1 behind the last row
    lengths: torch.Tensor     # [requests] tokens after the step, 0 for a finished request
    held: torch.Tensor        # [requests] blocks after the step
    ring_state: torch.Tensor  # [2] (first free, free) of the ring after the step
    status: torch.Tensor      # [1] 0, blocks missing (> 0), or a refusal (< 0) as drt_cache_plan lists them


def plan_cache(start: torch.Tensor, count: torch.Tensor, held: torch.Tensor, tables: torch.Tensor, ring: torch.Tensor,
               ring_state: torch.Tensor, *, block_size: int, max_rows: int, held_out: torch.Tensor | None = None,
               ring_state_out: torch.Tensor | None = None, stream: torch.cuda.Stream | None = None) -> CachePlan:
    """Block tables and slot maps of a step from the requests' lengths, without a host read.

    Request r holds start[r] tokens in held[r] blocks (tables[r, :held[r]]) and gets count[r] rows, or has
    finished (-1: its blocks go back). Blocks come from and go to the circular buffer `ring` whose free ids
    are ring_state[1] entries from ring_state[0] on. tables and ring are updated in place; held and
    ring_state too, unless their _out tensors are other ones. A call that cannot be served changes nothing
    and says why in `status` (drt_cache_plan)."""
    _need(isinstance(start, torch.Tensor) and start.is_cuda, "start must be a CUDA tensor")
    dev = start.device
    _ints(start, "start", dev)
    n = start.numel()
    _ints(count, "count", dev, (n,))
    _ints(held, "held", dev, (n,))
    _ints(ring, "ring", dev)
    _ints(ring_state, "ring_state", dev, (2,))
    _need(isinstance(tables, torch.Tensor) and tables.dtype == torch.int32 and tables.device == dev and tables.dim() == 2
          and tables.shape[0] == n and tables.stride(1) == 1 and (n <= 1 or tables.stride(0) >= tables.shape[1]),
          f"tables must be an int32 [{n}, width] tensor with contiguous rows on {dev}")
    _need(max_rows >= 0, "max_rows must be >= 0")
    held_out = held if held_out is None else _ints(held_out, "held_out", dev, (n,))
    ring_state_out = ring_state if ring_state_out is None else _ints(ring_state_out, "ring_state_out", dev, (2,))
    out = [torch.empty(m, dtype=torch.int32, device=dev) for m in (n + 1, max_rows, max_rows, n, 1)]
    row_start, slots, positions, lengths, status = out
    width = tables.shape[1]
    _launch(dev, stream, out, lambda s: _lib.load().drt_cache_plan(
        start.data_ptr(), count.data_ptr(), held.data_ptr(), held_out.data_ptr(), n, tables.data_ptr(),
        max(tables.stride(0), width), width, int(block_size), ring.data_ptr(), ring.numel(), ring_state.data_ptr(),
        ring_state_out.data_ptr(), row_start.data_ptr(), slots.data_ptr(), positions.data_ptr(), int(max_rows),
        lengths.data_ptr(), status.data_ptr(), s))
    return CachePlan(row_start, slots, positions, lengths, held_out, ring_state_out, status)


def cache_q8(blocks: int, kv_heads: int, block_size: int, dim: int = 128, *, dtype: torch.dtype = torch.int8, device="cuda"):
    """A new, empty 8-bit cache: (k_cache, v_cache, k_scale, v_scale) in the layout of the operators below."""
    _need(dtype in _CODES, "an 8-bit cache holds int8 or float8_e4m3fn")
    _need(block_size in (16, 32, 64, 128), "a block holds 16, 32, 64 or 128 tokens")
    k = torch.zeros(blocks, kv_heads, block_size, dim, dtype=torch.int8, device=device).view(dtype)
    v = torch.zeros(blocks, kv_heads, block_size // 16, dim, 16, dtype=torch.int8, device=device).view(dtype)
    scale = torch.zeros(2, blocks, kv_heads, dtype=torch.float32, device=device)
    return k, v, scale[0], scale[1]


def _cache_args(k_cache, v_cache, k_scale, v_scale, device):
    """(blocks, kv_heads, block, dim, code) of a cache on `device`."""
    _need(all(isinstance(t, torch.Tensor) and t.device == device and t.is_contiguous()
              for t in (k_cache, v_cache, k_scale, v_scale)), f"the cache must be contiguous tensors on {device}")
    _need(k_cache.dtype in _CODES and v_cache.dtype == k_cache.dtype, "k_cache and v_cache must be int8 or float8_e4m3fn")
    _need(k_cache.dim() == 4, "k_cache must be [blocks, kv_heads, block, dim]")
    blocks, heads, block, dim = k_cache.shape
    _need(block in (16, 32, 64, 128), "a block holds 16, 32, 64 or 128 tokens")
    _need(tuple(v_cache.shape) == (blocks, heads, block // 16, dim, 16), "v_cache must be [blocks, kv_heads, block / 16, dim, 16]")
    for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        _need(t.dtype == torch.float32 and tuple(t.shape) == (blocks, heads), f"{name} must be float32 [blocks, kv_heads]")
    return blocks, heads, block, dim, _CODES[k_cache.dtype]


def append_cache_q8(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    k_scale: torch.Tensor, v_scale: torch.Tensor, *, stream: torch.cuda.Stream | None = None) -> None:
    """Rows of K and V [rows, kv_heads, dim] (bf16 or f16, any row and head stride) into the slots of the cache.

    A block's scale covers its tokens: it grows with the largest value appended (the tokens already there are
    rounded anew), and a run of rows that begins a block starts it anew. Rows whose slot is -1 are skipped;
    slots are distinct and those of one block consecutive rows, as plan_cache gives them."""
    _need(isinstance(k, torch.Tensor) and k.is_cuda and k.dim() == 3, "k must be a CUDA tensor [rows, kv_heads, dim]")
    dev = k.device
    blocks, heads, block, dim, code = _cache_args(k_cache, v_cache, k_scale, v_scale, dev)
    rows = k.shape[0]
    for name, t in (("k", k), ("v", v)):
        _need(isinstance(t, torch.Tensor) and t.device == dev and t.dtype == k.dtype and tuple(t.shape) == (rows, heads, dim)
              and t.stride(2) == 1, f"{name} must be [rows, {heads}, {dim}] with a contiguous last dimension on {dev}")
    _need(k.dtype in (torch.bfloat16, torch.float16), "k and v must be bf16 or f16")
    _ints(slots, "slots", dev)
    _need(slots.numel() >= rows, "one slot per row")
    _launch(dev, stream, [], lambda s: _lib.load().drt_cache_append(
        k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), _TYPES[k.dtype], rows,
        slots.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), blocks, heads,
        block, dim, code, s))


def read_cache_q8(slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                  v_scale: torch.Tensor, *, dtype: torch.dtype = torch.bfloat16, stream: torch.cuda.Stream | None = None):
    """The K and V values of the listed slots, [slots, kv_heads, dim] each, rounded once to dtype (zeros for -1)."""
    _need(isinstance(slots, torch.Tensor) and slots.is_cuda, "slots must be a CUDA tensor")
    dev = slots.device
    _ints(slots, "slots", dev)
    blocks, heads, block, dim, code = _cache_args(k_cache, v_cache, k_scale, v_scale, dev)
    _need(dtype in _TYPES, "values are read as bfloat16, float16 or float32")
    k, v = (torch.empty(slots.numel(), heads, dim, dtype=dtype, device=dev) for _ in range(2))
    _launch(dev, stream, [k, v], lambda s: _lib.load().drt_cache_read(
        slots.data_ptr(), slots.numel(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
        blocks, heads, block, dim, code, k.data_ptr(), v.data_ptr(), _TYPES[dtype], s))
    return k, v


def attend_scratch(dim: int, device) -> torch.Tensor:
    """Scratch of one attend_cache_q8 call in flight (captured graphs that may run at once need one each)."""
    with torch.cuda.device(device):
        return torch.empty(int(_lib.load().drt_cache_attend_scratch_bytes(int(dim))), dtype=torch.uint8, device=device)


def attend_cache_q8(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                    v_scale: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor, row_start: torch.Tensor, *,
                    mask_block: int = 1, origin: torch.Tensor | None = None, scale: float | None = None, max_rows: int = 0,
                    out: torch.Tensor | None = None, lse: torch.Tensor | None = None, scratch: torch.Tensor | None = None,
                    stream: torch.cuda.Stream | None = None):
    """Attention of the rows of many requests over the 8-bit cache: (out, lse), both in row order.

    q [rows, heads, dim] (bf16 or f16); request r's rows row_start[r] .. row_start[r + 1] are the last of its
    lengths[r] tokens, all of them in the cache. mask_block 1 is causal, b > 1 lets a row see its whole block of
    b positions counted from origin[r] (the d2f_hybrid mask; the positions before origin see one another),
    0 shows every token. scale defaults to 1 / sqrt(dim). max_rows: a bound on a request's rows, if the
    caller knows one (1 for single-token decoding); it changes speed only. Rows behind the last request's
    are left as they are in `out` and `lse` (new ones: zeros)."""
    _need(isinstance(q, torch.Tensor) and q.is_cuda and q.dim() == 3 and q.dtype in (torch.bfloat16, torch.float16)
          and q.stride(2) == 1, "q must be a bf16 or f16 CUDA tensor [rows, heads, dim] with a contiguous last dimension")
    dev = q.device
    rows, heads, dim = q.shape
    blocks, kv_heads, block, kdim, code = _cache_args(k_cache, v_cache, k_scale, v_scale, dev)
    _need(dim == kdim and heads % kv_heads == 0, "q and the cache disagree on heads or dim")
    _ints(lengths, "lengths", dev)
    n = lengths.numel()
    _ints(row_start, "row_start", dev, (n + 1,))
    _need(isinstance(tables, torch.Tensor) and tables.dtype == torch.int32 and tables.device == dev and tables.dim() == 2
          and tables.shape[0] == n and tables.stride(1) == 1 and (n <= 1 or tables.stride(0) >= tables.shape[1]),
          f"tables must be an int32 [{n}, width] tensor with contiguous rows on {dev}")
    if origin is not None:
        _ints(origin, "origin", dev, (n,))
    made = []
    if out is None:
        out = torch.zeros(rows, heads, dim, dtype=q.dtype, device=dev)
        made.append(out)
    _need(out.dtype == q.dtype and out.device == dev and out.shape == q.shape and out.stride(2) == 1,
          "out must have q's shape and dtype and a contiguous last dimension")
    if lse is None:
        lse = torch.zeros(rows, heads, dtype=torch.float32, device=dev)
        made.append(lse)
    _need(lse.dtype == torch.float32 and lse.device == dev and tuple(lse.shape) == (rows, heads) and lse.is_contiguous(),
          "lse must be a contiguous float32 [rows, heads] tensor")
    if scratch is None:
        scratch = attend_scratch(dim, dev)
        made.append(scratch)
    with torch.cuda.device(dev):
        _need(scratch.device == dev and scratch.is_contiguous()
              and scratch.numel() * scratch.element_size() >= _lib.load().drt_cache_attend_scratch_bytes(dim),
              "scratch is too small (attend_scratch)")
    args = _lib.CacheAttendArgs(
        q=q.data_ptr(), q_row=q.stride(0), q_head=q.stride(1), out=out.data_ptr(), out_row=out.stride(0),
        out_head=out.stride(1), lse=lse.data_ptr(), k_cache=k_cache.data_ptr(), v_cache=v_cache.data_ptr(),
        k_scale=k_scale.data_ptr(), v_scale=v_scale.data_ptr(), blocks=blocks, tables=tables.data_ptr(),
        ld_tables=max(tables.stride(0), tables.shape[1]), lengths=lengths.data_ptr(), row_start=row_start.data_ptr(),
        origin=None if origin is None else origin.data_ptr(), scratch=scratch.data_ptr(), q_rows=rows, heads=heads,
        kv_heads=kv_heads, dim=dim, dtype=_TYPES[q.dtype], code=code, block=block, width=tables.shape[1], requests=n,
        mask_block=int(mask_block), max_rows=int(max_rows), scale=1 / math.sqrt(dim) if scale is None else float(scale))
    _launch(dev, stream, made, lambda s: _lib.load().drt_cache_attend(ctypes.byref(args), s))
    return out, lse


class TokenScores(NamedTuple):
    """Per row: of the given token, of the distribution, and of its likeliest tokens."""

    logprob: torch.Tensor      # f32 [rows]
    entropy: torch.Tensor      # f32 [rows], nats
    rank: torch.Tensor         # int32 [rows], 0 for the first argmax
    top_token: torch.Tensor    # int32 [rows, top], -1 behind the last of non-zero probability
    top_logprob: torch.Tensor  # f32 [rows, top]


def select_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0, temperature: float = 0.0,
                    exclude_token: int = -1, row_index: torch.Tensor | None = None, scratch: torch.Tensor | None = None,
                    stream: torch.cuda.Stream | None = None) -> TokenScores:
    """Log probabilities of given tokens (int32) under softmax(logits / T) of f32, bf16 or f16 rows [rows, vocab]
    (or of the rows row_index), with the entropy, the token's rank and the `top` <= 32 likeliest tokens.
    exclude_token counts as a logit of -inf; a token outside the vocabulary scores -inf with rank -1."""
    _need(isinstance(logits, torch.Tensor) and logits.is_cuda and logits.dim() == 2 and logits.dtype in _TYPES
          and logits.stride(1) == 1, "logits must be a row-major CUDA float32, bfloat16 or float16 [rows, vocab] tensor")
    dev = logits.device
    _ints(tokens, "tokens", dev)
    n = tokens.numel()
    if row_index is None:
        _need(n == logits.shape[0], "one token per logits row")
    else:
        _ints(row_index, "row_index", dev, (n,))
    _need(0 <= top <= 32, "top must be in [0, 32]")
    vocab, typ = logits.shape[1], _TYPES[logits.dtype]
    made = [torch.empty(n, dtype=torch.float32, device=dev), torch.empty(n, dtype=torch.float32, device=dev),
            torch.empty(n, dtype=torch.int32, device=dev), torch.empty(n, top, dtype=torch.int32, device=dev),
            torch.empty(n, top, dtype=torch.float32, device=dev)]
    out = TokenScores(*made)
    with torch.cuda.device(dev):
        size = int(_lib.load().drt_selector_logprobs_scratch_bytes(n, vocab, typ))
    if scratch is None:
        scratch = torch.empty(size, dtype=torch.uint8, device=dev)
        made.append(scratch)
    _need(scratch.device == dev and scratch.is_contiguous() and scratch.numel() * scratch.element_size() >= size,
          f"scratch must hold {size} bytes")
    _launch(dev, stream, made, lambda s: _lib.load().drt_selector_logprobs(
        logits.data_ptr(), typ, max(logits.stride(0), vocab), None if row_index is None else row_index.data_ptr(), n, vocab,
        tokens.data_ptr(), float(temperature), int(exclude_token), int(top), scratch.data_ptr(), out.logprob.data_ptr(),
        out.entropy.data_ptr(), out.rank.data_ptr(), out.top_token.data_ptr(), out.top_logprob.data_ptr(), s))
    return out
