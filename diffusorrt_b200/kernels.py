"""Kernel-level entry points on torch CUDA tensors (device memory and streams come from torch).

These call the C ABI directly with device pointers; they are the unit-level surface used by the
selector microbenchmark and the kernel parity tests, and the operators of a server that batches
requests: the paged 8-bit K/V cache (plan_cache, append_cache_q8, read_cache_q8, attend_cache_q8) and
the token scorer (select_logprobs).
"""
from __future__ import annotations

import functools
import math
import struct
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
# These run once or more per layer and step, so their host path is kept short: attributes are read once, messages
# are built only when a check fails, and outputs of one type share an allocation.
_TYPES = {torch.float32: _lib.TYPE_F32, torch.bfloat16: _lib.TYPE_BF16, torch.float16: _lib.TYPE_F16}
_CODES = {torch.int8: _lib.CODE_INT8, torch.float8_e4m3fn: _lib.CODE_E4M3}
_I32 = torch.int32
_ATTEND = struct.Struct("@PqqPqq5PqPq4P11if")  # CacheAttendArgs
_scratch_bytes: dict[tuple[int, int], int] = {}


def _check_ints(t, name: str, index: int, n: int | None = None) -> None:
    """t is a contiguous int32 vector (of n entries) on device `index` (-1: the CPU)."""
    if not (isinstance(t, torch.Tensor) and t.dtype is _I32 and t.get_device() == index and t.dim() == 1
            and t.is_contiguous() and (n is None or t.numel() == n)):
        raise ValueError(f"{name} must be a contiguous int32 vector{'' if n is None else f' of {n} entries'} on "
                         f"{'the CPU' if index < 0 else f'cuda:{index}'}")


def _check_tables(t, index: int, n: int) -> tuple[int, int]:
    """(width, row stride) of the block tables."""
    if isinstance(t, torch.Tensor) and t.dtype is _I32 and t.get_device() == index and t.dim() == 2:
        rows, width = t.shape
        ld, step = t.stride()
        if rows == n and step == 1 and (n <= 1 or ld >= width):
            return width, max(ld, width)
    raise ValueError(f"tables must be an int32 [{n}, width] tensor with contiguous rows on cuda:{index}")


def _launch(index: int, stream: torch.cuda.Stream | None, made, fn, *args) -> None:
    """fn(*args, stream) with device `index` current. Tensors made for the call belong to the current stream; when
    the work runs on another one, that waits for it and the allocator is told."""
    if stream is None:
        if torch.cuda.current_device() == index:
            _lib.check(fn(*args, _current_stream(index)))
        else:
            with torch.cuda.device(index):
                _lib.check(fn(*args, _current_stream(index)))
        return
    if stream.device.index != index:
        raise ValueError(f"the stream belongs to {stream.device}, the tensors to cuda:{index}")
    with torch.cuda.device(index):
        current = torch.cuda.current_stream(index)
        if stream != current and made:
            stream.wait_stream(current)  # memory that the allocator hands out may still be in use there
            for t in made:
                t.record_stream(stream)
        _lib.check(fn(*args, int(stream.cuda_stream)))


def _current_stream(index: int) -> int:
    return int(torch.cuda.current_stream(index).cuda_stream)


if hasattr(torch._C, "_cuda_getCurrentRawStream"):
    _current_stream = torch._C._cuda_getCurrentRawStream  # noqa: F811  (the same without a Stream object)


class CachePlan(NamedTuple):
    """A step's slot maps (all int32): request r's rows in the batch are row_start[r] .. row_start[r + 1]."""

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
    if not (isinstance(start, torch.Tensor) and start.is_cuda):
        raise ValueError("start must be a CUDA tensor")
    index, n = start.get_device(), start.numel()
    _check_ints(start, "start", index)
    _check_ints(count, "count", index, n)
    _check_ints(held, "held", index, n)
    _check_ints(ring, "ring", index)
    _check_ints(ring_state, "ring_state", index, 2)
    width, ld = _check_tables(tables, index, n)
    if max_rows < 0:
        raise ValueError("max_rows must be >= 0")
    if held_out is None:
        held_out = held
    else:
        _check_ints(held_out, "held_out", index, n)
    if ring_state_out is None:
        ring_state_out = ring_state
    else:
        _check_ints(ring_state_out, "ring_state_out", index, 2)
    made = torch.empty(2 * n + 2 * max_rows + 2, dtype=_I32, device=start.device)
    row_start, slots, positions, lengths, status = made.split_with_sizes((n + 1, max_rows, max_rows, n, 1))
    p = made.data_ptr()
    _launch(index, stream, (made,), _lib.load().drt_cache_plan, start.data_ptr(), count.data_ptr(), held.data_ptr(),
            held_out.data_ptr(), n, tables.data_ptr(), ld, width, block_size, ring.data_ptr(), ring.numel(),
            ring_state.data_ptr(), ring_state_out.data_ptr(), p, p + 4 * (n + 1), p + 4 * (n + 1 + max_rows), max_rows,
            p + 4 * (n + 1 + 2 * max_rows), p + 4 * (2 * n + 1 + 2 * max_rows))
    return CachePlan(row_start, slots, positions, lengths, held_out, ring_state_out, status)


def cache_q8(blocks: int, kv_heads: int, block_size: int, dim: int = 128, *, dtype: torch.dtype = torch.int8, device="cuda"):
    """A new, empty 8-bit cache: (k_cache, v_cache, k_scale, v_scale) in the layout of the operators below."""
    if dtype not in _CODES:
        raise ValueError("an 8-bit cache holds int8 or float8_e4m3fn")
    if block_size not in (16, 32, 64, 128):
        raise ValueError("a block holds 16, 32, 64 or 128 tokens")
    k = torch.zeros(blocks, kv_heads, block_size, dim, dtype=torch.int8, device=device).view(dtype)
    v = torch.zeros(blocks, kv_heads, block_size // 16, dim, 16, dtype=torch.int8, device=device).view(dtype)
    scale = torch.zeros(2, blocks, kv_heads, dtype=torch.float32, device=device)
    return k, v, scale[0], scale[1]


def _cache_args(k_cache, v_cache, k_scale, v_scale, index: int):
    """(blocks, kv_heads, block, dim, code) of a cache on device `index`."""
    for t in (k_cache, v_cache, k_scale, v_scale):
        if isinstance(t, torch.Tensor) and t.get_device() == index and t.is_contiguous():
            continue
        raise ValueError(f"the cache must be contiguous tensors on {'the CPU' if index < 0 else f'cuda:{index}'}")
    code = _CODES.get(k_cache.dtype)
    if code is None or v_cache.dtype is not k_cache.dtype:
        raise ValueError("k_cache and v_cache must be int8 or float8_e4m3fn")
    if k_cache.dim() != 4:
        raise ValueError("k_cache must be [blocks, kv_heads, block, dim]")
    blocks, heads, block, dim = k_cache.shape
    if block not in (16, 32, 64, 128):
        raise ValueError("a block holds 16, 32, 64 or 128 tokens")
    if v_cache.shape != (blocks, heads, block // 16, dim, 16):
        raise ValueError("v_cache must be [blocks, kv_heads, block / 16, dim, 16]")
    shape = (blocks, heads)
    if k_scale.shape != shape or v_scale.shape != shape or k_scale.dtype is not torch.float32 or v_scale.dtype is not torch.float32:
        raise ValueError("k_scale and v_scale must be float32 [blocks, kv_heads]")
    return blocks, heads, block, dim, code


def append_cache_q8(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    k_scale: torch.Tensor, v_scale: torch.Tensor, *, stream: torch.cuda.Stream | None = None) -> None:
    """Rows of K and V [rows, kv_heads, dim] (bf16 or f16, any row and head stride) into the slots of the cache.

    A block's scale covers its tokens: it grows with the largest value appended (the tokens already there are
    rounded anew), and a run of rows that begins a block starts it anew. Rows whose slot is -1 are skipped;
    slots are distinct and those of one block consecutive rows, as plan_cache gives them."""
    if not (isinstance(k, torch.Tensor) and k.is_cuda and k.dim() == 3):
        raise ValueError("k must be a CUDA tensor [rows, kv_heads, dim]")
    index = k.get_device()
    blocks, heads, block, dim, code = _cache_args(k_cache, v_cache, k_scale, v_scale, index)
    shape, dtype = k.shape, k.dtype
    rows = shape[0]
    if not (isinstance(v, torch.Tensor) and v.get_device() == index and v.dtype is dtype and v.shape == shape
            and shape[1] == heads and shape[2] == dim):
        raise ValueError(f"k and v must be [rows, {heads}, {dim}] of one type on cuda:{index}")
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise ValueError("k and v must be bf16 or f16")
    k_row, k_head, k_dim = k.stride()
    v_row, v_head, v_dim = v.stride()
    if k_dim != 1 or v_dim != 1:
        raise ValueError("k and v must have a contiguous last dimension")
    _check_ints(slots, "slots", index)
    if slots.numel() < rows:
        raise ValueError("one slot per row")
    _launch(index, stream, (), _lib.load().drt_cache_append, k.data_ptr(), k_row, k_head, v.data_ptr(), v_row, v_head,
            _TYPES[dtype], rows, slots.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(),
            v_scale.data_ptr(), blocks, heads, block, dim, code)


def read_cache_q8(slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                  v_scale: torch.Tensor, *, dtype: torch.dtype = torch.bfloat16, stream: torch.cuda.Stream | None = None):
    """The K and V values of the listed slots, [slots, kv_heads, dim] each, rounded once to dtype (zeros for -1)."""
    if not (isinstance(slots, torch.Tensor) and slots.is_cuda):
        raise ValueError("slots must be a CUDA tensor")
    index = slots.get_device()
    _check_ints(slots, "slots", index)
    blocks, heads, block, dim, code = _cache_args(k_cache, v_cache, k_scale, v_scale, index)
    if dtype not in _TYPES:
        raise ValueError("values are read as bfloat16, float16 or float32")
    n = slots.numel()
    made = torch.empty(2, n, heads, dim, dtype=dtype, device=slots.device)
    k, v = made.unbind(0)
    _launch(index, stream, (made,), _lib.load().drt_cache_read, slots.data_ptr(), n, k_cache.data_ptr(), v_cache.data_ptr(),
            k_scale.data_ptr(), v_scale.data_ptr(), blocks, heads, block, dim, code, k.data_ptr(), v.data_ptr(), _TYPES[dtype])
    return k, v


def _attend_bytes(dim: int, index: int) -> int:
    size = _scratch_bytes.get((index, dim))
    if size is None:
        with torch.cuda.device(index):
            size = _scratch_bytes[index, dim] = int(_lib.load().drt_cache_attend_scratch_bytes(int(dim)))
    return size


def attend_scratch(dim: int, device) -> torch.Tensor:
    """Scratch of one attend_cache_q8 call in flight (captured graphs that may run at once need one each)."""
    device = torch.device(device)
    index = torch.cuda.current_device() if device.index is None else device.index
    return torch.empty(_attend_bytes(dim, index), dtype=torch.uint8, device=torch.device("cuda", index))


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
    if not (isinstance(q, torch.Tensor) and q.is_cuda and q.dim() == 3):
        raise ValueError("q must be a CUDA tensor [rows, heads, dim]")
    index, dtype, shape = q.get_device(), q.dtype, q.shape
    rows, heads, dim = shape
    q_row, q_head, q_dim = q.stride()
    if q_dim != 1 or (dtype is not torch.bfloat16 and dtype is not torch.float16):
        raise ValueError("q must be bf16 or f16 with a contiguous last dimension")
    blocks, kv_heads, block, kdim, code = _cache_args(k_cache, v_cache, k_scale, v_scale, index)
    if dim != kdim or heads % kv_heads != 0:
        raise ValueError("q and the cache disagree on heads or dim")
    _check_ints(lengths, "lengths", index)
    n = lengths.numel()
    _check_ints(row_start, "row_start", index, n + 1)
    width, ld = _check_tables(tables, index, n)
    if origin is not None:
        _check_ints(origin, "origin", index, n)
    made = []
    if out is None:
        out = torch.zeros(rows, heads, dim, dtype=dtype, device=q.device)
        made.append(out)
    elif not (isinstance(out, torch.Tensor) and out.dtype is dtype and out.get_device() == index and out.shape == shape):
        raise ValueError("out must have q's shape and dtype on its device")
    out_row, out_head, out_dim = out.stride()
    if out_dim != 1:
        raise ValueError("out must have a contiguous last dimension")
    if lse is None:
        lse = torch.zeros(rows, heads, dtype=torch.float32, device=q.device)
        made.append(lse)
    elif not (isinstance(lse, torch.Tensor) and lse.dtype is torch.float32 and lse.get_device() == index
              and lse.shape == (rows, heads) and lse.is_contiguous()):
        raise ValueError("lse must be a contiguous float32 [rows, heads] tensor")
    if not (0 <= mask_block <= 1 << 24 and 0 <= max_rows < 1 << 31):
        raise ValueError("mask_block outside [0, 2^24] or max_rows outside [0, 2^31)")
    size = _attend_bytes(dim, index)
    if scratch is None:
        scratch = torch.empty(size, dtype=torch.uint8, device=q.device)
        made.append(scratch)
    elif not (scratch.get_device() == index and scratch.is_contiguous() and scratch.numel() * scratch.element_size() >= size):
        raise ValueError("scratch is too small (attend_scratch)")
    args = _ATTEND.pack(
        q.data_ptr(), q_row, q_head, out.data_ptr(), out_row, out_head, lse.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
        k_scale.data_ptr(), v_scale.data_ptr(), blocks, tables.data_ptr(), ld, lengths.data_ptr(), row_start.data_ptr(),
        0 if origin is None else origin.data_ptr(), scratch.data_ptr(), rows, heads, kv_heads, dim, _TYPES[dtype], code, block,
        width, n, mask_block, max_rows, 1 / math.sqrt(dim) if scale is None else scale)
    _launch(index, stream, made, _lib.load().drt_cache_attend, args)
    return out, lse


class TokenScores(NamedTuple):
    """Per row: of the given token, of the distribution, and of its likeliest tokens."""

    logprob: torch.Tensor      # f32 [rows]
    entropy: torch.Tensor      # f32 [rows], nats
    rank: torch.Tensor         # int32 [rows], 0 for the first argmax
    top_token: torch.Tensor    # int32 [rows, top], -1 behind the last of non-zero probability
    top_logprob: torch.Tensor  # f32 [rows, top]


@functools.lru_cache(maxsize=1024)
def _logprob_bytes(n: int, vocab: int, typ: int, index: int) -> int:
    with torch.cuda.device(index):
        return int(_lib.load().drt_selector_logprobs_scratch_bytes(n, vocab, typ))


def select_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0, temperature: float = 0.0,
                    exclude_token: int = -1, row_index: torch.Tensor | None = None, scratch: torch.Tensor | None = None,
                    stream: torch.cuda.Stream | None = None) -> TokenScores:
    """Log probabilities of given tokens (int32) under softmax(logits / T) of f32, bf16 or f16 rows [rows, vocab]
    (or of the rows row_index), with the entropy, the token's rank and the `top` <= 32 likeliest tokens.
    exclude_token counts as a logit of -inf; a token outside the vocabulary, or of a row_index
    outside the logits, scores -inf with rank -1."""
    if not (isinstance(logits, torch.Tensor) and logits.is_cuda and logits.dim() == 2):
        raise ValueError("logits must be a CUDA tensor [rows, vocab]")
    index = logits.get_device()
    typ = _TYPES.get(logits.dtype)
    ld, step = logits.stride()
    if typ is None or step != 1:
        raise ValueError("logits must be row-major float32, bfloat16 or float16")
    have, vocab = logits.shape
    _check_ints(tokens, "tokens", index)
    n = tokens.numel()
    if row_index is not None:
        _check_ints(row_index, "row_index", index, n)
    elif n != have:
        raise ValueError("one token per logits row")
    if not 0 <= top <= 32:
        raise ValueError("top must be in [0, 32]")
    if not -1 <= exclude_token < vocab:
        raise ValueError("exclude_token outside the vocabulary")
    size = _logprob_bytes(n, vocab, typ, index)
    words = n * (3 + 2 * top)
    # outputs in one allocation, the call's scratch in front of them
    own = (size + 3) // 4 if scratch is None else 0
    made = torch.empty(own + words, dtype=torch.float32, device=logits.device)
    if scratch is not None and not (scratch.get_device() == index and scratch.is_contiguous()
                                    and scratch.numel() * scratch.element_size() >= size):
        raise ValueError(f"scratch must hold {size} bytes")
    _, logprob, entropy, top_logprob, whole = made.split_with_sizes((own, n, n, n * top, n * (1 + top)))
    rank, top_token = whole.view(_I32).split_with_sizes((n, n * top))
    p = made.data_ptr()
    at = p + 4 * own
    _launch(index, stream, (made,) if scratch is None else (made, scratch), _lib.load().drt_selector_logprobs,
            logits.data_ptr(), typ, max(ld, vocab), have, 0 if row_index is None else row_index.data_ptr(), n, vocab,
            tokens.data_ptr(), temperature, exclude_token, top, p if scratch is None else scratch.data_ptr(), at, at + 4 * n,
            at + 4 * n * (2 + top), at + 4 * n * (3 + top), at + 8 * n)
    return TokenScores(logprob, entropy, rank, top_token.view(n, top), top_logprob.view(n, top))
