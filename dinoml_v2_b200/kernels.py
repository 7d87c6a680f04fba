"""Tensor-level wrappers over the C-ABI kernels (torch is used for device memory and streams only)."""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _native
from .gguf_blocks import qtype_of, row_bytes

_TORCH_DTYPE = {"float16": torch.float16, "float32": torch.float32, "bfloat16": torch.bfloat16}
_DTYPE_NAME = {v: k for k, v in _TORCH_DTYPE.items()}


def _stream_ptr(stream) -> int:
    if stream is None:
        stream = torch.cuda.current_stream()
    return int(stream.cuda_stream)


def _require_cuda(t: torch.Tensor, name: str) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (the GGUF quantized-linear path has no CPU implementation)")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _require_current_device(t: torch.Tensor, name: str) -> None:
    """A launch goes to the current device, whose kernels would take another device's addresses for their own."""
    if t.device.index != torch.cuda.current_device():
        raise ValueError(f"{name} is on {t.device}, the current device is cuda:{torch.cuda.current_device()}")


_binding = None


class _NoBinding:
    """Stands in for a native binding that does not load: every call is left to the wrapper's own path."""

    def __getattr__(self, name):
        return lambda *args: None


def _native_call(name: str):
    """A function of the native binding.  The binding is loaded on the first call."""
    global _binding
    if _binding is None:
        _binding = _native.binding() or _NoBinding()
    return getattr(_binding, name)


def dequantize_rows(blocks: torch.Tensor, qtype, n_per_row: int, dtype: str = "float32", out: torch.Tensor | None = None,
                    stream=None) -> torch.Tensor:
    """uint8 [rows, row_bytes] GGUF blocks -> dense [rows, n_per_row] (bit-exact dequantization)."""
    done = _native_call("dequantize")(blocks, qtype, n_per_row, dtype, out, stream)      # None: not the plain case, checked below
    if done is not None:
        if type(done) is int:
            _native.check(done, "libgguf_cuda_dequantize_rows_on_stream")
        return done
    q = qtype_of(qtype)
    _require_cuda(blocks, "blocks")
    if blocks.dtype != torch.uint8 or blocks.dim() != 2 or blocks.shape[1] != row_bytes(q, n_per_row):
        raise ValueError(f"blocks must be uint8 [rows, {row_bytes(q, n_per_row)}] for {q.name} with n_per_row={n_per_row}")
    rows = blocks.shape[0]
    if out is None:
        out = torch.empty((rows, n_per_row), dtype=_TORCH_DTYPE[dtype], device=blocks.device)
    _require_cuda(out, "out")
    rc = _native.lib().libgguf_cuda_dequantize_rows_on_stream(
        blocks.data_ptr(), q.value, rows, n_per_row, _native.DEQUANT_DTYPE[dtype], out.data_ptr(), _stream_ptr(stream))
    _native.check(rc, "libgguf_cuda_dequantize_rows_on_stream")
    return out


def gemm_rcr(a: torch.Tensor, b_quant: torch.Tensor, qtype, bias: torch.Tensor | None = None, *, variant: str = "auto",
             out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """a [..., K] x GGUF-encoded weight (uint8 [N, row_bytes]) -> [..., N], same dtype as `a`."""
    done = _native_call("linear")(a, b_quant, qtype, bias, variant, out, stream)          # None: not the plain case, checked below
    if done is not None:
        if type(done) is int:
            _native.check(done, "dinoml_b200_gguf_gemm_rcr")
        return done
    q = qtype_of(qtype)
    _require_cuda(a, "a")
    _require_cuda(b_quant, "b_quant")
    k = a.shape[-1]
    m = a.numel() // k
    n = b_quant.shape[0]
    if b_quant.dtype != torch.uint8 or b_quant.dim() != 2 or b_quant.shape[1] != row_bytes(q, k):
        raise ValueError(f"b_quant must be uint8 [N, {row_bytes(q, k)}] for {q.name} with K={k}")
    dtype = _DTYPE_NAME[a.dtype]
    if bias is not None:
        _require_cuda(bias, "bias")
        if bias.dtype != a.dtype or bias.numel() != n:
            raise ValueError("bias must have the activation dtype and N elements")
    if out is None:
        out = torch.empty(a.shape[:-1] + (n,), dtype=a.dtype, device=a.device)
    _require_cuda(out, "out")
    rc = _native.lib().dinoml_b200_gguf_gemm_rcr(
        a.data_ptr(), b_quant.data_ptr(), bias.data_ptr() if bias is not None else None, out.data_ptr(), q.value,
        _native.DINO_DTYPE[dtype], m, n, k, _native.variant_code(variant), _stream_ptr(stream))
    _native.check(rc, "dinoml_b200_gguf_gemm_rcr")
    return out


def interleave_rows8(b0, b1):
    """Row order the gated dual GEMM expects: rows 16t..16t+7 = rows 8t..8t+7 of b0, rows 16t+8..16t+15 = of b1.
    b0, b1: [N, row_bytes] (torch tensors or numpy arrays), N % 8 == 0; a b1 of ONE row (the reference's [1, K] broadcast,
    src/dinoml/kernels/families/dual_gemm.py:60-66) is repeated N times.  Blocks are not touched."""
    if b1.shape[0] == 1 and b0.shape[0] != 1 and b1.shape[1:] == b0.shape[1:]:
        b1 = b1.expand(b0.shape[0], -1) if isinstance(b1, torch.Tensor) else __import__("numpy").broadcast_to(b1, b0.shape)
    if b0.shape != b1.shape or b0.shape[0] % 8:
        raise ValueError("both weights must have the same shape (or b1 one row) and a row count that is a multiple of 8")
    n, rb = b0.shape
    if isinstance(b0, torch.Tensor):
        return torch.stack((b0.reshape(n // 8, 8, rb), b1.reshape(n // 8, 8, rb)), dim=1).reshape(2 * n, rb).contiguous()
    import numpy as np
    return np.ascontiguousarray(np.stack((b0.reshape(n // 8, 8, rb), b1.reshape(n // 8, 8, rb)), axis=1).reshape(2 * n, rb))


def interleave_bias8(bias0, bias1):
    """[2N] bias vector of the gated dual GEMM with bias: 8 values of bias0, the 8 matching values of bias1, ... - the order of
    `interleave_rows8`.  bias1 of one element (B1 [1, K]) is repeated."""
    return interleave_rows8(bias0.reshape(-1, 1), bias1.reshape(-1, 1)).reshape(-1)


def dual_gemm_rcr(a: torch.Tensor, b01_interleaved: torch.Tensor, qtype, activation: str = "silu", *, variant: str = "auto",
                  out: torch.Tensor | None = None, stream=None, bias01_interleaved: torch.Tensor | None = None) -> torch.Tensor:
    """act(a @ dequant(B0)^T [+ bias0]) * (a @ dequant(B1)^T [+ bias1]) in one launch; `b01_interleaved` =
    interleave_rows8(B0, B1), `bias01_interleaved` = interleave_bias8(bias0, bias1) in the activation dtype.
    a [..., K] -> [..., N] with N = rows of each matrix.  Mirrors dml.ops.dual_gemm_rcr_silu / _fast_gelu and their
    _bias_ forms of the reference (src/dinoml/ops/gemm.py:63-121) for GGUF weights."""
    done = _native_call("gated")(a, b01_interleaved, qtype, bias01_interleaved, variant, out, stream, activation)
    if done is not None:
        if type(done) is int:
            _native.check(done, "dinoml_b200_gguf_dual_gemm_rcr")
        return done
    q = qtype_of(qtype)
    _require_cuda(a, "a")
    _require_cuda(b01_interleaved, "b01_interleaved")
    k = a.shape[-1]
    m = a.numel() // k
    rows = b01_interleaved.shape[0]
    if b01_interleaved.dtype != torch.uint8 or b01_interleaved.dim() != 2 or b01_interleaved.shape[1] != row_bytes(q, k) or rows % 16:
        raise ValueError(f"b01_interleaved must be uint8 [2N, {row_bytes(q, k)}] with N % 8 == 0 for {q.name} with K={k}")
    n = rows // 2
    if activation not in _native.ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(_native.ACTIVATIONS)}")
    if out is None:
        out = torch.empty(a.shape[:-1] + (n,), dtype=a.dtype, device=a.device)
    _require_cuda(out, "out")
    if bias01_interleaved is not None:
        _require_cuda(bias01_interleaved, "bias01_interleaved")
        if bias01_interleaved.dtype != a.dtype or bias01_interleaved.numel() != 2 * n:
            raise ValueError("bias01_interleaved must have the activation dtype and 2N elements")
    rc = _native.lib().dinoml_b200_gguf_dual_gemm_rcr_bias(
        a.data_ptr(), b01_interleaved.data_ptr(), bias01_interleaved.data_ptr() if bias01_interleaved is not None else None,
        out.data_ptr(), None, 0, q.value, _native.DINO_DTYPE[_DTYPE_NAME[a.dtype]], m, n, k,
        _native.ACTIVATIONS[activation], _native.variant_code(variant), _stream_ptr(stream))
    _native.check(rc, "dinoml_b200_gguf_dual_gemm_rcr")
    return out


def profile_gemm_rcr(a, b_quant, qtype, out, *, variant: str, iterations: int, bias=None, stream=None) -> float:
    """Milliseconds per launch of one candidate (negative on failure), timed by the library with CUDA events."""
    q = qtype_of(qtype)
    k = a.shape[-1]
    return float(_native.lib().dinoml_profile_b200_gguf_gemm_rcr(
        a.data_ptr(), b_quant.data_ptr(), bias.data_ptr() if bias is not None else None, out.data_ptr(), q.value,
        _native.DINO_DTYPE[_DTYPE_NAME[a.dtype]], a.numel() // k, b_quant.shape[0], k, _native.variant_code(variant),
        int(iterations), _stream_ptr(stream)))


def select_variant(qtype, dtype: str, m: int, n: int, k: int) -> str:
    q = qtype_of(qtype)
    return _native.VARIANT_NAMES[_native.lib().dinoml_b200_gguf_gemm_rcr_select(q.value, _native.DINO_DTYPE[dtype], m, n, k)]


def variant_supports(variant: str, qtype, dtype: str, m: int, n: int, k: int) -> bool:
    """The library's own predicate: does this variant family serve the problem?"""
    q = qtype_of(qtype)
    family = _native.variant_code(variant) & 0xff
    return bool(_native.lib().dinoml_b200_gguf_variant_supports(family, q.value, _native.DINO_DTYPE[dtype], m, n, k))


def variant_configs(variant: str) -> int:
    """Number of tuning configurations of a variant family (valid: "family:1" .. "family:N")."""
    return int(_native.lib().dinoml_b200_gguf_variant_configs(_native.variant_code(variant) & 0xff))


class KVCache(NamedTuple):
    """A paged cache of keys and values in 8 bits: k, v [blocks, kv_heads, block_size, head_dim] (int8 or float8_e4m3fn), k_scale, v_scale [blocks, kv_heads]
    (float32).  A stored value stands for q * scale of its block and head.  Any sequence of four such tensors is a cache to the calls below."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


_KV_DTYPE = {"int8": torch.int8, "float8_e4m3fn": torch.float8_e4m3fn}
_KV_TYPE = {torch.int8: 1, torch.float8_e4m3fn: 2}
_KV_BLOCK_SIZES, _KV_HEAD_DIMS = (16, 32, 64, 128), (64, 128, 256)


def kv_cache(blocks: int, kv_heads: int, block_size: int, head_dim: int, dtype: str = "int8", device="cuda") -> KVCache:
    """An empty cache of `blocks` blocks of `block_size` tokens (16, 32, 64 or 128), head_dim 64, 128 or 256, values in int8 or float8_e4m3fn.  Small blocks
    have a scale of their own for fewer tokens, large ones are fewer copies and table entries."""
    if dtype not in _KV_DTYPE:
        raise ValueError(f"cache dtype must be one of {sorted(_KV_DTYPE)}, got {dtype!r}")
    if block_size not in _KV_BLOCK_SIZES or head_dim not in _KV_HEAD_DIMS or blocks < 1 or kv_heads < 1:
        raise ValueError(f"a cache has blocks of {_KV_BLOCK_SIZES} tokens and heads of {_KV_HEAD_DIMS} values, got {block_size} and {head_dim}")
    shape = (blocks, kv_heads, block_size, head_dim)
    k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(_KV_DTYPE[dtype]) for _ in range(2))
    return KVCache(k, v, *(torch.zeros(shape[:2], dtype=torch.float32, device=device) for _ in range(2)))


def _kv_struct(cache) -> _native.KvCache:
    k, v, k_scale, v_scale = cache
    for name, t in (("cache.k", k), ("cache.v", v), ("cache.k_scale", k_scale), ("cache.v_scale", v_scale)):
        _require_cuda(t, name)
        if t.device != k.device:
            raise ValueError("the tensors of a cache must be on one device")
    _require_current_device(k, "the cache")
    if k.dtype not in _KV_TYPE or k.dim() != 4 or v.dtype != k.dtype or v.shape != k.shape:
        raise ValueError("cache.k and cache.v must be int8 or float8_e4m3fn [blocks, kv_heads, block_size, head_dim] of one shape")
    if k.shape[2] not in _KV_BLOCK_SIZES or k.shape[3] not in _KV_HEAD_DIMS or k.shape[0] < 1 or k.shape[1] < 1:
        raise ValueError(f"a cache has blocks of {_KV_BLOCK_SIZES} tokens and heads of {_KV_HEAD_DIMS} values, got {tuple(k.shape)}")
    for t in (k_scale, v_scale):
        if t.dtype != torch.float32 or t.shape != k.shape[:2]:
            raise ValueError(f"cache scales must be float32 {tuple(k.shape[:2])}")
    return _native.KvCache(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), _KV_TYPE[k.dtype], *k.shape)


def _kv_ints(t: torch.Tensor, name: str, count: int, device) -> int:
    _require_cuda(t, name)
    if t.dtype != torch.int32 or t.shape != (count,) or t.device != device:
        raise ValueError(f"{name} must be int32 [{count}] on the device of the cache")
    return t.data_ptr()


def _kv_batch(cache, block_table: torch.Tensor, lengths, starts, rows: int) -> _native.KvBatch:
    device = cache[0].device
    if not block_table.is_cuda or block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.device != device or block_table.shape[1] < 1 \
            or block_table.stride(1) != 1 or (block_table.shape[0] > 1 and block_table.stride(0) < block_table.shape[1]):
        raise ValueError("block_table must be int32 [sequences, blocks] on the device of the cache, its rows contiguous")
    sequences = block_table.shape[0]
    if starts is None and rows != sequences:
        raise ValueError(f"without starts there is one row per sequence: {rows} rows, {sequences} sequences")
    return _native.KvBatch(block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
                           None if lengths is None else _kv_ints(lengths, "lengths", sequences, device),
                           None if starts is None else _kv_ints(starts, "starts", sequences + 1, device), sequences, rows)


def _kv_rows(t: torch.Tensor, name: str, device, heads, head_dim: int) -> None:
    if not t.is_cuda or t.device != device:
        raise ValueError(f"{name} must be a CUDA tensor on the device of the cache")
    if t.dim() != 3 or t.dtype not in _DTYPE_NAME or t.shape[2] != head_dim or (heads is not None and t.shape[1] != heads) or t.stride(2) != 1:
        raise ValueError(f"{name} must be [rows, {heads or 'heads'}, {head_dim}] in {sorted(_TORCH_DTYPE)}, its last dimension contiguous")


def _kv_zero(out, stream) -> None:
    """Rows without a sequence."""
    with torch.cuda.stream(stream):
        for t in out:
            t.zero_()


def kv_cache_write(cache, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor | None = None, *,
                   stream=None):
    """Quantizes new tokens into the cache, in place, and returns it.  k, v: [rows, kv_heads, head_dim], any row and head strides.  Rows are packed:
    sequence b has rows starts[b] .. starts[b + 1] - 1 (None: one row each) and `lengths[b]` tokens, these among them; position p of it is in slot
    p % block_size of block block_table[b, p // block_size].  A block's scale grows with its largest value; the tokens that are there already
    are brought to it.  Idle slots of a batch have length 0.  A non-finite value makes its block and head read as NaN."""
    done = _native_call("kv_write")(cache, k, v, block_table, lengths, starts, stream)
    if done is not None:                                                                  # None: not the plain case, checked below
        if type(done) is int:
            _native.check(done, "dinoml_b200_kv_cache_write")
        return done
    struct = _kv_struct(cache)
    device, heads, dim = cache[0].device, struct.kv_heads, struct.head_dim
    _kv_rows(k, "k", device, heads, dim)
    _kv_rows(v, "v", device, heads, dim)
    if v.dtype != k.dtype or v.shape != k.shape:
        raise ValueError("k and v must have one shape and dtype")
    batch = _kv_batch(cache, block_table, lengths, starts, k.shape[0])
    if k.shape[0] and batch.sequences:
        rc = _native.lib().dinoml_b200_kv_cache_write(
            ctypes.byref(struct), ctypes.byref(batch), k.data_ptr(), v.data_ptr(), _native.DINO_DTYPE[_DTYPE_NAME[k.dtype]], k.stride(0), k.stride(1),
            v.stride(0), v.stride(1), _stream_ptr(stream))
        _native.check(rc, "dinoml_b200_kv_cache_write")
    return cache


def kv_cache_read(cache, block_table: torch.Tensor, starts: torch.Tensor | None, rows: int, dtype: str = "bfloat16", *, begins: torch.Tensor | None = None,
                  out=None, stream=None):
    """Dense (k, v), each [rows, kv_heads, head_dim]: row starts[b] + j is position begins[b] + j of sequence b (begins None: from the first token; starts
    None: one row each).  Rows that no sequence has are zero.  `out`: two such tensors to fill."""
    done = _native_call("kv_read")(cache, block_table, starts, rows, dtype, begins, stream) if out is None else None
    if done is not None:                                                                  # None: not the plain case, checked below
        if type(done) is int:
            _native.check(done, "dinoml_b200_kv_cache_read")
        return done
    struct = _kv_struct(cache)
    device, shape = cache[0].device, (int(rows), struct.kv_heads, struct.head_dim)
    if dtype not in _TORCH_DTYPE:
        raise ValueError(f"dtype must be one of {sorted(_TORCH_DTYPE)}, got {dtype!r}")
    batch = _kv_batch(cache, block_table, None, starts, shape[0])
    begins_ptr = None if begins is None else _kv_ints(begins, "begins", batch.sequences, device)
    if out is None:
        out = tuple(torch.empty(shape, dtype=_TORCH_DTYPE[dtype], device=device) for _ in range(2))
    k, v = out
    for t in (k, v):
        _require_cuda(t, "out")
        if t.shape != shape or t.dtype != _TORCH_DTYPE[dtype] or t.device != device:
            raise ValueError(f"out must be two {dtype} tensors {shape} on the device of the cache")
    if shape[0] and batch.sequences:
        rc = _native.lib().dinoml_b200_kv_cache_read(ctypes.byref(struct), ctypes.byref(batch), begins_ptr, k.data_ptr(), v.data_ptr(),
                                                     _native.DINO_DTYPE[dtype], _stream_ptr(stream))
        _native.check(rc, "dinoml_b200_kv_cache_read")
    else:
        _kv_zero((k, v), stream)
    return k, v


def kv_cache_attention(q: torch.Tensor, cache, block_table: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor | None = None, *, scale: float | None = None,
                       window: int = 0, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """softmax(scale * q K^T) V over the cache, causal: a row at position p of its sequence sees positions max(0, p - window + 1) .. p (window 0: all up to p).
    q [rows, heads, head_dim], any row and head strides; heads is a multiple of kv_heads, head h reads cached head h // (heads // kv_heads); rows, lengths and
    starts as for `kv_cache_write`, whose tokens have to be in the cache.  scale None: head_dim ** -0.5.  A row that sees nothing is zero, and so is one that no sequence has."""
    done = _native_call("kv_attention")(q, cache, block_table, lengths, starts, scale, window, out, stream)
    if done is not None:                                                                  # None: not the plain case, checked below
        if type(done) is int:
            _native.check(done, "dinoml_b200_kv_cache_attention")
        return done
    struct = _kv_struct(cache)
    device = cache[0].device
    _kv_rows(q, "q", device, None, struct.head_dim)
    if q.shape[1] < 1 or q.shape[1] % struct.kv_heads:
        raise ValueError(f"q has {q.shape[1]} heads: a multiple of the cache's {struct.kv_heads} is wanted")
    if window < 0 or window > 0x7fffffff:
        raise ValueError("window must not be negative (0: none)")
    batch = _kv_batch(cache, block_table, lengths, starts, q.shape[0])
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=device)
    _require_cuda(out, "out")
    if out.shape != q.shape or out.dtype != q.dtype or out.device != device:
        raise ValueError("out must have the shape and dtype of q")
    if q.shape[0] and batch.sequences:
        rc = _native.lib().dinoml_b200_kv_cache_attention(
            ctypes.byref(struct), ctypes.byref(batch), q.data_ptr(), out.data_ptr(), _native.DINO_DTYPE[_DTYPE_NAME[q.dtype]], q.shape[1], q.stride(0),
            q.stride(1), struct.head_dim ** -0.5 if scale is None else float(scale), int(window), _stream_ptr(stream))
        _native.check(rc, "dinoml_b200_kv_cache_attention")
    else:
        _kv_zero((out,), stream)
    return out


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, *, residual: torch.Tensor | None = None, q8_0: bool = False,
             out: torch.Tensor | None = None, total: torch.Tensor | None = None, stream=None):
    """(y, total): total = x + residual, y = total / sqrt(mean(total^2) + eps) * weight over the last dimension, in float32 with one rounding at the end.
    weight [width] is float32 (as GGUF files hold it) or of x's dtype.  Without a residual total is None.  q8_0: y is uint8 [rows, width / 32 * 34], GGUF Q8_0
    blocks (`dequantize_rows` reads them).  `total` may be `residual` or x: the sum is then written in place."""
    done = _native_call("rms_norm")(x, weight, eps, residual, q8_0, stream) if out is None and total is None else None
    if done is not None:                                                                  # None: not the plain case, checked below
        if type(done) is int:
            _native.check(done, "dinoml_b200_rms_norm")
        return done
    _require_cuda(x, "x")
    _require_current_device(x, "x")
    _require_cuda(weight, "weight")
    if x.dtype not in _DTYPE_NAME or x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must be [..., width] in {sorted(_TORCH_DTYPE)}")
    width = x.shape[-1]
    rows = x.numel() // width
    if weight.shape != (width,) or weight.dtype not in (torch.float32, x.dtype) or weight.device != x.device:
        raise ValueError(f"weight must be [{width}] in float32 or the dtype of x, on its device")
    if residual is not None:
        _require_cuda(residual, "residual")
        if residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device:
            raise ValueError("residual must have the shape and dtype of x")
        if total is None:
            total = torch.empty_like(x)
    elif total is not None:
        raise ValueError("total is the sum with a residual: none is given")
    if total is not None:
        _require_cuda(total, "total")
        if total.shape != x.shape or total.dtype != x.dtype or total.device != x.device:
            raise ValueError("total must have the shape and dtype of x")
    if q8_0 and width % 32:
        raise ValueError(f"Q8_0 blocks hold 32 values: width {width} is no multiple")
    shape, dtype = ((rows, width // 32 * 34), torch.uint8) if q8_0 else (x.shape, x.dtype)
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=x.device)
    _require_cuda(out, "out")
    if out.shape != shape or out.dtype != dtype or out.device != x.device:
        raise ValueError(f"out must be {dtype} {tuple(shape)}")
    if rows:
        rc = _native.lib().dinoml_b200_rms_norm(
            x.data_ptr(), residual.data_ptr() if residual is not None else None, weight.data_ptr(), out.data_ptr(),
            total.data_ptr() if total is not None else None, _native.DINO_DTYPE[_DTYPE_NAME[x.dtype]], _native.DINO_DTYPE[_DTYPE_NAME[weight.dtype]], rows, width,
            float(eps), int(q8_0), _stream_ptr(stream))
        _native.check(rc, "dinoml_b200_rms_norm")
    return out, total


def release_stream(stream) -> None:
    """Gives back the workspaces that the library keeps for a stream (of the attention and of the linears), before the stream is destroyed.  Waits for the stream."""
    _native.check(_native.lib().dinoml_b200_release_stream(_stream_ptr(stream)), "dinoml_b200_release_stream")


def device_status() -> int:
    """Synchronizes and returns the status word written by bounded device-side waits (0 = none gave up; 16: one of the attention over the cache) and by the checks of
    what only the device sees (10: a block table, lengths, starts or begins pointed outside of the cache or of the rows).  Read once: it is 0 after that."""
    return int(_native.lib().dinoml_b200_gguf_device_status())
