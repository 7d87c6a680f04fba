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


class KVPool(NamedTuple):
    """Who has which blocks of a `KVCache`: block_table [sequences, table_blocks] (-1 behind a sequence's blocks), lengths [sequences] its tokens, free [blocks] a stack of
    which the first free_count [1] are free, all int32 on the device.  `kv_pool_step` changes them in place; block_table is what the cache's calls take."""
    block_table: torch.Tensor
    lengths: torch.Tensor
    free: torch.Tensor
    free_count: torch.Tensor
    block_size: int


class KVStep(NamedTuple):
    """One step's batch: lengths and starts as the cache's calls take them, positions and slots (block * block_size + place in it) of its rows, -1 of nobody's."""
    lengths: torch.Tensor
    starts: torch.Tensor | None
    positions: torch.Tensor
    slots: torch.Tensor


_POOL_SEQUENCES = 8192


def kv_pool(blocks: int, sequences: int, table_blocks: int, block_size: int, device="cuda") -> KVPool:
    """A pool of a cache's `blocks` blocks, all free, for `sequences` sequences (8192 at most) of up to table_blocks blocks.  Blocks are handed out from 0 on."""
    if block_size not in _KV_BLOCK_SIZES or blocks < 1 or table_blocks < 1 or not 1 <= sequences <= _POOL_SEQUENCES:
        raise ValueError(f"a pool has blocks of {_KV_BLOCK_SIZES} tokens and 1 to {_POOL_SEQUENCES} sequences, got {block_size} and {sequences}")
    if max(blocks, table_blocks) * block_size > 0x7fffffff:
        raise ValueError("a pool has less than 2^31 tokens")
    return KVPool(torch.full((sequences, table_blocks), -1, dtype=torch.int32, device=device), torch.zeros(sequences, dtype=torch.int32, device=device),
                  torch.arange(blocks - 1, -1, -1, dtype=torch.int32, device=device), torch.full((1,), blocks, dtype=torch.int32, device=device), int(block_size))


def kv_pool_step(pool, new: torch.Tensor, rows: int | None = None, *, drop: torch.Tensor | None = None, stream=None) -> KVStep:
    """One step of all sequences, in place: sequence b loses drop[b] tokens at its end (None: none; a request that is done: as many as it has, or more) and gets new[b].  Blocks
    go back before any is handed out; sequences that get as many as they lost get the same ones.  rows: of the packed batch, at least sum(new); those behind the last
    sequence are nobody's.  rows None: one row per sequence, new[b] 0 or 1, and starts None.  A sequence whose new tokens do not fit goes without them (its lengths entry is 0,
    it has no rows): the table's row is too short, or it wants blocks and those that the sequences up to it want are more than there are, or their rows more than `rows`.  The rows of those
    behind it come that much earlier: what a row is given (its token, say) goes by step.starts and positions, not by the running sum of `new`."""
    done = _native_call("kv_pool_step")(pool, new, rows, drop, stream)
    if done is not None:                                                                  # None: not the plain case, checked below
        if type(done) is int:
            _native.check(done, "dinoml_b200_kv_pool_step")
        return KVStep(*done)
    table, lengths, free, free_count, block_size = pool
    _require_cuda(lengths, "pool.lengths")
    _require_current_device(lengths, "the pool")
    device = lengths.device
    if not table.is_cuda or table.dtype != torch.int32 or table.dim() != 2 or table.device != device or min(table.shape) < 1 or table.stride(1) != 1 \
            or (table.shape[0] > 1 and table.stride(0) < table.shape[1]):
        raise ValueError("pool.block_table must be int32 [sequences, blocks] on the device of the pool, its rows contiguous")
    sequences = table.shape[0]
    if sequences > _POOL_SEQUENCES or block_size not in _KV_BLOCK_SIZES:
        raise ValueError(f"a pool has blocks of {_KV_BLOCK_SIZES} tokens and 1 to {_POOL_SEQUENCES} sequences, got {block_size} and {sequences}")
    if free.dim() != 1 or free.shape[0] < 1:
        raise ValueError("pool.free must be int32 [blocks]")
    if max(free.shape[0], table.shape[1]) * block_size > 0x7fffffff:
        raise ValueError("a pool has less than 2^31 tokens")
    _kv_ints(lengths, "pool.lengths", sequences, device)
    _kv_ints(free, "pool.free", free.shape[0], device)
    _kv_ints(free_count, "pool.free_count", 1, device)
    _kv_ints(new, "new", sequences, device)
    drop_ptr = None if drop is None else _kv_ints(drop, "drop", sequences, device)
    count = sequences if rows is None else int(rows)
    if not 0 <= count <= 0x7fffffff:
        raise ValueError(f"rows must be 0 to 2^31 - 1, got {rows}")
    step = KVStep(torch.empty(sequences, dtype=torch.int32, device=device), None if rows is None else torch.empty(sequences + 1, dtype=torch.int32, device=device),
                  *(torch.empty(count, dtype=torch.int32, device=device) for _ in range(2)))
    spare = step.lengths.data_ptr()                                                       # no rows: nothing is written there, but addresses are wanted
    struct = _native.KvPool(table.data_ptr(), table.stride(0), lengths.data_ptr(), free.data_ptr(), free_count.data_ptr(), table.shape[1], sequences, free.shape[0], block_size)
    rc = _native.lib().dinoml_b200_kv_pool_step(
        ctypes.byref(struct), new.data_ptr(), drop_ptr, count, step.lengths.data_ptr(), None if rows is None else step.starts.data_ptr(), step.positions.data_ptr() or spare,
        step.slots.data_ptr() or spare, _stream_ptr(stream))
    _native.check(rc, "dinoml_b200_kv_pool_step")
    return step


def rotary_frequencies(dim: int, base: float = 10000.0, *, scale: float = 1.0, factors=None, device="cuda") -> torch.Tensor:
    """Angles per position of the dim / 2 pairs of a rotated head, float64: scale * base ** (-2 i / dim), divided by factors[i] where there are some (a GGUF file's
    rope_freqs.weight)."""
    if dim < 2 or dim % 2:
        raise ValueError(f"pairs are of two values: dim {dim}")
    out = scale * float(base) ** (-2.0 * torch.arange(dim // 2, dtype=torch.float64) / dim)
    if factors is not None:
        factors = torch.as_tensor(factors).cpu().to(torch.float64)
        if factors.shape != out.shape:
            raise ValueError(f"factors must be [{dim // 2}]")
        out = out / factors
    return out.to(device)


def _apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two [rows, heads, head_dim] tensors of one dtype share no memory, as far as their addresses and strides tell: one behind the other, or other columns of rows that are equally far
    apart.  (Their storages may be two over one memory.)"""
    if not a.numel() or not b.numel():
        return True
    size = a.element_size()

    def inside(t):                                                                        # bytes from a row's first value to behind its last
        return ((t.shape[1] - 1) * t.stride(1) + t.shape[2]) * size

    def behind(t):
        return t.data_ptr() + (t.shape[0] - 1) * t.stride(0) * size + inside(t)

    if behind(a) <= b.data_ptr() or behind(b) <= a.data_ptr():
        return True
    pitch = a.stride(0) * size
    if a.shape[0] < 2 or b.stride(0) != a.stride(0) or max(inside(a), inside(b)) > pitch:
        return False
    gap = (b.data_ptr() - a.data_ptr()) % pitch
    return gap >= inside(a) and pitch - gap >= inside(b)


def _rotary_side(x: torch.Tensor, weight, out, name: str, like: torch.Tensor) -> _native.Heads:
    if not x.is_cuda or x.device != like.device or x.dim() != 3 or x.dtype != like.dtype or x.shape[0] != like.shape[0] or x.shape[2] != like.shape[2] or x.shape[1] < 1 \
            or x.stride(2) != 1:
        raise ValueError(f"{name} must be [rows, heads, head_dim], its last dimension contiguous, q and k of one dtype, device, number of rows and head_dim")
    if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device or out.stride(2) != 1:
        raise ValueError(f"out of {name} must have its shape and dtype, its last dimension contiguous")
    rows, heads, dim = x.shape
    if not (out.stride(1) >= dim or heads == 1) or not (out.stride(0) >= dim or rows == 1) or not (
            rows == 1 or heads == 1 or out.stride(0) >= (heads - 1) * out.stride(1) + dim or out.stride(1) >= (rows - 1) * out.stride(0) + dim):
        raise ValueError(f"out of {name} must not overlap itself")
    if (out.data_ptr(), out.stride()) != (x.data_ptr(), x.stride()) and not _apart(out, x):
        raise ValueError(f"out of {name} must be {name} itself or not overlap it")
    if weight is not None:
        _require_cuda(weight, f"{name}_weight")
        if weight.shape != (dim,) or weight.dtype not in (torch.float32, x.dtype) or weight.device != x.device:
            raise ValueError(f"{name}_weight must be [{dim}] in float32 or the dtype of {name}, on its device")
    return _native.Heads(x.data_ptr(), out.data_ptr(), None if weight is None else weight.data_ptr(), x.stride(0), x.stride(1), out.stride(0), out.stride(1), heads)


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, frequencies: torch.Tensor, *, q_weight: torch.Tensor | None = None,
           k_weight: torch.Tensor | None = None, eps: float = 1e-5, interleaved: bool = False, magnitude: float = 1.0, out=None, stream=None):
    """(q, k) turned by position: pairs (a, b) of every head become magnitude * (a cos - b sin, b cos + a sin), angle positions[row] * frequencies[i] in float64.  Pair i is
    (i, i + n) with n = len(frequencies), interleaved (2 i, 2 i + 1); values behind 2 n stay.  q_weight, k_weight [head_dim] (float32 or q's dtype): each head is first brought to
    x / sqrt(mean(x^2) + eps) * weight.  float32 inside, one rounding at the end.  q [rows, heads, head_dim], k [rows, kv_heads, head_dim] (None: q alone), any row and head strides; head_dim
    even, 512 at most; positions int32 [rows]; frequencies float64 (`rotary_frequencies`).  out: two tensors to fill (None: a new one), q and k themselves among them.  A row at a negative position is
    nobody's: zero, or left as it was where it is written in place."""
    done = _native_call("rotary")(q, k, positions, frequencies, q_weight, k_weight, eps, interleaved, magnitude, stream) if out is None else None
    if done is not None:                                                                  # None: not the plain case, checked below
        if type(done) is int:
            _native.check(done, "dinoml_b200_rotary")
        return done
    if q.dim() != 3 or q.dtype not in _DTYPE_NAME or not q.is_cuda:
        raise ValueError(f"q must be a CUDA tensor [rows, heads, head_dim] in {sorted(_TORCH_DTYPE)}")
    _require_current_device(q, "q")
    rows, _, dim = q.shape
    if dim < 2 or dim % 2 or dim > 512:
        raise ValueError(f"head_dim must be even and 512 at most, got {dim}")
    _kv_ints(positions, "positions", rows, q.device)
    _require_cuda(frequencies, "frequencies")
    if frequencies.dtype != torch.float64 or frequencies.dim() != 1 or 2 * frequencies.shape[0] > dim or frequencies.device != q.device:
        raise ValueError(f"frequencies must be float64 [{dim // 2} at most] on the device of q")
    if k is None and k_weight is not None:
        raise ValueError("k_weight is k's: none is given")
    given = (None, None) if out is None else tuple(out) if k is not None or isinstance(out, (tuple, list)) else (out, None)
    if len(given) != 2 or (k is None and given[1] is not None):
        raise ValueError("out must be two tensors, for q and for k")
    q_out, k_out = (torch.empty(x.shape, dtype=x.dtype, device=x.device) if o is None and x is not None else o for x, o in zip((q, k), given))
    side_q = _rotary_side(q, q_weight, q_out, "q", q)
    side_k = None if k is None else _rotary_side(k, k_weight, k_out, "k", q)
    if k is not None and not (_apart(q_out, k) and _apart(k_out, q) and _apart(q_out, k_out)):
        raise ValueError("what is written for one of q and k must not overlap the other")
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise ValueError("q_weight and k_weight must have one dtype")
    if rows:
        weight = q_weight if q_weight is not None else k_weight
        rc = _native.lib().dinoml_b200_rotary(
            ctypes.byref(side_q), None if side_k is None else ctypes.byref(side_k), positions.data_ptr(), frequencies.data_ptr() or None, frequencies.shape[0],
            _native.DINO_DTYPE[_DTYPE_NAME[q.dtype]], _native.DINO_DTYPE["float32" if weight is None else _DTYPE_NAME[weight.dtype]], rows, dim, float(eps), float(magnitude),
            int(bool(interleaved)), _stream_ptr(stream))
        _native.check(rc, "dinoml_b200_rotary")
    return q_out, k_out


def embedding(tokens: torch.Tensor, table: torch.Tensor, qtype, dtype: str = "bfloat16", *, scale: float = 1.0, out: torch.Tensor | None = None,
              stream=None) -> torch.Tensor:
    """Rows of a GGUF table (uint8 [vocabulary, row_bytes]) for tokens (int32 or int64, any shape): tokens.shape + [width] in `dtype`, each value the dequantized float32 times
    scale, rounded once.  Token -1 is nobody's, its row zero; so is that of any other token outside of the table, which `device_status()` tells."""
    done = _native_call("embedding")(tokens, table, qtype, dtype, scale, stream) if out is None else None
    if done is not None:                                                                  # None: not the plain case, checked below
        if type(done) is int:
            _native.check(done, "dinoml_b200_embedding")
        return done
    q = qtype_of(qtype)
    _require_cuda(tokens, "tokens")
    _require_cuda(table, "table")
    _require_current_device(table, "the table")
    if tokens.dtype not in (torch.int32, torch.int64) or tokens.device != table.device:
        raise ValueError("tokens must be int32 or int64 on the device of the table")
    if table.dtype != torch.uint8 or table.dim() != 2 or table.shape[0] < 1 or table.shape[1] < 1 or table.shape[1] % q.block_bytes:
        raise ValueError(f"table must be uint8 [vocabulary, row_bytes] with whole {q.name} blocks of {q.block_bytes} bytes")
    if dtype not in _TORCH_DTYPE:
        raise ValueError(f"dtype must be one of {sorted(_TORCH_DTYPE)}, got {dtype!r}")
    width = table.shape[1] // q.block_bytes * q.block_size
    shape = tuple(tokens.shape) + (width,)
    if out is None:
        out = torch.empty(shape, dtype=_TORCH_DTYPE[dtype], device=table.device)
    _require_cuda(out, "out")
    if tuple(out.shape) != shape or out.dtype != _TORCH_DTYPE[dtype] or out.device != table.device:
        raise ValueError(f"out must be {dtype} {shape} on the device of the table")
    if tokens.numel():
        rc = _native.lib().dinoml_b200_embedding(tokens.data_ptr(), tokens.element_size(), table.data_ptr(), table.shape[0], out.data_ptr(), q.value,
                                                 _native.DINO_DTYPE[dtype], tokens.numel(), width, float(scale), _stream_ptr(stream))
        _native.check(rc, "dinoml_b200_embedding")
    return out


_SAMPLE_VOCABULARY = 262144


def sample(logits: torch.Tensor, uniforms: torch.Tensor, *, temperature=1.0, top_k=None, top_p=None, min_p=None, stream=None):
    """(tokens int32 [rows], probabilities float32 [rows]): of every row of logits [rows, vocabulary] (262144 at most, any row stride) one token, chosen with its number of
    uniforms float32 [rows] in [0, 1).  Tokens are ordered by logit, the lowest index first among equals, their weights are exp((logit - largest) / temperature); kept are the first
    top_k (None or 0: all), of these the fewest whose weights are at least top_p of theirs (None or 1: all), of these those with at least min_p of the largest weight (None: all);
    the token is the first whose running sum is above uniforms[row] times the sum of the kept, its probability its share of that sum.  Temperature 0 takes the first.  Each setting is a number
    or a tensor [rows] (top_k int32, the others float32).  Logits of -inf are never chosen; a row with a NaN, without any other logit, or with a setting that is
    none gives -1 and 0 (`device_status()` tells of the last)."""
    done = _native_call("sample")(logits, uniforms, temperature, top_k, top_p, min_p, stream)
    if done is not None:                                                                  # None: not the plain case, checked below
        if type(done) is int:
            _native.check(done, "dinoml_b200_sample")
        return done
    if not logits.is_cuda or logits.dim() != 2 or logits.dtype not in _DTYPE_NAME or logits.shape[1] < 1 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError(f"logits must be a CUDA tensor [rows, vocabulary] in {sorted(_TORCH_DTYPE)}, its rows contiguous")
    _require_current_device(logits, "logits")
    rows, vocabulary = logits.shape
    if vocabulary > _SAMPLE_VOCABULARY or (rows > 1 and logits.stride(0) < vocabulary):
        raise ValueError(f"logits must have {_SAMPLE_VOCABULARY} columns at most, and rows that do not overlap")

    def per_row(t, name, dtype):
        _require_cuda(t, name)
        if t.dtype != dtype or t.shape != (rows,) or t.device != logits.device:
            raise ValueError(f"{name} must be {dtype} [{rows}] on the device of logits")
        return t.data_ptr()

    uniforms_ptr = per_row(uniforms, "uniforms", torch.float32)
    settings = _native.SampleSettings(None, None, None, None, 1.0, 0, 1.0, 0.0)
    for name, value, dtype in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32), ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32)):
        if value is None:
            if name == "temperature":
                raise ValueError("temperature must be a number or a tensor")
        elif isinstance(value, torch.Tensor):
            setattr(settings, name, per_row(value, name, dtype))
        elif name == "top_k":
            if value != int(value):
                raise ValueError(f"top_k must be a whole number, got {value}")
            settings.top_k_all = min(max(int(value), 0), 0x7fffffff)
        else:
            if not value >= 0:
                raise ValueError(f"{name} must not be negative, got {value}")
            setattr(settings, name + "_all", float(value))
    tokens, probabilities = (torch.empty(rows, dtype=t, device=logits.device) for t in (torch.int32, torch.float32))
    if rows:
        rc = _native.lib().dinoml_b200_sample(logits.data_ptr(), logits.stride(0), _native.DINO_DTYPE[_DTYPE_NAME[logits.dtype]], rows, vocabulary, uniforms_ptr,
                                              ctypes.byref(settings), tokens.data_ptr(), probabilities.data_ptr(), _stream_ptr(stream))
        _native.check(rc, "dinoml_b200_sample")
    return tokens, probabilities


def release_stream(stream) -> None:
    """Gives back the workspaces that the library keeps for a stream (of the attention and of the linears), before the stream is destroyed.  Waits for the stream."""
    _native.check(_native.lib().dinoml_b200_release_stream(_stream_ptr(stream)), "dinoml_b200_release_stream")


def device_status() -> int:
    """Synchronizes and returns the status word written by bounded device-side waits (0 = none gave up; 16: one of the attention over the cache) and by the checks of
    what only the device sees (10: a block table, lengths, starts or begins pointed outside of the cache or of the rows, a token outside of its table, a pool's numbers that cannot be, a row's
    sampling settings that are none).  Read once: it is 0 after that."""
    return int(_native.lib().dinoml_b200_gguf_device_status())
