"""The ``mode="mxfp4"`` side of :mod:`mlxturbo_amd.ops`.

MXFP4 (OCP Microscaling formats v1.0; the format of MLX's ``mode="mxfp4"``):
groups of 32 values along the last axis, 4-bit E2M1 codes packed eight to a
uint32 word (low bits first) and one E8M0 scale byte per group; no biases.  A
value is ``code * 2**(e - 127)``, ``e == 255`` is NaN.  The quantizer's choice of
a group's scale is the specification's; whether MLX's own takes the same byte for
every group is not pinned by any test here.

* quantize: ``e - 127 = floor(log2(max|w|)) - 2`` of the group, at least -127;
  codes are rounded to nearest, ties to even, and saturate at 6.  A group that
  holds a NaN or an infinity gets ``e = 255`` and zero codes.
* products: float sums over ``T(code * 2**(e - 127))`` with T the activations'
  type, what :func:`ops.dequantize` gives, rounded once to T.  In float16 a
  scale beyond 2**13 overflows as its dequantized values do.  qqmm multiplies
  codes and scales as they are, with no rounding to T before the sums.

The operators of :mod:`mlxturbo_amd.ops` call these for the mode; arguments and
errors are theirs.
"""

from __future__ import annotations

import math
import threading
from typing import Optional

import torch

from . import _lib, ops

GROUP_SIZE = 32
BITS = 4


def _scales(scales: torch.Tensor) -> torch.Tensor:
    """Scale bytes as uint8 (float8_e8m0fnu holds the same bytes)."""
    if scales.dtype == torch.uint8:
        return scales
    if scales.dtype == torch.float8_e8m0fnu:
        return scales.view(torch.uint8)
    raise ValueError(f"mxfp4 scales are uint8 exponents, got {scales.dtype}")


def _check(w: torch.Tensor, scales: torch.Tensor) -> int:
    """Shapes and types of a weight; returns its last dimension in values."""
    if w.dtype not in ops._CODE_DTYPES:
        raise ValueError(f"w must be uint32 packed codes, got {w.dtype}")
    if w.ndim < 1:
        raise ValueError("w must have at least one dimension")
    wshape = tuple(w.shape)
    K = wshape[-1] * 8
    want = (*wshape[:-1], K // GROUP_SIZE)
    if K % GROUP_SIZE or tuple(scales.shape) != want:
        raise ValueError(f"scales shape {tuple(scales.shape)} does not match w {wshape} "
                         f"in groups of {GROUP_SIZE} (expected {want})")
    return K


def _no_biases(biases) -> None:
    if biases is not None:
        raise NotImplementedError("mode='mxfp4': its codes have no biases")


def _elsewhere(dev: torch.device) -> bool:
    """Whether the tensors live on another device than the current one (launches
    and workspaces go by the current one)."""
    return dev.type == "cuda" and dev.index != torch._C._cuda_getDevice()


def _float_type(dtype: torch.dtype) -> None:
    if dtype not in ops._DTYPE_CODE:
        raise ValueError(f"mxfp4 operators take bfloat16, float16 or float32, got {dtype}")


def quantize(w: torch.Tensor):
    dev = ops._require_gpu(w)
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return quantize(w)
    if w.dtype not in ops._DTYPE_CODE:
        raise ValueError(f"w must be bfloat16, float16 or float32, got {w.dtype}")
    if w.ndim < 1:
        raise ValueError("w must have at least one dimension")
    K = w.shape[-1]
    if K == 0 or K % GROUP_SIZE:
        raise ValueError(f"the last dimension {K} must be a positive multiple of "
                         f"group_size={GROUP_SIZE}")
    lead = tuple(w.shape[:-1])
    N = math.prod(lead)
    wq = torch.empty((*lead, K // 8), dtype=torch.uint32, device=dev)
    s = torch.empty((*lead, K // GROUP_SIZE), dtype=torch.uint8, device=dev)
    if N == 0:
        return wq, s
    w_ = ops._aligned(w)
    rc = _lib.lib().mq_mxfp4_quantize(w_.data_ptr(), wq.data_ptr(), s.data_ptr(), N, K,
                                      ops._DTYPE_CODE[w.dtype], ops._stream_ptr(wq))
    _lib.check(rc, "quantize")
    return wq, s


def dequantize(w: torch.Tensor, scales: torch.Tensor, biases=None,
               dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    _no_biases(biases)
    dev = ops._require_gpu(w, scales)
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return dequantize(w, scales, dtype=dtype)
    scales = _scales(scales)
    K = _check(w, scales)
    dtype = torch.bfloat16 if dtype is None else dtype
    _float_type(dtype)
    out = torch.empty((*w.shape[:-1], K), dtype=dtype, device=dev)
    if out.numel() == 0:
        return out
    w_, s_ = ops._aligned(w), ops._aligned(scales)
    rc = _lib.lib().mq_mxfp4_dequantize(w_.data_ptr(), s_.data_ptr(), out.data_ptr(),
                                        out.numel() // K, K, ops._DTYPE_CODE[dtype],
                                        ops._stream_ptr(out))
    _lib.check(rc, "dequantize")
    return out


def _composed(x, w, scales, transpose: bool) -> torch.Tensor:
    """dequantize in x's type and one GPU GEMM, for what has no kernel."""
    deq = dequantize(w, scales, dtype=x.dtype)
    return torch.nn.functional.linear(x, deq) if transpose else torch.matmul(x, deq)


# A call's launches follow each other on the stream, as they share its workspace of
# these operators with the calls of other threads there.
_LAUNCH = threading.Lock()
_SCRATCH: dict = {}


def _scratch(dev: torch.device, stream: int, nbytes: int) -> torch.Tensor:
    """A workspace: the stream's, or in a capture one of the graph's own memory
    (graphs captured on one stream may be replayed on two at once)."""
    if torch.cuda.is_current_stream_capturing():
        return torch.empty(nbytes, dtype=torch.uint8, device=dev)
    buf = _SCRATCH.get((dev.index, stream))
    if buf is None or buf.numel() < nbytes:
        buf = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=dev)
        _SCRATCH[dev.index, stream] = buf
    return buf


def _launch(call, args, out, nbytes: int) -> int:
    """One call with a workspace of nbytes where it needs one; its status."""
    stream = ops._stream_ptr(out)
    if not nbytes:
        return call(*args, None, 0, stream)
    with _LAUNCH:
        ws = _scratch(out.device, stream, nbytes)
        return call(*args, ws.data_ptr(), ws.numel(), stream)


def _product(call, size, x, w, s, out, M: int, N: int, K: int) -> int:
    """One product call; its status."""
    return _launch(call, (x.data_ptr(), w.data_ptr(), s.data_ptr(), out.data_ptr(), M, N, K,
                          ops._DTYPE_CODE[out.dtype]), out,
                   size(M, N, K) if M > 16 else 0)   # up to 16 rows use none


def quantized_matmul(x, w, scales, biases, transpose: bool) -> torch.Tensor:
    _no_biases(biases)
    dev = ops._require_gpu(x, w, scales)
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return quantized_matmul(x, w, scales, None, transpose)
    if w.ndim != 2:
        raise NotImplementedError("batched w: only 2-D weights are on this path")
    scales = _scales(scales)
    Kq = _check(w, scales)
    _float_type(x.dtype)
    if x.ndim < 1:
        raise ValueError("x must have at least one dimension")
    K, N = (Kq, w.shape[0]) if transpose else (w.shape[0], Kq)
    if x.shape[-1] != K:
        raise ValueError(
            f"x last dimension {x.shape[-1]} does not match the quantized weight K={K}")
    if not transpose or x.dtype == torch.float32:
        return _composed(x, w, scales, transpose)
    lead = tuple(x.shape[:-1])
    M = math.prod(lead)
    out = torch.empty((*lead, N), dtype=x.dtype, device=dev)
    if M == 0 or N == 0:
        return out
    if K == 0:
        return out.zero_()
    x_, w_, s_ = ops._aligned(x), ops._aligned(w), ops._aligned(scales)
    lib = _lib.lib()
    rc = _product(lib.mq_mxfp4_matmul, lib.mq_mxfp4_matmul_workspace_size, x_, w_, s_, out, M, N, K)
    if rc == ops._EUNSUPPORTED:
        return _composed(x, w, scales, True)
    _lib.check(rc, "quantized_matmul")
    return out


def qqmm(x, w, scales) -> torch.Tensor:
    dev = ops._require_gpu(x, w, scales)
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return qqmm(x, w, scales)
    if w.ndim != 2:
        raise NotImplementedError("batched w: only 2-D weights are on this path")
    scales = _scales(scales)
    K = _check(w, scales)
    _float_type(x.dtype)
    if x.ndim < 1 or x.shape[-1] != K:
        raise ValueError(f"x {tuple(x.shape)} does not match the quantized weight K={K}")
    N = w.shape[0]
    lead = tuple(x.shape[:-1])
    M = math.prod(lead)
    out = torch.empty((*lead, N), dtype=x.dtype, device=dev)
    if M == 0 or N == 0:
        return out
    if K == 0:
        return out.zero_()
    rc = ops._EUNSUPPORTED
    if x.dtype != torch.float32:
        x_, w_, s_ = ops._aligned(x), ops._aligned(w), ops._aligned(scales)
        lib = _lib.lib()
        rc = _product(lib.mq_mxfp4_qqmm, lib.mq_mxfp4_qqmm_workspace_size, x_, w_, s_, out, M, N,
                      K)
    if rc == ops._EUNSUPPORTED:
        # in float, which holds what both sides' codes and scales stand for
        return _composed(dequantize(*quantize(x), dtype=torch.float32), w, scales,
                         True).to(x.dtype)
    _lib.check(rc, "qqmm")
    return out


def _gather_launch(x, flat, lhs, rhs, out, P, B, M, N, K, E, group_size, bits,
                   sorted_indices) -> None:
    """One mq_mxfp4_gather_qmm call on flattened, validated arguments (the
    signature of ops' launch of affine banks)."""
    x_ = ops._aligned(x)
    w_, s_ = (ops._aligned(t) for t in flat)
    lib = _lib.lib()
    args = (x_.data_ptr(), w_.data_ptr(), s_.data_ptr(), ops._ptr(lhs), rhs.data_ptr(),
            out.data_ptr(), P, B, M, N, K, E, ops._DTYPE_CODE[x.dtype])
    rc = _launch(lib.mq_mxfp4_gather_qmm, args, out,
                 lib.mq_mxfp4_gather_qmm_workspace_size(P, M))
    _lib.check(rc, "gather_qmm")


def gather_qmm(x, w, scales, biases, lhs_indices, rhs_indices, transpose: bool,
               sorted_indices: bool) -> torch.Tensor:
    _no_biases(biases)
    dev = ops._require_gpu(x, w, scales)
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return gather_qmm(x, w, scales, None, lhs_indices, rhs_indices, transpose,
                              sorted_indices)
    if x.ndim < 2 or w.ndim < 3:
        raise ValueError("gather_qmm needs x (..., M, K) and w (..., N, K*bits/32) with a batch dim")
    scales = _scales(scales)
    Kq = _check(w, scales)
    _float_type(x.dtype)
    K, N = (Kq, w.shape[-2]) if transpose else (w.shape[-2], Kq)
    if x.shape[-1] != K:
        raise ValueError(
            f"x last dimension {x.shape[-1]} does not match the quantized weight K={K}")
    M, bx, bw = x.shape[-2], tuple(x.shape[:-2]), tuple(w.shape[:-2])
    E, B = math.prod(bw), math.prod(bx)
    shape, P, lhs, rhs = ops._gather_pairs(dev, bx, bw, lhs_indices, rhs_indices)
    out = torch.empty((*shape, M, N), dtype=x.dtype, device=dev)
    if P == 0 or M == 0 or N == 0:
        return out
    if K == 0 or B == 0 or E == 0:
        return out.zero_()
    if w.ndim != 3:
        w, scales = w.reshape(E, *w.shape[-2:]), scales.reshape(E, *scales.shape[-2:])
    bank = [w, scales]
    kernels = transpose and x.dtype != torch.float32
    if kernels and M <= 16 and (
            E <= ops._GATHER_PREP_MAX_E
            or not _lib.lib().mq_mxfp4_gather_qmm_workspace_size(P, M)):
        try:
            _gather_launch(x, bank, lhs, rhs, out, P, B, M, N, K, E, GROUP_SIZE, BITS,
                           sorted_indices)
            return out
        except NotImplementedError:                  # beyond the kernels' address ranges
            kernels = False
    a = dict(x=x.reshape(B, M, K), flat=bank, lhs=lhs, rhs=rhs, P=P, B=B, M=M, N=N, K=K, E=E,
             dev=dev, transpose=transpose, shape=shape, dtype=x.dtype, launch=_gather_launch)
    if kernels:
        form = ops._gather_rows if M > 16 else ops._gather_slices
        try:
            return form(a, out, GROUP_SIZE, BITS, sorted_indices)
        except NotImplementedError:                  # the same
            pass
    return ops._gather_composed(a, out, lambda e: dequantize(w[e], scales[e], dtype=x.dtype))
