"""The dense gated feed-forward block's first half, and gradients past frozen weights.

* :func:`quantized_glu` - ``act(x Wg^T) * (x Wu^T)`` over affine matrices, in one
  launch where the sums need no splitting: the dense form of
  :func:`ops.gather_glu` (a dense model's MLP, mlx-lm's ``down(silu(gate(x)) *
  up(x))``, which the reference leaves to three MLX calls).
* :func:`ops.quantized_matmul`'s gradient of x.

The weights are constants: gradients go to x alone, as adapters below a quantized
layer are trained.  Sums are float; in the gradient of the block, the gate and up
products are kept in float between forward and backward (8 bytes per output), and the
products' inputs ``d u act'(g)`` and ``d act(g)`` are two 16-bit numbers each (the value
rounded, and the rest), in float16 scaled by rows, so that x's gradient is rounded once and in
range as that of float32 products is.
"""

from __future__ import annotations

import math
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _lib, ops

ACTIVATIONS = {"silu": _lib.MQ_ACT_SILU, "gelu_tanh": _lib.MQ_ACT_GELU_TANH}


def elsewhere(dev: torch.device) -> bool:
    """Whether the tensors live on another device than the current one (launches
    and workspaces go by the current one)."""
    return dev.type == "cuda" and dev.index != torch._C._cuda_getDevice()


def wants_grad(x: torch.Tensor) -> bool:
    return x.requires_grad and torch.is_grad_enabled()


def differentiated(x: torch.Tensor) -> bool:
    """Whether a call on x is part of a graph, or x has a forward-mode tangent."""
    return (x.requires_grad and torch.is_grad_enabled()
            or forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None)


def _workspace(nbytes: int, dev: torch.device) -> Optional[torch.Tensor]:
    """A call's own workspace: in a capture the graph's memory, and no two calls
    share one."""
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


def _room(ws: Optional[torch.Tensor]):
    return (ws.data_ptr(), ws.numel()) if ws is not None else (None, 0)


def note_leaf(x: torch.Tensor):
    """Refuses a capture that would end in an accumulator of another stream: a leaf's
    is made by the first graph of it that lives and keeps that graph's stream, and a
    captured backward that reaches it from another stream ends the process.  Returns the
    accumulator, which the caller holds until the graph does (else it and the note are gone)."""
    if not (x.is_leaf and x.requires_grad):
        return None
    node = torch.autograd.graph.get_gradient_edge(x).node
    meta = node.metadata
    stream = ops._stream_of(x.device)
    if torch.cuda.is_current_stream_capturing():
        if meta.get("mq_stream", stream) != stream:
            raise RuntimeError(
                "x is a leaf of a graph made on another stream that still lives, and its gradient "
                "cannot be captured: drop that graph, or pass x.detach().requires_grad_()")
    meta.setdefault("mq_stream", stream)
    return node


def _glu_forward(x, flat, act: int, group_size: int, bits: int, save: bool):
    """``(h, gate sums, up sums)`` of checked arguments, or None where no kernel takes
    them; x ``(M, K)``, ``flat`` the two matrices' six tensors."""
    dev, (M, K), N = x.device, x.shape, flat[0].shape[0]
    out = torch.empty((M, N), dtype=x.dtype, device=dev)
    g = torch.empty((M, N), dtype=torch.float32, device=dev) if save else None
    u = torch.empty_like(g) if save else None
    if M == 0 or N == 0:
        return out, g, u
    lib = _lib.lib()
    ws = None
    if M > 16:
        ws = _workspace(int(lib.mq_quantized_glu_workspace_size(M, N, K, group_size, bits)), dev)
    rc = lib.mq_quantized_glu(x.data_ptr(), *[t.data_ptr() for t in flat], out.data_ptr(),
                              ops._ptr(g), ops._ptr(u), M, N, K, group_size, bits,
                              ops._DTYPE_CODE[x.dtype], act, *_room(ws), ops._stream_ptr(out))
    if rc == ops._EUNSUPPORTED:
        return None
    _lib.check(rc, "quantized_glu")
    return out, g, u


def matmul_grad(d, w, scales, biases, group_size: int, bits: int) -> torch.Tensor:
    """``d @ dequantize(w)`` for d ``(M, N)`` in the scales' 16-bit type."""
    (M, N), K = d.shape, w.shape[1] * 32 // bits
    dx = torch.empty((M, K), dtype=d.dtype, device=d.device)
    if M == 0 or K == 0:
        return dx
    if N == 0:
        return dx.zero_()
    d = ops._aligned(d)
    lib = _lib.lib()
    ws = _workspace(int(lib.mq_quantized_matmul_grad_workspace_size(M, N, K, group_size, bits)),
                    d.device)
    rc = lib.mq_quantized_matmul_grad(d.data_ptr(), w.data_ptr(), scales.data_ptr(),
                                      biases.data_ptr(), dx.data_ptr(), M, N, K, group_size, bits,
                                      ops._DTYPE_CODE[d.dtype], *_room(ws), ops._stream_ptr(dx))
    if rc == ops._EUNSUPPORTED:                       # beyond the kernel's address ranges
        return ops._composed_qmm(d, w, scales, biases, False, group_size, bits)
    _lib.check(rc, "quantized_matmul_grad")
    return dx


def _glu_grad(d, g, u, flat, act: int, group_size: int, bits: int) -> torch.Tensor:
    (M, N), K = d.shape, flat[0].shape[1] * 32 // bits
    dx = torch.empty((M, K), dtype=d.dtype, device=d.device)
    if M == 0 or K == 0:
        return dx
    if N == 0:
        return dx.zero_()
    d = ops._aligned(d)
    lib = _lib.lib()
    ws = _workspace(int(lib.mq_quantized_glu_grad_workspace_size(M, N, K, group_size, bits)),
                    d.device)
    rc = lib.mq_quantized_glu_grad(d.data_ptr(), g.data_ptr(), u.data_ptr(),
                                   *[t.data_ptr() for t in flat], dx.data_ptr(), M, N, K,
                                   group_size, bits, ops._DTYPE_CODE[d.dtype], act, *_room(ws),
                                   ops._stream_ptr(dx))
    if rc == ops._EUNSUPPORTED:                       # beyond the kernel's address ranges
        with torch.enable_grad():
            gg, uu = g.detach().requires_grad_(), u.detach().requires_grad_()
            dg, du = torch.autograd.grad(_activation(gg, _name(act)) * uu, (gg, uu), d.float())
        for i, t in enumerate((dg, du)):              # float products, as the kernels' sums are
            w = ops.dequantize(*flat[3 * i:3 * i + 3], group_size, bits).float()
            out = torch.addmm(out, t, w) if i else torch.mm(t, w)
        return out.to(d.dtype)
    _lib.check(rc, "quantized_glu_grad")
    return dx


def _versions(ts) -> list:
    return [None if t.is_inference() else t._version for t in ts]


def _constants(ctx, ts) -> None:
    """Keeps the weights for the backward pass.  They are constants, so they go past the
    engine's saved tensors, whose packing and unpacking cost several us a step; like those
    they may not have changed by then."""
    ctx.flat, ctx.versions = ts, _versions(ts)


def _same_constants(ctx):
    if ctx.versions != _versions(ctx.flat):
        raise RuntimeError("a quantized weight needed for the gradient has been modified by an "
                           "inplace operation since the forward pass")
    return ctx.flat


def _first_order(backward):
    """``backward`` of kernels, which has no gradient of its own: asked for one
    (create_graph) it refuses a second pass, else it runs as it is."""
    twice = torch.autograd.function.once_differentiable(backward)
    return lambda ctx, d: (twice if torch.is_grad_enabled() else backward)(ctx, d)


class _Glu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, flat, act, group_size, bits):
        r = _glu_forward(x, flat, act, group_size, bits, True)
        if r is None:
            raise NotImplementedError("quantized_glu: no kernel of these sizes for the gradient")
        out, g, u = r
        ctx.args = act, group_size, bits
        ctx.save_for_backward(g, u)
        ctx.sums = (g, u) if forward_ad._current_level >= 0 else None
        _constants(ctx, flat)
        return out

    @staticmethod
    def jvp(ctx, t, *_):
        """h's tangent; those of the two products are rounded to their type."""
        (g, u), ctx.sums = ctx.sums, None
        act, *form = ctx.args
        tg, tu = (ops.quantized_matmul(t, *ctx.flat[i:i + 3], True, *form).float() for i in (0, 3))
        with torch.enable_grad():
            leaf = g.detach().requires_grad_()
            a = _activation(leaf, _name(act))
            da, = torch.autograd.grad(a, leaf, torch.ones_like(a))
        return (da * tg * u + a.detach() * tu).to(t.dtype)

    @staticmethod
    @_first_order
    def backward(ctx, d):
        g, u = ctx.saved_tensors
        return _glu_grad(d, g, u, _same_constants(ctx), *ctx.args), None, None, None, None


class _Matmul(torch.autograd.Function):
    """quantized_matmul of ``(M, K)`` rows by its own kernels, with x's gradient."""

    @staticmethod
    def forward(ctx, x, flat, group_size, bits):
        ctx.args = group_size, bits
        _constants(ctx, flat)
        return ops.quantized_matmul(x, *flat, True, group_size, bits)

    @staticmethod
    def jvp(ctx, t, *_):
        return ops.quantized_matmul(t, *ctx.flat, True, *ctx.args)

    @staticmethod
    @_first_order
    def backward(ctx, d):
        return matmul_grad(d, *_same_constants(ctx), *ctx.args), None, None, None


def quantized_matmul_differentiable(x, w, scales, biases, group_size: int, bits: int):
    """:func:`ops.quantized_matmul` of checked kernel-path arguments whose x is
    differentiated."""
    if wants_grad(x) and any(t.requires_grad for t in (scales, biases)):
        raise NotImplementedError("quantized_matmul: scales and biases are constants here; "
                                  "gradients go to x")
    leaf = note_leaf(x)
    flat = [ops._aligned(t) for t in (w, scales, biases)]
    x2 = x if x.ndim == 2 else x.reshape(-1, x.shape[-1])
    y = _Matmul.apply(x2, flat, group_size, bits)
    del leaf
    return y if x.ndim == 2 else y.reshape(*x.shape[:-1], w.shape[0])


def _name(act: int) -> str:
    return next(k for k, v in ACTIVATIONS.items() if v == act)


def _activation(g: torch.Tensor, activation: str) -> torch.Tensor:
    if activation == "silu":
        return torch.nn.functional.silu(g)
    return torch.nn.functional.gelu(g, approximate="tanh")


def _composed(x, gate, up, activation, group_size, bits, mode) -> torch.Tensor:
    """The block as its two products and the activation, for what has no kernel: the
    products are rounded to their type before the activation."""
    g, u = (ops.quantized_matmul(x, *m, group_size=group_size, bits=bits, mode=mode)
            for m in (gate, up))
    return (_activation(g.float(), activation) * u.float()).to(g.dtype)


def quantized_glu(x: torch.Tensor, gate, up, activation: str = "silu",
                  group_size: Optional[int] = None, bits: Optional[int] = None,
                  mode: str = "affine") -> torch.Tensor:
    """A dense gated feed-forward block up to its down projection:
    ``act(x @ dequantize(gate).T) * (x @ dequantize(up).T)`` for ``x`` ``(..., K)`` and
    ``gate`` and ``up`` ``(w, scales, biases)`` of one shape ``(N, K * bits / 32)``.
    ``activation``: "silu", or "gelu_tanh" (the tanh form).  Both products are summed
    in float, the activation and the product are float, and the result is rounded
    once (the three calls it replaces round three times).

    4- and 8-bit codes with bf16/fp16 activations in the scales' dtype run on the
    block's kernels: up to 16 rows (32 under :func:`ops.row_identity`) one that streams
    both matrices once, more on the MFMA tile; K in odd multiples of 32, which the tile does
    not take, in launches of 16 rows.  Other configurations run as two :func:`ops.quantized_matmul`
    and the activation, as does ``mode="mxfp4"`` (``(w, scales)``, or with None for
    the biases).

    Where ``x`` requires grad, so does the result: the backward pass gives x's
    gradient (``gate`` and ``up`` are constants; mxfp4 has none).  A forward-mode
    tangent of x gives the result's."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")
    group_size, bits = ops._format(group_size, bits, mode)
    gate, up = tuple(gate), tuple(up)
    if mode == "mxfp4":
        gate, up = ((*m, None)[:3] for m in (gate, up))
    if len(gate) != 3 or len(up) != 3:
        raise ValueError("gate and up are (w, scales, biases)")
    dev = ops._require_gpu(x, *gate, *up)
    if elsewhere(dev):
        with torch.cuda.device(dev):
            return quantized_glu(x, gate, up, activation, group_size, bits, mode)
    for name, i in (("w", 0), ("scales", 1)):
        if gate[i].shape != up[i].shape or gate[i].dtype != up[i].dtype:
            raise ValueError(f"gate and up differ: {name} {tuple(gate[i].shape)} {gate[i].dtype} "
                             f"and {tuple(up[i].shape)} {up[i].dtype}")
    if mode != "affine":
        if wants_grad(x):
            raise NotImplementedError(f"mode={mode!r}: gradients are affine weights' only")
        return _composed(x, gate, up, activation, group_size, bits, mode)
    for m in (gate, up):
        ops._check_mode(mode, m[2])
    w = gate[0]
    if w.ndim != 2:
        raise NotImplementedError("batched w: only 2-D weights are on this path")
    K = ops._check_quant(*gate, group_size, bits)
    if up[2].shape != up[1].shape or up[2].dtype != up[1].dtype:
        ops._check_quant(*up, group_size, bits)       # (the rest is the gate's: says what differs)
    if x.ndim < 1 or x.shape[-1] != K:
        raise ValueError(f"x {tuple(x.shape)} does not match the quantized weight K={K}")
    grad = differentiated(x)
    if wants_grad(x) and any(t.requires_grad for t in (*gate[1:], *up[1:])):
        raise NotImplementedError("quantized_glu: scales and biases are constants here; "
                                  "gradients go to x")
    if K == 0 or not (bits in (4, 8) and ops._kernel_dtype(x.dtype, gate[1].dtype)):
        return _composed(x, gate, up, activation, group_size, bits, mode)
    N, lead = w.shape[0], tuple(x.shape[:-1])
    x2 = x if x.ndim == 2 else x.reshape(math.prod(lead), K)
    flat = [ops._aligned(t) for t in (*gate, *up)]
    if grad:
        leaf = note_leaf(x)
        y = _Glu.apply(ops._aligned(x2), flat, ACTIVATIONS[activation], group_size, bits)
        del leaf
        return y if x.ndim == 2 else y.reshape(*lead, N)
    r = _glu_forward(ops._aligned(x2), flat, ACTIVATIONS[activation], group_size, bits, False)
    if r is None:
        return _composed(x, gate, up, activation, group_size, bits, mode)
    return r[0] if x.ndim == 2 else r[0].reshape(*lead, N)
