"""A token from a head's logits: temperature, top-k, top-p and min-p, from given
uniform numbers.

The step behind an ``lm_head`` product (:func:`ops.quantized_matmul`), as
:func:`ops.moe_route` is behind a router's: every row of logits is a sequence (or a
drafted position) with settings of its own.
"""

from __future__ import annotations

import math

import torch

from . import _lib, glu, ops


def _setting(name: str, v, lead: tuple, dev: torch.device, dtype: torch.dtype, least, most):
    """``(pointer or None, value, the tensor)`` of one setting."""
    if isinstance(v, torch.Tensor):
        # a tensor of the rows' own: nothing to convert
        if (v.dtype == dtype and v.shape == lead and v.get_device() == dev.index
                and v.is_contiguous()):
            return v.data_ptr(), 0, v
        ops._require_gpu(v)
        if v.device != dev:
            raise ValueError(f"{name} is on {v.device}, logits on {dev}")
        if dtype == torch.int32 and (v.dtype.is_floating_point or v.dtype == torch.bool):
            raise ValueError(f"{name} must be integers, got {v.dtype}")
        if v.dtype.is_complex or v.dtype == torch.bool:
            raise ValueError(f"{name} must be real numbers, got {v.dtype}")
        try:
            v = v.detach().expand(lead)
        except RuntimeError as exc:
            raise ValueError(f"{name} {tuple(v.shape)} does not broadcast to the rows "
                             f"{lead}") from exc
        if dtype == torch.int32 and v.dtype == torch.int64:
            v = v.clamp(-1, 2 ** 31 - 1)              # more words than any vocabulary has
        t = v.to(dtype).contiguous()
        return t.data_ptr(), 0, t
    v = int(v) if dtype == torch.int32 else float(v)
    if not least <= v <= most:
        raise ValueError(f"{name} must be in {least}..{most}, got {v}")
    return None, v, None


def sample(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0,
           min_p=0.0):
    """Tokens ``(...)`` int32 and their log probabilities ``(...)`` float32 for
    ``logits`` ``(..., V)`` (bfloat16, float16 or float32) and uniform numbers ``u``
    ``(...)`` float32 in [0, 1).

    A word's mass is ``exp((l - max) / temperature)``; words are in order of value,
    equal ones the lower index first.  Kept are the first ``top_k`` words (0: all), of
    those the words before which the mass is less than ``top_p`` of theirs (1: all), and
    of those the words of at least ``min_p`` of the most probable one's mass (0: all);
    always the first word.  The token is the first kept word, in index order, up to
    which the kept mass is more than ``u`` times all of it; its log probability is that
    among the kept.  ``temperature`` 0 takes the first word.  The settings are numbers,
    or tensors that broadcast to the rows.

    -inf masks a word, and so does NaN; a row with nothing left gives token -1 and
    -inf.  Masses are held in integers, so a row's result depends on the row alone.
    In tensors, which are not looked at on the host, a temperature below 0 or NaN is 0,
    top_k below 0 is 0, top_p outside (0, 1) is 1 or, at most 0, the first word alone,
    min_p below 0 is 0 and above 1 or NaN leaves the first word alone, and u is moved into
    [0, 1)."""
    dev = ops._require_gpu(logits, u)
    if glu.elsewhere(dev):
        with torch.cuda.device(dev):
            return sample(logits, u, temperature, top_k, top_p, min_p)
    if logits.dtype not in ops._DTYPE_CODE:
        raise ValueError(f"sample takes bfloat16, float16 or float32 logits, got {logits.dtype}")
    if logits.ndim < 1 or logits.shape[-1] == 0:
        raise ValueError("logits must have a vocabulary dimension")
    lead, V = tuple(logits.shape[:-1]), logits.shape[-1]
    if u.dtype != torch.float32 or tuple(u.shape) != lead:
        raise ValueError(f"u must be float32 {lead}, got {u.dtype} {tuple(u.shape)}")
    R = math.prod(lead)
    t = _setting("temperature", temperature, lead, dev, torch.float32, 0.0, math.inf)
    k = _setting("top_k", top_k, lead, dev, torch.int32, 0, 2 ** 31 - 1)
    p = _setting("top_p", top_p, lead, dev, torch.float32, 0.0, 1.0)
    m = _setting("min_p", min_p, lead, dev, torch.float32, 0.0, 1.0)
    tokens = torch.empty(lead, dtype=torch.int32, device=dev)
    logprobs = torch.empty(lead, dtype=torch.float32, device=dev)
    if R == 0:
        return tokens, logprobs
    # rows where they lie, if one stride leads from each to the next
    l, stride = logits, V
    if not l.is_contiguous():
        if l.stride(-1) != 1:
            l = l.contiguous()
        try:
            l = l.view(R, V)
        except RuntimeError:
            l = l.reshape(R, V)
        if R > 1:
            stride = l.stride(0)
    u_ = u.contiguous()
    lib = _lib.lib()
    ws = torch.empty(lib.mq_sample_workspace_size(R, V), dtype=torch.uint8, device=dev)
    rc = lib.mq_sample(l.data_ptr(), stride, R, V, ops._DTYPE_CODE[l.dtype], u_.data_ptr(),
                       *t[:2], *k[:2], *p[:2], *m[:2], tokens.data_ptr(), logprobs.data_ptr(),
                       ws.data_ptr(), ws.numel(), ops._stream_ptr(tokens))
    _lib.check(rc, "sample")
    return tokens, logprobs
