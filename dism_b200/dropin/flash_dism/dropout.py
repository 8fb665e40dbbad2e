"""Residual dropout from a counter-based generator; no mask is stored.  No counterpart in the reference."""
import torch
import cu_flash_dism as cu


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, threshold, seed, site):
        ctx.save_for_backward(seed)
        ctx.settings = threshold, site
        return cu.dropout(x.contiguous(), None if residual is None else residual.contiguous(), threshold, seed, site)

    @staticmethod
    def backward(ctx, dy):
        seed, = ctx.saved_tensors
        threshold, site = ctx.settings
        dx = None
        if ctx.needs_input_grad[0]:  # linear in dy: under create_graph the same operator again
            dx = _Dropout.apply(dy, None, threshold, seed, site) if torch.is_grad_enabled() else cu.dropout(dy.contiguous(), None, threshold, seed, site)
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


def dropout_add(x, residual, p, seed, *, site=0):
    """residual + dropout(x, p); with residual None just dropout(x, p).  float32, float16 or bfloat16, any shape; both of one type
    and shape.

    Element i (of the contiguous order) is kept when its 16-bit random number is at least round(65536 p), and scaled by
    65536 / (65536 - round(65536 p)).  The numbers are a function of (seed, site, i) alone: seed is a CUDA int64 tensor [2] of a key
    and an offset, read when the kernels run, and `site` (below 2^32) tells the calls of one step apart.  Advance the
    offset once a step, after the backward pass: seed[1] += 1, which a CUDA graph can capture too.  Autograd refuses a
    backward pass after the seed was changed in place, since its mask would differ from the forward's."""
    if not 0 <= p <= 1:
        raise ValueError('dropout probability must lie in [0, 1]')
    return _Dropout.apply(x, residual, round(65536 * p), seed, site)
