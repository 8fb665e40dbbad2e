"""Gated delta rule: the recurrent mixer beside DISM layers in a hybrid model, over whole sequences and one token at a time.

The reference's hybrid layers call such an operator of an outside package (dism_v3/python/flash_dism/hybrid_gdn.py,
pure_gdn.py); here it is part of the library.  Per value head, with a state S [D,DV]:

    S_t = exp(g_t) S_{t-1} + k_t u_t^T,   u_t = beta_t (v_t - exp(g_t) S_{t-1}^T k_t),   o_t = scale S_t^T q_t
"""
import torch
import cu_flash_dism as cu


def _ready(t):
    """Contiguous and 16-byte aligned, as the library wants its tensors; a copy only where it is needed."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _gate_type(g, beta):
    return g.dtype if g.dtype == beta.dtype and g.dtype in (torch.float32, torch.bfloat16) else torch.float32


def _backward(ctx, dout, dfinal=None):
    saved = ctx.saved_tensors
    types, gates, scale, shape = ctx.settings
    if dout is None:
        dout = torch.zeros(shape, dtype=torch.bfloat16, device=saved[0].device)
    dq, dk, dv, dg, dbeta, dinitial = cu.delta_backward(saved[0], saved[1], _ready(dout), scale, saved[2], gates, None if dfinal is None else _ready(dfinal),
                                                        ctx.needs_input_grad[5], saved[3] if len(saved) > 3 else None)
    return (dq, dk, dv, dg if gates is types[0] else dg.to(types[0]), dbeta if gates is types[1] else dbeta.to(types[1]), dinitial,
            None, None, None, None)


class _NotTwice(torch.autograd.Function):
    """Hands gradients on and refuses to be differentiated, whether or not what they depend on is a part of the graph."""
    @staticmethod
    def forward(ctx, anchor, *grads):
        return tuple(t.view_as(t) for t in grads)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError('the gradients of gated_delta_rule are not differentiable')


class _GatedDelta(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, initial_state, scale, final_state, starts, needed):
        gates = _gate_type(g, beta)
        q, k = _ready(q), _ready(k)
        out, final, saved = cu.delta_forward((q, k, _ready(v), _ready(g if gates is g.dtype else g.to(gates)),
                                              _ready(beta if gates is beta.dtype else beta.to(gates))), scale,
                                             None if initial_state is None else _ready(initial_state), final_state, starts, needed)
        if needed:
            ctx.save_for_backward(*((q, k, saved) if starts is None else (q, k, saved, starts)))
            ctx.settings = (g.dtype, beta.dtype), gates, scale, v.shape
            ctx.set_materialize_grads(False)
        return (out, final) if final_state else out

    @staticmethod
    def backward(ctx, *grads):
        if not torch.is_grad_enabled():
            return _backward(ctx, *grads)
        with torch.no_grad():  # create_graph=True
            result = _backward(ctx, *grads)
        present = iter(_NotTwice.apply(torch.zeros((), requires_grad=True), *[t for t in result if t is not None]))
        return tuple(t if t is None else next(present) for t in result)


_starts = {}
_captured = {}  # graphs hold the addresses of these


def _capturing(device):
    return device.type == 'cuda' and torch.cuda.is_current_stream_capturing()


def _host_starts(starts, device):
    """Document starts on the device, uploaded once for as long as the pack is among the last 32 or a captured graph reads it."""
    key = (tuple(starts), str(device))
    cached = _captured.get(key)
    if cached is None:
        cached = _starts.get(key)
    if _capturing(device):
        if cached is None:
            raise RuntimeError('document starts cannot be uploaded inside a capture: make the call once before it, or pass cu_seqlens on the device')
        _captured[key] = cached
        return cached
    if cached is None:
        if len(_starts) >= 32:
            _starts.pop(next(iter(_starts)), None)
        with torch.inference_mode(False):  # a training call may save what an evaluation has uploaded
            cached = _starts[key] = torch.tensor(starts, dtype=torch.int32).to(device)
    if device.type == 'cuda':
        cached.record_stream(torch.cuda.current_stream(device))  # dropped, its memory waits for this call's kernels
    return cached


def _documents(v, cu_seqlens, layout):
    """Device starts of the documents of a pack."""
    if cu_seqlens is not None and layout is not None:
        raise ValueError('provide either layout or cu_seqlens, not both')
    if layout is not None:
        starts = [0]
        for length in layout.lengths:
            starts.append(starts[-1] + length)
        if v.dim() != 4 or starts[-1] != v.size(1):
            raise ValueError('layout and operands differ in length')
        return _host_starts(starts, v.device)
    if cu_seqlens is None:
        return None
    if not (torch.is_tensor(cu_seqlens) and cu_seqlens.dim() == 1 and cu_seqlens.dtype == torch.int32 and cu_seqlens.numel() > 1):
        raise RuntimeError('cu_seqlens must be int32 [sequences+1]')
    if cu_seqlens.device.type == 'cpu':
        starts = cu_seqlens.tolist()
        if v.dim() != 4 or starts[0] != 0 or starts[-1] != v.size(1) or any(a > b for a, b in zip(starts, starts[1:])):
            raise RuntimeError('invalid cu_seqlens: starts at 0, ascending, ends at the number of positions')
        return _host_starts(starts, v.device)
    return cu_seqlens.contiguous()


def gated_delta_rule(q, k, v, g, beta, *, scale=None, initial_state=None, output_final_state=False, cu_seqlens=None, layout=None):
    """BF16 q, k [B,N,HK,D] and v [B,N,H,DV], log decay g and write strength beta [B,N,H] (float32 or bfloat16) -> BF16
    [B,N,H,DV]; with output_final_state=True also the FP32 state [sequences,H,D,DV] after each sequence's last position.

    H is a multiple of HK (value head h reads key head h // (H // HK)), D and DV in {32,64,128}, N any length.  Keys are meant to
    have length one at most; the caller normalises.  scale defaults to D ** -0.5.  g = -inf clears a finite state.  A pack is one
    batch row with either `layout` (a VarlenLayout) or `cu_seqlens`, int32 [documents+1]; documents may have any length, zero
    included.  On the CPU cu_seqlens is validated (and like a layout uploaded once, which has to happen before a
    capture); on the GPU it is read by the kernels only (so a captured graph can follow new
    lengths), must ascend, and rows outside [cu_seqlens[0], cu_seqlens[-1]) come out as zeros.  initial_state is FP32
    [sequences,H,D,DV].  All operands and the initial state are differentiable; gates receive gradients in their own type, with
    the relative accuracy of the bf16 operands.  Keeping the states for a backward takes 2 D DV / 64 + 2 DV + 184 bytes per position
    and head, and 4 D D + 4 D DV per segment and head where a long chain is cut (documents of a pack that are shorter than a segment add none), or 256 D
    per place of the device (two an SM) where chains are walked in shares."""
    starts = _documents(v, cu_seqlens, layout)
    needed = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or g.requires_grad or beta.requires_grad
                                          or initial_state is not None and initial_state.requires_grad)
    return _GatedDelta.apply(q, k, v, g, beta, initial_state, q.size(-1) ** -.5 if scale is None else float(scale),
                                   bool(output_final_state), starts, needed)


@torch.no_grad()
def gated_delta_step(q, k, v, g, beta, state, *, scale=None, slots=None):
    """One token for every row of a decoding batch: q, k BF16 [B,HK,D], v BF16 [B,H,DV], g and beta [B,H] -> BF16 [B,H,DV].

    `state` is FP32 [pool,H,D,DV], contiguous, and is updated in place.  `slots`, int32 [B] on the GPU, names the state of each
    row (default: state i for row i); a slot outside the pool marks a padding row, whose output is zero, and rows that name
    one slot are consecutive tokens of that sequence, in row order.  Everything is computed in 32 bits; not differentiable."""
    gates = _gate_type(g, beta)
    out = cu.delta_step((_ready(q), _ready(k), _ready(v), _ready(g.to(gates)), _ready(beta.to(gates))),
                        q.size(-1) ** -.5 if scale is None else float(scale), state, slots)
    if not state.is_inference():
        torch.autograd.graph.increment_version(state)  # a graph that has saved the state sees that it has changed
    return out
