"""The gated delta rule by chunks in 64 bits, differentiable: for sequences too long to walk token by token."""
import torch

import delta_reference as reference

# Relative root mean square of a rounding to bf16: half a step is 2^-8 of the power of two below the value, the error is uniform in it, and
# over values whose logarithm is uniform the mean of (power of two / value)^2 is 3 / (8 ln 2).
ROUNDING = 2 ** -8 / 3 ** .5 * (3 / (8 * 0.6931471805599453)) ** .5


def _document(q, k, v, g, beta, scale, s, chunk):
    """One sequence, [N,H,*] operands, state [H,D,DV]."""
    n, out = v.shape[0], []
    for begin in range(0, n, chunk):
        qc, kc, vc, gc, bc = (x[begin:begin + chunk].transpose(0, 1) for x in (q, k, v, g, beta))
        total = gc.cumsum(-1)
        size = total.shape[-1]
        later = torch.ones(size, size, dtype=torch.bool, device=v.device).tril()
        between = torch.exp((total[..., :, None] - total[..., None, :]).masked_fill(~later, -torch.inf))
        decay, tail = torch.exp(total)[..., None], torch.exp(total[..., -1:] - total)[..., None]
        mixed = (between * (kc @ kc.mT)).tril(-1) * bc[..., None, :]
        x = torch.linalg.solve_triangular(torch.eye(size, dtype=v.dtype, device=v.device) + mixed, vc - decay * (kc @ s), upper=False, unitriangular=True)
        u = bc[..., None] * x
        out.append((scale * (decay * (qc @ s) + (between * (qc @ kc.mT)) @ u)).transpose(0, 1))
        s = decay[..., -1:, :] * s + kc.mT @ (tail * u)
    return (torch.cat(out) if out else v), s


def sequences(q, k, v, g, beta, scale, initial=None, starts=None, chunk=64):
    """As delta_reference.sequences."""
    spans = [(b, 0, v.shape[1]) for b in range(v.shape[0])] if starts is None else [(0, a, b) for a, b in zip(starts, starts[1:])]
    groups = v.shape[2] // q.shape[2]
    q, k = (x.repeat_interleave(groups, 2) for x in (q, k))
    outs, finals = [], []
    for index, (b, begin, end) in enumerate(spans):
        s = v.new_zeros(v.shape[2], q.shape[3], v.shape[3]) if initial is None else initial[index]
        o, s = _document(*(x[b, begin:end] for x in (q, k, v, g, beta)), scale, s, chunk)
        outs.append(o)
        finals.append(s)
    if starts is None:
        return torch.stack(outs), torch.stack(finals)
    rows = lambda m: v.new_zeros(m, *v.shape[2:])
    return torch.cat([rows(starts[0]), *outs, rows(v.shape[1] - starts[-1])])[None], torch.stack(finals)


def norms(got, want, heads_axis):
    """Error of every head relative to its norm."""
    got, want = (x.detach().double().cpu().movedim(heads_axis, 0).flatten(1) for x in (got, want))
    assert got.shape == want.shape and torch.isfinite(got).all()
    return ((got - want).norm(dim=1) / want.norm(dim=1)).max().item()


def check_chunked_form():
    """Against the rule token by token; both in 64 bits."""
    for starts, n in ((None, 150), ([5, 70, 70, 199], 210)):
        x = reference.operands(3, 2 if starts is None else 1, n, 1, 2, 32, 64)
        sides = []
        for form in (reference.sequences, sequences):
            leaves = [t.double().requires_grad_() for t in x]
            out, final = form(*leaves, 32 ** -.5, None, starts)
            sides.append([out, final, *torch.autograd.grad(out.square().sum() + final.square().sum(), leaves)])
        for a, b in zip(*sides):
            assert (a - b).abs().max() <= 1e-11 * a.abs().max()
