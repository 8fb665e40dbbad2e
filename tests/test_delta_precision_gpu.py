"""Training calls of the gated delta rule (no state asked for) against 64 bits, in norm per head.

Tolerances count the roundings that each output goes through, added in quadrature (delta_chunked.ROUNDING each), twice that: output: S0, T, P, U, Y
and itself; gradients: those of the forward but the output's and P (S0, T, U, Y), then dS1, scaled dO, dX, T, dY, scaled dY, dP or dL and the result."""
import pytest
import torch

import delta_chunked as chunked
import delta_reference as reference

pytestmark = pytest.mark.gpu
OUT, GRAD = 2 * 6 ** .5 * chunked.ROUNDING, 2 * 12 ** .5 * chunked.ROUNDING


@pytest.fixture(scope='module')
def flash():
    import dism_b200
    dism_b200.install_dropin()
    import flash_dism
    return flash_dism


def check(flash, x, starts=None, form=chunked.sequences):
    """x: operands on the host."""
    dout = torch.randn(x[2].shape, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    exact = [t.cuda().double().requires_grad_() for t in x]
    want, _ = form(*exact, x[0].shape[-1] ** -.5, None, starts)
    want_grads = torch.autograd.grad(want, exact, dout.double())
    leaves = [t.cuda().requires_grad_() for t in x]
    cu = None if starts is None else torch.tensor(starts, dtype=torch.int32, device='cuda')
    out = flash.gated_delta_rule(*leaves, cu_seqlens=cu)
    grads = torch.autograd.grad(out, leaves, dout)
    errors = dict(out=chunked.norms(out, want, 2))
    for name, got, expected in zip(('q', 'k', 'v', 'g', 'beta'), grads, want_grads):
        errors['d' + name] = chunked.norms(got, expected, 2)
    print({name: f'{e:.2e}' for name, e in errors.items()})
    assert all(e <= (OUT if name == 'out' else GRAD) for name, e in errors.items()), errors


@pytest.mark.parametrize('n,d,dv', [(16384, 64, 64), (16384, 128, 128), (4099, 128, 64)])
def test_joins_of_segments_do_not_pile_up(flash, n, d, dv):
    """Slow decays and weak writes: a segment's transition matrix is close to one, and whatever a join of two segments rounds away stays
    for all that follow."""
    x = reference.operands(d, 1, n, 1, 1, d, dv, decay=1e-5)
    x[4] = (x[4].float() * .004).bfloat16()
    check(flash, x)
