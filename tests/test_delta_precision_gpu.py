"""The gated delta rule against 64 bits, in norm per head; above all training calls (no state asked for), whose kernels take single operands.

Tolerances count the roundings that each output goes through, added in quadrature (delta_chunked.ROUNDING each), twice that: output: S0, T, P, U, Y
and itself; gradients: those of the forward but the output's and P (S0, T, U, Y), then dS1, scaled dO, dX, T, dY, scaled dY, dP or dL and the result.
A final state: S0, Y, T, U and M as pairs, 2^-8 of the rounding above each, and the 64 additions in 32 bits of each chunk."""
import pytest
import torch

import delta_chunked as chunked
import delta_reference as reference

pytestmark = pytest.mark.gpu
OUT, GRAD = 2 * 6 ** .5 * chunked.ROUNDING, 2 * 12 ** .5 * chunked.ROUNDING
STATE = 2 * 5 ** .5 * chunked.ROUNDING * 2 ** -8 + 64 * 2 ** -24


@pytest.fixture(scope='module')
def flash():
    import dism_b200
    dism_b200.install_dropin()
    import flash_dism
    return flash_dism


def check(flash, x, starts=None, states=False, form=chunked.sequences):
    """x: operands on the host."""
    g = torch.Generator().manual_seed(1)
    dout = torch.randn(x[2].shape, generator=g).bfloat16().cuda()
    shape = (x[2].shape[0] if starts is None else len(starts) - 1, x[2].shape[2], x[0].shape[3], x[2].shape[3])
    initial, dfinal = (.3 * torch.randn(shape, generator=g).cuda() for _ in range(2)) if states else (None, None)
    more = [initial] if states else []
    exact = [t.cuda().double().requires_grad_() for t in x + more]
    want, want_state = form(*exact[:5], x[0].shape[-1] ** -.5, exact[5] if states else None, starts)
    want_grads = torch.autograd.grad([want, want_state] if states else want, exact, [dout.double(), dfinal.double()] if states else dout.double())
    leaves = [t.cuda().requires_grad_() for t in x + more]
    cu = None if starts is None else torch.tensor(starts, dtype=torch.int32, device='cuda')
    out = flash.gated_delta_rule(*leaves[:5], initial_state=leaves[5] if states else None, output_final_state=states, cu_seqlens=cu)
    out, final = out if states else (out, None)
    grads = torch.autograd.grad([out, final] if states else out, leaves, [dout, dfinal] if states else dout)
    errors = dict(out=chunked.norms(out, want, 2))
    for name, got, expected in zip(('q', 'k', 'v', 'g', 'beta', 'initial'), grads, want_grads):
        errors['d' + name] = chunked.norms(got, expected, 1 if name == 'initial' else 2)
    if states:
        errors['state'] = chunked.norms(final, want_state, 1)
    print({name: f'{e:.2e}' for name, e in errors.items()})
    assert all(e <= dict(out=OUT, state=STATE).get(name, GRAD) for name, e in errors.items()), errors


@pytest.mark.parametrize('n,d,dv', [(16384, 64, 64), (16384, 128, 128), (4099, 128, 64)])
def test_joins_of_segments_do_not_pile_up(flash, n, d, dv):
    """Slow decays and weak writes: a segment's transition matrix is close to one, and whatever a join of two segments rounds away stays
    for all that follow."""
    x = reference.operands(d, 1, n, 1, 1, d, dv, decay=1e-5)
    x[4] = (x[4].float() * .004).bfloat16()
    check(flash, x)


@pytest.mark.parametrize('starts', [[0, 700, 1300, 1301, 2500, 2564, 4000], [3, 1540, 1540, 3081, 4618, 4700], [0] + list(range(100, 1100)) + [4200]])
@pytest.mark.parametrize('states', [False, True])
def test_cut_documents_of_a_pack(flash, starts, states):
    """Several documents long enough to be cut, short and empty ones between them; what is kept of their segments lies without gaps."""
    x = reference.operands(len(starts), 1, starts[-1] + 20, 1, 2, 64, 64, decay=.01)
    check(flash, x, starts=starts, states=states)


def test_short_documents_take_no_room_for_segments():
    """262144 positions in 4096 documents, 16 heads of 128 x 128: such chains are cut, but only where a document is longer than a segment."""
    from dism_b200 import _lib
    lib = _lib.load()
    places = (262144 // 64 + 4096) * 16
    assert lib.dism_delta_saved(1, 4096, 262144, 16, 128, 128, 1, 0) <= 1.03 * places * (384 * 4 + 3 * 2560 * 2)
    assert lib.dism_delta_saved(1, 4096, 262144, 16, 128, 128, 0, 1) <= 1.03 * places * (384 * 4 + 2 * 2560 * 2 + 128 * 128 * 2 + 64 * 128 * 2)
    assert lib.dism_delta_backward_workspace(1, 4096, 262144, 16, 128, 128) <= 1.03 * places * (128 * 128 * 2 + 64 * 8 * 4)


def test_a_pack_seen_in_inference_mode_trains_afterwards(flash):
    x = [t.cuda() for t in reference.operands(2, 1, 90, 1, 1, 32, 32)]
    starts = torch.tensor([0, 33, 90], dtype=torch.int32)
    with torch.inference_mode():
        quiet = flash.gated_delta_rule(*x, cu_seqlens=starts)
    leaves = [t.requires_grad_() for t in x]
    out = flash.gated_delta_rule(*leaves, cu_seqlens=starts)
    assert torch.equal(out, quiet)
    assert all(torch.isfinite(t).all() for t in torch.autograd.grad(out, leaves, torch.ones_like(out)))
