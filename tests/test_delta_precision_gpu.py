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


def check(flash, x, starts=None, states=False, out_bound=OUT, grad_bound=GRAD, decay_terms=None):
    """x: operands on the host.  decay_terms: what the error of dg is measured by, from the exact gradients, instead of its norm."""
    g = torch.Generator().manual_seed(1)
    dout = torch.randn(x[2].shape, generator=g).bfloat16().cuda()
    shape = (x[2].shape[0] if starts is None else len(starts) - 1, x[2].shape[2], x[0].shape[3], x[2].shape[3])
    initial, dfinal = (.3 * torch.randn(shape, generator=g).cuda() for _ in range(2)) if states else (None, None)
    more = [initial] if states else []
    exact = [t.cuda().double().requires_grad_() for t in x + more]
    want, want_state = chunked.sequences(*exact[:5], x[0].shape[-1] ** -.5, exact[5] if states else None, starts)
    want_grads = torch.autograd.grad([want, want_state] if states else want, exact, [dout.double(), dfinal.double()] if states else dout.double())
    leaves = [t.cuda().requires_grad_() for t in x + more]
    cu = None if starts is None else torch.tensor(starts, dtype=torch.int32, device='cuda')
    out = flash.gated_delta_rule(*leaves[:5], initial_state=leaves[5] if states else None, output_final_state=states, cu_seqlens=cu)
    out, final = out if states else (out, None)
    grads = torch.autograd.grad([out, final] if states else out, leaves, [dout, dfinal] if states else dout)
    errors = dict(out=chunked.norms(out, want, 2))
    for name, got, expected in zip(('q', 'k', 'v', 'g', 'beta', 'initial'), grads, want_grads):
        errors['d' + name] = chunked.norms(got, expected, 1 if name == 'initial' else 2)
    bounds = dict(out=out_bound, state=STATE)
    if states:
        errors['state'] = chunked.norms(final, want_state, 1)
    if decay_terms:
        errors['dg'] = ((grads[3].double() - want_grads[3]).norm(dim=1) / decay_terms(exact, want_grads).norm(dim=1)).max().item()
        bounds['dg'] = chunked.ROUNDING
    print({name: f'{e:.2e}' for name, e in errors.items()})
    assert all(e <= bounds.get(name, grad_bound) for name, e in errors.items()), errors


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


@pytest.mark.parametrize('key_heads,heads', [(2, 2), (1, 3)])
@pytest.mark.parametrize('d,dv', [(32, 32), (32, 128), (64, 64), (64, 128), (128, 32), (128, 64), (128, 128)])
def test_training_at_every_width(flash, d, dv, key_heads, heads):
    """No state asked for, key heads shared and not."""
    check(flash, reference.operands(d + dv, 2, 333, key_heads, heads, d, dv, gates=torch.float32 if heads == 3 else torch.bfloat16))


@pytest.mark.parametrize('decay', [1e-4, .02, .5, 4.])
def test_training_at_any_decay(flash, decay):
    check(flash, reference.operands(7, 1, 700, 1, 2, 128, 128, decay=decay))


@pytest.mark.parametrize('d,dv,key_heads', [(64, 64, 1), (128, 128, 2), (128, 64, 1), (64, 128, 2)])
def test_training_on_cut_chains(flash, d, dv, key_heads):
    check(flash, reference.operands(d, 1, 3001, key_heads, 2, d, dv, decay=.02))


@pytest.mark.parametrize('d,dv,starts', [(128, 128, [0, 1, 2, 66, 130, 130, 257]), (64, 64, [0, 0, 64, 128, 200]), (32, 64, [4, 90, 300]), (128, 128, [0, 600, 2400])])
def test_training_on_packs(flash, d, dv, starts):
    check(flash, reference.operands(len(starts), 1, starts[-1], 2, 4, d, dv, decay=.1), starts=starts)


@pytest.mark.parametrize('d,dv', [(64, 64), (128, 128)])
@pytest.mark.parametrize('states', [False, True])
def test_shares_against_64_bits(flash, d, dv, states):
    """A few more chains than places, long enough to be walked in equal shares."""
    room = 2 * torch.cuda.get_device_properties(0).multi_processor_count
    check(flash, reference.operands(d, (room + 8) * 64 // (4 * dv), 577, 2, 4, d, dv, decay=.02), states=states)


def test_repeated_keys_in_training(flash):
    """One key for a whole chunk and write strengths of one, the worst case of the chunk's inverse: its rows cancel, so roundings are
    not small beside what is left of them, and each is counted in full (2^-8) and added.

    dg is what is left of larger terms: a factor on every state from position t on can be moved to q from t on and, inverted, to v, so dg_t is the sum
    over j >= t of q_j.dq_j - v_j.dv_j; and the kernels reach v_j.dv_j through k_j.dk_j, by adding beta_j dbeta_j and taking it away.  Each of these
    comes out of products of bf16 operands, so even with nothing else rounded one rounding of the terms, in quadrature over a chunk, is left
    in dg.  Here the terms are a hundred times dg (norms 2.4e2 and 2.4 for the first head): dg is held to one rounding of them."""
    x = reference.operands(11, 1, 200, 2, 2, 128, 64, decay=.02)
    x[1][:, 20:100] = x[1][:, 20:21]
    x[0][:, 50:] = x[1][:, 50:]
    x[4].fill_(1.)

    def terms(exact, grads):
        q, k, v, g, beta = exact
        each = (q * grads[0]).sum(-1).square() + (v * grads[2]).sum(-1).square() + 2 * (beta * grads[4]).square()
        chunks = torch.nn.functional.pad(each, (0, 0, 0, -each.shape[1] % 64)).unflatten(1, (-1, 64))
        return chunks.flip(2).cumsum(2).flip(2).flatten(1, 2)[:, :each.shape[1]].sqrt()
    check(flash, x, out_bound=6 * 2 ** -8, grad_bound=12 * 2 ** -8, decay_terms=terms)


def test_only_the_last_state_is_asked_for(flash):
    """A loss of the final state alone: no gradient reaches the output."""
    x = reference.operands(12, 2, 150, 1, 2, 64, 64)
    exact = [t.cuda().double().requires_grad_() for t in x]
    weight = torch.randn(2, 2, 64, 64, generator=torch.Generator().manual_seed(2)).cuda()
    want = torch.autograd.grad((chunked.sequences(*exact, 64 ** -.5)[1] * weight.double()).sum(), exact[1:])
    leaves = [t.cuda().requires_grad_() for t in x]
    got = torch.autograd.grad((flash.gated_delta_rule(*leaves, output_final_state=True)[1] * weight).sum(), leaves)
    assert not got[0].count_nonzero()
    assert all(chunked.norms(a, b, 2) <= GRAD for a, b in zip(got[1:], want))


@pytest.mark.parametrize('b,n,heads', [(75, 577, 4), (1, 4100, 2)])
def test_captured_training_step(flash, b, n, heads):
    """Walked in shares and cut into segments: replays follow new inputs, two graphs in turn do not disturb one another."""
    sets = [[t.cuda() for t in reference.operands(seed, b, n, 1, heads, 64, 64, decay=.02)] for seed in (1, 2)]
    dout = torch.randn_like(sets[0][2])

    def step(leaves):
        out = flash.gated_delta_rule(*leaves)
        return [out, *torch.autograd.grad(out, leaves, dout)]
    wanted = [step([t.clone().requires_grad_() for t in x]) for x in sets]
    wanted = [[t.detach() for t in w] for w in wanted]
    graphs = []
    for x in sets:
        held = [t.clone().requires_grad_() for t in x]
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            got = step(held)
        graphs.append((graph, held, got))
    for turn in range(4):
        graph, held, got = graphs[turn % 2]
        other = (turn // 2 + turn) % 2
        with torch.no_grad():
            for t, new in zip(held, sets[other]):
                t.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, w) for a, w in zip(got, wanted[other]))
