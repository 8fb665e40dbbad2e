"""Gated delta rule on the GPU against the 64-bit token-by-token rule.

Tolerances count roundings.  A bf16 rounding is off by at most 2^-8 of a value, a bf16 pair (value and remainder) by 2^-16.
Output: S0, Y, T, U, P and the result itself are rounded once each on the way: 6 * 2^-8 of the norm.  Gradients: S0 and X of the
forward (Y and T before X: 4), then dS1, scaled dO, dX, T, dY and scaled dY in the reverse chain, dP~ or dL~ and the result:
12 * 2^-8.  Final state: S0, Y, T and U as pairs, the product of the two remainders left out: 5 * 2^-16, and 64 additions in 32 bits
a chunk.  Every tensor is compared in norm per head, and every element with the same bound relative to the larger of itself and four times
the head's root mean square (a sum over a chunk can be smaller than its terms).
"""
import pytest
import torch

import delta_reference as reference

pytestmark = pytest.mark.gpu
OUT, GRAD, STATE = 6 * 2 ** -8, 12 * 2 ** -8, 5 * 2 ** -16 + 64 * 2 ** -24


@pytest.fixture(scope='module')
def flash():
    import dism_b200
    dism_b200.install_dropin()
    import flash_dism
    return flash_dism


@pytest.fixture(autouse=True)
def no_fault():
    """No bounded wait of the tensor-memory pipelines runs out in any test."""
    import ctypes
    from dism_b200 import _lib
    yield
    code = ctypes.c_int(-1)
    _lib.check(_lib.load().dism_delta_fault(ctypes.byref(code)))
    assert code.value == 0


def near(got, want, bound, heads_axis, what=''):
    got, want = (x.detach().double().cpu().movedim(heads_axis, 0).flatten(1) for x in (got, want))
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    error, norm = (got - want).norm(dim=1), want.norm(dim=1)
    assert (error <= bound * norm + 1e-30).all(), (what, (error / norm).max().item(), bound)
    level = torch.maximum(want.abs(), 4 * norm[:, None] / max(1, want.shape[1]) ** .5)
    assert ((got - want).abs() <= bound * level + 1e-30).all(), (what, 'elements', ((got - want).abs() / level).max().item(), bound)


def check(flash, seed, b, n, key_heads, heads, d, dv, gates=torch.bfloat16, starts=None, states=False, decay=.5, scale=None, change=None):
    x = reference.operands(seed, b, n, key_heads, heads, d, dv, gates, decay)
    if change:
        change(*x)
    sequences = b if starts is None else len(starts) - 1
    g = torch.Generator().manual_seed(seed + 1)
    dout = torch.randn(b, n, heads, dv, generator=g).bfloat16()
    initial = .3 * torch.randn(sequences, heads, d, dv, generator=g) if states else None
    dfinal = .3 * torch.randn(sequences, heads, d, dv, generator=g) if states else None
    factor = d ** -.5 if scale is None else scale
    exact = [t.double().requires_grad_() for t in x] + ([initial.double().requires_grad_()] if states else [])
    want, want_state = reference.sequences(*exact[:5], factor, exact[5] if states else None, starts)
    loss = (want * dout.double()).sum() + ((want_state * dfinal.double()).sum() if states else 0.)
    want_grads = torch.autograd.grad(loss, exact, allow_unused=True)

    leaves = [t.cuda().requires_grad_() for t in x]
    start = initial.cuda().requires_grad_() if states else None
    cu = None if starts is None else torch.tensor(starts, dtype=torch.int32, device='cuda')
    result = flash.gated_delta_rule(*leaves, scale=scale, initial_state=start, output_final_state=states, cu_seqlens=cu)
    out, final = result if states else (result, None)
    assert out.dtype == torch.bfloat16 and out.shape == want.shape
    near(out, want, OUT, 2, 'out')
    inputs = leaves + ([start] if states else [])
    grads = torch.autograd.grad([out, final] if states else [out], inputs, [dout.cuda(), dfinal.cuda()] if states else [dout.cuda()])
    for name, leaf, got, expected in zip(('q', 'k', 'v', 'g', 'beta', 'initial'), inputs, grads, want_grads):
        assert got.dtype == leaf.dtype and got.shape == leaf.shape
        near(got, expected, GRAD, 1 if name == 'initial' else 2, 'd' + name)
    if states:
        near(final, want_state, STATE, 1, 'final state')
    # without gradients nothing is kept, and the outputs are the same bits
    with torch.no_grad():
        again = flash.gated_delta_rule(*[t.detach() for t in leaves], scale=scale, initial_state=None if start is None else start.detach(),
                                       output_final_state=states, cu_seqlens=cu)
    assert torch.equal(again[0] if states else again, out)
    if states:
        assert torch.equal(again[1], final)


@pytest.mark.parametrize('n', [1, 2, 15, 16, 63, 64, 65, 127, 129, 200])
def test_lengths(flash, n):
    check(flash, n, 2, n, 2, 2, 64, 64)


@pytest.mark.parametrize('d', [32, 64, 128])
@pytest.mark.parametrize('dv', [32, 64, 128])
def test_widths_and_states(flash, d, dv):
    check(flash, d + dv, 2, 150, 1, 2, d, dv, states=True)


@pytest.mark.parametrize('gates', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('key_heads,heads', [(1, 4), (2, 6), (3, 3)])
def test_shared_key_heads(flash, gates, key_heads, heads):
    check(flash, heads, 1, 130, key_heads, heads, 64, 32, gates=gates, states=True)


@pytest.mark.parametrize('starts', [[0, 1, 2, 66, 130, 130, 257], [0, 0, 64, 128, 200], [0, 257], [0, 0, 0, 1]])
def test_packed_documents(flash, starts):
    check(flash, len(starts), 1, starts[-1], 2, 4, 32, 64, starts=starts, states=True)


@pytest.mark.parametrize('d,dv,starts', [(64, 64, None), (128, 64, None), (64, 128, [0, 1700, 1701, 1701, 2100]), (128, 128, [0, 600, 1750])])
def test_long_chains_are_cut_into_segments(flash, d, dv, starts):
    """Few heads and many chunks: the segments' transition matrices carry the state, and its gradient, from one to the next.  The state at
    a segment's start has one rounding more (M), which the bounds of the shorter cases leave room for."""
    check(flash, d + dv, 1, 2100 if starts is None else starts[-1], 1, 2, d, dv, starts=starts, states=True, decay=.02)


@pytest.mark.parametrize('decay', [0., .01, 4.])
def test_decays(flash, decay):
    check(flash, 7, 1, 320, 1, 2, 128, 64, states=True, decay=decay)


def test_repeated_keys_and_full_writes(flash):
    """One key for a whole chunk and beta of one: the worst case of the chunk's inverse."""
    def change(q, k, v, g, beta):
        k[:, 20:100] = k[:, 20:21]
        q[:, 50:] = k[:, 50:]
        beta.fill_(1.)
    check(flash, 11, 1, 160, 2, 2, 64, 64, states=True, decay=.02, change=change)


def test_beta_of_zero_and_scale(flash):
    def change(q, k, v, g, beta):
        beta[:, 10:90:3] = 0.
    check(flash, 12, 2, 100, 1, 2, 64, 64, change=change, scale=1.)


def test_cleared_state(flash):
    """g of minus infinity clears the state: the positions behind it are those of a sequence of their own."""
    x = reference.operands(3, 1, 150, 2, 2, 64, 64, torch.float32)
    x[3][:, 70] = -float('inf')
    leaves = [t.cuda().requires_grad_() for t in x]
    out, final = flash.gated_delta_rule(*leaves, output_final_state=True)
    want, want_state = reference.sequences(*[t.double() for t in x], 64 ** -.5)
    near(out, want, OUT, 2)
    near(final, want_state, STATE, 1)
    grads = torch.autograd.grad(out.float().square().sum() + final.square().sum(), leaves)
    assert all(torch.isfinite(t).all() for t in grads)
    rest, rest_state = flash.gated_delta_rule(*[t.detach()[:, 70:].contiguous() for t in leaves], output_final_state=True)
    near(out[:, 70:], rest.double(), 2 * OUT, 2)
    near(final, rest_state.double(), 2 * STATE, 1)
    assert (grads[3][:, 70] == 0).all()


def test_rows_outside_the_documents_are_zeros(flash):
    x = [t.cuda().requires_grad_() for t in reference.operands(5, 1, 200, 1, 2, 32, 32)]
    starts = [10, 50, 140]
    out = flash.gated_delta_rule(*x, cu_seqlens=torch.tensor(starts, dtype=torch.int32, device='cuda'))
    want, _ = reference.sequences(*[t.detach().double().cpu() for t in x], 32 ** -.5, None, starts)
    near(out, want, OUT, 2)
    assert not out[:, :10].count_nonzero() and not out[:, 140:].count_nonzero()
    for grad in torch.autograd.grad(out, x, torch.ones_like(out)):
        assert not grad[:, :10].count_nonzero() and not grad[:, 140:].count_nonzero() and torch.isfinite(grad).all()


@pytest.mark.parametrize('starts,n', [([1500, 1800, 3700], 4000), ([3990, 4000], 4100), ([0, 30], 4100)])
def test_rows_outside_the_documents_of_a_long_pack(flash, starts, n):
    """Long enough for chains cut into segments; the documents begin late or end early."""
    x = [t.cuda().requires_grad_() for t in reference.operands(5, 1, n, 1, 1, 64, 64)]
    out = flash.gated_delta_rule(*x, cu_seqlens=torch.tensor(starts, dtype=torch.int32, device='cuda'))
    dout = torch.randn_like(out)
    grads = torch.autograd.grad(out, x, dout)
    assert not out[:, :starts[0]].count_nonzero() and not out[:, starts[-1]:].count_nonzero()
    part = slice(starts[0], starts[-1])
    inner = [t.detach()[:, part].contiguous().requires_grad_() for t in x]
    want = flash.gated_delta_rule(*inner, cu_seqlens=torch.tensor(starts, dtype=torch.int32, device='cuda') - starts[0])
    near(out[:, part], want.double(), 2 * OUT, 2)
    for got, expected in zip(grads, torch.autograd.grad(want, inner, dout[:, part].contiguous())):
        assert not got[:, :starts[0]].count_nonzero() and not got[:, starts[-1]:].count_nonzero()
        near(got[:, part], expected.double(), 2 * GRAD, 2)


def test_mixed_gate_types_partial_gradients_and_second_order(flash):
    x = reference.operands(13, 1, 100, 1, 2, 64, 64, torch.float32, device='cuda')
    x[4] = x[4].bfloat16()
    leaves = [t.clone().requires_grad_() for t in x]
    out = flash.gated_delta_rule(*leaves)
    dout = torch.randn_like(out)
    every = torch.autograd.grad(out, leaves, dout)
    assert [t.dtype for t in every] == [t.dtype for t in x]
    only = x[1].clone().requires_grad_()
    again = flash.gated_delta_rule(x[0], only, *x[2:])
    assert torch.equal(again, out) and torch.equal(torch.autograd.grad(again, only, dout)[0], every[1])
    # a key shared by the batch: its gradient is the sum
    shared = x[1].clone().requires_grad_()
    two = flash.gated_delta_rule(*[t.expand(2, *t.shape[1:]) if t is not x[1] else shared.expand(2, *t.shape[1:]) for t in x])
    grad, = torch.autograd.grad(two, shared, dout.expand(2, *dout.shape[1:]))
    near(grad, 2 * every[1].double(), GRAD, 2)
    grad, = torch.autograd.grad(flash.gated_delta_rule(x[0], only, *x[2:]).float().sum(), only, create_graph=True)
    with pytest.raises(RuntimeError, match='not differentiable'):
        grad.sum().backward()


def test_first_call_inside_a_capture(flash):
    """A shape whose kernels have not run yet is captured at once."""
    x = [t.requires_grad_() for t in reference.operands(14, 1, 70, 2, 2, 64, 128, device='cuda')]
    dout = torch.randn_like(x[2])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = flash.gated_delta_rule(*x)
        grads = torch.autograd.grad(out, x, dout)
    graph.replay()
    torch.cuda.synchronize()
    want = flash.gated_delta_rule(*x)
    assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(want, x, dout)))


def test_a_step_counts_as_a_change_of_the_state(flash):
    x = reference.operands(15, 2, 1, 1, 1, 32, 32, device='cuda')
    state = torch.zeros(2, 1, 32, 32, device='cuda')
    before = state._version
    flash.gated_delta_step(*[t[:, 0] for t in x], state)
    assert state._version > before
    with torch.inference_mode():
        held = torch.zeros(2, 1, 32, 32, device='cuda')
        flash.gated_delta_step(*[t[:, 0] for t in x], held)
    assert torch.equal(held, state)


def test_host_and_device_starts_and_layout_agree(flash):
    x = [t.cuda() for t in reference.operands(6, 1, 768, 1, 1, 32, 32)]
    starts = torch.tensor([0, 256, 768], dtype=torch.int32)
    a = flash.gated_delta_rule(*x, cu_seqlens=starts)
    assert torch.equal(a, flash.gated_delta_rule(*x, cu_seqlens=starts.cuda()))
    assert torch.equal(a, flash.gated_delta_rule(*x, layout=flash.VarlenLayout.from_cu_seqlens(starts, 768)))
    single = torch.cat([flash.gated_delta_rule(*[t[:, i:j].contiguous() for t in x]) for i, j in ((0, 256), (256, 768))], 1)
    assert torch.equal(a, single)


def test_directional_differences(flash):
    """The kernels' gradients against central differences of the 64-bit rule along random directions."""
    x = reference.operands(21, 1, 90, 1, 2, 32, 32)
    leaves = [t.cuda().requires_grad_() for t in x]
    g = torch.Generator().manual_seed(1)
    dout = torch.randn(1, 90, 2, 32, generator=g).bfloat16()
    grads = torch.autograd.grad(flash.gated_delta_rule(*leaves), leaves, dout.cuda())
    f = lambda y: (reference.sequences(*y, 32 ** -.5)[0] * dout.double()).sum().item()
    for index, grad in enumerate(grads):
        direction = torch.randn(x[index].shape, generator=g).double()
        step = 1e-5
        moved = lambda sign: [t.double() + (sign * step * direction if i == index else 0.) for i, t in enumerate(x)]
        slope = (f(moved(1)) - f(moved(-1))) / (2 * step)
        assert abs((grad.double().cpu() * direction).sum().item() - slope) <= GRAD * grad.double().norm().item() * direction.norm().item()


def test_strides_and_alignment(flash):
    """Views that are not contiguous, or contiguous at an address that is not a multiple of 16, give the bits of their copies."""
    x = reference.operands(8, 2, 70, 2, 4, 32, 64, device='cuda')
    want = flash.gated_delta_rule(*x)
    views = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in x]
    assert torch.equal(want, flash.gated_delta_rule(*views))
    shifted = []
    for t in x:
        room = torch.empty(t.numel() + 1, dtype=t.dtype, device='cuda')
        room[1:] = t.flatten()
        shifted.append(room[1:].view(t.shape))
    assert torch.equal(want, flash.gated_delta_rule(*shifted))


def test_another_stream_and_graph_replay(flash):
    x = reference.operands(9, 1, 200, 2, 2, 64, 64, device='cuda')
    starts = torch.tensor([0, 70, 200], dtype=torch.int32, device='cuda')
    dout = torch.randn_like(x[2])

    def step(leaves):
        out, final = flash.gated_delta_rule(*leaves, output_final_state=True, cu_seqlens=starts)
        return [out, final, *torch.autograd.grad(out, leaves, dout)]
    fresh = lambda: [t.clone().requires_grad_() for t in x]
    want = step(fresh())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaves = fresh()
        got = step(leaves)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(leaves)
    for other in ([0, 70, 200], [0, 1, 200]):  # the captured launches follow the lengths of the replay
        starts.copy_(torch.tensor(other, dtype=torch.int32))
        want = step(fresh())
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_a_captured_pack_outlives_others_and_a_first_upload_inside_a_capture_is_refused(flash):
    x = [t.cuda() for t in reference.operands(12, 1, 200, 2, 2, 64, 64)]
    starts = torch.tensor([0, 71, 200], dtype=torch.int32)
    want = flash.gated_delta_rule(*x, cu_seqlens=starts)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = flash.gated_delta_rule(*x, cu_seqlens=starts)
        with pytest.raises(RuntimeError, match='inside a capture'):
            flash.gated_delta_rule(*x, cu_seqlens=torch.tensor([0, 72, 200], dtype=torch.int32))
    for i in range(80, 120):
        flash.gated_delta_rule(*x, cu_seqlens=torch.tensor([0, i, 200], dtype=torch.int32))
    taken = [torch.full((64,), 5, dtype=torch.int32, device='cuda') for _ in range(200)]
    got.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and len(taken) == 200


@pytest.mark.parametrize('n,d', [(200, 64), (2100, 64), (130, 32)])
def test_a_graph_can_be_walked_twice(flash, n, d):
    """The kept states are read only: a second backward pass of one forward gives the same gradients, chains cut or not."""
    x = [t.cuda().requires_grad_() for t in reference.operands(13, 1, n, 1, 2, d, 64)]
    out, final = flash.gated_delta_rule(*x, output_final_state=True)
    dout, dfinal = torch.randn_like(out), torch.randn_like(final)
    first = torch.autograd.grad((out, final), x, (dout, dfinal), retain_graph=True)
    second = torch.autograd.grad((out, final), x, (dout, dfinal))
    assert all(torch.equal(a, b) for a, b in zip(first, second))


@pytest.mark.parametrize('batch,key_heads,heads,n,d,dv', [(150, 1, 2, 513, 64, 64), (75, 2, 2, 576, 128, 128), (298, 1, 2, 520, 64, 64), (100, 3, 3, 700, 128, 64), (149, 1, 1, 650, 64, 128)])
def test_chains_in_shares(flash, batch, key_heads, heads, n, d, dv):
    """More chains than fit at once are walked in equal shares: the same numbers as from parts of the batch, which fit; also captured, and
    from two streams at once."""
    room = 2 * torch.cuda.get_device_properties(0).multi_processor_count
    x = [t.cuda() for t in reference.operands(15, batch, n, key_heads, heads, d, dv)]
    s0 = torch.randn(batch, heads, d, dv, device='cuda')
    dout, dfinal = torch.randn_like(x[2]), torch.randn_like(s0)

    def step(part, states=True):
        leaves = [t[part].clone().requires_grad_() for t in (*x, s0)]
        out = flash.gated_delta_rule(*leaves[:5], initial_state=leaves[5], output_final_state=states)
        outs, grads = (out, (dout[part], dfinal[part])) if states else ((out,), (dout[part],))
        return [*outs, *torch.autograd.grad(outs, leaves, grads)]
    assert batch * heads * (dv // 64) > room or room != 296
    for states in (True, False):
        whole = step(slice(None), states)
        third = (batch + 2) // 3
        parts = [step(slice(i, i + third), states) for i in range(0, batch, third)]
        assert all(torch.equal(a, torch.cat(b)) for a, b in zip(whole, zip(*parts)))
        if states:
            assert torch.equal(whole[0], flash.gated_delta_rule(*x, initial_state=s0, output_final_state=True)[0])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for stream in streams:
        with torch.cuda.stream(stream):
            got.append(flash.gated_delta_rule(*x, initial_state=s0))
    torch.cuda.synchronize()
    want = flash.gated_delta_rule(*x, initial_state=s0)
    assert all(torch.equal(a, want) for a in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = flash.gated_delta_rule(*x, initial_state=s0)
    for _ in range(2):
        captured.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, want)


def test_two_calls_at_once(flash):
    """Two streams, each with its own call in flight many times over, do not disturb one another."""
    sets = [[t.cuda().requires_grad_() for t in reference.operands(s, 1, 500, 2, 2, 64, 64)] for s in (1, 2)]
    step = lambda x: [flash.gated_delta_rule(*x)] + list(torch.autograd.grad(flash.gated_delta_rule(*x).square().sum(), x))
    want = [step(x) for x in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for x, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                got.append(step(x))
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_no_positions(flash):
    x = [t.cuda().requires_grad_() for t in reference.operands(1, 2, 0, 1, 2, 32, 32)]
    initial = torch.randn(2, 2, 32, 32, device='cuda', requires_grad=True)
    out, final = flash.gated_delta_rule(*x, initial_state=initial, output_final_state=True)
    assert out.shape == (2, 0, 2, 32) and torch.equal(final, initial)
    assert torch.equal(torch.autograd.grad(final.sum(), initial)[0], torch.ones_like(initial))


def test_long_sequence_keeps_its_state(flash):
    """16384 positions with slow decays: the state's error does not pile up."""
    torch.manual_seed(0)
    b, n, h, d = 1, 16384, 1, 64
    x = [t.cuda() for t in reference.operands(2, b, n, h, h, d, d, torch.float32, decay=.002)]
    out, final = flash.gated_delta_rule(*x, output_final_state=True)
    q, k, v, g, beta = (t.double() for t in x)
    s, rows = torch.zeros(h, d, d, dtype=torch.float64, device='cuda'), []
    for t in range(n):
        s = torch.exp(g[0, t])[:, None, None] * s
        u = beta[0, t][:, None] * (v[0, t] - torch.einsum('hij,hi->hj', s, k[0, t]))
        s = s + k[0, t][:, :, None] * u[:, None]
        rows.append(torch.einsum('hij,hi->hj', s, q[0, t]) * d ** -.5)
    near(out, torch.stack(rows)[None], OUT, 2)
    near(final, s[None], STATE, 1)


# ---- single tokens ---------------------------------------------------------------------------------
# In 32 bits: D products and additions in a sum, one rounding each: (D + 8) * 2^-24 of the norm; the output is rounded to bf16 besides.
@pytest.mark.parametrize('gates', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('batch,key_heads,heads,d,dv', [(1, 1, 1, 128, 128), (3, 2, 4, 64, 32), (5, 1, 3, 32, 64), (130, 1, 1, 32, 32)])
def test_single_tokens(flash, gates, batch, key_heads, heads, d, dv):
    state = .5 * torch.randn(batch, heads, d, dv, generator=torch.Generator().manual_seed(batch))
    exact, held = state.double(), state.cuda()
    for token in range(3):
        x = reference.operands(100 + token, batch, 1, key_heads, heads, d, dv, gates)
        want, exact = reference.sequences(*[t.double() for t in x], d ** -.5, exact)
        out = flash.gated_delta_step(*[t[:, 0].cuda() for t in x], held)
        near(out, want[:, 0], 2 ** -8 + (d + 8) * 2 ** -24, 1)
        near(held, exact, 3 * (d + 8) * 2 ** -24, 1)


def test_slots_padding_and_repeats(flash):
    """Rows name their states in any order; rows outside the pool are padding; a slot named twice takes its rows in order."""
    rows, pool, heads, d, dv = 150, 40, 2, 32, 64
    g = torch.Generator().manual_seed(4)
    slots = torch.full((rows,), -1, dtype=torch.int32)
    named = torch.randperm(pool, generator=g)[:30].to(torch.int32)
    slots[torch.randperm(rows, generator=g)[:30]] = named
    free = (slots < 0).nonzero().flatten()
    slots[free[0]], slots[free[1]], slots[free[2]] = named[3], named[3], named[7]
    slots[free[3]], slots[free[4]] = pool, 2 ** 31 - 1
    x = reference.operands(4, rows, 1, 1, heads, d, dv)
    state = torch.randn(pool, heads, d, dv, generator=g)
    exact, want = state.double(), torch.zeros(rows, heads, dv, dtype=torch.float64)
    for row in range(rows):
        if 0 <= slots[row] < pool:
            o, s = reference.sequences(*[t[row:row + 1].double() for t in x], d ** -.5, exact[slots[row]][None])
            exact[slots[row]], want[row] = s[0], o[0, 0]
    held = state.cuda()
    out = flash.gated_delta_step(*[t[:, 0].cuda() for t in x], held, slots=slots.cuda())
    near(out, want, 2 ** -8 + (d + 8) * 2 ** -24, 1)
    near(held, exact, 2 * (d + 8) * 2 ** -24, 1)
    untouched = torch.tensor([i for i in range(pool) if i not in set(slots.tolist())])
    assert torch.equal(held.cpu()[untouched], state[untouched])
    assert not out[(slots < 0).cuda()].count_nonzero()


def test_prompt_then_tokens(flash):
    """A ragged batch of prompts, their states scattered into a pool, then tokens one at a time, replayed from a graph: the
    outputs are those of the whole sequences at once."""
    heads, d, dv, more = 2, 64, 64, 5
    lengths = [3, 64, 100]
    whole = [reference.operands(30 + i, 1, m + more, 1, heads, d, dv) for i, m in enumerate(lengths)]
    prompts = [torch.cat([w[j][:, :m] for w, m in zip(whole, lengths)], 1).cuda() for j in range(5)]
    starts = torch.tensor([0, 3, 67, 167], dtype=torch.int32, device='cuda')
    _, states = flash.gated_delta_rule(*prompts, cu_seqlens=starts, output_final_state=True)
    pool, slots = torch.zeros(6, heads, d, dv, device='cuda'), torch.tensor([4, 0, 2], dtype=torch.int32, device='cuda')
    pool[slots.long()] = states
    tokens = [torch.cat([w[j][:, m] for w, m in zip(whole, lengths)]).cuda() for j in range(5)]
    keep = pool.clone()
    flash.gated_delta_step(*tokens, pool, slots=slots)
    pool.copy_(keep)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = flash.gated_delta_step(*tokens, pool, slots=slots)
    for step in range(more):
        for j in range(5):
            tokens[j].copy_(torch.cat([w[j][:, m + step] for w, m in zip(whole, lengths)]))
        graph.replay()
        for i, (w, m) in enumerate(zip(whole, lengths)):
            want, _ = reference.sequences(*[t[:, :m + step + 1].double() for t in w], d ** -.5)
            near(out[i][None], want[:, -1], 2 * 2 ** -8, 1)


def test_refusals_on_the_device(flash):
    import cu_flash_dism as cu
    x = [t.cuda() for t in reference.operands(1, 2, 8, 2, 4, 32, 32)]
    with pytest.raises(RuntimeError, match='multiple of the key heads'):
        flash.gated_delta_rule(x[0], x[1], x[2][:, :, :3].contiguous(), x[3][..., :3].contiguous(), x[4][..., :3].contiguous())
    with pytest.raises(RuntimeError, match='unsupported'):
        flash.gated_delta_rule(x[0][..., :16], x[1][..., :16], *x[2:])
    with pytest.raises(RuntimeError, match='device, dtype'):
        flash.gated_delta_rule(x[0].float(), *x[1:])
    with pytest.raises(RuntimeError, match='k: '):
        flash.gated_delta_rule(x[0], x[1][:, :7], *x[2:])
    with pytest.raises(RuntimeError, match='one batch row'):
        flash.gated_delta_rule(*x, cu_seqlens=torch.tensor([0, 8], dtype=torch.int32, device='cuda'))
    with pytest.raises(RuntimeError, match='initial state'):
        flash.gated_delta_rule(*x, initial_state=torch.zeros(1, 4, 32, 32, device='cuda'))
    single = [t[:1] for t in x]
    for bad in ([0, 5, 3, 8], [1, 8], [0, 7]):
        with pytest.raises(RuntimeError, match='invalid cu_seqlens'):
            flash.gated_delta_rule(*single, cu_seqlens=torch.tensor(bad, dtype=torch.int32))
    token = [t[:, 0].contiguous() for t in x]
    with pytest.raises(RuntimeError, match='state of its own'):
        flash.gated_delta_step(*token, torch.zeros(3, 4, 32, 32, device='cuda'))
    with pytest.raises(RuntimeError, match='slots'):
        flash.gated_delta_step(*token, torch.zeros(3, 4, 32, 32, device='cuda'), slots=torch.zeros(2, dtype=torch.int64, device='cuda'))
    with pytest.raises(RuntimeError, match='state'):
        flash.gated_delta_step(*token, torch.zeros(2, 4, 32, 32, device='cuda').bfloat16())
    with pytest.raises(RuntimeError, match='state'):
        flash.gated_delta_step(*token, torch.zeros(2, 4, 32, 64, device='cuda')[..., ::2])
    leaf = x[1].clone().requires_grad_()
    out = flash.gated_delta_rule(x[0], leaf, *x[2:])
    with torch.no_grad():
        leaf.mul_(2)
    with pytest.raises(RuntimeError, match='modified by an inplace'):
        out.sum().backward()
    assert cu.delta_step(token, 1., torch.zeros(2, 4, 32, 32, device='cuda')).shape == token[2].shape
