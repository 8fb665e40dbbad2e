"""Counter-based dropout against the generator in numpy: the mask bit for bit, values to the roundings they go through
(x * scale and the addition in 32 bits: 2 * 2^-24 of the terms; the result's own type: half a step)."""
import numpy as np
import pytest
import torch

import delta_reference as reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def flash():
    import dism_b200
    dism_b200.install_dropin()
    import flash_dism
    return flash_dism


def expected(x, residual, p, seed, site):
    threshold = round(65536 * p)
    keep = torch.from_numpy((reference.philox(x.numel(), *[int(s) for s in seed], site).astype(np.int64) >= threshold)).view(x.shape)
    y = torch.where(keep, x.double().cpu() * (65536 / (65536 - threshold) if threshold < 65536 else 0.), 0.)
    return (y if residual is None else y + residual.double().cpu()), keep


@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('count', [1, 7, 8, 9, 2047, 2048, 4103])
@pytest.mark.parametrize('p', [0., .1, .5, 1.])
def test_values_mask_and_gradients(flash, dtype, count, p):
    g = torch.Generator().manual_seed(count)
    x, residual, dy = (torch.randn(count, generator=g).to(dtype).cuda() for _ in range(3))
    seed = torch.tensor([-(1 << 62) + 12345, (7 << 32) + 3], device='cuda')
    half = torch.finfo(dtype).eps / 2
    for other in (None, residual):
        leaves = [t.clone().requires_grad_() for t in ((x,) if other is None else (x, other))]
        y = flash.dropout_add(leaves[0], None if other is None else leaves[1], p, seed, site=5)
        want, keep = expected(x, other, p, seed, 5)
        assert y.dtype == dtype
        terms = x.double().cpu().abs() * 2 + (0 if other is None else other.double().cpu().abs())
        assert ((y.detach().double().cpu() - want).abs() <= half * want.abs() + 2 * 2 ** -24 * terms).all()
        grads = torch.autograd.grad(y, leaves, dy)
        dx, _ = expected(dy, None, p, seed, 5)
        assert ((grads[0].double().cpu() - dx).abs() <= (half + 2 ** -23) * dx.abs()).all()
        assert torch.equal(grads[0].cpu() != 0, keep & (dy.cpu() != 0))
        if other is not None:
            assert torch.equal(grads[1], dy)


def test_share_of_kept_elements_sites_and_offsets(flash):
    """Shares within five standard deviations; different sites, offsets and keys draw different masks."""
    n = 1 << 20
    x = torch.ones(n, device='cuda')
    seed = torch.tensor([17, 0], device='cuda')
    masks = []
    for key, offset, site in ((17, 0, 0), (17, 0, 1), (17, 1, 0), (18, 0, 0)):
        seed.copy_(torch.tensor([key, offset]))
        y = flash.dropout_add(x, None, .25, seed, site=site)
        kept = (y != 0).double().mean().item()
        assert abs(kept - .75) <= 5 * (.75 * .25 / n) ** .5
        assert abs(y.double().mean().item() - 1) <= 5 * (.25 / .75 / n) ** .5
        masks.append(y != 0)
    for i in range(len(masks)):
        for j in range(i):
            both = (masks[i] & masks[j]).double().mean().item()
            assert abs(both - .75 ** 2) <= 5 * (.75 ** 2 * (1 - .75 ** 2) / n) ** .5


def test_alignment_and_strides_do_not_change_the_mask(flash):
    seed = torch.tensor([3, 9], device='cuda')
    x = torch.randn(33, 65, device='cuda').bfloat16()
    want = flash.dropout_add(x, x, .3, seed)
    room = torch.empty(33 * 65 + 1, dtype=torch.bfloat16, device='cuda')
    room[1:] = x.flatten()
    assert torch.equal(want, flash.dropout_add(room[1:].view(33, 65), x, .3, seed))
    assert torch.equal(want, flash.dropout_add(x.t().contiguous().t(), x, .3, seed))
    leaf = x.clone().requires_grad_()
    y = flash.dropout_add(leaf, None, .3, seed)
    a, = torch.autograd.grad(y, leaf, torch.ones_like(y), retain_graph=True)
    b, = torch.autograd.grad(y, leaf, torch.ones((), device='cuda', dtype=torch.bfloat16).expand(33, 65))
    assert torch.equal(a, b)


def test_graph_replay_follows_the_offset(flash):
    seed = torch.tensor([3, 0], device='cuda')
    x = torch.randn(5000, device='cuda').requires_grad_()
    dy = torch.randn(5000, device='cuda')
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(flash.dropout_add(x, x.detach(), .5, seed), x, dy)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = flash.dropout_add(x, x.detach(), .5, seed)
        dx, = torch.autograd.grad(y, x, dy)
        seed[1] += 1
    for offset in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert seed[1].item() == offset + 1
        _, keep = expected(x, None, .5, [3, offset], 0)
        assert torch.equal(dx.cpu() != 0, keep)
        assert torch.equal((y != x).cpu(), keep | (x.detach().cpu() != 0)) or torch.equal((y - x.detach() != 0).cpu(), keep)


def test_changed_seed_and_refusals(flash):
    seed = torch.tensor([1, 2], device='cuda')
    x = torch.randn(16, device='cuda', requires_grad=True)
    y = flash.dropout_add(x, None, .5, seed)
    seed[1] += 1
    with pytest.raises(RuntimeError, match='modified by an inplace'):
        y.sum().backward()
    with pytest.raises(RuntimeError, match='residual'):
        flash.dropout_add(x, x[:8], .5, seed)
    with pytest.raises(RuntimeError, match='residual'):
        flash.dropout_add(x, x.half(), .5, seed)
    with pytest.raises(RuntimeError, match='seed'):
        flash.dropout_add(x, None, .5, seed.int())
    with pytest.raises(RuntimeError, match='seed'):
        flash.dropout_add(x, None, .5, seed.cpu())
    with pytest.raises(RuntimeError, match='site'):
        flash.dropout_add(x, None, .5, seed, site=-1)
    with pytest.raises(ValueError, match='probability'):
        flash.dropout_add(x, None, 1.5, seed)
    with pytest.raises(RuntimeError, match='float32, float16 or bfloat16'):
        flash.dropout_add(x.double(), None, .5, seed)
    assert flash.dropout_add(x[:0], None, .5, seed).shape == (0,)
