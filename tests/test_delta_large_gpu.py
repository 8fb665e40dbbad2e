"""Tensors of more than 2^31 elements: the far end gives the bits of a call of its own."""
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


@pytest.fixture(autouse=True)
def room():
    if torch.cuda.mem_get_info()[0] < 70 << 30:
        pytest.skip('needs 70 GB')
    yield
    torch.cuda.empty_cache()


def test_training_far_into_a_batch(flash):
    b, n, heads, d, dv = 1100, 1024, 16, 64, 128
    assert b * n * heads * dv > 2 ** 31
    few = reference.operands(1, 2, n, 1, heads, d, dv, device='cuda')
    x = [t[:1].expand(b, *t.shape[1:]).contiguous() for t in few]
    for t, part in zip(x, few):
        t[-1] = part[1]
    leaves = [t.requires_grad_() for t in x]
    out = flash.gated_delta_rule(*leaves)
    dout = torch.empty_like(out).normal_(generator=torch.Generator(device='cuda').manual_seed(3))
    grads = torch.autograd.grad(out, leaves, dout)
    for row in (0, b - 1):
        alone = [t.detach()[row:row + 1].clone().requires_grad_() for t in x]
        want = flash.gated_delta_rule(*alone)
        assert torch.equal(out[row:row + 1], want)
        for got, expected in zip(grads, torch.autograd.grad(want, alone, dout[row:row + 1].clone())):
            assert torch.equal(got[row:row + 1], expected)


def test_one_long_pack(flash):
    """A single row of 1.1 million positions: its last document."""
    n, heads, d, dv = 1_100_000, 16, 64, 128
    part = 5000
    last = reference.operands(2, 1, part, 1, heads, d, dv, device='cuda')
    x = [torch.zeros(1, n, *t.shape[2:], dtype=t.dtype, device='cuda') for t in last]
    for t, p in zip(x, last):
        t[:, -part:] = p
    starts = torch.tensor([0, 70, n - part, n], dtype=torch.int32, device='cuda')
    out, states = flash.gated_delta_rule(*x, cu_seqlens=starts, output_final_state=True)
    want, state = flash.gated_delta_rule(*last, output_final_state=True)
    near = lambda a, b, bound: (a.double() - b.double()).norm() <= bound * b.double().norm()
    assert near(out[:, -part:], want, 2 ** -7) and near(states[2], state[0], 2 ** -14)  # cut elsewhere, hence not the same bits
    assert not out[:, :-part].count_nonzero()


def test_slots_far_into_a_pool(flash):
    pool, heads, d, dv = 140_000, 1, 128, 128
    x = [t[:, 0] for t in reference.operands(4, 3, 1, 1, heads, d, dv, device='cuda')]
    small = torch.randn(3, heads, d, dv, generator=torch.Generator(device='cuda').manual_seed(1), device='cuda')
    slots = torch.tensor([pool - 1, 131_072, 0], dtype=torch.int32, device='cuda')
    big = torch.zeros(pool, heads, d, dv, device='cuda')
    assert big.numel() > 2 ** 31
    big[slots.long()] = small
    out = flash.gated_delta_step(*x, big, slots=slots)
    assert torch.equal(out, flash.gated_delta_step(*x, small)) and torch.equal(big[slots.long()], small)
    assert not big[1:1000].count_nonzero() and not big[-1000:-1].count_nonzero()


def test_dropout_of_a_large_tensor(flash):
    """The mask's far end, which is that of the same elements' blocks in the generator's counter."""
    import numpy as np
    count, tail = 2 ** 31 + 4099, 5003
    x = torch.ones(count, dtype=torch.bfloat16, device='cuda')
    seed = torch.tensor([5, 6], device='cuda')
    y = flash.dropout_add(x, None, .5, seed, site=2)[-tail:].cpu()
    first = (count - tail) // 8
    blocks = np.arange(first, (count + 7) // 8, dtype=np.uint64)
    word, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = [blocks & word, np.full_like(blocks, 2), np.full_like(blocks, 6), np.zeros_like(blocks)]
    for turn in range(10):
        k0, k1 = (np.uint64((k + turn * w) & 0xFFFFFFFF) for k, w in ((5, 0x9E3779B9), (0, 0xBB67AE85)))
        p, r = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(r >> shift) ^ c[1] ^ k0, r & word, (p >> shift) ^ c[3] ^ k1, p & word]
    numbers = np.stack(c, 1).astype(np.uint32).view(np.uint16).reshape(-1)[count - tail - 8 * first:][:tail]
    assert torch.equal(y != 0, torch.from_numpy(numbers.astype(np.int64) >= 32768))
