"""Waits of the gated delta rule's kernels that run out: with a limit of no polls every wait does, although what it waits for arrives.  Outputs
that depend on them are NaN, the others are right, the code is reported, and the next call works."""
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


@pytest.fixture
def no_patience():
    """Sets the limit to nothing for the calls inside."""
    import contextlib
    import cu_flash_dism as cu
    from dism_b200 import _lib
    lib = _lib.load()

    @contextlib.contextmanager
    def limited():
        torch.cuda.synchronize()
        assert cu.delta_fault() == 0
        _lib.check(lib.dism_delta_wait_limit(0))
        try:
            yield
            torch.cuda.synchronize()
        finally:
            _lib.check(lib.dism_delta_wait_limit(-1))
    yield limited
    cu.delta_fault()


@pytest.mark.parametrize('b,n,key_heads,heads,d,dv', [(1, 64, 1, 1, 64, 64), (2, 200, 1, 2, 128, 128), (1, 1000, 2, 2, 64, 128), (8, 1500, 1, 2, 64, 64)])
def test_gradient_kernel_without_its_waits(flash, no_patience, b, n, key_heads, heads, d, dv):
    import cu_flash_dism as cu
    x = reference.operands(3, b, n, key_heads, heads, d, dv, device='cuda')
    dout = torch.randn_like(x[2])
    leaves = [t.requires_grad_() for t in x]
    want = flash.gated_delta_rule(*leaves)
    grads = torch.autograd.grad(want, leaves, dout)
    with no_patience():
        out = flash.gated_delta_rule(*leaves)
        lost = torch.autograd.grad(out, leaves, dout)
    assert 1 <= cu.delta_fault() <= 11 and cu.delta_fault() == 0
    assert torch.equal(out, want) and torch.equal(lost[2], grads[2])  # neither comes from the kernel that waits
    for index in (0, 1, 3, 4):
        assert lost[index].isnan().all(), index
    again = flash.gated_delta_rule(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(again, leaves, dout), grads)) and cu.delta_fault() == 0


def test_shares_without_their_waits(flash, no_patience):
    """Chains cut between two places: what the second place was to walk from the first one's state is NaN, all else as it should be."""
    import cu_flash_dism as cu
    room = 2 * torch.cuda.get_device_properties(0).multi_processor_count
    chains, chunks, n = room + 4, 9, 9 * 64 - 5
    x = reference.operands(4, chains // 2, n, 1, 2, 64, 64, device='cuda')
    dout = torch.randn_like(x[2])
    leaves = [t.requires_grad_() for t in x]
    with torch.no_grad():
        want, final = flash.gated_delta_rule(*leaves, output_final_state=True)
    grads = torch.autograd.grad(flash.gated_delta_rule(*leaves), leaves, dout)
    length = -(-chains * chunks // room)
    late = torch.zeros(chains, n, dtype=torch.bool)    # positions behind a cut, in the forward's walking order
    early = torch.zeros(chains, n, dtype=torch.bool)   # and before one, in the reverse's
    for place in range(1, -(-chains * chunks // length)):
        chain, first = divmod(place * length, chunks)
        if first:
            late[chain, first * 64:] = True
            early[chain, :(chunks - first) * 64] = True
    split = lambda t: t.view(chains // 2, 2, n).transpose(1, 2).cuda()
    assert late.any() and not late.all(1).any()
    with torch.no_grad(), no_patience():
        out, state = flash.gated_delta_rule(*leaves, output_final_state=True)
    assert cu.delta_fault() == 12 and cu.delta_fault() == 0
    lost = split(late)
    assert out[lost].isnan().all() and torch.equal(out[~lost], want[~lost])
    ended = lost[:, -1]
    assert state[ended].isnan().all() and torch.equal(state[~ended], final[~ended])
    kept = flash.gated_delta_rule(*leaves)
    with no_patience():
        dv = torch.autograd.grad(kept, leaves, dout)[2]
    assert cu.delta_fault() == 13 and cu.delta_fault() == 0
    lost = split(early)
    assert dv[lost].isnan().all() and torch.equal(dv[~lost], grads[2][~lost])
    kept = flash.gated_delta_rule(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(kept, leaves, dout), grads)) and cu.delta_fault() == 0


def test_the_fault_word_is_read_behind_all_streams(flash, no_patience):
    """A fault of a call that is still queued on a side stream is not missed."""
    import cu_flash_dism as cu
    x = reference.operands(5, 1, 64, 1, 1, 64, 64, device='cuda')
    leaves = [t.requires_grad_() for t in x]
    side = torch.cuda.Stream()
    with no_patience():
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            out = flash.gated_delta_rule(*leaves)
            torch.cuda._sleep(100_000_000)
            torch.autograd.grad(out, leaves, torch.ones_like(out))
        code = cu.delta_fault()
    assert 1 <= code <= 11
