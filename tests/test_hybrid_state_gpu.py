"""Residual dropout of the hybrid model across checkpoints and data-parallel ranks."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def make():
    import dism_b200
    dism_b200.install_dropin()
    from dism_b200.model import DismLM
    return lambda **more: DismLM(depth=2, width=128, heads=1, head_dim=128, vocab=128, delta_layers=(0, 1), dropout=.2, **more).cuda().bfloat16()


def test_a_resumed_model_draws_the_masks_of_the_first(make):
    torch.manual_seed(1)
    model = make()
    tokens = torch.randint(0, 128, (2, 100), device='cuda')
    model.dropout_seed[1] += 3
    kept = {k: t.clone() for k, t in model.state_dict().items()}
    want = model(tokens)
    other = make()
    other.load_state_dict(kept)
    assert torch.equal(other(tokens), want)


def test_ranks_draw_different_masks_from_one_seed(make):
    """Data-parallel replicas share their buffers; the rank is an attribute of the replica."""
    torch.manual_seed(2)
    models = [make(dropout_rank=rank) for rank in range(3)]
    for model in models[1:]:
        model.load_state_dict(models[0].state_dict())
    tokens = torch.randint(0, 128, (2, 100), device='cuda')
    outs = [model(tokens) for model in models]
    assert not any(torch.equal(outs[i], outs[j]) for i in range(3) for j in range(i))
    models[1].dropout_rank = 0
    assert torch.equal(models[1](tokens), outs[0])
    for model in models:
        model.eval()
    assert torch.equal(models[0](tokens), models[2](tokens))
