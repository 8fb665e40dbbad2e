"""The hybrid model: gated delta layers beside DISM layers, residual dropout, prompts and single tokens, all together."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def model_class():
    import dism_b200
    dism_b200.install_dropin()
    from dism_b200.model import DismLM
    return DismLM


def test_hybrid_step_trains_every_delta_parameter(model_class):
    torch.manual_seed(5)
    model = model_class(depth=3, width=256, heads=2, head_dim=128, vocab=512, delta_layers=(0, 2), dropout=.1).cuda().bfloat16()
    model.dropout_seed = torch.tensor([11, 0], device='cuda')
    tokens = torch.randint(0, 512, (2, 256), device='cuda')
    loss = model(tokens, tokens.roll(-1, 1))
    loss.backward()
    assert torch.isfinite(loss)
    for index in (0, 2):
        for name, parameter in model.blocks[index].mixer.named_parameters():
            assert parameter.grad is not None and torch.isfinite(parameter.grad).all() and parameter.grad.count_nonzero(), (index, name)
    again = model(tokens, tokens.roll(-1, 1))
    assert torch.equal(loss, again)  # the same offset draws the same masks
    model.dropout_seed[1] += 1
    assert not torch.equal(loss, model(tokens, tokens.roll(-1, 1)))
    model.eval()
    quiet = model(tokens, tokens.roll(-1, 1))
    model.dropout_seed[1] += 1
    assert torch.equal(quiet, model(tokens, tokens.roll(-1, 1)))


def test_a_captured_step_draws_new_masks(model_class):
    torch.manual_seed(6)
    model = model_class(depth=2, width=128, heads=1, head_dim=128, vocab=256, delta_layers=(0, 1), dropout=.2).cuda().bfloat16()
    model.dropout_seed = torch.tensor([3, 0], device='cuda')
    tokens = torch.randint(0, 256, (2, 300), device='cuda')
    parameters = list(model.parameters())

    def step():
        loss = model(tokens, tokens.roll(-1, 1))
        grads = torch.autograd.grad(loss, parameters)
        model.dropout_seed[1] += 1
        return loss.detach(), grads
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = [step() for _ in range(4)][2:]
        model.dropout_seed[1] -= 2
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grads = step()
    for want, want_grads in eager:
        graph.replay()
        torch.cuda.synchronize()
        # the operators are the same bits; torch's own embedding gradient adds in no fixed order
        assert torch.equal(loss, want)
        for got, expected in zip(grads[1:], want_grads[1:]):
            assert torch.equal(got, expected)


def test_prompts_and_tokens_agree_with_whole_sequences(model_class):
    """prefill + step give the logits of the forward pass over the whole sequence, to the bf16 rounding of the layers between: each of the
    two blocks adds a handful of roundings of 2^-8 to activations of order one, on both sides."""
    torch.manual_seed(7)
    model = model_class(depth=2, width=128, heads=2, head_dim=64, vocab=128, delta_layers=(0, 1)).cuda().bfloat16().eval()
    tokens = torch.randint(0, 128, (3, 70), device='cuda')
    with torch.no_grad():
        whole = model(tokens).double()
    logits, states = model.prefill(tokens[:, :65])
    scale = whole.square().mean().sqrt()
    bound = 24 * 2 ** -8
    assert (logits.double() - whole[:, 64]).square().mean().sqrt() <= bound * scale
    pools = [torch.zeros(5, *s.shape[1:], device='cuda') for s in states]
    slots = torch.tensor([4, 1, 2], dtype=torch.int32, device='cuda')
    for pool, state in zip(pools, states):
        pool[slots.long()] = state
    for t in range(65, 70):
        logits = model.step(tokens[:, t], pools, slots)
        assert (logits.double() - whole[:, t]).square().mean().sqrt() <= bound * scale


def test_a_model_with_dism_layers_does_not_step(model_class):
    model = model_class(depth=2, width=128, heads=2, head_dim=64, vocab=128, delta_layers=(1,)).cuda().bfloat16()
    with pytest.raises(NotImplementedError, match='DISM layers'):
        model.prefill(torch.zeros(1, 4, dtype=torch.long, device='cuda'))
