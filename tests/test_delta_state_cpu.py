"""Host side of the gated delta rule and of dropout that needs no device: what is kept from call to call, models and their states."""
import delta_chunked as chunked


def test_chunked_form_of_the_tests():
    chunked.check_chunked_form()


def test_wait_limit_arguments():
    from dism_b200 import _lib, build
    build.build()
    lib = _lib.load()
    assert lib.dism_abi_version() >= 11
    assert lib.dism_delta_wait_limit(1 << 17) == 1 and b'tries' in lib.dism_last_error()
    assert lib.dism_delta_wait_limit(5) == 0 and lib.dism_delta_wait_limit(-1) == 0


def test_starts_first_uploaded_in_inference_mode_serve_a_training_call():
    """An inference tensor cannot be saved for a backward pass."""
    import dism_b200
    import torch
    dism_b200.install_dropin()
    from flash_dism import delta
    with torch.inference_mode():
        first = delta._host_starts([0, 21, 64], torch.device('cpu'))
    assert not first.is_inference() and delta._host_starts([0, 21, 64], torch.device('cpu')) is first


def test_delta_layers_from_an_iterator_and_outside_the_model():
    import pytest
    import torch
    from dism_b200.model import DeltaLayer, DismLM
    make = lambda layers: DismLM(depth=4, width=64, heads=2, head_dim=32, vocab=64, delta_layers=layers)
    with torch.device('meta'):
        for layers in ((1, 3), (i for i in (1, 3)), range(1, 4, 2), {3, 1}):
            assert [type(b.mixer) is DeltaLayer for b in make(layers).blocks] == [False, True, False, True]
        for layers in ((4,), (-1,), (0, 9)):
            with pytest.raises(ValueError, match='delta_layers'):
                make(layers)
        with pytest.raises(TypeError):
            make((1.5,))


def test_states_have_to_be_one_per_block():
    import pytest
    import torch
    from dism_b200.model import DismLM
    model = DismLM(depth=3, width=64, heads=2, head_dim=32, vocab=64, delta_layers=range(3))
    states = [torch.zeros(1, 2, 32, 32) for _ in range(4)]
    for some in (states[:2], states, []):
        with pytest.raises(ValueError, match='one state per block'):
            model.step(torch.zeros(1, dtype=torch.long), some)
        with pytest.raises(ValueError, match='one state per block'):
            model.prefill(torch.zeros(1, 4, dtype=torch.long), some)


def test_checkpoints_hold_the_masks_key_and_offset():
    import torch
    from dism_b200.model import DismLM
    make = lambda p: DismLM(depth=1, width=64, heads=2, head_dim=32, vocab=64, delta_layers=(0,), dropout=p)
    trained, resumed = make(.1), make(.1)
    trained.dropout_seed[1] += 7
    assert not torch.equal(trained.dropout_seed, resumed.dropout_seed)
    resumed.load_state_dict(trained.state_dict())
    assert torch.equal(trained.dropout_seed, resumed.dropout_seed) and resumed.dropout_seed.dtype == torch.int64
    assert torch.equal(trained.bfloat16().dropout_seed, resumed.dropout_seed)
    # with and without dropout, either way round: the weights are the same model's
    quiet = make(0.)
    quiet.load_state_dict(trained.state_dict())
    other = make(.2)
    before = other.dropout_seed.clone()
    other.load_state_dict(quiet.state_dict())
    assert torch.equal(other.dropout_seed, before) and 'dropout_seed' not in quiet.state_dict()
    holder = torch.nn.ModuleDict(dict(m=make(0.)))
    holder.load_state_dict({f'm.{k}': t for k, t in trained.state_dict().items()})


def test_a_refused_step_leaves_the_states_version():
    """A graph that has saved the state may still be walked."""
    import dism_b200
    import pytest
    import torch
    dism_b200.install_dropin()
    import flash_dism
    q, gates, state = torch.zeros(1, 2, 32, dtype=torch.bfloat16), torch.zeros(1, 2), torch.zeros(1, 2, 32, 32)
    before = state._version
    with pytest.raises(RuntimeError, match='invalid device'):
        flash_dism.gated_delta_step(q, q, q, gates, gates, state)
    assert state._version == before
