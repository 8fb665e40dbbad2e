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
