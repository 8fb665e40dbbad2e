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
