"""Host side of the gated delta rule and of dropout that needs no device: what is kept from call to call, models and their states."""
import delta_chunked as chunked


def test_chunked_form_of_the_tests():
    chunked.check_chunked_form()
