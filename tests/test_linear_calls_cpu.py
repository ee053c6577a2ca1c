"""CPU: the dense-layer entries' refusals and bookkeeping that need no device."""
import pytest

from recflex_b200 import _lib

P = 1 << 20  # an aligned address that no refused call looks at


@pytest.mark.parametrize("status, device", [(P + 2, 0), (P, -1), (P, 64)])
def test_check_status_refuses(lib, status, device):
    assert lib.eb_linear_check_status(status, device, None) == _lib.EB_ERR_INVALID_ARG
