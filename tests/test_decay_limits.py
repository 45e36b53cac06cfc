"""Sizes at the ends of the decay operators' ranges, by status code at the C ABI; nothing is launched."""
import pytest

from rocm_flashinfer_contest_b200 import _lib
from test_decay_abi import PREFILL, call

UNS = _lib.GDN_ERR_UNSUPPORTED


@pytest.mark.parametrize("N,T,HV", [(2 ** 31 - 1, 256, 1), (2 ** 31 - 1, 2 ** 31 - 1, 1), (2 ** 31 - 2, 512, 1),
                                    (2 ** 31 - 1, 0, 2 ** 31 - 1), (2 ** 26, 1, 1)])
def test_prefill_refuses_more_sequences_than_a_grid_has(N, T, HV):
    """The number of segments, T / 256 + N, does not fit 32 bits here; it was taken for a negative, small one."""
    assert call("gdn_decay_prefill_fwd", PREFILL, dict(N=N, T=T, H=1, HV=HV, ws=64, wsb=2 ** 40)) == UNS
