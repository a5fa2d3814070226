"""Requests past what the paged cache's and the logits' kernels count in are refused before any launch, on a host without a GPU."""

import pytest

from chunkkv_amd import _native
from tests.test_paged_host import ADJUST, NEXT, _with

MOST = 2**31 - 1


@pytest.mark.parametrize("fn,base", [("ckv_adjust_logits", ADJUST), ("ckv_next_tokens", NEXT)])
def test_two_histories_of_the_most_tokens(fn, base):
    """The kernel walks the pairs of both lists, 2048 at a time, with 32-bit numbers: from 2^31 - 2048 pairs on it would pass them and never end."""
    call = getattr(_native.lib(), fn)
    for n, m in ((MOST, MOST), (MOST - 1, MOST), (MOST - 2, MOST - 2), (MOST - 4092, MOST), (MOST, MOST - 4092)):
        assert n // 2 + m // 2 > MOST - 2048
        assert call(*_with(base, np=n, p_row=n, ng=m, g_row=m)) == _native.CKV_ERR_TOO_LARGE, (n, m)
    # the lists alone may be as long: what is refused then is something else
    assert call(*_with(base, np=MOST, p_row=MOST, ng=3, logits=None)) == _native.CKV_ERR_INVALID_ARGUMENT
    assert call(*_with(base, np=MOST, p_row=MOST, ng=0, row=99)) == _native.CKV_ERR_OUT_OF_RANGE
