"""A call whose query rows per K/V head (queries x heads of a group) pass 31 bits is refused before any CUDA call: the kernels count them in 32."""
import ctypes

import pytest

import gpt2_b200 as G
from test_kv8_abi import cache


@pytest.mark.parametrize("Hq,Tq", [(8, 2 ** 31 - 1), (4 * 2 ** 20, 2 ** 12), (4, 2 ** 31 - 1)])
def test_more_query_rows_than_31_bits(lib, Hq, Tq):
    c = cache()
    c.work_bytes = 1 << 50
    assert lib.gpt2_kv8_attend_b200(16, 2 ** 40, 8, 16, 2 ** 40, 8, ctypes.byref(c), 0, Hq, Tq, None, None, 0, 0, None) == G.EINVAL
