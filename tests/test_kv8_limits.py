"""What the 8-bit KV cache refuses at the ends of its ranges, without a GPU."""
import ctypes as C

import pytest

from hllm_b200 import _lib
from tests.test_kv8 import attention_args, cache


@pytest.mark.parametrize("max_blocks", [(2 ** 31 - 4097) // 16 + 1, (2 ** 31 - 1) // 16])
def test_rows_whose_tiles_would_pass_32_bits_are_refused(max_blocks):
    """The last tile of such a row ends past 2^31 - 1, where its key numbers turn negative."""
    call = _lib.lib().hllm_b200_kv8_attention
    assert call(C.byref(cache()), *attention_args(max_blocks=max_blocks)) == _lib.INVALID_REQUEST
    assert "max_blocks" in _lib.last_error()
