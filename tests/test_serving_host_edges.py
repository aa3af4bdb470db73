"""More of the serving calls' argument checks, through the C ABI without a GPU (every check
comes before the device is looked for)."""
import ctypes

import pytest

from mini_tensorrt_b200 import _lib
from tests.test_serving_host import A, paged, prompt


@pytest.mark.parametrize("field", ["k_pages", "v_pages", "table", "kv_len"])
def test_prompt_call_with_paged_arguments_refused(field):
    """The sizes of a call with pages are not those of a prompt's, so a struct kept for both
    would have the rows written past the workspace."""
    a = prompt(**{field: A})
    assert _lib.lib().mtrtq_prompt_attention(ctypes.byref(a), None, 0, None) == _lib.ERR_INVALID_ARG
    assert "NULL" in _lib.last_error()


@pytest.mark.parametrize("over", [{}, {"dtype": _lib.DTYPE_BF16}, {"x_dtype": _lib.DTYPE_BF16, "dtype": _lib.DTYPE_BF16}])
def test_prompt_call_with_a_whole_cache_refused(over):
    a = paged(**over)
    assert _lib.lib().mtrtq_attention_workspace_bytes(ctypes.byref(a)) > 0  # of the paged call
    assert _lib.lib().mtrtq_prompt_attention(ctypes.byref(a), A, 1 << 40, None) == _lib.ERR_INVALID_ARG
    assert "NULL" in _lib.last_error()


def test_beam_vocabulary_near_2_31_refused():
    """Places in a row are counted in 32 bits, a block's beyond its end included."""
    lib, most = _lib.lib(), 2 ** 31 - 2 ** 14
    for beams, vocab in ((1, most + 1), (1, 2 ** 31 - 1), (2, most // 2 + 1), (32, most // 32 + 1)):
        assert lib.mtrtq_beam_workspace_bytes(1, beams, vocab) == -1
        assert lib.mtrtq_beam_select(A, vocab, A, A, -1, 1, beams, vocab, A, A, A, A, A, 1 << 40, None) == _lib.ERR_INVALID_ARG
    assert lib.mtrtq_beam_workspace_bytes(1, 1, most) > 0 and lib.mtrtq_beam_workspace_bytes(1, 32, most // 32) > 0


@pytest.mark.parametrize("over", [{"out_head": 0}, {"out_head": 8}, {"out_row": 8}, {"out_head": 0, "dtype": _lib.DTYPE_BF16}])
def test_heads_or_rows_of_out_that_overlap_refused(over):
    """Heads of 16 dimensions that start 8 apart, or at the same place, would be written by
    several blocks in no order."""
    for make, fn in ((prompt, _lib.lib().mtrtq_prompt_attention), (paged, _lib.lib().mtrtq_paged_attention)):
        assert fn(ctypes.byref(make(**over)), None, 0, None) == _lib.ERR_INVALID_ARG
        assert "overlap" in _lib.last_error()


def test_strides_of_a_single_row_or_head_of_out_say_nothing():
    one = {"rows": 1, "batch": 1, "heads": 1, "kv_heads": 1}
    for over in ({"out_row": 0}, {"out_head": 0}, {"out_row": 0, "out_head": 0}):
        a = prompt(**one, **over)
        assert _lib.lib().mtrtq_attention_workspace_bytes(ctypes.byref(a)) > 0
