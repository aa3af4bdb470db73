"""PagedDecoder's passes over chunks of prompts."""
import numpy as np
import pytest

from mini_tensorrt_b200 import gpt2, paged, serving
from tests.test_paged_decoder import LENS, SMALL, prompts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("beams", [1, 3])
def test_prompts_that_are_done_are_left_out(cuda_device, monkeypatch, beams):
    """Each pass has the prompts with tokens left and no others, and the tokens that come out
    are those of whole prompts."""
    dec = paged.PagedDecoder(gpt2.random_weights(SMALL, seed=5), "fp32", 16, cuda_device)
    ps = prompts(6, LENS)
    whole = dec.generate(ps, 6, beams=beams)
    real, seen = serving.paged_attention, []

    def noted(q, k, v, kp, vp, table, kv_len, cu_rows, **kw):
        seen.append((cu_rows.diff().tolist(), kv_len.tolist()))
        assert table.shape[0] == kv_len.shape[0]
        return real(q, k, v, kp, vp, table, kv_len, cu_rows, **kw)

    monkeypatch.setattr(serving, "paged_attention", noted)
    got = dec.generate(ps, 6, beams=beams, chunk=7, use_graph=False)
    want = []
    for begin in range(0, max(LENS), 7):
        live = [n for n in LENS if n > begin]
        want.append(([min(7, n - begin) for n in live], [min(begin + 7, n) for n in live]))
    assert seen[: len(want) * SMALL.n_layer] == [w for w in want for _ in range(SMALL.n_layer)]
    np.testing.assert_array_equal(got["tokens"], whole["tokens"])
