"""PagedDecoder in bf16 mode, decoding: every token that it chose and every score, against the
CPU decoder run over the same tokens."""
import numpy as np
import pytest

from mini_tensorrt_b200 import gpt2, matmulq, paged
from oracle.gpt2_decode import OracleDecoder
from tests.test_paged_decoder import LENS, SMALL, prompts

pytestmark = pytest.mark.gpu
NEW = 12


@pytest.mark.parametrize("page,beams,graph", [(16, 1, True), (32, 1, False), (16, 3, True)])
def test_decoded_tokens_and_scores(cuda_device, page, beams, graph):
    """bf16 mode's logits are off by up to e = 2e-2 (|logit| + their rms), so the token that a
    greedy step takes is at most 2 e below the largest, and a sum of log-probabilities is off
    by at most 2 e for each token (a logit and the log-sum, which moves no more than its
    largest term). Of a beam the score alone is bounded that way."""
    w = gpt2.random_weights(SMALL, seed=5)
    ps = prompts(6, LENS)
    got = paged.PagedDecoder(w, "bf16", page, cuda_device).generate(ps, NEW, beams=beams, use_graph=graph)
    for b, p in enumerate(ps):
        for beam in range(beams):
            tokens = got["tokens"][b, beam]
            forced = np.concatenate([p, tokens]).astype(np.int32)
            ref, total, slack = OracleDecoder(w, 1, len(forced)), 0.0, 0.0
            for pos in range(len(forced) - 1):
                logits = ref.step(forced[None, pos], pos)[1][0].astype(np.float64)
                if pos < len(p) - 1:
                    continue
                chosen = tokens[pos - len(p) + 1]
                e = 2e-2 * (np.abs(logits).max() + np.sqrt(np.mean(logits ** 2)))
                if beams == 1:
                    assert logits.max() - logits[chosen] <= 2 * e
                total += logits[chosen] - logits.max() - np.log(np.exp(logits - logits.max()).sum())
                slack += 2 * e
            assert abs(got["scores"][b, beam] - total) <= slack
    assert matmulq.read_device_status() == 0
