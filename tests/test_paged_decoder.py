"""Serving GPT-2 from the paged cache (mini_tensorrt_b200.paged): page bookkeeping on the
CPU; on the GPU the tokens of requests of different lengths against the reference's decoder
restated on the CPU, one request at a time, and beam search against a plain one over the
same decoder's logits."""
import numpy as np
import pytest
import torch

from mini_tensorrt_b200 import gpt2, matmulq, paged
from oracle.gpt2_decode import OracleDecoder
from tests.conftest import rel_err

SMALL = gpt2.GPT2Config(n_layer=2, d_model=128, n_head=4, d_ff=512, vocab=1000, n_pos=128)


@pytest.mark.parametrize("lens,beams,new,page", [([1], 1, 1, 16), ([16, 17, 5], 3, 20, 16), ([64, 1], 8, 70, 32)])
def test_assign_pages(lens, beams, new, page):
    table, owned, count = paged.assign_pages(lens, beams, new, page)
    assert table.shape == owned.shape == (len(lens) * beams, max(-(-(p + new) // page) for p in lens))
    used = []
    for b, p in enumerate(lens):
        rows = owned[b * beams:(b + 1) * beams]
        full = p // page
        assert (rows[:, :full] == rows[0, :full]).all()          # the prompt's full pages are shared
        used += rows[0, :full].tolist() + rows[:, full:].ravel().tolist()
        assert (table[b * beams:(b + 1) * beams] == rows[0]).all()  # all read the first beam's at first
    assert sorted(used) == list(range(count))                     # every page once


def prompts(seed, lens):
    r = np.random.default_rng(seed)
    return [r.integers(0, SMALL.vocab, n, dtype=np.int32) for n in lens]


LENS = [5, 33, 1, 16, 47]


@pytest.mark.gpu
@pytest.mark.parametrize("page,chunk,graph", [(16, None, True), (32, 7, True), (128, 16, False)])
def test_greedy_matches_the_oracle(cuda_device, page, chunk, graph):
    w = gpt2.random_weights(SMALL, seed=5)
    ps = prompts(6, LENS)
    got = paged.PagedDecoder(w, "fp32", page, cuda_device).generate(ps, 20, chunk=chunk, use_graph=graph)
    for b, p in enumerate(ps):
        want = OracleDecoder(w, 1, len(p) + 20).generate(p[None], 20)
        np.testing.assert_array_equal(got["tokens"][b, 0], want[0])
    assert matmulq.read_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["fp32", "bf16"])
def test_packed_logits_match_the_oracle(cuda_device, mode):
    """Every position of every prompt in one packed pass; the tolerances are the decoder's:
    1e-4 in fp32 mode, 2e-2 in bf16 mode."""
    w = gpt2.random_weights(SMALL, seed=5)
    ps = prompts(7, LENS)
    got = paged.PagedDecoder(w, mode, 32, cuda_device).logits(ps)
    for p, g in zip(ps, got):
        ref = OracleDecoder(w, 1, len(p))
        want = np.stack([ref.step(p[None, i], i)[1][0] for i in range(len(p))])
        assert rel_err(g.cpu().numpy(), want) <= (1e-4 if mode == "fp32" else 2e-2)


def plain_beam_search(w, prompt, new, beams, eos):
    """Beam search over the oracle's logits, every beam's whole history run again each
    step: scores in 64 bits, ties to the lowest beam and token."""
    live = [(0.0, list(prompt), False)]
    for _ in range(new):
        cand = []
        for i, (score, toks, ended) in enumerate(live):
            if ended:
                cand.append((-score, i, eos, True))
                continue
            dec = OracleDecoder(w, 1, len(toks))
            for pos, t in enumerate(toks):
                _, logits = dec.step(np.array([t], np.int32), pos)
            x = logits[0].astype(np.float64)
            lp = x - (x.max() + np.log(np.exp(x - x.max()).sum()))
            for t in np.argsort(-lp, kind="stable")[:beams]:
                cand.append((-(score + lp[t]), i, int(t), int(t) == eos))
        cand.sort(key=lambda c: c[:3])
        live = [(-s, live[i][1] + [t], e) for s, i, t, e in cand[:beams]]
    return [t[len(prompt):] for _, t, _ in live], [s for s, _, _ in live]


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [True, False])
def test_beam_search_matches_a_plain_one(cuda_device, graph):
    w = gpt2.random_weights(SMALL, seed=8)
    ps = prompts(9, [3, 18, 15])
    dec = paged.PagedDecoder(w, "fp32", 16, cuda_device)
    # a token that the best beams do take, so that some end early
    eos = int(dec.generate(ps, 4, beams=4)["tokens"][0, 1, 2])
    got = dec.generate(ps, 6, beams=4, eos=eos, use_graph=graph)
    for b, p in enumerate(ps):
        tokens, scores = plain_beam_search(w, p, 6, 4, eos)
        # sums of up to six log-probabilities of some -7 each, logits off by up to 1e-4 of
        # their largest
        np.testing.assert_allclose(got["scores"][b], scores, rtol=1e-4)
        np.testing.assert_array_equal(got["tokens"][b], np.array(tokens))
    assert matmulq.read_device_status() == 0


@pytest.mark.gpu
def test_one_beam_is_greedy_and_bf16_runs(cuda_device):
    w = gpt2.random_weights(SMALL, seed=5)
    ps = prompts(6, LENS)
    dec = paged.PagedDecoder(w, "bf16", 32, cuda_device)
    a, b = dec.generate(ps, 12), dec.generate(ps, 12, use_graph=False, chunk=9)
    assert a["tokens"].shape == (5, 1, 12) and (a["scores"] < 0).all()
    assert (a["tokens"][:, :, 0] == b["tokens"][:, :, 0]).mean() >= 0.8  # bf16: near ties may differ
    g = dec.generate(ps, 12, beams=3)
    assert (g["scores"][:, 0] >= a["scores"][:, 0] - 0.2).all()
    assert (np.diff(g["scores"], axis=1) <= 0).all()


@pytest.mark.gpu
def test_refusals(cuda_device):
    dec = paged.PagedDecoder(gpt2.random_weights(SMALL, seed=5), "fp32", 32, cuda_device)
    for ps, new in (([[]], 3), ([[1, 2], [5] * 129], 1), ([[1, 1000]], 2), ([[1] * 120], 20), ([], 2), ([[1]], 0)):
        with pytest.raises(ValueError):
            dec.generate(ps, new)
    with pytest.raises(ValueError):
        paged.PagedDecoder(gpt2.random_weights(SMALL, seed=5), page_size=8)
    with pytest.raises(ValueError):
        paged.PagedDecoder(gpt2.random_weights(SMALL, seed=5), mode="int8")
