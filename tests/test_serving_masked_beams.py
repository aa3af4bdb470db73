"""Beam selection where masks leave few tokens or scores tie by rounding: exactly the
candidates that 32-bit scores and the order of their indices give."""
import math

import numpy as np
import pytest
import torch

from mini_tensorrt_b200 import serving
from tests.test_serving import F32, INF, make_gen, randn

pytestmark = pytest.mark.gpu

LOWEST = torch.finfo(F32).min
MASKS = (-INF, LOWEST)
SIZES = [(1, 1, 5), (1, 4, 50257), (3, 8, 50257), (2, 16, 4097), (1, 32, 33), (40, 4, 9000), (2, 32, 20000), (1, 3, 1)]


def expected(logits, scores, done, eos):
    """(parent, token) of the best, scores rounded as the kernel rounds them: the log-sum to
    32 bits, then one rounding for each of the two sums."""
    B, W = scores.shape
    x = logits.double().cpu().numpy().reshape(B, W, -1)
    V = x.shape[2]
    s, out = scores.cpu().numpy(), []
    for b in range(B):
        total = np.full((W, V), -np.inf, np.float32)
        for w in range(W):
            if done[b, w]:
                if eos >= 0:
                    total[w, eos] = s[b, w]
            elif s[b, w] > -np.inf and x[b, w].max() > -np.inf:
                top = x[b, w].max()
                lse = np.float32(top + np.log(np.exp(x[b, w] - top).sum()))
                with np.errstate(over="ignore"):
                    total[w] = s[b, w] + (x[b, w].astype(np.float32) - lse)
        at = np.argsort(-total.reshape(-1), kind="stable")[:W]
        out.append([(int(i) // V, int(i) % V) for i in at])
    return out


def pairs(got):
    return [list(zip(p, t)) for p, t in zip(got[1].tolist(), got[2].tolist())]


@pytest.mark.parametrize("B,W,V", SIZES)
@pytest.mark.parametrize("left", [0, 1, 2, 7])
@pytest.mark.parametrize("mask", [-INF, LOWEST], ids=["inf", "lowest"])
def test_masks_that_leave_few_tokens(cuda_device, B, W, V, left, mask):
    """Every row keeps `left` tokens, whole numbers apart so that rounding does not order them."""
    gen = torch.Generator().manual_seed(W + V + left)
    logits = torch.full((B * W, V), mask)
    for r in range(B * W):
        at = torch.randperm(V, generator=gen)[: min(left, V)]
        logits[r, at] = 2.0 * torch.randperm(len(at), generator=gen).float()
    logits = logits.cuda()
    scores = -32.0 * torch.stack([torch.randperm(W, generator=gen) for _ in range(B)]).float().cuda()
    done = torch.zeros((B, W), dtype=torch.uint8, device="cuda")
    if W > 2:
        scores[0, 1] = -INF
        done[:, 2] = 1
    got = serving.beam_select(logits, scores, done, V - 1)
    assert pairs(got) == expected(logits, scores, done, V - 1)


@pytest.mark.parametrize("W,V", [(2, 50257), (8, 50257), (5, 6000), (32, 12000)])
@pytest.mark.parametrize("hidden", [0, 9, 4999])
@pytest.mark.parametrize("two", [False, True])
def test_scores_that_tie_by_rounding(cuda_device, W, V, hidden, two):
    """Scores of some -1e8 are 8 apart, so logits that differ by a thousandth give the same, and
    the lowest indices win whatever their logits; also with a beam before it that has three
    tokens of that score, and where a mask hides the first ones. (A log-sum between 4 and 12
    takes 8 off, one below 4 nothing.)"""
    logits = 1e-3 * randn(make_gen(W + V), W, V)
    logits[:, :hidden] = -INF
    assert 4.1 < math.log(V - hidden) < 11.9
    scores = torch.full((1, W), -INF, device="cuda")
    scores[0, 0] = -1e8
    if two:
        scores[0, :2] = torch.tensor([-1e8 - 8, -1e8])
        logits[0, hidden + 3:] = -INF
    done = torch.zeros((1, W), dtype=torch.uint8, device="cuda")
    got = serving.beam_select(logits, scores, done)
    assert pairs(got) == expected(logits, scores, done, -1)
    assert (got[0] == -1e8 - 8).all()


def test_masks_cost_no_more_than_other_logits(cuda_device):
    """Once looked through again by one block for every beam: 40 to 120 times as long."""
    B, W, V = 4, 8, 50257
    scores, done = -torch.rand((B, W), device="cuda"), torch.zeros((B, W), dtype=torch.uint8, device="cuda")
    ws = torch.zeros(1 << 24, dtype=torch.uint8, device="cuda")

    def took(logits):
        times = []
        for _ in range(9):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(10):
                serving.beam_select(logits, scores, done, workspace=ws)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return sorted(times)[4]

    plain = randn(make_gen(1), B * W, V)
    masked = {}
    for mask in MASKS:
        masked[mask] = plain.clone()
        masked[mask][:, 1:] = mask
    usual = took(plain)
    scores[:, 1:] = -INF
    for x in masked.values():
        assert took(x) < 10 * usual


@pytest.mark.parametrize("mask", [-INF, LOWEST], ids=["inf", "lowest"])
@pytest.mark.parametrize("beam", [0, 17, 31])
def test_one_beam_of_many_in_use(cuda_device, mask, beam):
    """Its chunks come after hundreds of others', and ties start in the middle of one."""
    W, V = 32, 50257
    logits = randn(make_gen(beam), W, V)
    logits[beam] = -INF
    logits[beam, 30000:] = mask
    logits[beam, 40000:40005] = torch.tensor([4.0, 8.0, 0.0, 2.0, 6.0], device="cuda")
    scores = torch.full((1, W), -INF, device="cuda")
    scores[0, beam] = -3.0
    done = torch.zeros((1, W), dtype=torch.uint8, device="cuda")
    got = serving.beam_select(logits, scores, done)
    want = expected(logits, scores, done, -1)
    assert pairs(got) == want
    first = [(beam, 40000 + i) for i in (1, 4, 0, 3, 2)]
    assert want[0][:5] == first and want[0][5] == ((beam, 30000) if mask == LOWEST else (0, 0))
