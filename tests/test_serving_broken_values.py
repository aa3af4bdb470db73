"""What NaN and infinities in q, k and the scores do to the serving operators' results: the
rows and beams that meet them, and only those. Expected values follow from the formulas (a
sum with a NaN is NaN, a NaN score counts as -infinity), so they are compared exactly."""
import pytest
import torch

from mini_tensorrt_b200 import matmulq, serving
from tests.test_serving import INF, NAN, TYPES, Paged, i32, make_gen, offsets, randn, rows

pytestmark = pytest.mark.gpu

# (heads, lengths): long tiles that are cut between CTAs, also with groups of heads; tiles of
# one block each, which never are; short prompts and a few rows
PROMPTS = [((12, 12, 64), [515, 140]), ((5, 1, 64), [700, 300, 90]), ((25, 25, 64), [100] * 8), ((4, 2, 128), [600, 64]),
           ((4, 4, 64), [40, 3]), ((2, 2, 64), [6, 1])]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads,lens", PROMPTS, ids=str)
@pytest.mark.parametrize("bad", [NAN, INF])
def test_prompt_rows_of_broken_q(cuda_device, kind, heads, lens, bad):
    """A row whose q has a NaN is NaN, and so is one whose q is infinite where the first key,
    which every row sees, is positive (its largest score is +infinity). No other row feels it."""
    H, KV, D = heads
    q, k, v = rows(make_gen(21), sum(lens), H, KV, D, kind)
    cu, held = i32(offsets(lens)), TYPES[kind][1]
    k[offsets(lens)[:-1], :, 5] = 1.0
    clean = serving.prompt_attention(q, k, v, cu, out_dtype=held).clone()
    hit = sorted({x for a, n in zip(offsets(lens), lens) for x in (a, a + n // 2, a + n - 1)})
    q[hit, :, 5] = bad
    got = serving.prompt_attention(q, k, v, cu, out_dtype=held)
    assert got[hit].isnan().all()
    rest = [x for x in range(sum(lens)) if x not in hit]
    assert torch.equal(got[rest], clean[rest])
    assert matmulq.read_device_status() == 0


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads,lens", PROMPTS, ids=str)
@pytest.mark.parametrize("many", [1, 128, 10000])
def test_prompt_keys_that_are_nan(cuda_device, kind, heads, lens, many):
    """The first keys of a request are NaN, up to all of them: every row sees one, so every row
    of the request is NaN, also where others of the row's scores are fine. The next request
    keeps its bits."""
    H, KV, D = heads
    q, k, v = rows(make_gen(22), sum(lens), H, KV, D, kind)
    cu, held = i32(offsets(lens)), TYPES[kind][1]
    clean = serving.prompt_attention(q, k, v, cu, out_dtype=held).clone()
    k[: min(many, lens[0])] = NAN
    got = serving.prompt_attention(q, k, v, cu, out_dtype=held)
    assert got[: lens[0]].isnan().all()
    assert torch.equal(got[lens[0]:], clean[lens[0]:])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads,lens", [((12, 12, 64), [515, 700]), ((4, 2, 128), [600, 130])], ids=str)
def test_prompt_later_keys_that_are_nan(cuda_device, kind, heads, lens):
    """A block of NaN keys in the middle: the rows from it on are NaN, the rows before keep
    their bits."""
    H, KV, D = heads
    q, k, v = rows(make_gen(23), sum(lens), H, KV, D, kind)
    cu, held = i32(offsets(lens)), TYPES[kind][1]
    clean = serving.prompt_attention(q, k, v, cu, out_dtype=held).clone()
    k[256:384] = NAN
    got = serving.prompt_attention(q, k, v, cu, out_dtype=held)
    assert got[256:lens[0]].isnan().all()
    keep = [*range(256), *range(lens[0], sum(lens))]
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads", [(4, 4, 64), (8, 2, 128)], ids=str)
@pytest.mark.parametrize("new,lens", [([1, 1, 1], [900, 33, 128]), ([130, 1, 5], [700, 40, 5])], ids=str)
def test_paged_rows_of_broken_q(cuda_device, kind, heads, new, lens):
    """The same over a cache, with parts of long requests joined."""
    args = (new, lens, *heads, 32, kind)
    clean, s = Paged(*args, seed=24), Paged(*args, seed=24)
    want = clean.run()
    hit = [0, sum(new) - 1]
    s.q[hit, :, 5] = NAN
    got = s.run()
    assert got[hit].isnan().all()
    assert torch.equal(got[1:-1], want[1:-1])


@pytest.mark.parametrize("W,V", [(2, 50257), (4, 7), (8, 9000)])
@pytest.mark.parametrize("nan", [NAN, -NAN])
def test_beam_that_is_done_with_a_nan_score(cuda_device, W, V, nan):
    """Its one candidate has a NaN score, which counts as -infinity: it comes after every
    candidate with a score, and at its index among those without."""
    logits = randn(make_gen(24), W, V)
    scores = torch.full((1, W), -INF, device="cuda")
    scores[0, 0], scores[0, 1] = -1.0, nan
    done = torch.zeros((1, W), dtype=torch.uint8, device="cuda")
    done[0, 1] = 1
    keep = torch.zeros(V, dtype=torch.bool, device="cuda")
    keep[5] = True
    logits[0] = torch.where(keep, logits[0], torch.full_like(logits[0], -INF))  # one candidate in all
    out_scores, parent, token, _ = serving.beam_select(logits, scores, done, 3)
    at = (parent.long() * V + token)[0].tolist()
    assert at == [5, *[t for t in range(W + 1) if t != 5][: W - 1]]
    assert out_scores[0, 0] == -1.0 and (out_scores[0, 1:] == -INF).all()
