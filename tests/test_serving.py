"""The serving operators on the GPU against their formulas in 64 bits.

Tolerances, from the arithmetic alone. Let S be a row's largest scale * sqrt(sum q^2 k^2)
over its keys and V the largest |v| in its view; rounding errors of independent terms add
as the root of their number, and six standard deviations are allowed.
* f32 (unit roundoff u = 2^-24): a score of D products is off by about u sqrt(D) S, a
  weight by as much of itself, the sums over n keys by u sqrt(n):
  |error| <= u V (6 sqrt(D) S + 6 sqrt(n) + 16).
* bf16 (a rounding is off by up to 2 u of the value, u = 2^-9, and by less than u in the
  mean): the output is rounded once, up to 2 u |ref| <= u (|ref| + V); the weights once each,
  which leaves u V for their sum; and f32 rows round q (u S / sqrt(3) standard deviation on a
  score, as much of itself on a weight): |error| <= u (|ref| + V (2 + 4 S)), 4 = 6 / sqrt(3)
  rounded up, without the S term for bf16 rows; and over a whole output the errors' norm is at most 2^-8 of the result's
  (2^-7 with f32 rows).
"""
import math

import pytest
import torch

from mini_tensorrt_b200 import _lib, matmulq, serving

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")
F32, BF16 = torch.float32, torch.bfloat16
TYPES = {"f32": (F32, F32), "bf16": (BF16, BF16), "mixed": (F32, BF16)}
HEADS = [(12, 12, 64), (8, 2, 128), (6, 2, 80), (5, 1, 64), (3, 3, 8), (4, 4, 128), (7, 7, 40), (16, 1, 64)]


def randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def make_gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def offsets(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def reference(q, k, v, visible, scale):
    """Rows q [m, H, D] over keys k, v [n, KV, D], row i over the first visible[i]: the
    output, and the S and V of the tolerances for every row and head."""
    H, D = q.shape[1:]
    n = torch.tensor(list(visible), device=q.device)[:, None, None]
    kk = k.double().repeat_interleave(H // k.shape[1], 1)
    vv = v.double().repeat_interleave(H // k.shape[1], 1)
    hidden = torch.arange(k.shape[0], device=q.device) >= n  # [m, 1, keys]
    s = torch.einsum("mhd,nhd->mhn", q.double(), kk) * scale
    p = torch.softmax(s.masked_fill(hidden, -INF), 2).masked_fill(hidden, 0.0)
    out = torch.einsum("mhn,nhd->mhd", p, vv)
    S = torch.einsum("mhd,nhd->mhn", q.double() ** 2, kk ** 2).sqrt() * scale
    V = vv.abs().amax(2).T.expand(len(n), -1, -1)
    top = lambda x: x.masked_fill(hidden, 0.0).amax(2, keepdim=True) if x.shape[2] else x.new_zeros(len(n), H, 1)
    return out, top(S), top(V)


def near(got, ref, S, V, kind, D, visible):
    got = got.double()
    n = torch.tensor([max(1, x) for x in visible], dtype=torch.float64, device=got.device)[:, None, None]
    if kind == "f32":
        bound = 2.0 ** -24 * V * (6 * math.sqrt(D) * S + 6 * n.sqrt() + 16)
    else:
        bound = 2.0 ** -9 * (ref.abs() + V * (2 + (4 * S if kind == "mixed" else 0)))
    assert torch.isfinite(got).all()
    worst = ((got - ref).abs() - bound).max()
    assert worst <= 0, f"off by {worst.item():.3e} more than allowed"
    if kind != "f32" and ref.norm() > 0:
        rel = ((got - ref).norm() / ref.norm()).item()
        assert rel <= (2.0 ** -8 if kind == "bf16" else 2.0 ** -7), rel


def rows(gen, T, H, KV, D, kind, order="fused"):
    """q, k, v as views of one projection's rows, of [heads, rows, dim] tensors, or of
    rows with a gap between them."""
    x = TYPES[kind][0]
    if order == "fused":
        p = randn(gen, T, (H + 2 * KV) * D)
        p[:, : H * D] *= 1.5
        q, k, v = p.to(x).split([H * D, KV * D, KV * D], 1)
        return q.view(T, H, D), k.view(T, KV, D), v.view(T, KV, D)
    if order == "heads_first":
        return tuple(randn(gen, n, T, D).to(x).transpose(0, 1) for n in (H, KV, KV))
    return tuple(randn(gen, T, n + 1, D + 8).to(x)[:, 1:, :D] for n in (H, KV, KV))


# ---- whole prompts ------------------------------------------------------------------------------

LENS = [[1], [2, 1, 0, 3], [128, 127, 129], [0, 65, 300, 1, 17], [515]]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("lens", LENS, ids=str)
def test_prompt(cuda_device, kind, heads, lens):
    H, KV, D = heads
    q, k, v = rows(make_gen(len(lens) + H), sum(lens), H, KV, D, kind)
    got = serving.prompt_attention(q, k, v, i32(offsets(lens)), out_dtype=TYPES[kind][1])
    assert got.dtype == TYPES[kind][1] and got.shape == q.shape
    for a, n in zip(offsets(lens), lens):
        s = slice(a, a + n)
        if n:
            held = TYPES[kind][1]
            near(got[s], *reference(q[s], k[s].to(held), v[s].to(held), range(1, n + 1), D ** -0.5), kind, D,
                 range(1, n + 1))
    assert matmulq.read_device_status() == 0


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("order", ["heads_first", "gaps"])
def test_prompt_strides_out_and_scale(cuda_device, kind, order):
    """Other orders in memory, the caller's out (itself strided) and scale, rows outside
    every request left alone."""
    H, KV, D, lens, scale = 6, 3, 64, [70, 1, 133], 0.31
    T = sum(lens)
    q, k, v = rows(make_gen(3), T + 9, H, KV, D, kind, order)
    held = TYPES[kind][1]
    space = torch.full((H, T + 9, D), 7.0, dtype=held, device="cuda")
    out = space.transpose(0, 1)
    at = [x + 4 for x in offsets(lens)]  # rows 0..3 and the last 5 belong to nobody
    got = serving.prompt_attention(q, k, v, i32(at), out=out, scale=scale)
    assert got is out
    for a, n in zip(at, lens):
        s = slice(a, a + n)
        near(got[s], *reference(q[s], k[s].to(held), v[s].to(held), range(1, n + 1), scale), kind, D, range(1, n + 1))
    assert (out[:4] == 7).all() and (out[T + 4:] == 7).all()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads", [(4, 4, 64), (8, 2, 128)], ids=str)
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
def test_prompt_hidden_values_have_no_effect(cuda_device, kind, heads, bad):
    """What a later token, or another request, holds does not reach a row."""
    H, KV, D = heads
    lens, at = [200, 150], 131
    q, k, v = rows(make_gen(4), 350, H, KV, D, kind)
    cu = i32(offsets(lens))
    held = TYPES[kind][1]
    clean = serving.prompt_attention(q, k, v, cu, out_dtype=held).clone()
    k[at], v[at, :, 3] = bad, bad
    k[200 + at], v[200 + at] = bad, bad
    got = serving.prompt_attention(q, k, v, cu, out_dtype=held)
    for a, n in ((0, at), (200, at)):
        assert torch.equal(got[a:a + n], clean[a:a + n])
    # the rows that see it do feel it
    assert not torch.isfinite(got[at:200].float()).all() and not torch.isfinite(got[200 + at:].float()).all()


@pytest.mark.parametrize("kind", TYPES)
def test_prompt_infinite_values_arrive(cuda_device, kind):
    """A row that sees an infinite v gets it, in its dimension alone."""
    q, k, v = rows(make_gen(5), 140, 2, 2, 64, kind)
    held = TYPES[kind][1]
    cu = i32([0, 140])
    clean = serving.prompt_attention(q, k, v, cu, out_dtype=held).clone()
    v[133, 0, 7] = INF
    got = serving.prompt_attention(q, k, v, cu, out_dtype=held)
    assert torch.equal(got[:133], clean[:133])
    assert (got[133:, 0, 7] == INF).all()
    got[133:, 0, 7] = clean[133:, 0, 7]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("kind", TYPES)
def test_prompt_large_scores(cuda_device, kind):
    """Scores of thousands and a maximum that keeps rising: no overflow on the way."""
    H, D, n = 2, 64, 400
    q, k, v = rows(make_gen(6), n, H, H, D, kind)
    q, k = q.clone(), k.clone()
    q[..., 0], k[..., 0] = 64.0, torch.linspace(-500, 500, n, device="cuda")[:, None].to(k.dtype)
    held = TYPES[kind][1]
    got = serving.prompt_attention(q, k, v, i32([0, n]), out_dtype=held)
    near(got, *reference(q, k.to(held), v.to(held), range(1, n + 1), D ** -0.5), kind, D, range(1, n + 1))


# ---- new tokens over pages ----------------------------------------------------------------------


class Paged:
    """A paged cache of random requests, with NaN in every place that no token has, and
    page numbers out of range in the columns that no token needs."""

    def __init__(self, new, lens, H, KV, D, page, kind, seed=0, hold=False, order="fused"):
        gen = make_gen(seed)
        self.new, self.lens, self.kind, self.D = new, lens, kind, D
        held = TYPES[kind][1]
        used = [-(-n // page) for n in lens]
        width = max(1, max(used))
        P = sum(used) + 2
        order_ = torch.randperm(P, generator=torch.Generator().manual_seed(seed)).tolist()
        self.kp = torch.full((P, KV, page, D), NAN, dtype=held, device="cuda")
        self.vp = self.kp.clone()
        self.q, self.k, self.v = rows(gen, sum(new), H, KV, D, kind, order)
        table, self.keys, self.values = [], [], []
        for b, (m, n) in enumerate(zip(new, lens)):
            pages = [order_.pop() for _ in range(used[b])]
            table.append(pages + [-1 if b % 2 else P + 5] * (width - used[b]))
            a = offsets(new)[b]
            old = max(0, n - m)
            lost = max(0, m - n)  # new rows before the request's first position
            k = torch.cat([randn(gen, old, KV, D).to(held), self.k[a + lost:a + m].to(held)])
            v = torch.cat([randn(gen, old, KV, D).to(held), self.v[a + lost:a + m].to(held)])
            i = torch.arange(n if hold else old, device="cuda")
            if len(i):
                at = i32(pages).long()[i // page]
                self.kp[at, :, i % page], self.vp[at, :, i % page] = k[:len(i)], v[:len(i)]
            self.keys.append(k)
            self.values.append(v)
        self.table, self.kv_len, self.cu = i32(table), i32(lens), i32(offsets(new))
        self.page = page

    def run(self, **kw):
        return serving.paged_attention(self.q, self.k, self.v, self.kp, self.vp, self.table, self.kv_len, self.cu, **kw)

    def verify(self, got, scale=None):
        scale = self.D ** -0.5 if scale is None else scale
        for b, (m, n) in enumerate(zip(self.new, self.lens)):
            a = offsets(self.new)[b]
            visible = [n - m + t + 1 for t in range(m)]
            if m:
                near(got[a:a + m], *reference(self.q[a:a + m], self.keys[b], self.values[b], visible, scale), self.kind,
                     self.D, visible)
            if n:
                i = torch.arange(n, device="cuda")
                at = self.table[b].long()[i // self.page]
                assert torch.equal(self.kp[at, :, i % self.page], self.keys[b])
                assert torch.equal(self.vp[at, :, i % self.page], self.values[b])
        assert matmulq.read_device_status() == 0


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("page", [16, 128])
def test_decode(cuda_device, kind, heads, page):
    lens = [1, 2, 16, 17, 127, 128, 129, 700]
    s = Paged([1] * len(lens), lens, *heads, page, kind)
    s.verify(s.run())


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads", [(4, 2, 64), (8, 4, 128), (6, 3, 40)], ids=str)
@pytest.mark.parametrize("new,lens", [([1] * 6, [1, 2, 255, 256, 257, 900]), ([1], [3000]),
                                      ([4, 0, 0, 0, 0, 1], [610, 9, 0, 5, 33, 2])], ids=str)
def test_decode_pairs_of_heads(cuda_device, kind, heads, new, lens):
    """Tiles of two rows, also where one request has more tokens than the others together."""
    H, KV, D = heads
    s = Paged(new, lens, H, KV, D, 32, kind, seed=len(new))
    s.verify(s.run())


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads", [(2, 2, 64), (4, 2, 128), (8, 2, 128)], ids=str)
def test_decode_key_of_minus_infinity_has_no_weight(cuda_device, kind, heads):
    """An infinite element of a key makes a score of -infinity where q is negative there: the
    token counts for nothing, as if it were not there."""
    H, KV, D = heads
    x = Paged([1, 1], [200, 70], H, KV, D, 16, kind, seed=8)
    x.q[..., 5] = -x.q[..., 5].abs() - 0.1
    at = [x.table[b, 2].item() for b in range(2)]
    for page in at:
        x.kp[page, :, 7, 5] = INF
    got = x.run()
    for b, n in enumerate(x.lens):
        keep = torch.arange(n, device="cuda") != 39
        near(got[b:b + 1], *reference(x.q[b:b + 1], x.keys[b][keep], x.values[b][keep], [n - 1], D ** -0.5), kind, D, [n - 1])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads", [(12, 12, 64), (8, 2, 128), (6, 2, 80), (5, 1, 64)], ids=str)
@pytest.mark.parametrize("page", [32, 64])
def test_chunks(cuda_device, kind, heads, page):
    """Chunks of every size beside single tokens and requests that wait."""
    s = Paged([1, 0, 5, 130, 64, 0, 33, 257], [900, 40, 5, 131, 500, 0, 34, 400], *heads, page, kind, seed=1)
    s.verify(s.run())


@pytest.mark.parametrize("kind", TYPES)
def test_long_caches(cuda_device, kind):
    """Work split over a long axis, with few rows and one request much longer."""
    s = Paged([1, 1, 3], [9001, 33, 5000], 4, 2, 64, 32, kind, seed=2)
    s.verify(s.run())


@pytest.mark.parametrize("kind", TYPES)
def test_many_requests(cuda_device, kind):
    lens = [1 + (37 * i) % 90 for i in range(300)]
    s = Paged([1 if i % 7 else 0 for i in range(300)], lens, 4, 4, 32, 16, kind, seed=3)
    s.verify(s.run())


@pytest.mark.parametrize("kind", TYPES)
def test_rows_that_see_nothing_are_zero(cuda_device, kind):
    """kv_len smaller than the new rows: the first ones have no position."""
    s = Paged([4, 3, 2], [2, 0, 2], 4, 2, 64, 16, kind, seed=4)
    got = s.run(out=torch.full(s.q.shape, 9.0, dtype=s.kp.dtype, device="cuda"))
    s.verify(got)
    assert (got[:2] == 0).all() and (got[4:7] == 0).all()


@pytest.mark.parametrize("kind", TYPES)
def test_pages_that_hold_the_tokens_already(cuda_device, kind):
    s = Paged([1, 40, 7], [77, 90, 7], 6, 3, 64, 16, kind, seed=5, hold=True)
    s.k = s.v = None
    s.verify(s.run(scale=0.2), scale=0.2)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("order", ["heads_first", "gaps"])
def test_paged_strides(cuda_device, kind, order):
    s = Paged([1, 40, 7], [77, 90, 7], 6, 3, 64, 16, kind, seed=6, order=order)
    # pages that are slices of a larger buffer, K and V interleaved
    both = torch.full((s.kp.shape[0], 2, *s.kp.shape[1:]), NAN, dtype=s.kp.dtype, device="cuda")
    both[:, 0], both[:, 1] = s.kp, s.vp
    s.kp, s.vp = both[:, 0], both[:, 1]
    s.verify(s.run())


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("bad", [NAN, INF])
def test_chunk_hidden_values_have_no_effect(cuda_device, kind, bad):
    """A later token of the same chunk does not reach the rows before it."""
    args = ([150, 3], [400, 60], 8, 2, 64, 32, kind)
    s, t = Paged(*args, seed=7), Paged(*args, seed=7)
    clean = s.run()
    t.k[[99, 152]], t.v[[99, 152]] = bad, bad
    got = t.run()
    assert torch.equal(got[:99], clean[:99]) and torch.equal(got[150:152], clean[150:152])
    assert not torch.isfinite(got[99:150].float()).all() and not torch.isfinite(got[152:].float()).any()


@pytest.mark.parametrize("kind", TYPES)
def test_repeated_calls_give_the_same_bits(cuda_device, kind):
    s = Paged([1, 1, 60, 1], [3000, 17, 900, 444], 8, 2, 128, 64, kind, seed=8)
    first = s.run().clone()
    for _ in range(3):
        assert torch.equal(s.run(), first)


def test_offsets_past_32_bits(cuda_device):
    """Pages whose elements lie past 2^31, read and written."""
    P, KV, page, D = 17000, 8, 128, 128
    kp, vp = (torch.empty((P, KV, page, D), dtype=BF16, device="cuda") for _ in range(2))
    assert kp.numel() > 2 ** 31
    for new in ([1, 1], [80, 1]):
        s = Paged(new, [300, 140], 16, KV, D, page, "bf16", seed=9)
        far = [P - 1 - i for i in range(s.kp.shape[0])]
        kp[far], vp[far] = s.kp, s.vp
        s.table = torch.where((s.table >= 0) & (s.table < len(far)), P - 1 - s.table, s.table)
        s.kp, s.vp = kp, vp
        s.verify(s.run())


def test_another_stream_and_a_graph(cuda_device):
    """On a stream of its own, then captured: replays read the lengths of the moment."""
    s = Paged([1, 1], [40, 600], 8, 2, 64, 16, "mixed", seed=10)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = s.run(stream=side)
    side.synchronize()
    s.verify(got)
    out = torch.empty_like(got)
    ws = torch.zeros(1 << 26, dtype=torch.uint8, device="cuda")
    s.kv_len.copy_(i32([39, 599]))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        s.run(out=out, workspace=ws)
    s.kv_len.copy_(i32([40, 600]))
    torch.cuda.synchronize()
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, got)


def test_malformed_bounds_stay_in_bounds(cuda_device):
    """cu_rows out of range or decreasing, lengths past the table: clamped, no fault."""
    s = Paged([3, 4, 5], [50, 60, 70], 4, 2, 64, 16, "f32", seed=11)
    for kind in ("f32", "mixed"):
        s = Paged([3, 4, 5], [50, 60, 70], 4, 2, 64, 16, kind, seed=11)
        s.kv_len.copy_(i32([1 << 30, -5, 70]))
        s.cu.copy_(i32([-7, 3, 1, 1 << 30]))
        s.run()
        serving.prompt_attention(s.q, s.k, s.v, s.cu, out_dtype=TYPES[kind][1])
        torch.cuda.synchronize()


# ---- refusals of the Python layer ------------------------------------------------------------------


def test_python_refusals(cuda_device):
    s = Paged([1, 1], [5, 9], 4, 2, 64, 16, "mixed", seed=12)

    def refused(**over):
        d = dict(q=s.q, k=s.k, v=s.v, k_pages=s.kp, v_pages=s.vp, table=s.table, kv_len=s.kv_len, cu_rows=s.cu)
        d.update(over)
        with pytest.raises((ValueError, _lib.MtrtqError)):
            serving.paged_attention(**d)

    refused(q=s.q.half())
    refused(q=s.q[0])
    refused(k=None)
    refused(v=s.v[:, :1])
    refused(k=s.k.bfloat16())
    refused(k_pages=s.kp.float())
    refused(k_pages=s.kp[..., :32], v_pages=s.vp[..., :32])
    refused(k_pages=s.kp.transpose(1, 2), v_pages=s.vp.transpose(1, 2))
    refused(table=s.table.long())
    refused(table=s.table[:1])
    refused(kv_len=s.kv_len[:1])
    refused(cu_rows=s.cu[:2])
    refused(cu_rows=s.cu.cpu())
    refused(scale=-1.0)
    refused(out=torch.empty_like(s.q))
    with pytest.raises(_lib.MtrtqError):
        serving.prompt_attention(s.q.bfloat16(), s.k.bfloat16(), s.v.bfloat16(), s.cu, out_dtype=F32)
    with pytest.raises(ValueError):
        serving.prompt_attention(s.q, s.k, s.v[:1], s.cu)
    assert serving.prompt_attention(s.q[:0], s.k[:0], s.v[:0], i32([0, 0])).shape == (0, 4, 64)


def test_small_workspace_is_refused(cuda_device):
    s = Paged([1, 1], [5, 9], 4, 2, 64, 16, "mixed", seed=13)
    with pytest.raises(_lib.MtrtqError) as e:
        s.run(workspace=torch.zeros(16, dtype=torch.uint8, device="cuda"))
    assert e.value.status == _lib.ERR_WORKSPACE


# ---- beam search --------------------------------------------------------------------------------


def select_reference(logits, scores, done, eos):
    """Candidates in 64 bits, [requests, beams * vocab]."""
    B, W = scores.shape
    x = logits.double().view(B, W, -1)
    x = torch.where(x.isnan(), torch.full_like(x, -INF), x)
    total = scores.double()[:, :, None] + torch.log_softmax(x, 2)
    total = torch.where(total.isnan(), torch.full_like(total, -INF), total)
    for b, w in done.nonzero().tolist():
        total[b, w] = -INF
        if eos >= 0:
            total[b, w, eos] = scores[b, w].double()
    return total.view(B, -1)


def check_select(logits, scores, done, eos, got):
    """Every output is a candidate with its own score, and the scores are the best: to
    the rounding of a sum of three f32 numbers (the log of the sum is off by an ulp of
    itself too: 4 * 2^-24 of the largest of them). Candidates apart by more than that are
    in order, equal ones in order of their index."""
    out_scores, parent, token, out_done = got
    B, W = scores.shape
    V = logits.shape[1]
    total = select_reference(logits, scores, done, eos)
    at = parent.long() * V + token.long()
    assert ((parent >= 0) & (parent < W) & (token >= 0) & (token < V)).all()
    assert all(len(set(r)) == W for r in at.tolist())
    exact = total.gather(1, at)
    finite = logits[torch.isfinite(logits)].abs().max() if torch.isfinite(logits).any() else torch.zeros(())
    size = finite.double().cpu().item() + math.log(V) + scores[torch.isfinite(scores)].abs().max().item()
    tol = 4 * 2.0 ** -24 * size
    assert torch.equal(exact == -INF, out_scores == -INF)
    live = exact != -INF
    assert ((out_scores.double() - exact)[live].abs() <= tol).all()
    best = total.sort(1, descending=True).values[:, :W]
    assert torch.equal(best == -INF, exact == -INF)
    assert ((best - exact)[live].abs() <= 2 * tol).all()
    assert torch.equal(out_done != 0, (done.gather(1, parent.long()) != 0) | (token == eos))
    dead = out_scores == -INF
    same = out_scores[:, 1:] == out_scores[:, :-1]
    assert (at[:, 1:] > at[:, :-1])[same].all()
    return at, dead


@pytest.mark.parametrize("B,W,V", [(1, 1, 1), (1, 1, 50257), (3, 4, 50257), (2, 8, 1000), (5, 5, 7), (1, 32, 33),
                                   (2, 16, 4097), (70, 3, 130), (1, 2, 200000), (2, 3, 1)])
def test_beam_select(cuda_device, B, W, V):
    gen = make_gen(B + W + V)
    if V < W and V * W < W:
        pytest.skip("fewer candidates than beams")
    logits, scores = randn(gen, B * W, V) * 3, -20 * torch.rand((B, W), generator=gen, device="cuda")
    done = (torch.rand((B, W), generator=gen, device="cuda") < 0.2).to(torch.uint8)
    for eos in (0, V - 1, -1):
        d = done if eos >= 0 else torch.zeros_like(done)
        check_select(logits, scores, d, eos, serving.beam_select(logits, scores, d, eos))


def test_beam_select_first_step_and_unused_beams(cuda_device):
    """Only beam 0 is in use: its own best tokens, in order; with a vocabulary smaller
    than the beams the rest are candidates of -inf, lowest index first."""
    logits, scores = randn(make_gen(1), 4, 1000), torch.tensor([[0.0, -INF, -INF, -INF]], device="cuda")
    done = torch.zeros((1, 4), dtype=torch.uint8, device="cuda")
    got = serving.beam_select(logits, scores, done)
    check_select(logits, scores, done, -1, got)
    assert (got[1] == 0).all() and torch.equal(got[2][0].long(), logits[0].topk(4).indices)
    got = serving.beam_select(logits[:, :3].contiguous(), scores, done)
    assert got[1].tolist() == [[0, 0, 0, 1]] and got[2][0, 3] == 0 and got[0][0, 3] == -INF


@pytest.mark.parametrize("W,V", [(4, 50257), (8, 64), (16, 5000), (32, 4096)])
def test_beam_select_ties_go_to_the_lowest(cuda_device, W, V):
    """Equal logits everywhere, and a few larger equal ones far apart."""
    logits = torch.zeros((2 * W, V), device="cuda")
    scores = torch.zeros((2, W), device="cuda")
    done = torch.zeros((2, W), dtype=torch.uint8, device="cuda")
    _, parent, token, _ = serving.beam_select(logits, scores, done)
    assert (parent == 0).all() and torch.equal(token[0].cpu(), torch.arange(W, dtype=torch.int32))
    logits[W:, [V - 1, V // 2, 5]] = 2.0
    _, parent, token, _ = serving.beam_select(logits, scores, done)
    assert (parent[0] == 0).all() and torch.equal(token[0].cpu(), torch.arange(W, dtype=torch.int32))
    want = [(w, t) for w in range(W) for t in (5, V // 2, V - 1)][:W]
    assert list(zip(parent[1].tolist(), token[1].tolist())) == want


def test_beam_select_two_zeros_are_equal(cuda_device):
    logits = torch.zeros((1, 100), device="cuda")
    logits[0, ::2] = -0.0
    got = serving.beam_select(logits, torch.zeros((1, 1), device="cuda"), torch.zeros((1, 1), dtype=torch.uint8, device="cuda"))
    assert got[2].item() == 0


@pytest.mark.parametrize("V", [300, 50257])
def test_beam_select_masked_and_broken_logits(cuda_device, V):
    """Tokens forbidden by -inf or the type's lowest value, NaN logits, whole rows of
    them, an infinite logit (its row has no candidates: inf - inf)."""
    gen = make_gen(2)
    W = 4
    logits, scores = randn(gen, 3 * W, V), -torch.rand((3, W), generator=gen, device="cuda")
    done = torch.zeros((3, W), dtype=torch.uint8, device="cuda")
    logits[:, ::3] = -INF
    logits[1, :] = torch.finfo(F32).min
    logits[2, 100:] = torch.finfo(F32).min
    logits[4, 50], logits[5, :], logits[6, :] = NAN, NAN, -INF
    logits[9, 17] = INF
    check_select(logits, scores, done, -1, serving.beam_select(logits, scores, done))
    done[2, 1] = 1
    check_select(logits, scores, done, 5, serving.beam_select(logits, scores, done, 5))


def test_beam_select_strides_and_out(cuda_device):
    gen = make_gen(3)
    wide = randn(gen, 6, 1003)
    logits = wide[:, 1:1001]  # rows that are not 16-byte aligned
    scores, done = -torch.rand((2, 3), generator=gen, device="cuda"), torch.zeros((2, 3), dtype=torch.uint8, device="cuda")
    out = (torch.empty((2, 3), device="cuda"), i32([[0] * 3] * 2), i32([[0] * 3] * 2), torch.empty_like(done))
    got = serving.beam_select(logits, scores, done, 7, out=out)
    assert got[0] is out[0]
    check_select(logits, scores, done, 7, got)
    again = serving.beam_select(logits.contiguous(), scores, done, 7)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    with pytest.raises(ValueError):
        serving.beam_select(logits, scores.double(), done)
    with pytest.raises(ValueError):
        serving.beam_select(logits[:5], scores, done)
    with pytest.raises(ValueError):
        serving.beam_select(logits, scores, done.bool())
    with pytest.raises(_lib.MtrtqError):
        serving.beam_select(logits, scores, done, 1000)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("W,page,D,lens", [(1, 16, 64, [20, 31]), (4, 16, 8, [0, 15, 16, 17]), (7, 64, 80, [100, 1]),
                                           (12, 32, 128, [70]), (32, 16, 64, [24])])
def test_beam_reorder(cuda_device, dtype, W, page, D, lens):
    gen = make_gen(W)
    B, L, KV = len(lens), 3, 2
    width = max(lens) // page + 2
    P = B * W * width + 3
    owned = torch.randperm(P, generator=torch.Generator().manual_seed(W))[:B * W * width].view(B * W, width).int().cuda()
    table = owned.clone()
    parent = torch.randint(0, W, (B, W), generator=gen, device="cuda", dtype=torch.int32)
    kp, vp = randn(gen, L, P, KV, page, D).to(dtype), randn(gen, L, P, KV, page, D).to(dtype)
    n = i32(lens)
    for _ in range(2):
        want_table, want = table.clone(), [kp.clone(), vp.clone()]
        for b in range(B):
            full, rest = divmod(lens[b], page)
            for i in range(W):
                r, s = b * W + i, b * W + int(parent[b, i])
                want_table[r, :full] = table[s, :full]
                want_table[r, full:] = owned[r, full:]
                for new, old in zip(want, (kp, vp)):
                    new[:, owned[r, full].long(), :, :rest] = old[:, owned[s, full].long(), :, :rest]
        serving.beam_reorder(parent, table, owned, n, kp, vp)
        assert torch.equal(table, want_table) and torch.equal(kp, want[0]) and torch.equal(vp, want[1])
        parent = parent.flip(1).contiguous()


def test_beam_reorder_out_of_range(cuda_device):
    """Parents outside the beams count as the beam itself; pages outside the cache and
    lengths outside the table touch nothing."""
    gen = make_gen(0)
    kp, vp = randn(gen, 4, 2, 16, 8), randn(gen, 4, 2, 16, 8)
    k0, v0 = kp.clone(), vp.clone()
    owned = i32([[0, 1], [2, 3]])
    table = owned.clone()
    serving.beam_reorder(i32([[-1, 2]]), table, owned, i32([20]), kp, vp)
    assert torch.equal(kp, k0) and torch.equal(vp, v0) and torch.equal(table, owned)
    bad = i32([[0, 99], [2, -4]])
    serving.beam_reorder(i32([[1, 0]]), table, bad, i32([20]), kp, vp)
    assert torch.equal(kp, k0) and torch.equal(vp, v0) and table.tolist() == [[2, 99], [0, -4]]
    for n in (-3, 1 << 30):
        table.copy_(owned)
        serving.beam_reorder(i32([[1, 0]]), table, owned, i32([n]), kp, vp)
        assert torch.equal(kp, k0) and torch.equal(vp, v0)


def test_beam_reorder_refusals(cuda_device):
    kp = torch.zeros((2, 4, 2, 16, 8), device="cuda")
    owned = i32([[0, 1], [2, 3]])
    ok = dict(parent=i32([[0, 1]]), table=owned, owned=owned, kv_len=i32([3]), k_pages=kp, v_pages=kp)
    for over in ({"parent": i32([[0, 1]]).long()}, {"table": owned[:1]}, {"owned": owned[:, :1]}, {"kv_len": i32([3, 3])},
                 {"k_pages": kp.half()}, {"v_pages": kp[:1]}, {"k_pages": kp[:, :, :, :8], "v_pages": kp[:, :, :, :8]}):
        with pytest.raises((ValueError, _lib.MtrtqError)):
            serving.beam_reorder(**{**ok, **over})
