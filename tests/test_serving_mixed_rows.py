"""Calls in which few requests have most of the rows: a chunk of a prompt beside single tokens
or beside requests that wait. Some requests then run in one kernel, some in another."""
import pytest
import torch

from mini_tensorrt_b200 import matmulq, serving
from tests.test_serving import BF16, F32, TYPES, Paged, i32, make_gen, near, offsets, reference, rows

pytestmark = pytest.mark.gpu

HEADS = [(4, 4, 64), (4, 2, 64), (8, 2, 128), (8, 1, 40)]
# few rows on average (with the group); requests of up to 18 tokens and of 63 to 66, around the
# numbers where the kernel changes, and of none
MIXES = {"decode": ([1] * 40, [7 + 31 * i for i in range(40)]),
         "chunk_beside_decode": ([1] * 30 + [40] + [1] * 33, [3 + 11 * i for i in range(64)]),
         "chunk_beside_waiting": ([0] * 50 + [3, 65, 0, 1], [9] * 50 + [500, 777, 80, 130]),
         "around": ([4, 5, 15, 16, 17, 18] + [0, 1] * 30, [4, 300, 15, 140, 129, 18] + [20, 33] * 30),
         "longer": ([63, 64, 65, 66, 1] + [0] * 150, [63, 100, 65, 300, 7] + [20] * 150),
         "only_chunks": ([0] * 60 + [20, 21, 0], [5] * 60 + [600, 21, 8]),
         "before_the_first": ([0] * 60 + [20, 6, 2], [5] * 60 + [11, 3, 1])}


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("mix", MIXES)
def test_mixed_rows(cuda_device, kind, heads, mix):
    new, lens = MIXES[mix]
    s = Paged(new, lens, *heads, 16, kind, seed=41)
    space = torch.full((s.q.shape[0] + 8, *s.q.shape[1:]), 7.0, dtype=s.kp.dtype, device="cuda")
    got = s.run(out=space[4:-4])
    s.verify(got)
    assert (space[:4] == 7).all() and (space[-4:] == 7).all()
    assert torch.equal(s.run(), got)


@pytest.mark.parametrize("kind", TYPES)
def test_mixed_rows_with_pages_that_hold_the_tokens(cuda_device, kind):
    new, lens = MIXES["around"]
    s = Paged(new, lens, 6, 3, 64, 32, kind, seed=42, hold=True)
    s.k = s.v = None
    s.verify(s.run(scale=0.2), scale=0.2)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads", [(4, 4, 64), (8, 2, 128)], ids=str)
def test_mixed_prompts(cuda_device, kind, heads):
    H, KV, D = heads
    lens = [1] * 30 + [0] * 90 + [150, 16, 17]
    q, k, v = rows(make_gen(43), sum(lens), H, KV, D, kind)
    held = TYPES[kind][1]
    got = serving.prompt_attention(q, k, v, i32(offsets(lens)), out_dtype=held)
    for a, n in zip(offsets(lens), lens):
        s = slice(a, a + n)
        if n:
            near(got[s], *reference(q[s], k[s].to(held), v[s].to(held), range(1, n + 1), D ** -0.5), kind, D,
                 range(1, n + 1))
    assert matmulq.read_device_status() == 0


@pytest.mark.parametrize("kind", TYPES)
def test_mixed_rows_in_a_graph(cuda_device, kind):
    """The bounds are read by each replay: requests change kernels from one to the next."""
    new, lens = MIXES["chunk_beside_waiting"]
    s = Paged(new, lens, 4, 2, 64, 16, kind, seed=44)
    out, ws = torch.empty_like(s.run()), torch.zeros(1 << 26, dtype=torch.uint8, device="cuda")
    want = s.run().clone()
    s.cu.copy_(i32([min(x, 33) for x in range(len(new))] + [69]))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        s.run(out=out, workspace=ws)
    s.cu.copy_(i32(offsets(new)))
    for _ in range(2):
        out.zero_()
        g.replay()
        assert torch.equal(out, want)


@pytest.mark.parametrize("x,held,heads", [(F32, BF16, (12, 12, 64)), (BF16, BF16, (16, 8, 64)), (F32, F32, (12, 12, 64)),
                                          (F32, F32, (8, 2, 128))], ids=str)
def test_requests_that_wait_cost_a_chunk_little(cuda_device, x, held, heads):
    """511 requests without rows beside a chunk of 512 tokens over 8192: once 5 to 36 times as
    long as the chunk alone, which ran in tiles of a row or two."""
    H, KV, D = heads
    m, n, page = 512, 8192, 64
    p = torch.randn((m, (H + 2 * KV) * D), generator=make_gen(45), device="cuda").to(x)
    q, k, v = p.split([H * D, KV * D, KV * D], 1)
    q, k, v = q.view(m, H, D), k.view(m, KV, D), v.view(m, KV, D)
    kp, vp = (torch.zeros((n // page, KV, page, D), dtype=held, device="cuda") for _ in range(2))
    table = torch.arange(n // page, dtype=torch.int32, device="cuda").repeat(512, 1)
    ws = torch.zeros(1 << 27, dtype=torch.uint8, device="cuda")

    def took(lens, cu):
        lens, cu, times = i32(lens), i32(cu), []
        call = lambda: serving.paged_attention(q, k, v, kp, vp, table[:len(lens)], lens, cu, workspace=ws)
        for _ in range(7):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(5):
                call()
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return sorted(times)[3]

    alone = took([n], [0, m])
    assert took([16] * 511 + [n], [0] * 512 + [m]) < 3 * alone
