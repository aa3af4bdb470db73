"""The serving operators at the ends of what they accept: groups of up to 128 heads (one token
fills a tile slot from 65 on) and 1024 requests."""
import pytest
import torch

from mini_tensorrt_b200 import _lib, matmulq, serving
from tests.test_serving import INF, NAN, TYPES, Paged, i32, make_gen, near, offsets, reference, rows

pytestmark = pytest.mark.gpu

GROUPS = [(24, 1, 64), (64, 2, 64), (48, 1, 40), (64, 1, 128), (65, 1, 64), (96, 1, 128), (128, 1, 64), (256, 2, 128)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads", GROUPS, ids=str)
@pytest.mark.parametrize("lens", [[1, 2, 0, 131], [300]], ids=str)
def test_prompt_wide_groups(cuda_device, kind, heads, lens):
    H, KV, D = heads
    q, k, v = rows(make_gen(31), sum(lens), H, KV, D, kind)
    held = TYPES[kind][1]
    got = serving.prompt_attention(q, k, v, i32(offsets(lens)), out_dtype=held)
    for a, n in zip(offsets(lens), lens):
        s = slice(a, a + n)
        if n:
            near(got[s], *reference(q[s], k[s].to(held), v[s].to(held), range(1, n + 1), D ** -0.5), kind, D,
                 range(1, n + 1))
    assert matmulq.read_device_status() == 0


# Two tokens whose first sees whole blocks of 128 keys, and so on: neighbouring slots that see
# different numbers of blocks.
CHUNKS = [([2, 2, 3, 1], [129, 257, 130, 128]), ([5, 0, 2], [385, 7, 1025]), ([130], [260])]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads", GROUPS, ids=str)
@pytest.mark.parametrize("new,lens", CHUNKS, ids=str)
def test_paged_wide_groups(cuda_device, kind, heads, new, lens):
    s = Paged(new, lens, *heads, 32, kind, seed=32)
    s.verify(s.run())


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads", [(64, 1, 64), (65, 1, 64), (128, 1, 128)], ids=str)
@pytest.mark.parametrize("bad", [NAN, INF])
def test_wide_groups_hidden_values(cuda_device, kind, heads, bad):
    """The last token of each request is broken: the rows before keep their bits, its own
    row's dimension is what it holds."""
    new, lens = CHUNKS[0]
    a, b = Paged(new, lens, *heads, 16, kind, seed=33), Paged(new, lens, *heads, 16, kind, seed=33)
    want = a.run()
    last = [x - 1 for x in offsets(new)[1:]]
    b.v[last, :, 3] = bad
    got = b.run()
    before = [x for x in range(sum(new)) if x not in last]
    assert torch.equal(got[before], want[before])
    assert not torch.isfinite(got[last, :, 3].float()).any()
    got[last, :, 3] = want[last, :, 3]
    assert torch.equal(got, want)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads", [(2, 2, 64), (4, 1, 32)], ids=str)
def test_most_requests(cuda_device, kind, heads):
    B = _lib.MAX_BATCH
    s = Paged([3 if i % 97 == 5 else i % 5 != 0 for i in range(B)], [3 + (41 * i) % 150 for i in range(B)], *heads, 16,
              kind, seed=34)
    s.verify(s.run())
    q, k, v = s.q, s.k, s.v
    got = serving.prompt_attention(q, k, v, s.cu, out_dtype=s.kp.dtype)
    for a, n in zip(offsets(s.new), s.new):
        if n == 3:
            r = slice(a, a + n)
            near(got[r], *reference(q[r], k[r].to(got.dtype), v[r].to(got.dtype), range(1, n + 1), s.D ** -0.5), kind,
                 s.D, range(1, n + 1))
