"""f32 rows over a bf16 cache: q keeps 16 bits on the tensor cores, so that scores of tens are
right to a thousandth.

Tolerance: as in tests/test_serving.py for bf16 (u = 2^-9), with what is left of q's roundings
in place of one to bf16. The first plane cuts q by less than 2^-7 of itself, the second rounds
that by up to 2^-9: a score of S is off by 2^-16 S / sqrt(3) in the mean, a weight by as much of
itself, six standard deviations of which are 2^-14.2 S < u S / 32:
|error| <= u (|ref| + V (2 + S / 32)), and the errors' norm is at most 2^-8 of the result's."""
import pytest
import torch

from mini_tensorrt_b200 import matmulq, serving
from tests.test_serving import BF16, F32, INF, NAN, Paged, i32, make_gen, offsets, reference, rows

pytestmark = pytest.mark.gpu


def near(got, ref, S, V):
    got = got.double()
    assert ((got - ref).abs() <= 2.0 ** -9 * (ref.abs() + V * (2 + S / 32))).all()
    assert (got - ref).norm() <= 2.0 ** -8 * ref.norm()


@pytest.mark.parametrize("heads", [(4, 4, 64), (8, 2, 128), (6, 2, 80), (5, 1, 40), (24, 1, 64), (65, 1, 128)], ids=str)
@pytest.mark.parametrize("lens", [[3, 128, 129], [700], [1] * 40 + [200]], ids=["few", "long", "many"])
@pytest.mark.parametrize("factor", [1, 10])
def test_prompts(cuda_device, heads, lens, factor):
    H, KV, D = heads
    q, k, v = rows(make_gen(51), sum(lens), H, KV, D, "mixed")
    q *= factor
    got = serving.prompt_attention(q, k, v, i32(offsets(lens)), out_dtype=BF16)
    for a, n in zip(offsets(lens), lens):
        s = slice(a, a + n)
        near(got[s], *reference(q[s], k[s].to(BF16), v[s].to(BF16), range(1, n + 1), D ** -0.5))
    assert matmulq.read_device_status() == 0


@pytest.mark.parametrize("heads", [(4, 4, 64), (8, 2, 128), (12, 2, 80), (32, 1, 64), (128, 1, 128)], ids=str)
@pytest.mark.parametrize("new,lens", [([1, 1, 1], [900, 33, 128]), ([130, 1, 0, 70, 257], [700, 40, 9, 70, 1500]),
                                      ([0] * 40 + [60, 1, 2], [7] * 40 + [1111, 50, 2])], ids=["decode", "chunks", "waiting"])
@pytest.mark.parametrize("factor", [1, 10])
def test_paged(cuda_device, heads, new, lens, factor):
    s = Paged(new, lens, *heads, 32, "mixed", seed=52)
    s.q *= factor
    got = s.run()
    for b, (m, n) in enumerate(zip(new, lens)):
        a = offsets(new)[b]
        if m:
            near(got[a:a + m], *reference(s.q[a:a + m], s.keys[b], s.values[b], [n - m + t + 1 for t in range(m)],
                                          s.D ** -0.5))


@pytest.mark.parametrize("heads", [(2, 2, 64), (8, 2, 128)], ids=str)
@pytest.mark.parametrize("value", [1.0, 1.00390625, 0.3, 1e-30, 3e38])
def test_infinite_keys_meet_both_planes(cuda_device, heads, value):
    """An infinite element of a key makes a score of the infinity that q's sign there gives,
    whether or not q's second plane has anything left: -infinity counts for nothing, +infinity
    makes the row NaN; so does a zero q."""
    H, KV, D = heads
    n, at = 200, 70
    q, k, v = rows(make_gen(53), n, H, KV, D, "mixed")
    q, k = q.clone(), k.clone()
    q[..., 5] = -value
    k[..., 5] = 0.0
    q[150, :, 5], q[160, :, 5], q[170, :, 5] = value, 0.0, -0.0
    k[at, :, 5] = INF
    got = serving.prompt_attention(q, k, v, i32([0, n]), out_dtype=BF16)
    assert got[[150, 160, 170]].isnan().all()
    keep = torch.arange(n, device="cuda") != at
    fine = [i for i in range(n) if i not in (150, 160, 170)]
    ref, S, V = reference(q, k[keep].to(BF16), v[keep].to(BF16), [i + 1 - (i >= at) for i in range(n)], D ** -0.5)
    near(got[fine], ref[fine], S[fine], V[fine])


@pytest.mark.parametrize("heads", [(2, 2, 64), (8, 2, 128)], ids=str)
def test_infinite_and_nan_q_meet_both_planes(cuda_device, heads):
    """An infinite q gives the infinity of its key's sign (counting for nothing where it is
    negative), and the largest numbers stay finite."""
    H, KV, D = heads
    n = 150
    q, k, v = rows(make_gen(54), n, H, KV, D, "mixed")
    q, k = q.clone(), k.clone()
    k[..., 5] = -1.0
    k[3, :, 5] = 2.0
    q[40, :, 5], q[50, :, 5] = INF, NAN
    q[60], q[60, :, 5] = 0.0, torch.finfo(F32).max
    k[4, :, 5] = -2.0 ** -126
    got = serving.prompt_attention(q, k, v, i32([0, n]), out_dtype=BF16)
    assert got[[40, 50]].isnan().all()  # +infinity at key 3
    k[:, :, 5] = -k[:, :, 5].abs()
    want = serving.prompt_attention(q, k, v, i32([0, n]), out_dtype=BF16)
    assert torch.isfinite(got[61:].float()).all() and torch.isfinite(want[:40].float()).all()
    # only key 4 has more than -3e38 there
    torch.testing.assert_close(want[60], v[4].to(BF16).repeat_interleave(H // KV, 0), rtol=0, atol=0)
