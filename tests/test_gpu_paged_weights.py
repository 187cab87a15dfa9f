"""GPU tests of the weights that attention over pages multiplies V with: as exact as float32 asks, whatever the queries' type."""
import pytest
import torch

from oracle import paged_ref as P
from test_gpu_paged import BF16, DEV, E4M3, FP32, SCALE, TYPE_IDS, TYPES, A, make, values  # noqa: F401

pytestmark = pytest.mark.gpu


def bounds(ref, ref_lse, terms, dtype):
    """`oracle.paged_ref.bounds` with the weights in 16 bits instead of 8: float32's roundings of logits, weights and sums, the rounding of o itself (2^-8 of it
    in bfloat16, 2^-24 in float32), and of a weight that is held as two bfloat16 terms.  The second of them is what the first leaves, at most 2^-7 of the
    weight, and is rounded by half a step, 2^-8 of itself: 2^-15 of the weight."""
    tol, _ = P.bounds(ref, ref_lse, terms, FP32)
    if dtype == BF16:
        tol = tol + 1.01 * (2.0 ** -15 * terms[0] + 2.0 ** -8 * ref.abs())
    return tol


@pytest.mark.parametrize("dtype,storage", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("lens,h,g,sq,w", [
    ([40, 7, 300], 8, 1, 1, 0),                 # one block of columns, short rows
    ([900, 1000], 16, 2, 1, 0),                 # sixteen wavefronts
    ([5000, 700], 16, 2, 1, 0),                 # cut
    ([300, 33], 8, 1, 3, 20),                   # two blocks
    ([4000, 100], 8, 1, 4, 0),
    ([300, 50], 8, 1, 5, 0),                    # three
    ([4000, 100], 8, 1, 6, 3000),
    ([300, 50], 8, 1, 8, 0),                    # four
    ([4000, 129], 8, 1, 8, 0),
])
def test_weights_in_sixteen_bits(A, dtype, storage, lens, h, g, sq, w):  # noqa: F811
    """Sums of many keys cancel, so an error of the weights stands out against a result that is small."""
    print(f"case {dtype} {storage} lens={lens} H={h} G={g} Sq={sq} window={w}", flush=True)
    cache, table, n, q, sinks, _, _ = make(A, 41 + sum(lens) + sq, lens, h, g, sq, 16, dtype, storage)
    o = A.paged_attention(q.to(DEV), cache, table, n, sinks.to(DEV), SCALE, w or None).cpu().double()
    ref, ref_lse, terms = P.attention(q, *values(cache), table.cpu(), n.cpu(), sinks, SCALE, w)
    over = (o - ref).abs() - bounds(ref, ref_lse, terms, dtype)
    assert bool((over <= 0).all()), float(over.max())


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("n", [20, 700, 3000])
def test_infinities_that_every_query_sees(A, dtype, n):  # noqa: F811
    """A weight times infinity is infinity with its sign, in the columns that hold one, whatever the weight; the other columns are as without it.  bfloat16's V
    stands in float32's cache as the same numbers."""
    cache, table, m, q, sinks, k, v = make(A, 43 + n, [n], 8, 2, 1, 16, dtype, dtype)
    v = v.clone()
    v[0, :, 5] = v[0, :, 5].sign()                        # (a finite row for comparison)
    A.paged_cache_write(cache, k.to(DEV), v.to(DEV), table, [0])
    plain = A.paged_attention(q.to(DEV), cache, table, m, sinks.to(DEV), SCALE)
    v[0, :, 5, 3], v[0, :, 5, 40] = float("inf"), -float("inf")
    A.paged_cache_write(cache, k.to(DEV), v.to(DEV), table, [0])
    o = A.paged_attention(q.to(DEV), cache, table, m, sinks.to(DEV), SCALE)
    assert bool((o[..., 3] == float("inf")).all()) and bool((o[..., 40] == -float("inf")).all())
    others = [i for i in range(64) if i not in (3, 40)]
    assert torch.equal(o[..., others], plain[..., others])
