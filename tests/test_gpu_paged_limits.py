"""GPU tests of attention over pages at the longest tables, 2^30 tokens, of which all but the first and the last page are missing."""
import pytest
import torch

from oracle import paged_ref as P
from test_gpu_paged import BF16, DEV, SCALE, TYPE_IDS, TYPES, A, make, values  # noqa: F401

pytestmark = pytest.mark.gpu
LONGEST, PAGE = 1 << 30, 1024


def both_ends(A, dtype, storage, sq):  # noqa: F811
    """A cache of two pages, the table of a row of 2048 tokens and that of a row of 2^30 which has only its ends."""
    cache, table, n, q, sinks, k, v = make(A, 51 + sq, [2 * PAGE], 4, 1, sq, PAGE, dtype, storage)
    far = torch.full((1, LONGEST // PAGE), -1, dtype=torch.int32, device=DEV)
    far[0, 0], far[0, -1] = table[0, 0], table[0, 1]
    return cache, table, far, n, q, sinks, k, v


@pytest.mark.parametrize("dtype,storage", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("sq", [1, 5])
def test_the_last_query_sees_the_first_key(A, dtype, storage, sq):  # noqa: F811
    """Without a window, and with one of 2^30, the query at position 2^30 - 1 sees key 0; with one of 2^30 - 1 it does not."""
    print(f"case {dtype} {storage} Sq={sq}", flush=True)
    cache, table, far, n, q, sinks, k, v = both_ends(A, dtype, storage, sq)
    # a first key that outweighs the others
    k[:, :, 0], v[:, :, 0] = q[:, :1, -1] * 2, 9.0
    A.paged_cache_write(cache, k.to(DEV), v.to(DEV), table, [0])
    for far_window, window in ((None, 0), (LONGEST, 0), (LONGEST - 1, 2 * PAGE - 1)):
        o, lse = A.paged_attention_forward(q.to(DEV), cache, far, [LONGEST], sinks.to(DEV), SCALE, far_window)
        ref, ref_lse, terms = P.attention(q, *values(cache), table.cpu(), n.cpu(), sinks, SCALE, window)
        tol, tol_lse = P.bounds(ref, ref_lse, terms, dtype)
        assert bool(((o.cpu().double() - ref).abs() <= tol).all()) and bool(((lse.cpu().double() - ref_lse).abs() <= tol_lse).all()), far_window


def test_an_infinite_first_value(A):  # noqa: F811
    """Rows that not every query sees: without a window both do, with one of 2^30 - 1 only the query at 2^30 - 2."""
    cache, table, far, n, q, sinks, k, v = both_ends(A, BF16, BF16, 2)
    v[0, 0, 0, 7] = float("inf")
    A.paged_cache_write(cache, k.to(DEV), v.to(DEV), table, [0])
    for window, seen in ((None, (True, True)), (LONGEST - 1, (True, False))):
        o = A.paged_attention(q.to(DEV), cache, far, [LONGEST], sinks.to(DEV), SCALE, window)
        others = [i for i in range(64) if i != 7]
        assert torch.isfinite(o[..., others]).all()
        for i, s in enumerate(seen):
            assert bool(((o[0, i, :, 7] == float("inf")) == s).all()), (window, i)
