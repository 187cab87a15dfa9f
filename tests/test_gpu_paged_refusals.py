"""GPU tests of what the calls of the cache in pages refuse where they go past the dispatcher."""
import pytest
import torch
from torch.autograd import forward_ad

from test_gpu_paged import BF16, DEV, E4M3, SCALE, A  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grad", [True, False])
def test_tangents(A, grad):  # noqa: F811
    """A forward-mode tangent is refused under torch.no_grad() too, and nothing is written; without one the same tensors pass."""
    cache, table, n = A.paged_cache(4, 2, 16), torch.zeros(1, 2, dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    q, k = torch.ones(1, 16, 1, 64, dtype=BF16, device=DEV), torch.ones(1, 2, 1, 64, dtype=BF16, device=DEV)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        for call in (lambda d: A.paged_attention(d(q), cache, table, n, None, SCALE),
                     lambda d: A.paged_attention_forward(q, cache, table, n, d(torch.zeros(16, device=DEV)), SCALE),
                     lambda d: A.paged_cache_write(cache, k, d(k), table, n - 1),
                     lambda d: A.paged_cache_read(A.PagedCache(cache.k, d(cache.v)), table, n, 4)):
            with pytest.raises(RuntimeError, match="no gradient"):
                call(lambda t: forward_ad.make_dual(t, torch.ones_like(t)))
            assert not cache.k.any()
        for call in (lambda d: A.paged_attention(d(q), cache, table, n, None, SCALE), lambda d: A.paged_cache_write(cache, d(k), d(k), table, n - 1)):
            call(lambda t: forward_ad.unpack_dual(forward_ad.make_dual(t, torch.ones_like(t))).primal)
        assert bool((cache.k[0, :, 0] == 1).all())


@pytest.mark.parametrize("storage", [BF16, E4M3])
def test_a_cache_made_in_inference_mode(A, storage):  # noqa: F811
    """Outside of inference mode its writes are refused, as torch refuses such a tensor's in-place operations, and then nothing has been written; reads go on."""
    with torch.inference_mode():
        cache = A.paged_cache(2, 1, 16, storage)
    table, k, n = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.ones(1, 1, 4, 64, dtype=BF16, device=DEV), torch.full((1,), 4, dtype=torch.int32, device=DEV)
    with torch.no_grad(), pytest.raises(RuntimeError, match="inference"):
        A.paged_cache_write(cache, k, k, table, n - 4)
    for t in cache:
        assert t is None or not t.view(torch.uint8).any()
    with torch.no_grad():
        assert not A.paged_cache_read(cache, table, n, 4)[0].any()
    with torch.inference_mode():
        A.paged_cache_write(cache, k, k, table, n - 4)
        assert torch.equal(A.paged_cache_read(cache, table, n, 4)[1], k)


def test_written_caches_have_a_new_version(A):  # noqa: F811
    cache = A.paged_cache(2, 1, 16, E4M3)
    table, k = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.ones(1, 1, 4, 64, dtype=BF16, device=DEV)
    before = [t._version for t in cache]
    A.paged_cache_write(cache, k, k, table, [0])
    assert all(t._version == v + 1 for t, v in zip(cache, before))
