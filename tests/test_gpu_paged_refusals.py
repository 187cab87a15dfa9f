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


@pytest.mark.parametrize("dtype", [torch.complex64, torch.float16, torch.uint64])
def test_tables_and_lengths_that_are_no_integers(A, dtype):  # noqa: F811
    """Complex numbers lost their imaginary part, numbers of 64 bits without a sign theirs above 2^63."""
    cache, table, n = A.paged_cache(4, 2, 16), torch.zeros(1, 2, dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    q, k = torch.ones(1, 16, 1, 64, dtype=BF16, device=DEV), torch.ones(1, 2, 1, 64, dtype=BF16, device=DEV)
    odd = lambda x: x.cpu().to(dtype).to(DEV)
    for text, call in (("integer", lambda: A.paged_attention(q, cache, odd(table), n, None, SCALE)),
                       ("integer", lambda: A.paged_attention(q, cache, table, odd(n), None, SCALE)),
                       ("integer", lambda: A.paged_attention(q, cache, table, n, None, SCALE, None, odd(n))),
                       ("integer", lambda: A.paged_cache_read(cache, table, odd(n), 4)),
                       ("integer", lambda: A.paged_cache_write(cache, k, k, table, odd(n))),
                       ("integer", lambda: A.paged_cache_write(cache, k, k, table, n, odd(n)))):
        with pytest.raises(RuntimeError, match=text):
            call()
    assert not cache.k.any()


@pytest.mark.parametrize("dtype", [torch.int8, torch.uint8, torch.int16, torch.uint16, torch.uint32, torch.int64])
def test_integers_of_other_widths(A, dtype):  # noqa: F811
    cache, n = A.paged_cache(4, 2, 16), torch.full((1,), 20, dtype=torch.int32, device=DEV)
    table = torch.tensor([[3, 1]], dtype=torch.int32, device=DEV)
    k = torch.randn(1, 2, 20, 64, device=DEV).to(BF16)
    q = torch.randn(1, 16, 1, 64, device=DEV).to(BF16)
    as_is = lambda x: x.cpu().to(dtype).to(DEV)
    A.paged_cache_write(cache, k, k, as_is(table), as_is(n - 20), as_is(n))
    assert torch.equal(A.paged_cache_read(cache, as_is(table), as_is(n), 20)[0], k)
    assert torch.equal(A.paged_attention(q, cache, as_is(table), as_is(n), None, SCALE), A.paged_attention(q, cache, table, n, None, SCALE))
