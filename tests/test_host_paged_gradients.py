"""Host-only: the calls of the cache in pages have no gradient in either mode, whatever torch.no_grad() says about the other."""
import pytest
import torch
from torch.autograd import forward_ad

import oregon_gpt_oss_patching_amd as A


def _calls(dual):
    cache, table, n = A.paged_cache(4, 2, 16, device="cpu"), torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q, k = torch.zeros(1, 16, 1, 64, dtype=torch.bfloat16), torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16)
    return {
        "q": lambda: A.paged_attention(dual(q), cache, table, n, None, 0.125),
        "q, lse": lambda: A.paged_attention_forward(dual(q), cache, table, n, None, 0.125),
        "sinks": lambda: A.paged_attention(q, cache, table, n, dual(torch.zeros(16)), 0.125),
        "cache of attention": lambda: A.paged_attention(q, A.PagedCache(dual(cache.k), cache.v), table, n, None, 0.125),
        "k": lambda: A.paged_cache_write(cache, dual(k), k, table, n),
        "v": lambda: A.paged_cache_write(cache, k, dual(k), table, n),
        "cache of reading": lambda: A.paged_cache_read(A.PagedCache(cache.k, dual(cache.v)), table, n, 4),
    }


@pytest.mark.parametrize("name", sorted(_calls(None)))
@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(name, grad):
    """torch.no_grad() does not speak of forward mode: the tangent would be dropped without a word."""
    with forward_ad.dual_level(), torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="no gradient"):
        _calls(lambda t: forward_ad.make_dual(t, torch.ones_like(t)))[name]()


@pytest.mark.parametrize("name", sorted(_calls(None)))
def test_what_no_grad_takes_back(name):
    """A tensor that requires a gradient is nobody's under torch.no_grad(): the call goes on (and finds tensors of the CPU)."""
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU only"):
        _calls(lambda t: t.detach().requires_grad_())[name]()
