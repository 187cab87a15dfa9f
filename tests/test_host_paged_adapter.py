"""Host-only: what hip_flash_attention(paged=) refuses before anything is written."""
from types import SimpleNamespace

import pytest
import torch

import oregon_gpt_oss_patching_amd as A

MODULE = SimpleNamespace(sinks=torch.zeros(16), sliding_window=None, layer_idx=0)


def _state(start):
    ints = torch.ones(1, dtype=torch.int32)
    return A.PagedState([A.paged_cache(4, 2, 16, device="cpu")], torch.zeros(1, 2, dtype=torch.int32), start, ints)


@pytest.mark.parametrize("start", [None, torch.zeros(1, dtype=torch.int32)])
@pytest.mark.parametrize("keys", [0, 1, 9])
def test_keys_of_the_past_are_refused(start, keys):
    """With past_key_values the layer's keys are the whole past's, which would be written again from `start` on."""
    q, k = torch.zeros(1, 16, 3, 64, dtype=torch.bfloat16), torch.zeros(1, 2, keys, 64, dtype=torch.bfloat16)
    with torch.no_grad(), pytest.raises(RuntimeError, match="as many as queries"):
        A.hip_flash_attention(MODULE, q, k, k, None, 0.125, paged=_state(start))


def test_as_many_keys_as_queries_pass():
    q, k = torch.zeros(1, 16, 3, 64, dtype=torch.bfloat16), torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16)
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU only"):
        A.hip_flash_attention(MODULE, q, k, k, None, 0.125, paged=_state(None))


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_lengths_as_a_mask_are_refused(dtype):
    """Without pages a 1-D attention_mask of integers is the rows' lengths, and seqlens= is refused with them: neither is dropped."""
    x = torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16)
    with torch.no_grad(), pytest.raises(RuntimeError, match="lengths as attention_mask"):
        A.hip_flash_attention(MODULE, x, x, x, torch.full((1,), 2, dtype=dtype), 0.125, paged=_state(None))


def test_other_masks_are_ignored_as_without_pages():
    q, k = torch.zeros(1, 16, 3, 64, dtype=torch.bfloat16), torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16)
    for mask in (torch.ones(1, 3, dtype=torch.int64), torch.zeros(1, 1, 3, 3), torch.zeros(3)):
        with torch.no_grad(), pytest.raises(RuntimeError, match="GPU only"):
            A.hip_flash_attention(MODULE, q, k, k, mask, 0.125, paged=_state(None))
