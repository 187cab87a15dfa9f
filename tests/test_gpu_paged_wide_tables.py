"""GPU tests of tables far wider than their rows: the same division of work as with a table that fits, and the same results."""
import ctypes

import pytest
import torch

from oregon_gpt_oss_patching_amd import _lib
from test_gpu_paged import BF16, DEV, E4M3, FP32, SCALE, TYPE_IDS, TYPES, A, check, make  # noqa: F401

pytestmark = pytest.mark.gpu
CODE = {BF16: _lib.DTYPE_BF16, FP32: _lib.DTYPE_FP32, E4M3: _lib.DTYPE_E4M3}


def _strides(s, t):
    s.b, s.h, s.s = t.stride(0), t.stride(1), t.stride(2)


def shares(cache, table, n, q):
    """(first share, how many) of each unit, which the kernel leaves at the scratch's beginning; None where there is no scratch."""
    p = _lib.PagedParams()
    p.struct_size = ctypes.sizeof(p)
    p.dtype, p.storage, p.sinks_dtype, p.D, p.scale = CODE[q.dtype], CODE[cache.k.dtype], _lib.DTYPE_FP32, 64, SCALE
    p.B, p.H, p.Sq = q.shape[0], q.shape[1], q.shape[2]
    p.pages, p.G, p.page_size = cache.k.shape[:3]
    p.table_width, p.table_stride = table.shape[1], table.stride(0)
    p.k_pages, p.v_pages, p.page_table, p.seqlens = cache.k.data_ptr(), cache.v.data_ptr(), table.data_ptr(), n.data_ptr()
    _strides(p.k_page_stride, cache.k)
    _strides(p.v_page_stride, cache.v)
    if cache.k_exp is not None:
        p.k_exp, p.v_exp = cache.k_exp.data_ptr(), cache.v_exp.data_ptr()
        _strides(p.k_exp_stride, cache.k_exp)
        _strides(p.v_exp_stride, cache.v_exp)
    o = torch.empty_like(q)
    p.q, p.o = q.data_ptr(), o.data_ptr()
    _strides(p.q_stride, q)
    _strides(p.o_stride, o)
    lib = _lib.load()
    p.scratch_bytes = lib.gptoss_attn_paged_workspace_bytes(ctypes.byref(p))
    if not p.scratch_bytes:
        return None
    scratch = torch.full((p.scratch_bytes // 4,), -1, dtype=torch.int32, device=DEV)
    p.scratch = scratch.data_ptr()
    assert lib.gptoss_attn_paged_fwd(ctypes.byref(p), torch.cuda.current_stream().cuda_stream) == 0
    pairs = p.Sq * p.H // p.G
    blocks = -(-pairs // (16 * min(-(-pairs // 16), 2 if q.dtype == FP32 else 4)))
    return scratch[:2 * p.B * blocks].view(-1, 2).tolist()


@pytest.mark.parametrize("dtype,storage", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("lens,h,g,sq", [
    ([2049], 64, 8, 1),
    ([2049], 64, 8, 5),
    ([5000], 64, 8, 1),
    ([6000, 700, 0, 2500], 32, 4, 1),
    ([6000, 700, 0, 2500], 32, 4, 4),
    ([4000, 3999] * 4, 16, 2, 1),
    ([2600] + [5, 900] * 40, 16, 2, 1),              # more units than a wavefront has lanes
    ([7000], 8, 1, 17),                              # blocks of pairs, each with keys of its own
])
def test_shares_follow_the_lengths(A, dtype, storage, lens, h, g, sq):  # noqa: F811
    print(f"case {dtype} {storage} rows={len(lens)} H={h} G={g} Sq={sq}", flush=True)
    cache, table, n, q, sinks, _, _ = make(A, 91 + sum(lens) + sq, lens, h, g, sq, 16, dtype, storage)
    q = q.to(DEV)
    fits = shares(cache, table, n, q)
    for width in (10000, 131072):
        wide = torch.cat([table, torch.full((len(lens), width // 16 - table.shape[1]), -1, dtype=torch.int32, device=DEV)], dim=1)
        assert shares(cache, wide, n, q) == fits
    check(A, cache, wide, n, q.cpu(), sinks)
    # shares in a row, one at least for each unit
    at = 0
    for first, count in fits:
        assert first == at and count >= 1
        at += count
    assert at > len(fits)
