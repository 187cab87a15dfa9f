"""GPU tests of attention over pages where a row's work is cut into shares: each number of column blocks, few and many shares, windows that begin inside a row.
Each case is checked to be cut (it asks for scratch), and one beside it not to be."""
import ctypes

import pytest
import torch

from oregon_gpt_oss_patching_amd import _lib
from test_gpu_paged import BF16, DEV, E4M3, FP32, TYPE_IDS, TYPES, A, check, make  # noqa: F401

pytestmark = pytest.mark.gpu
CODE = {BF16: _lib.DTYPE_BF16, FP32: _lib.DTYPE_FP32, E4M3: _lib.DTYPE_E4M3}


def scratch_bytes(cache, table, q, window=0, max_len=0):
    """Scratch that the library asks for: none where rows are not cut."""
    p = _lib.PagedParams()
    p.struct_size = ctypes.sizeof(p)
    p.dtype, p.storage, p.D, p.scale = CODE[q.dtype], CODE[cache.k.dtype], 64, 0.125
    p.B, p.H, p.Sq = q.shape[0], q.shape[1], q.shape[2]
    p.pages, p.G, p.page_size = cache.k.shape[:3]
    p.table_width, p.window, p.max_len = table.shape[1], window, max_len
    return _lib.load().gptoss_attn_paged_workspace_bytes(ctypes.byref(p))


@pytest.mark.parametrize("dtype,storage", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("lens,h,g,sq,w", [
    ([5000, 3000, 40], 16, 2, 1, 0),            # one block of columns (8 pairs)
    ([5000, 77], 16, 2, 3, 0),                  # 24 pairs: two blocks, few shares
    ([9000], 8, 1, 4, 0),                       # 32 pairs: two blocks, many shares of a row
    ([6000] + [2500, 31] * 8, 16, 2, 4, 0),     # the same in a batch
    ([5000, 77], 16, 2, 5, 0),                  # 40: three
    ([9000], 8, 1, 8, 0),                       # 64: four
    ([5000, 333], 17, 1, 1, 0),                 # 17 heads: the second block holds one
    ([9000, 5200], 8, 1, 1, 2500),              # windows: shares that begin inside a row
    ([5200, 8000, 2700, 100], 16, 2, 1, 2900),
    ([9000, 5200], 16, 2, 3, 2500),
    ([5200, 100, 7001], 8, 1, 5, 2047),
    ([6000, 2400], 8, 1, 8, 2333),
    ([5000, 4100], 8, 1, 20, 1999),             # several blocks of pairs, each with keys of its own
])
def test_cut_rows(A, dtype, storage, lens, h, g, sq, w):  # noqa: F811
    print(f"case {dtype} {storage} lens={lens} H={h} G={g} Sq={sq} window={w}", flush=True)
    cache, table, n, q, sinks, _, _ = make(A, 81 + sum(lens) + sq + w, lens, h, g, sq, 16, dtype, storage, 1)
    assert scratch_bytes(cache, table, q, w) > 0
    check(A, cache, table, n, q, sinks, w)
    # queries that start elsewhere, the last of them behind some of the rows
    check(A, cache, table, n, q, sinks, w, [max(-2, x - sq - 1 + 2 * i) for i, x in enumerate(lens)])


@pytest.mark.parametrize("dtype,storage", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("sq,w", [(1, 0), (3, 0), (3, 2100)])
def test_missing_pages_of_cut_rows(A, dtype, storage, sq, w):  # noqa: F811
    """Entries that name no page, whole shares of them among them."""
    lens = [5000, 2600]
    cache, table, n, q, sinks, _, _ = make(A, 83 + sq, lens, 16, 2, sq, 16, dtype, storage)
    table[0, 40:140] = -1
    table[0, 200] = 10 ** 6
    table[1, :100] = -1
    table[0, 311] = -1
    assert scratch_bytes(cache, table, q, w) > 0
    check(A, cache, table, n, q, sinks, w)


@pytest.mark.parametrize("dtype,storage", TYPES, ids=TYPE_IDS)
def test_what_is_cut(A, dtype, storage):  # noqa: F811
    """Short rows take no scratch; the same rows under a longest length that is given as short do not either."""
    cache, table, n, q, sinks, _, _ = make(A, 85, [250, 33], 16, 2, 3, 16, dtype, storage)
    assert scratch_bytes(cache, table, q) == 0
    wide = torch.cat([table, torch.full((2, 1000), -1, dtype=torch.int32, device=DEV)], dim=1)
    assert scratch_bytes(cache, wide, q) > 0 and scratch_bytes(cache, wide, q, 0, 256) == 0
    for t, max_len in ((table, None), (wide, None), (wide, 256)):
        check(A, cache, t, n, q, sinks, 0, None, max_len)
