"""Host-only checks of the page tables: the parameter block mirrors the header, arguments are refused with their codes before anything is launched.  No kernel is launched."""
import ctypes
import os
import re

import pytest
import torch

import oregon_gpt_oss_patching_amd as A
from oregon_gpt_oss_patching_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
UPDATE, MAP = 0, 1


def test_struct_mirror_matches_header_field_order():
    text = open(os.path.join(ROOT, "include", "gptoss_attn.h")).read()
    body = re.search(r"typedef struct gptoss_attn_table_params \{(.*?)\} gptoss_attn_table_params;", text, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = []
    for decl in body.split(";"):
        for part in decl.strip().split(","):
            if part.strip():
                names.append(re.findall(r"[A-Za-z_][A-Za-z_0-9]*", part)[-1])
    assert names == [f[0] for f in _lib.TableParams._fields_]


def _params():
    """A block that passes (fake addresses, never dereferenced)."""
    p = _lib.TableParams()
    p.struct_size = ctypes.sizeof(p)
    p.B, p.table_width, p.page_size, p.pages, p.total, p.table_stride = 3, 4, 16, 10, 5, 4
    for f in ("page_table", "have", "want", "seqlens", "left", "row", "position", "first", "slot", "used"):
        setattr(p, f, 0x1000)
    return p


@pytest.mark.parametrize("field,value,code,calls", [
    (None, None, 0, (UPDATE, MAP)), ("struct_size", 8, -9, (UPDATE, MAP)), ("B", 0, -5, (UPDATE, MAP)), ("B", 16385, -5, (UPDATE, MAP)), ("page_size", 8, -11, (UPDATE, MAP)),
    ("page_size", 48, -11, (UPDATE, MAP)), ("page_size", 2048, -11, (UPDATE, MAP)), ("table_width", 0, -11, (UPDATE, MAP)), ("table_width", 2 ** 26 + 1, -11, (UPDATE, MAP)),
    ("table_stride", 3, -11, (UPDATE,)), ("table_stride", 0, 0, (MAP,)), ("table_stride", -4, -11, (UPDATE, MAP)), ("pages", 0, -11, (UPDATE,)), ("pages", 2 ** 30 + 1, -11, (UPDATE,)),
    ("total", -1, -5, (MAP,)), ("total", 2 ** 30 + 1, -5, (MAP,)), ("total", 0, 0, (MAP,)), ("page_table", None, -2, (UPDATE, MAP)), ("have", None, -2, (UPDATE, MAP)),
    ("want", 0x1002, -7, (UPDATE, MAP)), ("seqlens", None, -2, (UPDATE,)), ("left", None, -2, (UPDATE,)), ("row", None, -2, (MAP,)), ("position", 0x1001, -7, (MAP,)),
    ("first", None, -2, (MAP,)), ("used", None, -2, (MAP,)), ("slot", None, -2, (MAP,)), ("slot", 0x1004, -7, (MAP,)),
])
def test_validate(field, value, code, calls):
    for call in calls:
        p = _params()
        if field:
            setattr(p, field, value)
        assert _lib.load().gptoss_attn_table_validate(ctypes.byref(p), call) == code
        if code:
            name = "gptoss_attn_token_map" if call else "gptoss_attn_page_table_update"
            assert getattr(_lib.load(), name)(ctypes.byref(p), None) == code
    assert _lib.load().gptoss_attn_table_validate(None, 0) == -1


@pytest.mark.parametrize("rows,width,pages,need", [
    (128, 256, 1000, 0), (129, 256, 1000, 16 * 32 * 4), (32, 257, 1000, 0), (33, 257, 1000, 16 * 32 * 4), (16, 2048, 33, 0), (17, 2048, 33, 16 * 2 * 4), (5000, 100, 1 << 19, 16 << 16),
    (5000, 100, (1 << 19) + 1, 0), (0, 100, 100, 0),
])
def test_update_scratch(rows, width, pages, need):
    """A launch that sets the pool's bits takes sixteen copies of them; pools of more than 2^19 pages are looked at in parts, by one workgroup."""
    p = _params()
    p.B, p.table_width, p.table_stride, p.pages = rows, width, width, pages
    lib = _lib.load()
    assert lib.gptoss_attn_table_workspace_bytes(ctypes.byref(p)) == need and lib.gptoss_attn_table_workspace_bytes(None) == 0
    if need:
        assert lib.gptoss_attn_table_validate(ctypes.byref(p), UPDATE) == lib.gptoss_attn_page_table_update(ctypes.byref(p), None) == -10
        p.scratch, p.scratch_bytes = 0x1000, need - 1
        assert lib.gptoss_attn_table_validate(ctypes.byref(p), UPDATE) == -10
        p.scratch_bytes = need
        assert lib.gptoss_attn_table_validate(ctypes.byref(p), UPDATE) == 0


@pytest.mark.parametrize("mutate,code", [
    (lambda p: None, 0), (lambda p: setattr(p, "page_table", None), 0), (lambda p: setattr(p, "start", None), 0), (lambda p: setattr(p, "table_width", 0), 0), (lambda p: setattr(p, "B", 2), -5),
    (lambda p: setattr(p, "Sq", 0), -5), (lambda p: setattr(p, "k", None), -2), (lambda p: setattr(p, "pages", 0), -11), (lambda p: setattr(p, "page_size", 24), -11),
    (lambda p: setattr(p, "k_pages", 0x1008), -7), (lambda p: setattr(p.v_stride, "s", 8), -8),
])
def test_write_by_slots_validate(mutate, code):
    p = _lib.PagedParams()
    p.struct_size = ctypes.sizeof(p)
    p.B, p.G, p.Sq, p.D, p.pages, p.page_size = 1, 2, 5, 64, 10, 16
    for f in ("k_pages", "v_pages", "k", "v"):
        setattr(p, f, 0x1000)
    for name in ("k_stride", "v_stride", "k_page_stride", "v_page_stride"):
        s = getattr(p, name)
        s.b, s.h, s.s = 2 * 16 * 64, 16 * 64, 64
    mutate(p)
    lib = _lib.load()
    assert lib.gptoss_attn_paged_validate(ctypes.byref(p), 3) == code
    if code:
        assert lib.gptoss_attn_paged_write_slots(ctypes.byref(p), 0x1000, None) == code
    else:
        assert lib.gptoss_attn_paged_write_slots(ctypes.byref(p), None, None) == -2
        assert lib.gptoss_attn_paged_write_slots(ctypes.byref(p), 0x1004, None) == -7


def test_cpu_tensors_are_refused():
    t, n = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    cache, k = A.paged_cache(4, 2, 16, device="cpu"), torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: A.page_table_update(t, n, n, 4, 16), lambda: A.token_map(t, n, n, 4, 16), lambda: A.paged_cache_write_tokens(cache, k, k, torch.zeros(3, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()
    with pytest.raises(RuntimeError, match="no gradient"):
        A.paged_cache_write_tokens(cache, k.requires_grad_(), k, torch.zeros(3, dtype=torch.int64))


def test_traced_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        t, n = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
        got, left = A.page_table_update(t, n, n, 4, 16)
        assert got.shape == (2,) and left.shape == (1,) and got.dtype == left.dtype == torch.int32
        m = A.token_map(t, n, n, 7, 16)
        assert [tuple(x.shape) for x in m] == [(7,), (7,), (7,), (7,), (1,)] and m.slot.dtype == torch.int64
        cache, k = A.paged_cache(4, 2, 16), torch.zeros(7, 2, 64, dtype=torch.bfloat16, device="cuda")
        assert A.paged_cache_write_tokens(cache, k, k, m.slot) is None


def test_states_of_packed_rows_are_refused_what_the_map_says_already():
    from types import SimpleNamespace
    module, n = SimpleNamespace(layer_idx=0, sliding_window=None, sinks=None), torch.zeros(2, dtype=torch.int32)
    cache, table = A.paged_cache(4, 2, 16, device="cpu"), torch.zeros(2, 3, dtype=torch.int32)
    tokens = A.TokenMap(*(torch.zeros(5, dtype=torch.int32) for _ in range(5)))
    q, k = torch.zeros(1, 4, 5, 64, dtype=torch.bfloat16), torch.zeros(1, 2, 5, 64, dtype=torch.bfloat16)
    for state, rows, match in ((A.PagedState([cache], table, n, n, tokens=tokens), 1, "start must be None"), (A.PagedState([cache], table, None, n, tokens=tokens), 2, "one batch row"),
                               (A.PagedState([cache], table, None, n, counts=n, tokens=tokens), 1, "counts=")):
        with pytest.raises(RuntimeError, match=match):
            state.attend(module, q.expand(rows, -1, -1, -1), k.expand(rows, -1, -1, -1), k.expand(rows, -1, -1, -1), 0.125)
