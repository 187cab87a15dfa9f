"""Host-only checks of the key / value cache in pages: the parameter block mirrors the header, arguments are refused with the documented codes
before anything is launched, and the Python calls refuse what the kernels cannot take.  No kernel is launched."""
import ctypes
import os
import re

import pytest
import torch

import oregon_gpt_oss_patching_amd as A
from oregon_gpt_oss_patching_amd import _lib
from oracle import paged_ref as P

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FWD, WRITE, READ = 0, 1, 2


def test_struct_mirror_matches_header_field_order():
    text = open(os.path.join(ROOT, "include", "gptoss_attn.h")).read()
    body = re.search(r"typedef struct gptoss_attn_paged_params \{(.*?)\} gptoss_attn_paged_params;", text, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = []
    for decl in body.split(";"):
        for part in decl.strip().split(","):
            if part.strip():
                names.append(re.findall(r"[A-Za-z_][A-Za-z_0-9]*", part)[-1])
    assert names == [f[0] for f in _lib.PagedParams._fields_]


def _params(storage=_lib.DTYPE_BF16, dtype=_lib.DTYPE_BF16):
    """A block that passes (fake, aligned addresses, never dereferenced)."""
    p = _lib.PagedParams()
    p.struct_size = ctypes.sizeof(_lib.PagedParams)
    p.dtype, p.storage, p.sinks_dtype = dtype, storage, _lib.DTYPE_FP32
    p.B, p.H, p.G, p.Sq, p.D = 2, 16, 2, 1, 64
    p.pages, p.page_size, p.table_width, p.table_stride, p.scale = 10, 16, 4, 4, 0.125
    for f in ("k_pages", "v_pages", "k_exp", "v_exp", "page_table", "seqlens", "start", "q", "o", "lse", "k", "v", "scratch"):
        setattr(p, f, 0x1000)
    p.scratch_bytes = 1 << 40
    for name in ("q_stride", "o_stride", "k_stride", "v_stride", "k_page_stride", "v_page_stride", "k_exp_stride", "v_exp_stride"):
        s = getattr(p, name)
        s.b, s.h, s.s = 2 * 16 * 64, 16 * 64, 64
    return p


def _validate(p, call):
    return _lib.load().gptoss_attn_paged_validate(ctypes.byref(p), call)


@pytest.mark.parametrize("call", [FWD, WRITE, READ])
@pytest.mark.parametrize("dtype,storage", [(0, 0), (0, 2), (1, 1), (1, 2)])
def test_validate_accepts_good_params(call, dtype, storage):
    assert _validate(_params(storage, dtype), call) == 0


ALL = (FWD, WRITE, READ)


@pytest.mark.parametrize("mutate,code,calls", [
    (lambda p: setattr(p, "struct_size", 8), -9, ALL),
    (lambda p: setattr(p, "dtype", 2), -6, ALL),
    (lambda p: setattr(p, "storage", 1), -6, ALL),               # float32 pages of a bfloat16 model
    (lambda p: setattr(p, "storage", 7), -6, ALL),
    (lambda p: setattr(p, "D", 128), -3, ALL),
    (lambda p: setattr(p, "G", 0), -4, ALL),
    (lambda p: setattr(p, "H", 15), -4, (FWD,)),
    (lambda p: setattr(p, "B", 0), -5, ALL),
    (lambda p: setattr(p, "Sq", 0), -5, ALL),
    (lambda p: setattr(p, "Sq", 2 ** 30 + 1), -5, ALL),
    (lambda p: setattr(p, "pages", 0), -11, ALL),
    (lambda p: setattr(p, "page_size", 8), -11, ALL),
    (lambda p: setattr(p, "page_size", 48), -11, ALL),
    (lambda p: setattr(p, "page_size", 2048), -11, ALL),
    (lambda p: setattr(p, "table_width", 0), -11, ALL),
    (lambda p: setattr(p, "table_stride", -4), -11, ALL),
    (lambda p: setattr(p, "table_width", 2 ** 26 + 1), -11, ALL),
    (lambda p: setattr(p, "k_pages", None), -2, ALL),
    (lambda p: setattr(p, "v_pages", 0x1008), -7, ALL),
    (lambda p: setattr(p, "page_table", None), -2, ALL),
    (lambda p: setattr(p, "page_table", 0x1002), -7, ALL),
    (lambda p: setattr(p, "seqlens", None), -2, (FWD, READ)),
    (lambda p: setattr(p, "start", None), -2, (WRITE,)),
    (lambda p: setattr(p, "start", 0x1002), -7, ALL),
    (lambda p: setattr(p.k_page_stride, "s", 32), -8, ALL),
    (lambda p: setattr(p.v_page_stride, "s", 68), -7, ALL),
    (lambda p: setattr(p.v_page_stride, "s", 2 ** 24 + 64), -8, ALL),
    (lambda p: setattr(p, "k", None), -2, (WRITE, READ)),
    (lambda p: setattr(p.v_stride, "s", 0), -8, (WRITE, READ)),
    (lambda p: setattr(p, "q", 0x1004), -7, (FWD,)),
    (lambda p: setattr(p, "o", None), -2, (FWD,)),
    (lambda p: setattr(p, "lse", 0x1002), -7, (FWD,)),
    (lambda p: setattr(p, "sinks_dtype", 2), -6, (FWD,)),
    (lambda p: setattr(p, "window", -1), -5, (FWD,)),
    (lambda p: setattr(p, "max_len", -1), -5, (FWD,)),
    (lambda p: setattr(p, "scale", 0.0), -5, (FWD,)),
    (lambda p: setattr(p, "scale", float("nan")), -5, (FWD,)),
    (lambda p: setattr(p, "scratch", 0x1004), -7, (FWD,)),
])
def test_validate_error_codes(mutate, code, calls):
    names = {FWD: "gptoss_attn_paged_fwd", WRITE: "gptoss_attn_paged_write", READ: "gptoss_attn_paged_read"}
    for call in calls:
        p = _params()
        mutate(p)
        assert _validate(p, call) == code
        assert getattr(_lib.load(), names[call])(ctypes.byref(p), None) == code      # the call itself, before any launch
    assert _lib.status_string(code) not in ("ok", "unknown status")


def test_e4m3_needs_its_exponents():
    for call in ALL:
        p = _params(_lib.DTYPE_E4M3)
        p.v_exp = None
        assert _validate(p, call) == -2


@pytest.mark.parametrize("storage", [_lib.DTYPE_BF16, _lib.DTYPE_E4M3])
def test_page_strides_of_32_bits(storage):
    """A page's stride in bytes is below 2^32; what is longer, or runs backwards, is refused."""
    most = 2 ** 31 - 8 if storage == _lib.DTYPE_BF16 else 2 ** 32 - 16
    for call in ALL:
        for name in ("k_page_stride", "v_page_stride") + (("k_exp_stride", "v_exp_stride") if storage == _lib.DTYPE_E4M3 else ()):
            p = _params(storage)
            getattr(p, name).b = most
            assert _validate(p, call) == 0
            for bad in (2 ** 32, -64):
                getattr(p, name).b = bad
                assert _validate(p, call) == -8


def test_paged_adapter_refuses_other_lengths():
    """hip_flash_attention(paged=) takes the rows' lengths from the state alone."""
    import oregon_gpt_oss_patching_amd as A
    x = torch.zeros(1, 1, 1, 64)
    state = A.PagedState([], torch.zeros(1, 1, dtype=torch.int32), None, torch.ones(1, dtype=torch.int32))
    for name in ("seqlens", "doc_start"):
        with pytest.raises(RuntimeError, match="neither seqlens nor doc_start"):
            A.hip_flash_attention(None, x, x, x, None, 0.125, paged=state, **{name: torch.ones(1, dtype=torch.int32)})


def test_null_params():
    for call in ALL:
        assert _lib.load().gptoss_attn_paged_validate(None, call) == -1
    assert _lib.load().gptoss_attn_paged_workspace_bytes(None) == 0
    with pytest.raises(_lib.GptossAttnError):
        raise _lib.GptossAttnError("gptoss_attn_paged_fwd", -11, _lib.status_string(-11))


def _cpu_cache(**kw):
    return A.paged_cache(4, 2, 16, device="cpu", **kw)


def test_cpu_tensors_are_refused():
    cache, table, n = _cpu_cache(), torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q, k = torch.zeros(1, 16, 1, 64, dtype=torch.bfloat16), torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU only"):
        A.paged_attention(q, cache, table, n, None, 0.125)
    with pytest.raises(RuntimeError, match="GPU only"):
        A.paged_cache_write(cache, k, k, table, n)
    with pytest.raises(RuntimeError, match="GPU only"):
        A.paged_cache_read(cache, table, n, 4)


def test_gradients_are_refused():
    cache, table, n = _cpu_cache(), torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q = torch.zeros(1, 16, 1, 64, dtype=torch.bfloat16, requires_grad=True)
    k = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        A.paged_attention(q, cache, table, n, None, 0.125)
    with pytest.raises(RuntimeError, match="no gradient"):
        A.paged_cache_write(cache, k.detach(), k, table, n)
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU only"):      # allowed as far as gradients go
        A.paged_attention(q, cache, table, n, None, 0.125)


def test_forward_gradients_are_refused():
    cache, table, n = _cpu_cache(), torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q = torch.zeros(1, 16, 1, 64, dtype=torch.bfloat16)
    with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError, match="no gradient"):
        A.paged_attention(torch.autograd.forward_ad.make_dual(q, q), cache, table, n, None, 0.125)


def test_paged_cache_allocates_and_refuses():
    c = _cpu_cache(storage=torch.float8_e4m3fn)
    assert c.k.shape == (4, 2, 16, 64) and c.k_exp.shape == (4, 2, 16) and c.k_exp.dtype == torch.uint8
    assert _cpu_cache().k_exp is None
    with pytest.raises(RuntimeError, match="power of two"):
        A.paged_cache(4, 2, 24, device="cpu")
    with pytest.raises(RuntimeError, match="storage"):
        A.paged_cache(4, 2, 16, storage=torch.float16, device="cpu")


def test_vmap_is_refused():
    cache, table, n = _cpu_cache(), torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q = torch.zeros(3, 1, 16, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="vmapped"):
        torch.vmap(lambda x: A.paged_attention(x, cache, table, n, None, 0.125))(q)


def test_traced_shapes():
    """The shape-only implementations give the operators' shapes and types."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        cache = A.paged_cache(9, 2, 32, storage=torch.float8_e4m3fn)
        table, n = torch.zeros(3, 2, dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
        q = torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
        o, lse = A.paged_attention_forward(q, cache, table, n, None, 0.125)
        assert o.shape == (3, 2, 16, 64) and o.dtype == torch.bfloat16 and lse.shape == (3, 16, 2) and lse.dtype == torch.float32
        k, v = A.paged_cache_read(cache, table, n, 40, dtype=torch.float32)
        assert k.shape == v.shape == (3, 2, 40, 64) and k.dtype == torch.float32
        assert A.paged_cache_write(cache, k[:, :, :2], v[:, :, :2], table, n) is None


def test_oracle_quantiser_agrees_with_the_types_own_rounding():
    """Numbers between -448 and 448 rounded by torch's conversion, the row's power of two held at 1 by a 448."""
    x = torch.linspace(-448, 448, 64 * 301, dtype=torch.float64).view(-1, 64).clone()
    x = torch.cat([x, x / 448 * 0.02])
    x[:, 0] = 448.0
    y, s = P.quantise(x)
    assert bool((s == 0).all())
    assert torch.equal(y.float(), x.float().to(torch.float8_e4m3fn).float())


def test_oracle_quantiser_powers_of_two():
    for top, s in ((448.0, 0), (448.0000001, 1), (224.0, -1), (1.75, -8), (1.76, -7), (1.0, -8), (2.0 ** -70, -64), (0.0, -64), (3.3e38, 120)):
        x = torch.zeros(1, 64, dtype=torch.float64)
        x[0, 5] = -top
        y, e = P.quantise(x)
        assert int(e) == s, (top, int(e))
        assert abs(float(y[0, 5]) * 2.0 ** s + top) <= max(top * 2.0 ** -4, 2.0 ** (s - 10))
    x = torch.zeros(1, 64, dtype=torch.float64)
    x[0, 0], x[0, 1], x[0, 2] = float("inf"), float("nan"), 7.0
    y, e = P.quantise(x)
    assert torch.isnan(y[0, :2]).all() and float(y[0, 2]) == 448.0 and int(e) == -6


def test_oracle_attention_is_the_eager_one_where_both_apply():
    """A pool whose pages lie in order is a contiguous cache."""
    from oracle import eager_ref as E
    for n, sq, w, seed in ((37, 3, 0, 1), (48, 1, 9, 2)):
        q, k, v, sinks, _ = E.make_inputs(seed, 1, 8, 2, sq, 64, torch.float32, skv=48)
        pool = [t[0].view(2, 3, 16, 64).transpose(0, 1).double() for t in (k, v)]
        o, lse, _ = P.attention(q, *pool, torch.tensor([[0, 1, 2]]), [n], sinks, 0.125, w)
        ref = E.eager_attention(q.double(), k.double()[:, :, :n], v.double()[:, :, :n], sinks.double(), 0.125, w or None, n - sq)
        assert float((o - ref).abs().max()) < 1e-5
        ref_lse = E.logsumexp_rows(q.double(), k.double()[:, :, :n], sinks.double(), 0.125, w or None, n - sq)
        assert float((lse - ref_lse).abs().max()) < 1e-5
