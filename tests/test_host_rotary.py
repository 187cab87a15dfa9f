"""Host-only checks of the rotary positions: the parameter block mirrors the header, arguments are refused before anything is launched, frequencies are
those of the formulas, the model's function is swapped and put back.  No kernel is launched."""
import ctypes
import math
import os
import re

import pytest
import torch

import oregon_gpt_oss_patching_amd as A
from oregon_gpt_oss_patching_amd import _lib
from oracle import rotary_ref as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_mirror_matches_header_field_order():
    text = open(os.path.join(ROOT, "include", "gptoss_attn.h")).read()
    body = re.search(r"typedef struct gptoss_attn_rotary_params \{(.*?)\} gptoss_attn_rotary_params;", text, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = []
    for decl in body.split(";"):
        for part in decl.strip().split(","):
            if part.strip():
                names.append(re.findall(r"[A-Za-z_][A-Za-z_0-9]*", part)[-1])
    assert names == [f[0] for f in _lib.RotaryParams._fields_]


def _params(tables=False):
    """A block that passes (fake addresses, never dereferenced)."""
    p = _lib.RotaryParams()
    p.struct_size = ctypes.sizeof(p)
    p.position_bytes, p.B, p.H, p.G, p.S, p.D, p.R, p.scale = 8, 2, 8, 2, 5, 64, 64, 1.0
    for f in ("q", "k", "q_out", "k_out") + (("cos_table", "sin_table") if tables else ("positions", "frequencies")):
        setattr(p, f, 0x1000)
    return p


@pytest.mark.parametrize("tables", [False, True])
def test_validate_accepts_good_params(tables):
    assert _lib.load().gptoss_attn_rotary_validate(ctypes.byref(_params(tables))) == 0


@pytest.mark.parametrize("field,value,code", [
    ("struct_size", 8, -9), ("dtype", 2, -6), ("dtype", -1, -6), ("B", 0, -5), ("S", 0, -5), ("H", 0, -4), ("G", 0, -4), ("H", 2 ** 20 + 1, -4), ("D", 0, -3), ("D", 257, -3),
    ("R", 0, -3), ("R", 66, -3), ("R", 31, -3), ("q", None, -2), ("k_out", None, -2), ("q", 0x1001, -7), ("positions", None, -2), ("frequencies", None, -2),
    ("positions", 0x1004, -7), ("frequencies", 0x1004, -7), ("position_bytes", 2, -6), ("cos_table", 0x1000, -2), ("B", 2 ** 24, -5), ("S", 2 ** 30, -5),
])
def test_validate_error_codes(field, value, code):
    p = _params()
    setattr(p, field, value)
    if field == "B" and value == 2 ** 24:
        p.S = 2
    assert _lib.load().gptoss_attn_rotary_validate(ctypes.byref(p)) == code
    assert _lib.load().gptoss_attn_rotary(ctypes.byref(p), None) == code


@pytest.mark.parametrize("field,value,code", [("sin_table", None, -2), ("table_dtype", 2, -6), ("sin_table", 0x1001, -7), ("positions", 0x1000, -2)])
def test_validate_tables(field, value, code):
    p = _params(True)
    setattr(p, field, value)
    assert _lib.load().gptoss_attn_rotary_validate(ctypes.byref(p)) == code


def test_null_params():
    assert _lib.load().gptoss_attn_rotary_validate(None) == -1 and _lib.load().gptoss_attn_rotary(None, None) == -1


def test_frequencies():
    f = A.rotary_frequencies(64, 10000.0, device="cpu")
    assert f.scale == 1.0 and f.frequencies.dtype == torch.float64
    assert torch.allclose(f.frequencies, 10000.0 ** (-torch.arange(32).double() / 32), rtol=1e-14)
    assert torch.equal(A.rotary_frequencies(64, 10000.0, factor=8.0, device="cpu").frequencies, f.frequencies / 8)
    for bad in (dict(rotary_dim=0), dict(rotary_dim=7), dict(theta=1.0), dict(factor=0.0), dict(original_length=0), dict(original_length=4096, beta_slow=40.0)):
        with pytest.raises(RuntimeError):
            A.rotary_frequencies(**bad, device="cpu")


@pytest.mark.parametrize("truncate", [True, False])
@pytest.mark.parametrize("theta,factor,length", [(150000.0, 32.0, 4096), (10000.0, 4.0, 2048), (500.0, 16.0, 100)])
def test_scaled_frequencies_are_the_models(theta, factor, length, truncate):
    """Those that transformers computes for the same parameters, in float32."""
    transformers = pytest.importorskip("transformers")
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    config = transformers.GptOssConfig(num_hidden_layers=1, head_dim=64, max_position_embeddings=int(factor * length),
                                       rope_parameters=dict(rope_type="yarn", rope_theta=theta, factor=factor, beta_fast=32.0, beta_slow=1.0, truncate=truncate,
                                                            original_max_position_embeddings=length))
    want, scale = ROPE_INIT_FUNCTIONS["yarn"](config, torch.device("cpu"))
    got = A.rotary_frequencies(64, theta, factor=factor, original_length=length, truncate=truncate, device="cpu")
    assert abs(got.scale - scale) < 1e-12 and torch.allclose(got.frequencies.float(), want, rtol=3e-6, atol=0.0)
    assert abs(got.scale - (0.1 * math.log(factor) + 1.0)) < 1e-12


def test_oracle_is_the_models_embedding():
    """transformers' own function in 64 bits, and the pairs' other order after a permutation."""
    M = pytest.importorskip("transformers.models.gpt_oss.modeling_gpt_oss")
    gen = torch.Generator().manual_seed(0)
    q, k = torch.randn(2, 4, 9, 64, generator=gen).double(), torch.randn(2, 2, 9, 64, generator=gen).double()
    rope = A.rotary_frequencies(64, 150000.0, factor=32.0, original_length=4096, device="cpu")
    positions = torch.randint(0, 10000, (2, 9), generator=gen)
    z = R.of_positions(positions, rope.frequencies, rope.scale)
    for got, want in zip(M.apply_rotary_pos_emb(q, k, z.real, z.imag), (R.turn(q, z), R.turn(k, z))):
        assert float((got - want).abs().max()) < 1e-13
    order = torch.arange(64).view(2, 32).t().flatten()
    assert torch.equal(R.turn(q[..., order], z, True), R.turn(q, z)[..., order])


def test_cpu_tensors_gradients_and_transforms_are_refused():
    rope, x, at = A.rotary_frequencies(64, device="cpu"), torch.randn(1, 2, 3, 64), torch.arange(3)
    with pytest.raises(RuntimeError, match="GPU only"):
        A.rotary(x, x, at, rope)
    with pytest.raises(RuntimeError, match="GPU only"):
        A.rotary(x.clone().requires_grad_(), x, at, rope)
    with pytest.raises(RuntimeError, match="no gradient"):
        A.rotary(x, x, at, A.Rotary(rope.frequencies.clone().requires_grad_()))
    with pytest.raises(RuntimeError, match="vmapped"):
        torch.vmap(lambda y: A.rotary(y, y, at, rope)[0])(x[None])
    with torch.autograd.forward_ad.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        A.rotary(torch.autograd.forward_ad.make_dual(x, x), x, at, rope)


def test_traced_shapes_stay_symbols():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.symbolic_shapes import DimDynamic, ShapeEnv, StatelessSymbolicContext
    env = ShapeEnv()
    mode = FakeTensorMode(shape_env=env)
    ctx = StatelessSymbolicContext(dynamic_sizes=[DimDynamic.DYNAMIC, DimDynamic.DYNAMIC])
    b, s = mode.from_tensor(torch.empty((3, 100), device="meta"), symbolic_context=ctx, static_shapes=False).shape
    with mode, torch.no_grad():
        q, k = (torch.empty((b, n, s, 64), dtype=torch.bfloat16, device="cuda") for n in (64, 8))
        out = A.rotary(q, k, torch.empty((b, s), dtype=torch.int64, device="cuda"), A.Rotary(torch.empty(32, dtype=torch.float64, device="cuda")))
    for x, n in zip(out, (64, 8)):
        assert tuple(map(str, x.shape)) == (str(b), str(n), str(s), "64") and x.dtype == torch.bfloat16 and x.transpose(1, 2).is_contiguous()
    assert not env.replacements and not [g for g in env.guards if "Eq" in str(g.expr)]


@pytest.mark.parametrize("which", [0, 1])
def test_a_result_asks_for_a_gradient_where_its_tensor_does(which):
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = [torch.empty((2, n, 5, 64), dtype=torch.bfloat16, device="cuda", requires_grad=i == which) for i, n in enumerate((8, 2))]
        out = A.rotary(*x, torch.empty((2, 5), dtype=torch.int64, device="cuda"), A.Rotary(torch.empty(32, dtype=torch.float64, device="cuda")))
    assert [y.requires_grad for y in out] == [which == 0, which == 1]


def test_the_models_function_is_swapped_and_put_back():
    M = pytest.importorskip("transformers.models.gpt_oss.modeling_gpt_oss")
    from oregon_gpt_oss_patching_amd.patching import patch_flash_attention, unpatch_flash_attention
    before = M.apply_rotary_pos_emb
    try:
        patch_flash_attention()
        assert M.apply_rotary_pos_emb is before
        patch_flash_attention(rotary=True)
        patch_flash_attention(rotary=True)
        assert M.apply_rotary_pos_emb is A.hip_rotary_pos_emb
        patch_flash_attention()
        assert M.apply_rotary_pos_emb is before
        M.apply_rotary_pos_emb = mine = lambda *a: a           # somebody's own is left alone, and comes back
        patch_flash_attention()
        assert M.apply_rotary_pos_emb is mine
        patch_flash_attention(rotary=True)
        unpatch_flash_attention()
        assert M.apply_rotary_pos_emb is mine
        unpatch_flash_attention()
        assert M.apply_rotary_pos_emb is mine
    finally:
        unpatch_flash_attention()
        M.apply_rotary_pos_emb = before
