"""GPU tests of caches in 8 bits that a program fills itself: any byte is the power of two that it says, and 255 is NaN."""
import pytest
import torch

from oracle import paged_ref as P
from test_gpu_paged import BF16, DEV, E4M3, FP32, SCALE, A  # noqa: F401

pytestmark = pytest.mark.gpu
SEEN = torch.arange(256, dtype=torch.uint8)


def rows(codes, exps):
    """What rows of codes (..., 64) with a byte each stand for, in 64 bits: infinite from 2^128 on."""
    x = codes.float().double() * torch.exp2(exps.double() - 127)[..., None]
    x = torch.where(x.abs() >= 2.0 ** 128, torch.sign(x) * float("inf"), x)
    return torch.where((exps == 255)[..., None], torch.full_like(x, float("nan")), x)


def cache_of(A, k, ke, v, ve):  # noqa: F811
    """One head, pages of 64 tokens in order: rows (n, 64) of codes and (n) bytes."""
    def pages(x):
        pad = -len(x) % 64
        return torch.cat([x.view(torch.uint8), x.new_zeros((pad, *x.shape[1:])).view(torch.uint8)]).view(-1, 1, 64, *x.shape[1:]).to(DEV)
    return A.PagedCache(pages(k).view(E4M3), pages(v).view(E4M3), pages(ke), pages(ve)), torch.arange(-(-len(k) // 64), dtype=torch.int32, device=DEV)[None]


def same(got, want):
    return torch.equal(got.double().nan_to_num(nan=7e200, posinf=8e200, neginf=-8e200), want.double().nan_to_num(nan=7e200, posinf=8e200, neginf=-8e200))


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_every_byte_read_back(A, dtype):  # noqa: F811
    """All 256 codes under all 256 bytes; what the type does not hold is rounded once."""
    codes = SEEN.repeat(256).view(E4M3).view(1024, 64)
    exps = SEEN.repeat_interleave(4)
    cache, table = cache_of(A, codes, exps, codes.flip(0), exps.flip(0))
    k, v = A.paged_cache_read(cache, table, [1024], 1024, None, dtype)
    want = rows(codes, exps).to(FP32).to(dtype)
    assert same(k.cpu()[0, 0], want) and same(v.cpu()[0, 0], want.flip(0))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("byte", [0, 1, 2, 60, 240])
@pytest.mark.parametrize("n", [50, 3000])
def test_attention_under_small_and_large_powers(A, dtype, byte, n):  # noqa: F811
    """Keys of 2^(byte - 127) under queries of its inverse, values of 2^(byte - 127)."""
    gen = torch.Generator().manual_seed(71 + byte + n)
    k, v = ((torch.randn(n, 64, generator=gen) * 60).to(E4M3) for _ in range(2))
    exps = torch.full((n,), byte, dtype=torch.uint8)
    q = (torch.randn(1, 4, 1, 64, generator=gen).double() * 2.0 ** (121 - byte)).to(dtype)
    cache, table = cache_of(A, k, exps, v, exps)
    o, lse = A.paged_attention_forward(q.to(DEV), cache, table, [n], None, SCALE)
    pools = [torch.cat([rows(x, exps), torch.zeros(-n % 64, 64, dtype=torch.float64)]).view(-1, 1, 64, 64) for x in (k, v)]
    ref, ref_lse, terms = P.attention(q, *pools, table.cpu(), [n], None, SCALE)
    tol, tol_lse = P.bounds(ref, ref_lse, terms, dtype)
    # next to 2^-126, in place of the bound's 1e-37: steps are 2^-133 in bfloat16 and 2^-149 in float32, half of one for each row's numbers, half of one
    # for o and one for each sum
    tol = tol - 1e-37 + 2.0 ** -133 + (n + 64) * 2.0 ** -149
    assert float(ref.abs().max()) > 10 * float(tol.max())
    assert bool(((o.cpu().double() - ref).abs() <= tol).all()) and bool(((lse.cpu().double() - ref_lse).abs() <= tol_lse).all())


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("byte,code", [(255, 0x38), (255, 0), (254, 0x38), (254, 0x48), (248, 0x7e), (247, 0x78), (247, 0x7f)])
@pytest.mark.parametrize("heads", [1, 8, 16])
def test_values_that_only_a_later_query_sees(A, dtype, byte, code, heads):  # noqa: F811
    """A row of V that is infinite or NaN by its byte: queries that do not see it are as if it were not there."""
    gen = torch.Generator().manual_seed(77)
    n, sq = 60, 4
    k, v = ((torch.randn(n, 64, generator=gen) * 60).to(E4M3) for _ in range(2))
    exps = torch.full((n,), 120, dtype=torch.uint8)
    q = torch.randn(1, heads, sq, 64, generator=gen).to(dtype).to(DEV)
    clean, table = cache_of(A, k, exps, v, exps)
    want = A.paged_attention(q, clean, table, [n], None, SCALE)
    bad, bad_exps = v.view(torch.uint8).clone(), exps.clone()
    bad[58], bad_exps[58] = 0x30, byte
    bad[58, 5:9] = code
    broken, _ = cache_of(A, k, exps, bad.view(E4M3), bad_exps)
    value = rows(bad.view(E4M3), bad_exps)[58]
    o = A.paged_attention(q, broken, table, [n], None, SCALE)
    # queries at 56, 57, 58, 59: the first two do not see the row
    assert torch.equal(o[:, :2], want[:, :2])
    for i in range(2, sq):
        for d in range(64):
            if not torch.isfinite(value[d]):
                x = o[0, i, :, d].float().cpu()
                assert bool(torch.isnan(x).all()) if torch.isnan(value[d]) else bool((x == float(value[d])).all()), (i, d)
