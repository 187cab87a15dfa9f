"""GPU tests of the cache in pages in 4 bits (e2m1 numbers, a power of two for each 32): writes and reads bit by bit, attention within the bounds of its
roundings (oracle/paged_ref.py), against the definition in 64 bits.  Every slot that holds no token of the call is NaN."""
import pytest
import torch

from oracle import paged_ref as P
from test_gpu_paged import BF16, DEV, FP32, SCALE, A, make, new_table, poison  # noqa: F401

pytestmark = pytest.mark.gpu
E2M1 = torch.float4_e2m1fn_x2
BOTH = pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])


def values(cache):
    """The pools' values in 64 bits on the CPU."""
    return [P.values4(x.view(torch.uint8).cpu(), e.cpu()) for x, e in ((cache.k, cache.k_exp), (cache.v, cache.v_exp))]


def bounds(ref, ref_lse, terms, dtype):
    """`oracle.paged_ref.bounds`, with a bfloat16 query's weights as two bfloat16 terms: 2^-15 of a weight and not 2^-8."""
    tol, tol_lse = P.bounds(ref, ref_lse, terms, FP32)
    if dtype == BF16:
        tol = tol + 1.01 * (2.0 ** -15 * terms[0] + 2.0 ** -8 * ref.abs())
    return tol, tol_lse


def check(A, cache, table, n, q, sinks, window=0, start=None, max_len=None, scale=SCALE):  # noqa: F811
    args = (q.to(DEV), cache, table, n, None if sinks is None else sinks.to(DEV), scale, window or None,
            None if start is None else torch.tensor(start, dtype=torch.int32, device=DEV), max_len)
    o, lse = A.paged_attention_forward(*args)
    again, lse2 = A.paged_attention_forward(*args)
    assert torch.equal(o, again) and torch.equal(lse, lse2) and torch.equal(o, A.paged_attention(*args))
    ref, ref_lse, terms = P.attention(q, *values(cache), table.cpu(), n.cpu(), sinks, scale, window, start)
    assert o.dtype == q.dtype and o.shape == ref.shape and lse.shape == ref_lse.shape
    tol, tol_lse = bounds(ref, ref_lse, terms, q.dtype)
    o, lse = o.cpu().double(), lse.cpu().double()
    assert torch.isfinite(o).all()
    over = (o - ref).abs() - tol
    assert bool((over <= 0).all()), (float(over.max()), [int(x) for x in torch.nonzero(over == over.max())[0]])
    none = torch.isinf(ref_lse)
    assert torch.equal(none, torch.isinf(lse)) and bool(((lse - ref_lse).abs() <= tol_lse)[~none].all()), float((lse - ref_lse).abs()[~none].max())
    return o, lse


def same(got, want):
    return torch.equal(got.double().nan_to_num(nan=7e200, posinf=8e200, neginf=-8e200), want.double().nan_to_num(nan=7e200, posinf=8e200, neginf=-8e200))


# ---- writing and reading ---------------------------------------------------------------------------------------------
@BOTH
@pytest.mark.parametrize("lens,g,ps,token_major", [([1], 1, 16, False), ([1, 15, 16, 17], 2, 16, False), ([40, 0, 133], 8, 32, True), ([300, 299], 3, 64, False), ([1025, 7], 2, 1024, True)])
def test_write_then_read(A, dtype, lens, g, ps, token_major):  # noqa: F811
    print(f"case {dtype} lens={lens} G={g} page={ps} token_major={token_major}", flush=True)
    gen = torch.Generator().manual_seed(1)
    table, pages = new_table(gen, lens, ps, 1)
    cache = A.paged_cache(pages, g, ps, E2M1)
    if token_major:
        cache = A.PagedCache(*(t.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(t.dtype) for t in cache))
    poison(cache)
    longest = max(lens)
    k, v = (torch.randn(len(lens), g, longest, 64, generator=gen).to(dtype) for _ in range(2))
    t, n = table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    A.paged_cache_write(cache, k.to(DEV), v.to(DEV), t, torch.zeros_like(n), n)
    gk, gv = A.paged_cache_read(cache, t, n, longest + 3, None, dtype)
    assert gk.dtype == dtype and gk.shape == (len(lens), g, longest + 3, 64)
    for got, x in ((gk, k), (gv, v)):
        want = torch.zeros(got.shape, dtype=torch.float64)
        for b, m in enumerate(lens):
            want[b, :, :m] = P.stored_rows(x[b, :, :m], E2M1)
        assert torch.equal(got.cpu().double(), want)
    free = cache.k.shape[0] * ps - sum(lens)
    for x in values(cache):
        nan = torch.isnan(x)
        assert int(nan.all(-1).sum()) == free * g and int(nan.any(-1).sum()) == free * g
    assert A.paged_cache_read(cache, t, n, 1)[0].dtype == BF16


@BOTH
def test_codes_of_every_bfloat16_number(A, dtype):  # noqa: F811
    """All 65536 bfloat16 numbers among 32 whose largest one sets different powers of two, infinities and NaN among them; halves of a row apart."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF16).view(1024, 64)
    gen = torch.Generator().manual_seed(2)
    mixed = x.reshape(-1)[torch.randperm(65536, generator=gen)].view(1024, 64)
    near = (torch.randn(2048, 2, 32, generator=gen) * torch.exp2(torch.randint(-70, 100, (2048, 2, 1), generator=gen).float())).to(BF16).view(2048, 64)
    # all ties and their neighbours under a largest number of 4 to 7.5
    ties = torch.tensor([0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 6.5, 7.0]).repeat(3)[:31]
    rows = torch.cat([torch.cat([ties * s, torch.tensor([t])]) for s in (1, 0.99, 1.01, -1) for t in (4.0, 6.0, 6.96, 7.0)]).view(-1, 64).to(BF16)
    rows = torch.cat([x, mixed, near, rows, rows * 2.0 ** -66, rows * 2.0 ** 120]).to(dtype).view(1, 1, -1, 64)
    if dtype == FP32:
        more = torch.stack([torch.full((64,), t) for t in (1e-42, 3.4e38, 7 * 2.0 ** 125, 7.0000005, 7.0, -6.9999995, 2.0 ** -64, 0.24999999, 0.25)])
        rows = torch.cat([rows, torch.randn(1, 1, 1024, 64, generator=gen) * 3, more[None, None]], dim=2)
    m = rows.shape[2]
    cache = poison(A.paged_cache(-(-m // 64), 1, 64, E2M1))
    table = torch.arange(cache.k.shape[0], dtype=torch.int32, device=DEV)[None]
    A.paged_cache_write(cache, rows.to(DEV), rows.flip(2).to(DEV), table, [0])
    y, s = P.quantise4(rows[0, 0])
    exps = cache.k_exp.cpu().view(-1, 2)[:m]
    assert torch.equal(exps.long(), s + 127)
    got = P.values4(cache.k.view(torch.uint8).cpu().view(-1, 32)[:m], exps)
    want = y * torch.exp2(s.double()).repeat_interleave(32, -1)
    assert same(got, want)
    assert torch.equal(cache.v.view(torch.uint8).cpu().view(-1, 32)[:m].flip(0), cache.k.view(torch.uint8).cpu().view(-1, 32)[:m])
    for t in (BF16, FP32):
        assert same(A.paged_cache_read(cache, table, [m], m, None, t)[0].cpu()[0, 0], want)


def cache_of(A, k, ke, v, ve):  # noqa: F811
    """One head, pages of 64 tokens in order: rows (n, 32) of codes and (n, 2) bytes."""
    def pages(x):
        return torch.cat([x, x.new_zeros((-len(x) % 64, *x.shape[1:]))]).view(-1, 1, 64, *x.shape[1:]).to(DEV)
    return A.PagedCache(pages(k).view(E2M1), pages(v).view(E2M1), pages(ke), pages(ve)), torch.arange(-(-len(k) // 64), dtype=torch.int32, device=DEV)[None]


@BOTH
def test_every_byte_read_back(A, dtype):  # noqa: F811
    """All codes in every place of a pair under all 256 bytes, another in the row's other half; what the type does not hold is rounded once."""
    codes = torch.arange(256, dtype=torch.uint8).view(8, 32).repeat(256, 1)
    first = torch.arange(256, dtype=torch.uint8).repeat_interleave(8)
    exps = torch.stack([first, first.flip(0)], -1)
    m = len(codes)
    cache, table = cache_of(A, codes, exps, codes.flip(0), exps.flip(0))
    k, v = A.paged_cache_read(cache, table, [m], m, None, dtype)
    want = P.values4(codes, exps).to(FP32).to(dtype)
    assert same(k.cpu()[0, 0], want) and same(v.cpu()[0, 0], want.flip(0))


def test_write_positions(A):  # noqa: F811
    """Starts in the middle of pages, padding, positions in front of 0 and behind the table, entries that name no page."""
    ps, g, s = 16, 2, 20
    gen = torch.Generator().manual_seed(3)
    table = torch.tensor([[3, 1, 7], [0, -1, 5], [2, 99, 4], [6, 8, 9]], dtype=torch.int32)
    start, new = [14, 10, -5, 40], [20, 17, 20, 0]
    k, v = (torch.randn(4, g, s, 64, generator=gen).to(BF16) for _ in range(2))
    cache = poison(A.paged_cache(10, g, ps, E2M1))
    A.paged_cache_write(cache, k.to(DEV), v.to(DEV), table.to(DEV), start, new)
    want = [torch.full((10, g, ps, 64), float("nan"), dtype=torch.float64) for _ in range(2)]
    for b in range(4):
        for i in range(new[b]):
            p = P.page_of(table[b].tolist(), start[b] + i, ps, 10)
            if p is not None:
                want[0][p, :, (start[b] + i) % ps] = P.stored_rows(k[b, :, i], E2M1)
                want[1][p, :, (start[b] + i) % ps] = P.stored_rows(v[b, :, i], E2M1)
    for got, w in zip(values(cache), want):
        assert same(got, w)


@pytest.mark.parametrize("counts,g,ps", [([1], 1, 16), ([5, 0, 40, 1], 8, 16), ([300, 7], 3, 64)])
def test_tokens_by_slots(A, counts, g, ps):  # noqa: F811
    gen = torch.Generator().manual_seed(sum(counts))
    table, pages = new_table(gen, counts, ps)
    t, total = table.to(DEV), sum(counts) + 2
    k, v = (torch.randn(total, g, 64, generator=gen).to(BF16).to(DEV) for _ in range(2))
    m = A.token_map(t, [0] * len(counts), counts, total, ps)
    cache = poison(A.paged_cache(pages, g, ps, E2M1))
    A.paged_cache_write_tokens(cache, k, v, m.slot)
    gk, gv = A.paged_cache_read(cache, t, counts, max(counts))
    at = 0
    for b, n in enumerate(counts):
        for got, x in ((gk, k), (gv, v)):
            assert torch.equal(got[b, :, :n].cpu().double(), P.stored_rows(x[at:at + n].transpose(0, 1).cpu(), E2M1))
        at += n
    free = pages * ps - sum(counts)
    assert all(int(torch.isnan(x).all(-1).sum()) == free * g for x in values(cache))


# ---- attention -------------------------------------------------------------------------------------------------------
@BOTH
@pytest.mark.parametrize("lens,h,g,sq,ps,w", [
    ([1], 8, 8, 1, 16, 0),
    ([1, 2, 31, 32, 33, 63, 64, 65], 8, 1, 1, 16, 0),
    ([127, 128, 129, 255, 256, 257, 1000], 8, 2, 1, 32, 0),
    ([0, 5, 0], 8, 2, 1, 16, 0),
    ([2049], 64, 8, 1, 64, 0),
    ([700, 90], 64, 1, 1, 128, 0),
    ([700, 90], 17, 1, 1, 16, 0),
    ([300, 301], 6, 2, 5, 16, 0),
    ([50, 3, 0, 2], 8, 2, 4, 16, 0),
    ([600, 333, 64], 16, 2, 8, 16, 0),
    ([600, 333, 64], 16, 2, 9, 64, 0),
    ([140, 139], 8, 2, 140, 16, 0),
    ([1500, 100, 129, 128, 127], 64, 8, 1, 16, 128),
    ([1500, 100, 17], 8, 2, 1, 64, 1),
    ([400, 77], 8, 2, 6, 16, 33),
    ([90, 333], 8, 1, 70, 32, 50),
    ([40, 41], 8, 2, 1, 16, 5000),
    ([3000, 48], 24, 2, 4, 1024, 0),
])
def test_attention(A, dtype, lens, h, g, sq, ps, w):  # noqa: F811
    print(f"case {dtype} lens={lens} H={h} G={g} Sq={sq} page={ps} window={w}", flush=True)
    cache, table, n, q, sinks, _, _ = make(A, 5 + sum(lens) + sq, lens, h, g, sq, ps, dtype, E2M1, 2)
    check(A, cache, table, n, q, sinks, w)


@BOTH
def test_attention_over_long_and_short_rows(A, dtype):  # noqa: F811
    lens = [9000, 3, 1, 4100, 64, 0, 700]
    cache, table, n, q, sinks, _, _ = make(A, 6, lens, 16, 2, 1, 16, dtype, E2M1)
    check(A, cache, table, n, q, sinks)
    for max_len in (9000, 100):
        check(A, cache, table, n, q, sinks, 0, None, max_len)
    wide = torch.cat([table, torch.full((len(lens), 4000), -1, dtype=torch.int32, device=DEV)], dim=1)
    check(A, cache, wide, n, q, sinks)


@BOTH
@pytest.mark.parametrize("lens,h,g,sq,width,w", [
    ([1024, 300, 1, 0], 16, 2, 1, 64, 0),
    ([256, 17, 255], 8, 8, 1, 16, 0),
    ([250] * 40, 16, 8, 1, 16, 0),
    ([2300, 40, 1153], 40, 1, 1, 144, 0),
    ([600, 31], 24, 2, 4, 38, 0),
    ([2900] + [0, 37, 64, 1200, 1] * 14, 12, 3, 1, 190, 0),
    ([2100, 5] * 35, 6, 3, 3, 140, 500),
    ([30, 0, 77] * 367, 4, 2, 1, 100, 0),
    ([1300] + [3] * 11, 4, 1, 40, 100, 0),
    ([1536, 7], 8, 1, 1, 96, 0),
    ([1600, 7], 8, 1, 1, 100, 0),
    ([2304, 90] + [40] * 14, 16, 8, 1, 144, 0),
    ([3456, 1000] + [40] * 31, 16, 8, 1, 216, 0),
    ([832, 31], 24, 2, 2, 52, 0),
    ([1152, 900] + [31] * 14, 24, 8, 6, 72, 0),
])
def test_attention_divisions(A, dtype, lens, h, g, sq, width, w):  # noqa: F811
    """Sizes on both sides of what decides how the work is divided."""
    print(f"case {dtype} rows={len(lens)} H={h} G={g} Sq={sq} width={width} window={w}", flush=True)
    cache, table, n, q, sinks, _, _ = make(A, 23 + sum(lens) + sq, lens, h, g, sq, 16, dtype, E2M1)
    wide = torch.full((len(lens), width), -1, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    check(A, cache, wide, n, q, sinks, w)


@BOTH
@pytest.mark.parametrize("ps", [16, 64])
@pytest.mark.parametrize("lens,h,g,sq,keys,w", [
    # pairs (a query and a head of a KV head's group) of a row: 20, 40, 64, 65, 96; few keys in all, then so many that each unit has all pairs that fit
    ([500, 90], 8, 2, 5, 512, 0), ([500, 90], 8, 2, 5, 1 << 18, 0),
    ([500, 90], 8, 1, 5, 512, 0), ([500, 90], 8, 1, 5, 1 << 18, 0),
    ([700, 8, 0], 8, 1, 8, 704, 0), ([700, 8, 0], 8, 1, 8, 1 << 18, 0),
    ([700, 66], 5, 1, 13, 704, 0), ([700, 66], 5, 1, 13, 1 << 18, 0),
    ([130, 300], 24, 2, 8, 320, 0), ([130, 300], 24, 2, 8, 1 << 18, 0),
    # no unit is cut
    ([830, 3, 64] + [5] * 50, 24, 8, 7, 832, 0),
    ([830, 3, 64] + [5] * 50, 40, 8, 8, 832, 0),
    ([830, 3, 64] + [5] * 50, 56, 8, 8, 832, 0),
    ([830, 3, 64] + [5] * 50, 64, 8, 8, 832, 0),
    # windows
    ([1000, 140, 128, 129], 64, 8, 8, 1024, 128),
    ([600, 140, 128, 129] + [9] * 260, 32, 8, 8, 640, 128),
    ([600, 140, 128, 129] + [9] * 260, 64, 8, 8, 640, 128),
])
def test_attention_units_of_few_and_many_pairs(A, dtype, lens, h, g, sq, keys, w, ps):  # noqa: F811
    print(f"case {dtype} rows={len(lens)} H={h} G={g} Sq={sq} keys={keys} window={w} page={ps}", flush=True)
    cache, table, n, q, sinks, _, _ = make(A, 29 + sum(lens) + sq, lens, h, g, sq, ps, dtype, E2M1)
    wide = torch.full((len(lens), keys // ps), -1, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    check(A, cache, wide, n, q, sinks, w)


@BOTH
def test_missing_pages_and_lengths_beyond_the_table(A, dtype):  # noqa: F811
    lens = [200, 150, 96, 300]
    cache, table, n, q, sinks, _, _ = make(A, 9, lens, 8, 2, 2, 16, dtype, E2M1)
    table[0, 1] = -1
    table[0, 5:7] = 10 ** 6
    table[1, 0] = -2 ** 31
    table[1, 9] = 2 ** 31 - 1
    table[2, :] = -1
    check(A, cache, table, n, q, sinks)
    check(A, cache, table, n, q, sinks, 40)
    o, _ = check(A, cache, table[:, :6], n, q, sinks)
    assert not o[2].any()
    check(A, cache, table, torch.tensor([-1, 2 ** 31 - 1, -2 ** 31, 299], dtype=torch.int32, device=DEV), q, sinks, 16)


@BOTH
@pytest.mark.parametrize("w", [0, 20])
def test_queries_that_start_elsewhere(A, dtype, w):  # noqa: F811
    lens, start = [100, 37, 64, 10, 5], [96, 30, 64, -3, 90]
    cache, table, n, q, sinks, _, _ = make(A, 10, lens, 8, 2, 9, 16, dtype, E2M1)
    o, lse = check(A, cache, table, n, q, sinks, w, start)
    assert not o[0, 4:].any() and not o[2].any() and not o[4].any() and not o[3, :3].any()
    assert torch.equal(lse[2], sinks.double()[:, None].expand(-1, 9).to(torch.float32).double())


@BOTH
def test_sinks(A, dtype):  # noqa: F811
    cache, table, n, q, sinks, _, _ = make(A, 11, [300, 0, 33], 8, 2, 1, 16, dtype, E2M1)
    check(A, cache, table, n, q, None)
    check(A, cache, table, n, q, torch.full((8,), float("-inf")))
    check(A, cache, table, n, q, sinks.float() + 1e-3)
    check(A, cache, table, n, q, torch.tensor([100.0, -100.0, 1e30, -1e30, 0.0, 5.0, -5.0, 30.0]))
    check(A, cache, table, n, q, sinks, scale=1.0)


@BOTH
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_rows_that_no_query_or_only_a_later_one_sees(A, dtype, bad):  # noqa: F811
    """NaN or infinity in the key and value of a token (NaN in 4 bits): queries that do not see it are as if it were not there."""
    lens, sq, ps, w = [75, 40], 4, 16, 10
    cache, table, n, q, sinks, k, v = make(A, 12, lens, 8, 2, sq, ps, dtype, E2M1)
    clean, _ = A.paged_attention_forward(q.to(DEV), cache, table, n, sinks.to(DEV), SCALE, w)
    for pos in (73, 64, 60):
        broken = A.PagedCache(*(t.view(torch.uint8).clone().view(t.dtype) for t in cache))
        x = torch.full((2, 2, 1, 64), bad, device=DEV).to(dtype)
        A.paged_cache_write(broken, x, x, table, [pos, 0], [1, 0])
        got, lse = A.paged_attention_forward(q.to(DEV), broken, table, n, sinks.to(DEV), SCALE, w)
        see = {73: [2, 3], 64: [0, 1, 2], 60: []}[pos]
        blind = [i for i in range(sq) if i not in see]
        assert torch.isfinite(got[0, blind]).all() and torch.isfinite(lse[0][:, blind]).all(), (pos, got[0, blind])
        ref, ref_lse, terms = P.attention(q, *values(broken), table.cpu(), n.cpu(), sinks, SCALE, w)
        assert bool(((got.cpu().double() - ref).abs() <= bounds(ref, ref_lse, terms, q.dtype)[0])[0, blind].all())
        assert torch.equal(got[1], clean[1])
        assert torch.isnan(got[0, see]).all() and torch.isnan(lse[0][:, see]).all()


@BOTH
@pytest.mark.parametrize("byte", [0, 1, 2, 60, 240])
@pytest.mark.parametrize("n", [50, 3000])
def test_attention_under_small_and_large_powers(A, dtype, byte, n):  # noqa: F811
    """Keys of 2^(byte - 127) under queries of its inverse, values of 2^(byte - 127); the halves' bytes differ by one."""
    gen = torch.Generator().manual_seed(71 + byte + n)
    k, v = (torch.randint(0, 256, (n, 32), generator=gen).to(torch.uint8) for _ in range(2))
    exps = torch.full((n, 2), byte, dtype=torch.uint8)
    exps[:, 1] += 1
    q = (torch.randn(1, 4, 1, 64, generator=gen).double() * 2.0 ** (124 - byte)).to(dtype)
    cache, table = cache_of(A, k, exps, v, exps)
    o, lse = A.paged_attention_forward(q.to(DEV), cache, table, [n], None, SCALE)
    pools = [torch.cat([P.values4(x, exps), torch.zeros(-n % 64, 64, dtype=torch.float64)]).view(-1, 1, 64, 64) for x in (k, v)]
    ref, ref_lse, terms = P.attention(q, *pools, table.cpu(), [n], None, SCALE)
    tol, tol_lse = bounds(ref, ref_lse, terms, dtype)
    # next to 2^-126, in place of the bound's 1e-37: steps are 2^-133 in bfloat16 and 2^-149 in float32, half of one for each row's numbers, half of one
    # for o and one for each sum
    tol = tol - 1e-37 + 2.0 ** -133 + (n + 64) * 2.0 ** -149
    assert float(ref.abs().max()) > 10 * float(tol.max())
    assert bool(((o.cpu().double() - ref).abs() <= tol).all()) and bool(((lse.cpu().double() - ref_lse).abs() <= tol_lse).all())


@BOTH
@pytest.mark.parametrize("byte,code", [(255, 2), (255, 0), (254, 4), (254, 7), (254, 3), (253, 6), (253, 15), (253, 5), (252, 7)])
@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("heads", [1, 8, 16])
def test_values_that_only_a_later_query_sees(A, dtype, byte, code, half, heads):  # noqa: F811
    """Half a row of V that is infinite or NaN by its byte: queries that do not see it are as if it were not there, and the other half is a row's like any."""
    gen = torch.Generator().manual_seed(77)
    n, sq = 60, 4
    k, v = (torch.randint(0, 256, (n, 32), generator=gen).to(torch.uint8) for _ in range(2))
    exps = torch.full((n, 2), 125, dtype=torch.uint8)
    q = torch.randn(1, heads, sq, 64, generator=gen).to(dtype).to(DEV)
    clean, table = cache_of(A, k, exps, v, exps)
    want = A.paged_attention(q, clean, table, [n], None, SCALE)
    bad, bad_exps = v.clone(), exps.clone()
    bad[58, 16 * half:16 * half + 16], bad_exps[58, half] = 0x11, byte
    bad[58, 16 * half + 3:16 * half + 6] = code | code << 4
    broken, _ = cache_of(A, k, exps, bad, bad_exps)
    value = P.values4(bad, bad_exps)[58]
    o = A.paged_attention(q, broken, table, [n], None, SCALE)
    assert torch.equal(o[:, :2], want[:, :2])
    for i in range(2, sq):
        for d in range(64):
            x = o[0, i, :, d].float().cpu()
            if not torch.isfinite(value[d]):
                assert bool(torch.isnan(x).all()) if torch.isnan(value[d]) else bool((x == float(value[d])).all()), (i, d)
            elif d // 32 != half:
                assert torch.equal(o[0, i, :, d], want[0, i, :, d]), (i, d)


@BOTH
def test_infinite_queries(A, dtype):  # noqa: F811
    cache, table, n, q, sinks, k, v = make(A, 27, [40], 4, 1, 1, 16, dtype, E2M1)
    k = k.clone()
    k[..., 9] = -1 - k[..., 9].abs()
    A.paged_cache_write(cache, k.to(DEV), v.to(DEV), table, [0])
    plain = A.paged_attention(q.to(DEV), cache, table, n, sinks.to(DEV), SCALE)
    q[:, 2, :, 9] = float("inf")
    o, lse = A.paged_attention_forward(q.to(DEV), cache, table, n, sinks.to(DEV), SCALE)
    assert not o[:, :, 2].any() and torch.equal(lse[0, 2].cpu(), sinks[2:3].float())
    for h in (0, 1, 3):
        assert torch.equal(o[:, :, h], plain[:, :, h])


@BOTH
def test_layouts(A, dtype):  # noqa: F811
    """A pool with the heads of a token side by side, one layer's slice of a larger pool, exponents with strides of their own, q out of a projection's layout, 64-bit and strided
    tables, float16."""
    lens = [130, 77, 5]
    cache, table, n, q, sinks, _, _ = make(A, 13, lens, 8, 2, 2, 32, dtype, E2M1, 2)
    o, lse = check(A, cache, table, n, q, sinks)
    raw = [t.view(torch.uint8) for t in cache]
    as_cache = lambda ts: A.PagedCache(ts[0].view(E2M1), ts[1].view(E2M1), ts[2], ts[3])
    tm = as_cache([t.transpose(1, 2).contiguous().transpose(1, 2) for t in raw])
    layers = as_cache([torch.stack([t, t, t], dim=1)[:, 1] for t in raw])
    odd = as_cache(raw[:2] + [torch.nn.functional.pad(t, (1, 2))[..., 1:3] for t in raw[2:]])
    q2 = q.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)
    t2 = torch.cat([table, table], dim=1)[:, :table.shape[1]]
    for c, qq, t, m in ((tm, q, table, n), (layers, q, table.long(), n.long()), (odd, q, table, n), (cache, q2, t2, n), (cache, q, table.t().contiguous().t(), n)):
        got, glse = A.paged_attention_forward(qq.to(DEV), c, t, m, sinks.to(DEV), SCALE)
        assert torch.equal(got.cpu().double(), o) and torch.equal(glse.cpu().double(), lse)
        assert all(torch.equal(x, y) for x, y in zip(A.paged_cache_read(c, t, m, 130), A.paged_cache_read(cache, table, n, 130)))
    if dtype == BF16:
        assert A.paged_attention(q.half().to(DEV), cache, table, n, sinks.to(DEV), SCALE).dtype == torch.float16


def test_shared_prefix(A):  # noqa: F811
    cache, table, n, q, sinks, _, _ = make(A, 14, [128, 200], 8, 2, 1, 16, BF16, E2M1)
    table[0, :8] = table[1, :8]
    check(A, cache, table, n, q, sinks)
    o, _ = check(A, cache, table[1:].expand(2, -1), torch.tensor([200, 200], dtype=torch.int32, device=DEV), q[1:].expand(2, -1, -1, -1), sinks)
    assert torch.equal(o[0], o[1])


def test_pool_beyond_32_bit_offsets(A):  # noqa: F811
    """Pages beyond 2^32 bytes, next to each other in a row and far from each other in one tile."""
    g, ps = 8, 16
    pages = (2 ** 32 // (g * ps * 32)) + 40
    cache = A.PagedCache(*(torch.empty(pages, g, ps, 32, dtype=torch.uint8, device=DEV).view(E2M1) for _ in range(2)),
                         *(torch.empty(pages, g, ps, 2, dtype=torch.uint8, device=DEV) for _ in range(2)))
    few = torch.tensor([pages - 1, 0, pages - 20, 5, pages // 2, pages - 3, 1, pages - 7], dtype=torch.int32, device=DEV)
    table = few.view(2, 4)
    gen = torch.Generator().manual_seed(15)
    k, v = (torch.randn(2, g, 64, 64, generator=gen).to(BF16) for _ in range(2))
    n = torch.tensor([64, 59], dtype=torch.int32, device=DEV)
    A.paged_cache_write(cache, k.to(DEV), v.to(DEV), table, [0, 0], n)
    gk, gv = A.paged_cache_read(cache, table, n, 64)
    for got, x in ((gk, k), (gv, v)):
        assert torch.equal(got[0].cpu().double(), P.stored_rows(x[0], E2M1)) and torch.equal(got[1, :, :59].cpu().double(), P.stored_rows(x[1, :, :59], E2M1))
    q, sinks = torch.randn(2, 16, 1, 64, generator=gen).to(BF16), torch.randn(16, generator=gen)
    o, lse = A.paged_attention_forward(q.to(DEV), cache, table, n, sinks.to(DEV), SCALE)
    small = A.PagedCache(*(t.view(torch.uint8)[few.long()].clone().view(t.dtype) for t in cache))
    t8 = torch.arange(8, dtype=torch.int32, device=DEV).view(2, 4)
    check(A, small, t8, n, q, sinks)
    o2, lse2 = A.paged_attention_forward(q.to(DEV), small, t8, n, sinks.to(DEV), SCALE)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)


def test_under_inference_mode_and_compiled(A):  # noqa: F811
    cache, table, n, q, sinks, k, v = make(A, 28, [300, 20], 8, 2, 1, 16, BF16, E2M1, 2)
    q, sinks, k, v = q.to(DEV), sinks.to(DEV), k.to(DEV), v.to(DEV)
    start = torch.tensor([3, 7], dtype=torch.int32, device=DEV)

    def calls(k):
        A.paged_cache_write(cache, k, v, table, start)
        kk, vv = A.paged_cache_read(cache, table, n, 300)
        return (kk, vv, A.paged_attention(q, cache, table, n, sinks, SCALE, 40), *A.paged_attention_forward(q, cache, table, n, sinks, SCALE))

    with torch.no_grad():
        want = calls(k)
        got = [torch.compile(calls, fullgraph=True, backend="aot_eager")(k)]
    with torch.inference_mode():
        got.append(calls(k))
    for out in got:
        assert all(torch.equal(x, y) for x, y in zip(out, want))


def test_refusals(A):  # noqa: F811
    cache = A.paged_cache(4, 2, 16, E2M1)
    table, n = torch.zeros(1, 2, dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    q = torch.zeros(1, 16, 1, 64, dtype=BF16, device=DEV)
    for text, c in (
        ("exponents", cache._replace(k_exp=None)),
        ("side by side", cache._replace(k_exp=cache.k_exp[..., 0])),
        ("side by side", cache._replace(v_exp=cache.v_exp.transpose(2, 3).contiguous().transpose(2, 3))),
        ("uint8", cache._replace(v_exp=cache.v_exp.int())),
        ("page_size, 32", cache._replace(k=cache.k.view(torch.uint8)[..., :16].view(E2M1), v=cache.v.view(torch.uint8)[..., :16].view(E2M1))),
        ("does not go with", cache._replace(v=torch.zeros(4, 2, 16, 32, dtype=BF16, device=DEV))),
        ("v_exp is on", cache._replace(v_exp=cache.v_exp.cpu())),
    ):
        with pytest.raises(RuntimeError, match=text):
            A.paged_attention(q, c, table, n, None, SCALE)
    with pytest.raises(RuntimeError, match="does not go with|unsupported"):
        A.paged_attention(q.double(), cache, table, n, None, SCALE)


# ---- streams, graphs, layers -----------------------------------------------------------------------------------------
@BOTH
def test_graph_of_a_decoding_step(A, dtype):  # noqa: F811
    """Embedding, tables, write and attention captured once; replays follow what changes on the GPU, with eager work between them."""
    b, h, g, ps, pages = 3, 16, 2, 16, 80
    gen = torch.Generator().manual_seed(17)
    rope = A.rotary_frequencies(64, 150000.0, factor=32.0, original_length=4096)
    lens = torch.tensor([700, 33, 15], dtype=torch.int32, device=DEV)
    sinks = torch.randn(h, generator=gen).to(dtype).to(DEV)
    past = [torch.randn(b, g, 700, 64, generator=gen).to(dtype).to(DEV) for _ in range(2)]
    q, k, v = (torch.zeros(b, x, 1, 64, dtype=dtype, device=DEV) for x in (h, g, g))

    def begin():
        table = torch.full((b, 60), -1, dtype=torch.int32, device=DEV)
        A.page_table_update(table, [0] * b, lens, pages, ps)
        cache = poison(A.paged_cache(pages, g, ps, E2M1))
        A.paged_cache_write(cache, *past, table, [0] * b, lens)
        return table, cache, lens.clone()

    def step(table, cache, at):
        n, _ = A.page_table_update(table, at, at + 1, pages, ps)
        qq, kk = A.rotary(q, k, at[:, None], rope)
        A.paged_cache_write(cache, kk, v, table, at)
        return A.paged_attention_forward(qq, cache, table, n, sinks, SCALE)

    table, cache, at = begin()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(table, cache, at)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = step(table, cache, at)
    fresh = begin()
    for x, y in zip((table, at, *cache), (fresh[0], fresh[2], *fresh[1])):
        x.view(torch.uint8).copy_(y.view(torch.uint8))
    eager = begin()
    for i in range(4):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=gen))
        graph.replay()
        want, want_lse = step(*eager)
        torch.cuda.synchronize()
        assert torch.equal(o, want) and torch.equal(lse, want_lse) and torch.equal(table, eager[0]), i
        ref, ref_lse, terms = P.attention(A.rotary(q, k, at[:, None], rope)[0].cpu(), *values(cache), table.cpu(), (at + 1).cpu(), sinks.cpu(), SCALE)
        assert bool(((o.cpu().double() - ref).abs() <= bounds(ref, ref_lse, terms, dtype)[0]).all()), i
        at += 1
        eager[2].add_(1)


def test_calls_on_two_streams(A):  # noqa: F811
    cache, table, n, q, sinks, _, _ = make(A, 18, [6000, 20, 3000], 16, 2, 1, 16, BF16, E2M1)
    q, sinks = q.to(DEV), sinks.to(DEV)
    n2 = (n // 2).contiguous()
    want = [A.paged_attention(q, cache, table, m, sinks, SCALE) for m in (n, n2)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for i, m in enumerate((n, n2)):
            with torch.cuda.stream(streams[i]):
                got[i].append(A.paged_attention(q, cache, table, m, sinks, SCALE))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


@pytest.mark.parametrize("window", [None, 32])
def test_prompt_chunks_and_decoding(A, window):  # noqa: F811
    """A prompt in two chunks and tokens one by one, each against the definition on what the pages hold.  attention()'s bound is that of its own tests: 2e-2 and half
    a step of the result."""
    g, h, ps, total = 2, 16, 16, 150
    gen = torch.Generator().manual_seed(19)
    q, k, v = (torch.randn(1, x, total, 64, generator=gen).to(BF16).to(DEV) for x in (h, g, g))
    sinks = torch.randn(h, generator=gen).to(BF16).to(DEV)
    cache = poison(A.paged_cache(12, g, ps, E2M1))
    table = torch.randperm(12, generator=gen).to(torch.int32)[None, :10].to(DEV)
    at = 0
    for size in (70, 61, 1, 1, 1, 5, 11):
        A.paged_cache_write(cache, k[:, :, at:at + size], v[:, :, at:at + size], table, [at])
        qs, end = q[:, :, at:at + size], at + size
        if size > 8:
            kk, vv = A.paged_cache_read(cache, table, [end], end)
            o = A.attention(qs, kk, vv, sinks, SCALE, window, at)
        else:
            o = A.paged_attention(qs, cache, table, [end], sinks, SCALE, window)
        ref, ref_lse, terms = P.attention(qs.cpu(), *values(cache), table.cpu(), [end], sinks.cpu(), SCALE, window or 0)
        tol = 2e-2 + 2.0 ** -8 * ref.abs() if size > 8 else bounds(ref, ref_lse, terms, BF16)[0]
        assert bool(((o.cpu().double() - ref).abs() <= tol).all()), at
        at = end


def test_layers_with_a_paged_state(A):  # noqa: F811
    """Layers through hip_flash_attention(paged=): prompts back to back through a map of their tokens, then tokens one by one, tables built on the GPU."""
    from types import SimpleNamespace
    g, h, ps, b, pages = 2, 16, 16, 3, 30
    gen = torch.Generator().manual_seed(25)
    sinks = torch.randn(h, generator=gen).to(BF16).to(DEV)
    modules = [SimpleNamespace(sinks=sinks, sliding_window=w, layer_idx=i) for i, w in enumerate((32, None))]
    caches = [poison(A.paged_cache(pages, g, ps, E2M1)) for _ in modules]
    table = torch.full((b, 9), -1, dtype=torch.int32, device=DEV)
    have, lens = torch.zeros(b, dtype=torch.int32, device=DEV), torch.tensor([90, 1, 37], dtype=torch.int32, device=DEV)
    for step in range(4):
        n, _ = A.page_table_update(table, have, lens, pages, ps)
        assert torch.equal(n, lens)
        if step == 0:
            tokens = A.token_map(table, have, lens, 130, ps)
            state, shape = A.PagedState(caches, table, None, n, tokens=tokens), (1, 130)
        else:
            state, shape = A.PagedState(caches, table, have, n), (b, 1)
        for module in modules:
            q, k, v = (torch.randn(*shape, x, 64, generator=gen).to(BF16).to(DEV).transpose(1, 2) for x in (h, g, g))
            o, _ = A.hip_flash_attention(module, q, k, v, None, SCALE, paged=state)
            cache = caches[module.layer_idx]
            if step == 0:
                kk, vv = A.paged_cache_read(cache, table, n, 90)
                at = 0
                for r, c in enumerate(lens.tolist()):
                    for x, y in ((kk, k), (vv, v)):
                        assert torch.equal(x[r, :, :c].cpu().double(), P.stored_rows(y[0, :, at:at + c].cpu(), E2M1))
                    at += c
                continue
            ref, ref_lse, terms = P.attention(q.cpu(), *values(cache), table.cpu(), n.cpu(), sinks.cpu(), SCALE, module.sliding_window or 0)
            assert bool(((o.cpu().double() - ref).abs() <= bounds(ref, ref_lse, terms, BF16)[0]).all()), (step, module.layer_idx)
        have, lens = n, n + 1


def test_float16_goes_through_bfloat16(A):  # noqa: F811
    """Tokens and queries in float16 are those in bfloat16, rounded; results come back in float16."""
    lens, g, ps = [70, 33], 2, 16
    cache, table, n, q, sinks, _, _ = make(A, 41, lens, 8, g, 1, ps, BF16, E2M1)
    gen = torch.Generator().manual_seed(5)
    k, v = (torch.randn(40, g, 64, generator=gen).to(torch.float16).to(DEV) for _ in range(2))
    a, b = A.paged_cache(4, g, ps, E2M1), A.paged_cache(4, g, ps, E2M1)
    slots = torch.randperm(64, generator=gen)[:40].to(DEV)
    A.paged_cache_write_tokens(a, k, v, slots)
    A.paged_cache_write_tokens(b, k.to(BF16), v.to(BF16), slots)
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))
    half, sinks = q.to(DEV, torch.float16), sinks.to(DEV)
    o = A.paged_attention(half, cache, table, n, sinks, 0.125)
    assert o.dtype == torch.float16 and torch.equal(o, A.paged_attention(half.to(BF16), cache, table, n, sinks, 0.125).to(torch.float16))
    got = A.paged_cache_read(cache, table, n, 70, dtype=torch.float16)
    assert all(x.dtype == torch.float16 and torch.equal(x, y.to(torch.float16)) for x, y in zip(got, A.paged_cache_read(cache, table, n, 70)))


def test_float16_beside_a_tie(A):  # noqa: F811
    """What the documents say of float16 numbers next to the middle between two codes: as they are, rounded to bfloat16 first; as float32, to the nearest code of their own."""
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    row = torch.cat([t * (1 + torch.tensor([-2.0, -1.0, 1.0, 2.0]) * 2.0 ** -10) for t in ties] + [torch.tensor([6.0, 0.0, 1.0, 2.0])])
    x = torch.cat([row, -row]).to(torch.float16).view(1, 1, 64).to(DEV)
    table, n = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    for given, counts in ((x, x.to(BF16)), (x.float(), x)):
        cache = A.paged_cache(1, 1, 16, E2M1)
        A.paged_cache_write_tokens(cache, given, given, torch.zeros(1, dtype=torch.int64, device=DEV))
        got = A.paged_cache_read(cache, table, n, 1, None, FP32)[0].cpu().double().view(64)
        assert torch.equal(got, P.stored_rows(counts.cpu().view(1, 64), E2M1)[0])
