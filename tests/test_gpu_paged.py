"""GPU tests of the key / value cache in pages: writes and reads bit by bit, attention within bounds that follow from its roundings
(oracle/paged_ref.py), against the definition in 64 bits.  Every slot that holds no token of the call is NaN."""
import pytest
import torch

from oracle import paged_ref as P

pytestmark = pytest.mark.gpu
DEV, SCALE = "cuda", 0.125
BF16, FP32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
TYPES = [(BF16, BF16), (BF16, E4M3), (FP32, FP32), (FP32, E4M3)]
TYPE_IDS = ["bf16", "bf16-e4m3", "fp32", "fp32-e4m3"]


@pytest.fixture(scope="module")
def A():
    import oregon_gpt_oss_patching_amd as A_
    from oregon_gpt_oss_patching_amd import _lib
    _lib.load()
    return A_


def poison(cache):
    cache.k.view(torch.uint8).fill_(0xff)          # NaN in all three types
    cache.v.view(torch.uint8).fill_(0xff)
    if cache.k_exp is not None:
        cache.k_exp.fill_(0xff)
        cache.v_exp.fill_(0xff)
    return cache


def new_cache(A, pages, g, ps, storage, token_major=False):
    if not token_major:
        return poison(A.paged_cache(pages, g, ps, storage))
    # (pages, page_size, G, 64) underneath: a page's tokens with their heads side by side
    k, v = (torch.zeros(pages, ps, g, 64, device=DEV, dtype=storage).transpose(1, 2) for _ in range(2))
    e = [torch.zeros(pages, ps, g, device=DEV, dtype=torch.uint8).transpose(1, 2) for _ in range(2)] if storage == E4M3 else [None, None]
    return poison(A.PagedCache(k, v, *e))


def values(cache):
    """The pools' values in 64 bits on the CPU."""
    out = []
    for x, e in ((cache.k, cache.k_exp), (cache.v, cache.v_exp)):
        x = x.cpu().float().double()
        out.append(x if e is None else x * torch.exp2(e.cpu().double() - 127)[..., None])
    return out


def new_table(gen, lens, ps, extra=0):
    """Pages in no order for rows of these lengths, -1 behind them, and how many pages there are."""
    used = [-(-n // ps) for n in lens]
    order = torch.randperm(sum(used) + 2, generator=gen).to(torch.int32)
    table = torch.full((len(lens), max(used + [1]) + extra), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    return table, sum(used) + 2


def make(A, seed, lens, h, g, sq, ps, dtype, storage, extra=0, token_major=False):
    """A poisoned pool with rows of these lengths written through paged_cache_write, q and sink logits."""
    gen = torch.Generator().manual_seed(seed)
    table, pages = new_table(gen, lens, ps, extra)
    cache = new_cache(A, pages, g, ps, storage, token_major)
    longest = max(max(lens), 1)
    k, v = (torch.randn(len(lens), g, longest, 64, generator=gen).to(dtype) for _ in range(2))
    t = table.to(DEV)
    zero = torch.zeros(len(lens), dtype=torch.int32, device=DEV)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    A.paged_cache_write(cache, k.to(DEV), v.to(DEV), t, zero, n)
    q = torch.randn(len(lens), h, sq, 64, generator=gen).to(dtype)
    sinks = torch.randn(h, generator=gen).to(dtype)
    return cache, t, n, q, sinks, k, v


def check(A, cache, table, n, q, sinks, window=0, start=None, max_len=None, scale=SCALE):
    o, lse = A.paged_attention_forward(q.to(DEV), cache, table, n, None if sinks is None else sinks.to(DEV), scale, window or None,
                                       None if start is None else torch.tensor(start, dtype=torch.int32, device=DEV), max_len)
    again, lse2 = A.paged_attention_forward(q.to(DEV), cache, table, n, None if sinks is None else sinks.to(DEV), scale, window or None,
                                            None if start is None else torch.tensor(start, dtype=torch.int32, device=DEV), max_len)
    assert torch.equal(o, again) and torch.equal(lse, lse2)
    alone = A.paged_attention(q.to(DEV), cache, table, n, None if sinks is None else sinks.to(DEV), scale, window or None,
                              None if start is None else torch.tensor(start, dtype=torch.int32, device=DEV), max_len)
    assert torch.equal(o, alone)
    ref, ref_lse, terms = P.attention(q, *values(cache), table.cpu(), n.cpu(), sinks, scale, window, start)
    assert o.dtype == q.dtype and o.shape == ref.shape and lse.shape == ref_lse.shape
    tol, tol_lse = P.bounds(ref, ref_lse, terms, q.dtype)
    o, lse = o.cpu().double(), lse.cpu().double()
    assert torch.isfinite(o).all()
    over = (o - ref).abs() - tol
    assert bool((over <= 0).all()), (float(over.max()), [int(x) for x in torch.nonzero(over == over.max())[0]])
    none = torch.isinf(ref_lse)
    assert torch.equal(none, torch.isinf(lse)) and bool(((lse - ref_lse).abs() <= tol_lse)[~none].all()), float((lse - ref_lse).abs()[~none].max())
    return o, lse


# ---- writing and reading ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,storage", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("lens,g,ps,token_major", [
    ([1], 1, 16, False),
    ([1, 15, 16, 17], 2, 16, False),
    ([40, 0, 133], 8, 32, True),                       # an empty row between two
    ([300, 299], 3, 64, False),
    ([1025, 7], 2, 1024, True),
])
def test_write_then_read(A, dtype, storage, lens, g, ps, token_major):
    print(f"case {dtype} {storage} lens={lens} G={g} page={ps} token_major={token_major}", flush=True)
    cache, table, n, _, _, k, v = make(A, 1, lens, g, g, 1, ps, dtype, storage, 1, token_major)
    longest = max(lens) + 3                            # rows behind every sequence
    gk, gv = A.paged_cache_read(cache, table, n, longest, None, dtype)
    assert gk.dtype == dtype and gk.shape == (len(lens), g, longest, 64)
    for got, x in ((gk, k), (gv, v)):
        want = torch.zeros(got.shape, dtype=torch.float64)
        for b, m in enumerate(lens):
            want[b, :, :m] = P.stored_rows(x[b, :, :m], storage)
        assert torch.equal(got.cpu().double(), want)
    # nothing else of the pool is touched: as many NaN rows as slots without a token
    free = cache.k.shape[0] * ps - sum(lens)
    for x in values(cache):
        nan = torch.isnan(x)
        assert int(nan.all(-1).sum()) == free * g and int(nan.any(-1).sum()) == free * g


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_e4m3_codes_of_every_bfloat16_number(A, dtype):
    """All 65536 bfloat16 numbers among rows whose largest one sets different powers of two, infinities and NaN among them."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF16).view(1024, 64)
    gen = torch.Generator().manual_seed(2)
    mixed = x.reshape(-1)[torch.randperm(65536, generator=gen)].view(1024, 64)
    near = (torch.randn(1024, 64, generator=gen) * torch.exp2(torch.randint(-70, 100, (1024, 1), generator=gen).float())).to(BF16)
    rows = torch.cat([x, mixed, near]).to(dtype).view(1, 1, -1, 64)
    if dtype == FP32:
        rows = torch.cat([rows, torch.randn(1, 1, 1024, 64, generator=gen) * 3, torch.full((1, 1, 1, 64), 1e-42)], dim=2)
    m = rows.shape[2]
    cache = new_cache(A, -(-m // 64), 1, 64, E4M3)
    table = torch.arange(cache.k.shape[0], dtype=torch.int32, device=DEV)[None]
    A.paged_cache_write(cache, rows.to(DEV), rows.flip(2).to(DEV), table, [0])
    y, s = P.quantise(rows[0, 0])
    codes, exps = cache.k.cpu().view(-1, 64)[:m], cache.k_exp.cpu().view(-1)[:m]
    assert torch.equal(exps.long(), s + 127)
    assert torch.equal(codes.float().nan_to_num(nan=1000.0).double(), y.nan_to_num(nan=1000.0))
    assert torch.equal(cache.v.cpu().view(-1, 64)[:m].flip(0).view(torch.uint8), codes.view(torch.uint8))
    for t in (BF16, FP32):
        got = A.paged_cache_read(cache, table, [m], m, None, t)[0].cpu().double().view(-1, 64)
        want = y * torch.exp2(s.double())[:, None]
        assert torch.equal(got.nan_to_num(nan=1e39), want.nan_to_num(nan=1e39))


def test_write_positions(A):
    """Starts in the middle of pages, padding behind the new tokens, positions in front of 0 and behind the table, entries that name no page."""
    ps, g, s = 16, 2, 20
    gen = torch.Generator().manual_seed(3)
    table = torch.tensor([[3, 1, 7], [0, -1, 5], [2, 99, 4], [6, 8, 9]], dtype=torch.int32)      # a pool of 10
    start, new = [14, 10, -5, 40], [20, 17, 20, 0]
    k, v = (torch.randn(4, g, s, 64, generator=gen).to(BF16) for _ in range(2))
    cache = new_cache(A, 10, g, ps, BF16)
    A.paged_cache_write(cache, k.to(DEV), v.to(DEV), table.to(DEV), start, new)
    want = [torch.full((10, g, ps, 64), float("nan"), dtype=torch.float64) for _ in range(2)]
    for b in range(4):
        for i in range(new[b]):
            p = P.page_of(table[b].tolist(), start[b] + i, ps, 10)
            if p is not None:
                want[0][p, :, (start[b] + i) % ps] = k[b, :, i].double()
                want[1][p, :, (start[b] + i) % ps] = v[b, :, i].double()
    for got, w in zip(values(cache), want):
        assert torch.equal(got.nan_to_num(nan=1e39), w.nan_to_num(nan=1e39))
    # the rows back, from in front of 0 on
    gk, _ = A.paged_cache_read(cache, table.to(DEV), [34, 27, 15, 48], 60, [-3, 0, 5, 0])
    for b, (n, first) in enumerate(zip([34, 27, 15, 48], [-3, 0, 5, 0])):
        for i in range(60):
            pos = first + i
            p = P.page_of(table[b].tolist(), pos, ps, 10) if pos < n else None
            w = torch.zeros(g, 64, dtype=torch.float64) if p is None else want[0][p, :, pos % ps]
            assert torch.equal(gk[b, :, i].cpu().double().nan_to_num(nan=1e39), w.nan_to_num(nan=1e39)), (b, i)


def test_strided_sources_and_float16(A):
    """Values as a transposed view, keys cut out of a wider tensor, a source whose rows are not aligned; float16 as bfloat16."""
    gen = torch.Generator().manual_seed(4)
    wide = torch.randn(2, 5, 4, 3, 64, generator=gen).to(BF16).to(DEV)
    table = torch.tensor([[1], [0]], dtype=torch.int32, device=DEV)
    for k in (wide[:, :, :2, 1].transpose(1, 2), wide[:, :, 1:3, 0].transpose(1, 2), torch.randn(2, 2, 5, 65, device=DEV).to(BF16)[..., 1:],
              torch.randn(2, 2, 5, 64, device=DEV).half()):
        cache = new_cache(A, 2, 2, 16, BF16)
        A.paged_cache_write(cache, k, k, table, [0, 3])
        got = A.paged_cache_read(cache, table, [5, 8], 5, [0, 3], k.dtype)[0]
        assert torch.equal(got, k.to(BF16).to(k.dtype))


@pytest.mark.parametrize("dtype,storage", TYPES, ids=TYPE_IDS)
def test_dimensions_of_one_and_addresses_between_16_bytes(A, dtype, storage):
    """Strides of dimensions with one element say nothing, whatever they are; rows on other addresses are copied."""
    gen = torch.Generator().manual_seed(26)
    table = torch.tensor([[1, 0]], dtype=torch.int32, device=DEV)
    for g, h, s in ((1, 1, 1), (2, 8, 1), (1, 4, 3)):
        k, v, q = (torch.randn(1, x, s, 64, generator=gen).to(dtype).to(DEV) for x in (g, g, h))

        def odd(x, strides, at=0):
            y = torch.empty(x.numel() * 2 + 64, dtype=dtype, device=DEV)[at:].as_strided(x.shape, strides)
            y.copy_(x)
            return y

        want = None
        for at in (0, 1):
            st = lambda x: (7, 5 if x.shape[1] == 1 else 64 * s, 3 if s == 1 else 64, 1)
            kk, vv, qq = (odd(x, st(x), at) for x in (k, v, q))
            cache = A.paged_cache(2, g, 16, storage)
            A.paged_cache_write(cache, kk, vv, table, [5])
            o = A.paged_attention(qq, cache, table, [5 + s], None, SCALE, None, [5])
            if want is None:
                plain = A.paged_cache(2, g, 16, storage)
                A.paged_cache_write(plain, k, v, table, [5])
                want = A.paged_attention(q, plain, table, [5 + s], None, SCALE, None, [5])
            for x, y in zip(cache, plain):
                assert x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8))
            assert torch.equal(o, want)


def test_under_inference_mode(A):
    with torch.inference_mode():
        cache = A.paged_cache(2, 1, 16, E4M3)
        table, k = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.ones(1, 1, 4, 64, dtype=BF16, device=DEV)
        A.paged_cache_write(cache, k, k, table, [0])
        assert torch.equal(A.paged_cache_read(cache, table, [4], 4)[0], k)
        assert torch.equal(A.paged_attention(k[:, :, :1], cache, table, [4], torch.full((1,), -float("inf"), device=DEV), SCALE), k[:, :, :1])


# ---- attention -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,storage", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("lens,h,g,sq,ps,w", [
    ([1], 8, 8, 1, 16, 0),                             # a single key, a head of its own for each
    ([1, 2, 31, 32, 33, 63, 64, 65], 8, 1, 1, 16, 0),  # around the tiles' ends
    ([127, 128, 129, 255, 256, 257, 1000], 8, 2, 1, 32, 0),
    ([0, 5, 0], 8, 2, 1, 16, 0),                       # rows without a token
    ([2049], 64, 8, 1, 64, 0),
    ([700, 90], 64, 1, 1, 128, 0),                     # 64 heads on one
    ([700, 90], 17, 1, 1, 16, 0),                      # 17: the second block of columns holds one
    ([300, 301], 6, 2, 5, 16, 0),                      # groups of three heads
    ([50, 3, 0, 2], 8, 2, 4, 16, 0),                   # more queries than tokens
    ([600, 333, 64], 16, 2, 8, 16, 0),                 # 64 pairs
    ([600, 333, 64], 16, 2, 9, 64, 0),                 # 72
    ([140, 139], 8, 2, 140, 16, 0),                    # a prompt's worth of queries
    ([1500, 100, 129, 128, 127], 64, 8, 1, 16, 128),   # windows
    ([1500, 100, 17], 8, 2, 1, 64, 1),
    ([400, 77], 8, 2, 6, 16, 33),
    ([90, 333], 8, 1, 70, 32, 50),
    ([40, 41], 8, 2, 1, 16, 5000),                     # a window beyond the row
])
def test_attention(A, dtype, storage, lens, h, g, sq, ps, w):
    print(f"case {dtype} {storage} lens={lens} H={h} G={g} Sq={sq} page={ps} window={w}", flush=True)
    cache, table, n, q, sinks, _, _ = make(A, 5 + sum(lens) + sq, lens, h, g, sq, ps, dtype, storage, 2)
    check(A, cache, table, n, q, sinks, w)


@pytest.mark.parametrize("dtype,storage", TYPES, ids=TYPE_IDS)
def test_attention_over_long_and_short_rows(A, dtype, storage):
    """Rows whose work is divided among many workgroups beside rows of one tile; with and without the longest length given, also too short."""
    lens = [9000, 3, 1, 4100, 64, 0, 700]
    cache, table, n, q, sinks, _, _ = make(A, 6, lens, 16, 2, 1, 16, dtype, storage)
    o, _ = check(A, cache, table, n, q, sinks)
    for max_len in (9000, 100):
        check(A, cache, table, n, q, sinks, 0, None, max_len)
    # a table far wider than the rows
    wide = torch.cat([table, torch.full((len(lens), 4000), -1, dtype=torch.int32, device=DEV)], dim=1)
    check(A, cache, wide, n, q, sinks)


@pytest.mark.parametrize("dtype,storage", TYPES, ids=TYPE_IDS)
def test_attention_many_rows(A, dtype, storage):
    gen = torch.Generator().manual_seed(7)
    lens = torch.randint(0, 200, (300,), generator=gen).tolist()
    cache, table, n, q, sinks, _, _ = make(A, 8, lens, 4, 1, 1, 16, dtype, storage)
    check(A, cache, table, n, q, sinks)


@pytest.mark.parametrize("dtype,storage", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("lens,h,g,sq,width,w", [
    ([1024, 300, 1, 0], 16, 2, 1, 64, 0),                         # rows that many wavefronts walk without a second launch
    ([256, 17, 255], 8, 8, 1, 16, 0),
    ([250] * 40, 16, 8, 1, 16, 0),
    ([2300, 40, 1153], 40, 1, 1, 144, 0),                         # 40 pairs: three blocks of columns, cut
    ([600, 31], 24, 2, 4, 38, 0),                                 # 48, not cut (bfloat16)
    ([2900] + [0, 37, 64, 1200, 1] * 14, 12, 3, 1, 190, 0),       # 71 rows, more than a wavefront has lanes
    ([2100, 5] * 35, 6, 3, 3, 140, 500),
    ([30, 0, 77] * 367, 4, 2, 1, 100, 0),                         # 1101 rows in a table of 1600 tokens
    ([1300] + [3] * 11, 4, 1, 40, 100, 0),                        # blocks of pairs beside rows
    ([1536, 7], 8, 1, 1, 96, 0),                                  # codes are walked alone for longer than other rows
    ([2304, 90] + [40] * 14, 16, 8, 1, 144, 0),
    ([3456, 1000] + [40] * 31, 16, 8, 1, 216, 0),
    ([832, 31], 24, 2, 2, 52, 0),
    ([1152, 900] + [31] * 14, 24, 8, 6, 72, 0),
])
def test_attention_divisions(A, dtype, storage, lens, h, g, sq, width, w):
    """Sizes on both sides of what decides how the work is divided."""
    print(f"case {dtype} {storage} rows={len(lens)} H={h} G={g} Sq={sq} width={width} window={w}", flush=True)
    cache, table, n, q, sinks, _, _ = make(A, 23 + sum(lens) + sq, lens, h, g, sq, 16, dtype, storage)
    wide = torch.full((len(lens), width), -1, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    check(A, cache, wide, n, q, sinks, w)


@pytest.mark.parametrize("dtype,storage", TYPES, ids=TYPE_IDS)
def test_missing_pages_and_lengths_beyond_the_table(A, dtype, storage):
    """Entries of -1 and beyond the pool inside a row: their keys are invisible; a row of nothing else sees nothing.  A length behind the table's end is the
    table's end."""
    lens = [200, 150, 96, 300]
    cache, table, n, q, sinks, _, _ = make(A, 9, lens, 8, 2, 2, 16, dtype, storage)
    table[0, 1] = -1
    table[0, 5:7] = 10 ** 6
    table[1, 0] = -2 ** 31
    table[1, 9] = 2 ** 31 - 1
    table[2, :] = -1
    check(A, cache, table, n, q, sinks)
    check(A, cache, table, n, q, sinks, 40)
    narrow = table[:, :6]
    o, _ = check(A, cache, narrow, n, q, sinks)
    assert not o[2].any()
    check(A, cache, table, torch.tensor([-1, 2 ** 31 - 1, -2 ** 31, 299], dtype=torch.int32, device=DEV)[:4], q, sinks, 16)


@pytest.mark.parametrize("dtype,storage", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("w", [0, 20])
def test_queries_that_start_elsewhere(A, dtype, storage, w):
    """Right-padded new tokens: each row's queries from a position of its own, the last of them behind the sequence or in front of it."""
    lens, start = [100, 37, 64, 10, 5], [96, 30, 64, -3, 90]
    cache, table, n, q, sinks, _, _ = make(A, 10, lens, 8, 2, 9, 16, dtype, storage)
    o, lse = check(A, cache, table, n, q, sinks, w, start)
    assert not o[0, 4:].any() and not o[2].any() and not o[4].any() and not o[3, :3].any()
    assert torch.equal(lse[2], sinks.double()[:, None].expand(-1, 9).to(torch.float32).double())


@pytest.mark.parametrize("dtype,storage", TYPES, ids=TYPE_IDS)
def test_sinks(A, dtype, storage):
    """None (a logit of 0), -inf (no sink; a row without keys then has lse -inf), float32 and bfloat16 logits, very large ones."""
    lens = [300, 0, 33]
    cache, table, n, q, sinks, _, _ = make(A, 11, lens, 8, 2, 1, 16, dtype, storage)
    check(A, cache, table, n, q, None)
    check(A, cache, table, n, q, torch.full((8,), float("-inf")))
    check(A, cache, table, n, q, sinks.float() + 1e-3)
    check(A, cache, table, n, q, torch.tensor([100.0, -100.0, 1e30, -1e30, 0.0, 5.0, -5.0, 30.0]))
    check(A, cache, table, n, q, sinks, scale=1.0)


@pytest.mark.parametrize("dtype,storage", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_rows_that_no_query_or_only_a_later_one_sees(A, dtype, storage, bad):
    """NaN or infinity in the key and value of a token: queries that do not see it are as if it were not there, those that do give NaN where it
    is a NaN."""
    lens, sq, ps, w = [75, 40], 4, 16, 10
    cache, table, n, q, sinks, k, v = make(A, 12, lens, 8, 2, sq, ps, dtype, storage)
    clean, _ = A.paged_attention_forward(q.to(DEV), cache, table, n, sinks.to(DEV), SCALE, w)
    for pos in (73, 64, 60):
        # queries at 71, 72, 73, 74 see 10 keys each: 73 is seen by the last two, 64 by the first three, 60 by none
        broken = A.PagedCache(*(None if t is None else t.clone() for t in cache))
        x = torch.full((2, 2, 1, 64), bad, device=DEV).to(dtype)
        A.paged_cache_write(broken, x, x, table, [pos, 0], [1, 0])
        got, lse = A.paged_attention_forward(q.to(DEV), broken, table, n, sinks.to(DEV), SCALE, w)
        see = {73: [2, 3], 64: [0, 1, 2], 60: []}[pos]
        blind = [i for i in range(sq) if i not in see]
        assert torch.isfinite(got[0, blind]).all() and torch.isfinite(lse[0][:, blind]).all(), (pos, got[0, blind])
        ref, ref_lse, terms = P.attention(q, *values(broken), table.cpu(), n.cpu(), sinks, SCALE, w)
        tol, _ = P.bounds(ref, ref_lse, terms, q.dtype)
        assert bool(((got.cpu().double() - ref).abs() <= tol)[0, blind].all())
        assert torch.equal(got[1], clean[1])
        if storage == E4M3 or bad != bad:                                  # (an infinity is NaN in 8 bits)
            assert torch.isnan(got[0, see]).all() and torch.isnan(lse[0][:, see]).all()


@pytest.mark.parametrize("dtype,storage", TYPES, ids=TYPE_IDS)
def test_infinite_queries(A, dtype, storage):
    """A query with an infinity where all keys are negative has logits of -inf alone: no weight but the sink's."""
    cache, table, n, q, sinks, k, v = make(A, 27, [40], 4, 1, 1, 16, dtype, storage)
    k = k.clone()
    k[..., 9] = -1 - k[..., 9].abs()
    A.paged_cache_write(cache, k.to(DEV), v.to(DEV), table, [0])
    plain = A.paged_attention(q.to(DEV), cache, table, n, sinks.to(DEV), SCALE)
    q[:, 2, :, 9] = float("inf")
    o, lse = A.paged_attention_forward(q.to(DEV), cache, table, n, sinks.to(DEV), SCALE)
    assert not o[:, :, 2].any() and torch.equal(lse[0, 2].cpu(), sinks[2:3].float())
    for h in (0, 1, 3):
        assert torch.equal(o[:, :, h], plain[:, :, h])


def test_positions_at_the_end_of_the_longest_table(A):
    """2^30 tokens: the last one exists, positions behind it do not, whatever they are."""
    table = torch.full((1, 1 << 20), -1, dtype=torch.int32, device=DEV)
    table[0, -1] = 0
    cache, n = A.paged_cache(1, 1, 1024), [1 << 30]
    k = torch.ones(1, 1, 1, 64, dtype=BF16, device=DEV)
    A.paged_cache_write(cache, k, k, table, [(1 << 30) - 1])
    assert bool((cache.k[0, 0, -1] == 1).all()) and not cache.k[0, 0, :-1].any()
    sinks = torch.full((1,), -float("inf"), device=DEV)
    assert torch.equal(A.paged_attention(k, cache, table, n, sinks, SCALE, 1, [(1 << 30) - 1]), k)
    for start in (1 << 30, 2 ** 31 - 1, -1, -2 ** 31):
        assert not A.paged_attention(k, cache, table, n, sinks, SCALE, 1, [start]).any()


@pytest.mark.parametrize("dtype,storage", TYPES, ids=TYPE_IDS)
def test_layouts(A, dtype, storage):
    """A pool with the heads of a token side by side, one layer's slice of a larger pool, q out of a projection's layout, 64-bit and strided tables."""
    lens = [130, 77, 5]
    cache, table, n, q, sinks, _, _ = make(A, 13, lens, 8, 2, 2, 32, dtype, storage, 2)
    o, lse = check(A, cache, table, n, q, sinks)
    tm = A.PagedCache(*(None if t is None else t.transpose(1, 2).contiguous().transpose(1, 2) for t in cache))
    layers = A.PagedCache(*(None if t is None else torch.stack([t, t, t], dim=1)[:, 1] for t in cache))
    q2 = q.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)
    t2 = torch.cat([table, table], dim=1)[:, :table.shape[1]]
    for c, qq, t, m in ((tm, q, table, n), (layers, q, table.long(), n.long()), (cache, q2, t2, n), (cache, q, table.t().contiguous().t(), n)):
        got, glse = A.paged_attention_forward(qq.to(DEV), c, t, m, sinks.to(DEV), SCALE)
        assert torch.equal(got.cpu().double(), o) and torch.equal(glse.cpu().double(), lse)
    if dtype == BF16:
        half = A.paged_attention(q.half().to(DEV), cache, table, n, sinks.to(DEV), SCALE)
        assert half.dtype == torch.float16


@pytest.mark.parametrize("storage", [BF16, E4M3])
def test_shared_prefix(A, storage):
    """Rows whose tables begin with the same pages."""
    cache, table, n, q, sinks, _, _ = make(A, 14, [128, 200], 8, 2, 1, 16, BF16, storage)
    table[0, :8] = table[1, :8]
    check(A, cache, table, n, q, sinks)
    same = table[1:].expand(2, -1)
    o, _ = check(A, cache, same, torch.tensor([200, 200], dtype=torch.int32, device=DEV), q[1:].expand(2, -1, -1, -1), sinks)
    assert torch.equal(o[0], o[1])


@pytest.mark.parametrize("dtype,storage", TYPES, ids=TYPE_IDS)
def test_pool_beyond_32_bit_offsets(A, dtype, storage):
    """Pages whose elements lie beyond 2^31 (4- and 2-byte types) and 2^32 bytes (codes)."""
    g, ps = 8, 128
    pages = (2 ** 32 // (g * ps * 64)) + 40
    empty = [torch.empty(pages, g, ps, 64, dtype=storage, device=DEV) for _ in range(2)]
    exps = [torch.empty(pages, g, ps, dtype=torch.uint8, device=DEV) if storage == E4M3 else None for _ in range(2)]
    cache = A.PagedCache(*empty, *exps)
    table = torch.tensor([[pages - 1, 0, pages - 20], [5, pages // 2, pages - 3]], dtype=torch.int32, device=DEV)
    gen = torch.Generator().manual_seed(15)
    k, v = (torch.randn(2, g, 300, 64, generator=gen).to(dtype) for _ in range(2))
    n = torch.tensor([300, 290], dtype=torch.int32, device=DEV)
    A.paged_cache_write(cache, k.to(DEV), v.to(DEV), table, [0, 0], n)
    gk, gv = A.paged_cache_read(cache, table, n, 300, None, dtype)
    for got, x in ((gk, k), (gv, v)):
        assert torch.equal(got[0].cpu().double(), P.stored_rows(x[0], storage)) and torch.equal(got[1, :, :290].cpu().double(), P.stored_rows(x[1, :, :290], storage))
    q, sinks = torch.randn(2, 16, 1, 64, generator=gen).to(dtype), torch.randn(16, generator=gen)
    o, lse = A.paged_attention_forward(q.to(DEV), cache, table, n, sinks.to(DEV), SCALE)
    small = table.flatten().long()
    few = A.PagedCache(*(None if t is None else t[small].clone() for t in cache))
    check(A, few, torch.arange(6, dtype=torch.int32, device=DEV).view(2, 3), n, q, sinks)
    o2, lse2 = A.paged_attention_forward(q.to(DEV), few, torch.arange(6, dtype=torch.int32, device=DEV).view(2, 3), n, sinks.to(DEV), SCALE)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)


def test_refusals(A):
    cache = A.paged_cache(4, 2, 16)
    table, n = torch.zeros(1, 2, dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    q, k = torch.zeros(1, 16, 1, 64, dtype=BF16, device=DEV), torch.zeros(1, 2, 1, 64, dtype=BF16, device=DEV)
    from oregon_gpt_oss_patching_amd._lib import GptossAttnError
    for text, call in (
        ("does not go with", lambda: A.paged_attention(q.float(), cache, table, n, None, SCALE)),
        ("does not go with", lambda: A.paged_cache_write(cache, k.float(), k.float(), table, n)),
        ("does not go with", lambda: A.paged_cache_read(cache, table, n, 4, None, torch.float32)),
        ("must be", lambda: A.paged_attention(q[..., :32], cache, table, n, None, SCALE)),
        ("one integer per", lambda: A.paged_attention(q, cache, table, n.repeat(2), None, SCALE)),
        ("one integer per", lambda: A.paged_attention(q, cache, table, n.float(), None, SCALE)),
        ("page_table", lambda: A.paged_attention(q, cache, table[0], n, None, SCALE)),
        ("page_table", lambda: A.paged_attention(q, cache, table.repeat(2, 1), n, None, SCALE)),
        ("one logit per", lambda: A.paged_attention(q, cache, table, n, torch.zeros(3, device=DEV), SCALE)),
        ("sinks is on", lambda: A.paged_attention(q, cache, table, n, torch.zeros(16), SCALE)),
        ("q is on", lambda: A.paged_attention(q.cpu(), cache, table, n, None, SCALE)),
        ("k is on", lambda: A.paged_cache_write(cache, k.cpu(), k.cpu(), table, n)),
        ("for this cache", lambda: A.paged_cache_write(cache, q, q, table, n)),
        ("both be", lambda: A.paged_cache_write(cache, k, q, table, n)),
        ("max_len", lambda: A.paged_cache_read(cache, table, n, 0)),
        ("rows of 64 must be contiguous", lambda: A.paged_attention(q, A.PagedCache(*(torch.zeros(4, 2, 16, 128, dtype=BF16, device=DEV)[..., ::2] for _ in range(2))), table, n, None, SCALE)),
        ("exponents", lambda: A.paged_attention(q, A.PagedCache(cache.k.to(E4M3), cache.v.to(E4M3)), table, n, None, SCALE)),
        ("must not be negative", lambda: A.paged_attention(q, cache, table, n, None, SCALE, -3)),
    ):
        with pytest.raises(RuntimeError, match=text):
            call()
    for status, call in (
        (-4, lambda: A.paged_attention(q[:, :15], cache, table, n, None, SCALE)),
        (-5, lambda: A.paged_attention(q, cache, table, n, None, 0.0)),
        (-5, lambda: A.paged_attention(q[:, :, :0], cache, table, n, None, SCALE)),
        (-11, lambda: A.paged_attention(q, A.PagedCache(cache.k[:, :, :8], cache.v[:, :, :8]), table, n, None, SCALE)),
        (-11, lambda: A.paged_attention(q, cache, table[:, :0], n, None, SCALE)),
    ):
        with pytest.raises(GptossAttnError) as e:
            call()
        assert e.value.status == status


def test_the_operators_are_called_where_something_watches(A):
    """Python's calls go past the dispatcher only where nobody stands there: modes, a profiler and the compiler see the operators, and what comes out is the same.  Gradients are
    refused either way; a parameter's are nobody's under no_grad."""
    from torch.utils._python_dispatch import TorchDispatchMode
    cache, table, n, q, sinks, k, v = make(A, 28, [300, 20], 8, 2, 1, 16, BF16, E4M3, 2)
    q, sinks, k, v = q.to(DEV), torch.nn.Parameter(sinks.to(DEV)), k.to(DEV), v.to(DEV)
    start = torch.tensor([3, 7], dtype=torch.int32, device=DEV)

    def calls(k):
        A.paged_cache_write(cache, k, v, table, start)
        kk, vv = A.paged_cache_read(cache, table, n, 300)
        o = A.paged_attention(q, cache, table, n, sinks, SCALE, 40)
        return (kk, vv, o, *A.paged_attention_forward(q, cache, table, n, sinks, SCALE))

    seen = []

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    names = ["paged_write", "paged_read", "paged_fwd", "paged_fwd"]
    with torch.no_grad():
        want = calls(k)
        with Watch():
            got = [calls(k)]
        assert [x for x in seen if "paged" in x] == [f"gptoss_attn.{x}.default" for x in names]
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
            got.append(calls(k))
        assert {e.key for e in prof.key_averages()} >= {f"gptoss_attn::{x}" for x in names}
        got.append(torch.compile(calls, fullgraph=True, backend="aot_eager")(k))
        with torch.autocast("cuda", torch.bfloat16):
            got.append(calls(k))
    for out in got:
        assert all(torch.equal(x, y) for x, y in zip(out, want))
    with pytest.raises(RuntimeError, match="no gradient"):
        A.paged_attention(q, cache, table, n, sinks, SCALE)
    with pytest.raises(RuntimeError, match="no gradient"):
        A.paged_cache_write(cache, k.clone().requires_grad_(), v, table, start)
    with torch.no_grad(), pytest.raises(RuntimeError, match="vmap"):
        torch.vmap(lambda x: A.paged_attention(x, cache, table, n, None, SCALE))(q[None])


# ---- streams and graphs ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,storage", TYPES, ids=TYPE_IDS)
def test_graph_of_a_decoding_step(A, dtype, storage):
    """Write and attention captured once; replays follow positions, tables and tokens that change on the GPU, with eager work between them."""
    lens, h, g, ps = [700, 33], 16, 2, 16
    cache, table, n, q, sinks, _, _ = make(A, 16, lens, h, g, 1, ps, dtype, storage, 3)
    free = [i for i in range(cache.k.shape[0]) if i not in table.flatten().tolist()]
    table[0, 44], table[1, 3] = free[0], free[1]            # room for what is written below
    gen = torch.Generator().manual_seed(17)
    q, sinks = q.to(DEV), sinks.to(DEV)
    k, v = (torch.zeros(2, g, 1, 64, dtype=dtype, device=DEV) for _ in range(2))
    start = n.clone()

    def step():
        A.paged_cache_write(cache, k, v, table, start)
        return A.paged_attention_forward(q, cache, table, start + 1, sinks, SCALE)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    saved = A.PagedCache(*(None if t is None else t.clone() for t in cache))
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = step()
    for t, s in zip(cache, saved):
        if t is not None:
            t.copy_(s)
    eager = A.PagedCache(*(None if t is None else t.clone() for t in cache))
    for i in range(4):
        new = [torch.randn(2, g, 1, 64, generator=gen).to(dtype).to(DEV) for _ in range(2)]
        k.copy_(new[0])
        v.copy_(new[1])
        graph.replay()
        A.paged_cache_write(eager, *new, table, start)
        want, want_lse = A.paged_attention_forward(q, eager, table, start + 1, sinks, SCALE)
        torch.cuda.synchronize()
        assert torch.equal(o, want) and torch.equal(lse, want_lse), i
        start += 1


def test_calls_on_two_streams(A):
    """Calls that run at the same time, each with scratch of its own, give what they give alone."""
    cache, table, n, q, sinks, _, _ = make(A, 18, [6000, 20, 3000], 16, 2, 1, 16, BF16, BF16)
    q, sinks = q.to(DEV), sinks.to(DEV)
    n2 = (n // 2).contiguous()
    want = [A.paged_attention(q, cache, table, m, sinks, SCALE) for m in (n, n2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for i, m in enumerate((n, n2)):
            with torch.cuda.stream(streams[i]):
                got[i].append(A.paged_attention(q, cache, table, m, sinks, SCALE))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


@pytest.mark.parametrize("storage", [BF16, E4M3])
def test_two_graphs_that_share_a_pool(A, storage):
    """Two captured calls of different divisions whose scratch comes from one memory pool, replayed in turn with eager calls between them."""
    cache, table, n, q, sinks, _, _ = make(A, 24, [5000, 20, 3000], 16, 2, 1, 16, BF16, storage)
    q, sinks = q.to(DEV), sinks.to(DEV)
    args = [(q, table, n, None), (q[:2].contiguous(), table[:2].contiguous(), n[:2].contiguous(), 700)]

    def call(i):
        x, t, m, window = args[i]
        return A.paged_attention_forward(x, cache, t, m, sinks, SCALE, window)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(0)
        call(1)
    side.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for i in range(2):
        with torch.cuda.graph(graphs[i], pool=graphs[0].pool() if i else None):
            outs.append(call(i))
    for step in range(4):
        n.copy_(torch.tensor([5000 - 900 * step, 20, 3000 - 70 * step]))
        args[1][2].copy_(n[:2])
        for i in range(2):
            graphs[i].replay()
            got = [x.clone() for x in outs[i]]
            want = call(i)
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(got, want)), (step, i)


# ---- as they are used together ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("storage", [BF16, E4M3])
@pytest.mark.parametrize("window", [None, 32])
def test_prompt_chunks_and_decoding(A, storage, window):
    """A prompt in two chunks and tokens one by one: chunks through attention() on what paged_cache_read gives, tokens through paged_attention, each against
    the definition on what the pages hold.  attention()'s bound is that of its own tests: 2e-2 and half a step of the result."""
    g, h, ps, total = 2, 16, 16, 150
    gen = torch.Generator().manual_seed(19)
    q, k, v = (torch.randn(1, x, total, 64, generator=gen).to(BF16).to(DEV) for x in (h, g, g))
    sinks = torch.randn(h, generator=gen).to(BF16).to(DEV)
    cache = new_cache(A, 12, g, ps, storage)
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
        tol = 2e-2 + 2.0 ** -8 * ref.abs() if size > 8 else P.bounds(ref, ref_lse, terms, BF16)[0]
        assert bool(((o.cpu().double() - ref).abs() <= tol).all()), at
        at = end


@pytest.mark.parametrize("storage", [BF16, E4M3])
def test_layers_with_a_paged_state(A, storage):
    """A layer through hip_flash_attention(paged=): a padded prompt, padded chunks of different lengths, single tokens.  Each against the definition, on
    what the pages hold, and the prompt against attention() itself."""
    from types import SimpleNamespace
    g, h, ps, b = 2, 16, 16, 2
    gen = torch.Generator().manual_seed(25)
    sinks = torch.randn(h, generator=gen).to(BF16).to(DEV)
    modules = [SimpleNamespace(sinks=sinks, sliding_window=w, layer_idx=i) for i, w in enumerate((32, None))]
    caches = [new_cache(A, 24, g, ps, storage) for _ in modules]
    table = torch.randperm(24, generator=gen).to(torch.int32)[:22].view(2, 11).to(DEV)
    start = torch.zeros(b, dtype=torch.int32)
    for step, counts in enumerate(([90, 37], [7, 3], [1, 1], [1, 1], [0, 5])):
        s, counts = max(counts), torch.tensor(counts, dtype=torch.int32)
        seqlens = start + counts
        state = A.PagedState(caches, table, None if step == 0 else start.to(DEV), seqlens.to(DEV), None if step in (0, 2, 3) else counts.to(DEV))
        for module in modules:
            q, k, v = (torch.randn(b, s, x, 64, generator=gen).to(BF16).to(DEV).transpose(1, 2) for x in (h, g, g))
            o, none = A.hip_flash_attention(module, q, k, v, None, SCALE, paged=state)
            assert none is None
            if step == 0:
                assert torch.equal(o, A.attention(q, k, v, sinks, SCALE, module.sliding_window, None, counts.to(DEV)))
                kk, vv = A.paged_cache_read(caches[module.layer_idx], table, seqlens.to(DEV), s)
                for x, y in ((kk, k), (vv, v)):
                    for r in range(b):
                        c = int(counts[r])
                        assert torch.equal(x[r, :, :c].cpu().double(), P.stored_rows(y[r, :, :c].cpu(), storage))
                continue
            ref, ref_lse, terms = P.attention(q.cpu(), *values(caches[module.layer_idx]), table.cpu(), seqlens, sinks.cpu(), SCALE,
                                              module.sliding_window or 0, start)
            assert bool(((o.cpu().double() - ref).abs() <= P.bounds(ref, ref_lse, terms, BF16)[0]).all()), (step, module.layer_idx)
        start = seqlens
    with pytest.raises(RuntimeError, match="neither seqlens nor doc_start"):
        A.hip_flash_attention(modules[0], q, k, v, None, SCALE, paged=state, seqlens=seqlens)


def test_patched_model_decodes_on_pages(A):
    """A patched two-layer model: a padded prompt and tokens one by one on pages give, up to the roundings of the type, the logits of whole rows at once.
    In float32: two runs whose sums are ordered differently differ by the order of 1e-6 of logits near 1; a key too few or too many moves them by 1e-2."""
    from transformers import GptOssConfig, GptOssForCausalLM
    from oregon_gpt_oss_patching_amd import patching
    cfg = GptOssConfig(vocab_size=512, hidden_size=256, intermediate_size=256, num_hidden_layers=2,
                       num_attention_heads=16, num_key_value_heads=4, head_dim=64, num_local_experts=2,
                       num_experts_per_tok=2, sliding_window=32, max_position_embeddings=512,
                       layer_types=["sliding_attention", "full_attention"], attn_implementation="eager")
    torch.manual_seed(0)
    model = GptOssForCausalLM(cfg).to(DEV, FP32).eval()
    lens, total = torch.tensor([50, 71]), 6
    ids = torch.randint(0, 512, (2, 80), device=DEV)
    table = torch.arange(10, dtype=torch.int32, device=DEV).view(2, 5)
    caches = [A.paged_cache(10, 4, 16, FP32) for _ in range(2)]
    patching.patch_flash_attention()
    try:
        with torch.no_grad():
            whole = model(ids, use_cache=False).logits
            s = int(lens.max())
            state = A.PagedState(caches, table, None, lens.to(DEV))
            out = model(ids[:, :s], use_cache=False, paged=state).logits
            for r in range(2):
                assert torch.allclose(out[r, :lens[r]], whole[r, :lens[r]], rtol=1e-4, atol=1e-4)
            at = lens.to(DEV)
            for _ in range(total):
                state = A.PagedState(caches, table, at, at + 1)
                new = ids.gather(1, at[:, None])
                out = model(new, position_ids=at[:, None], use_cache=False, paged=state).logits[:, 0]
                want = whole[torch.arange(2, device=DEV), at]
                assert torch.allclose(out, want, rtol=1e-4, atol=1e-4), float((out - want).abs().max())
                at = at + 1
    finally:
        patching.unpatch_flash_attention()
