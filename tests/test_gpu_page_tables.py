"""GPU tests of the page tables built on the device and of writing by slots: every number against the definition, a row at a time (oracle/tables_ref.py)."""
import random

import pytest
import torch

from oracle import paged_ref as P
from oracle import tables_ref as T

pytestmark = pytest.mark.gpu
DEV, BF16, FP32, E4M3 = "cuda", torch.bfloat16, torch.float32, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def A():
    import oregon_gpt_oss_patching_amd as A_
    from oregon_gpt_oss_patching_amd import _lib
    _lib.load()
    return A_


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


def tables_of(rng, have, ps, pages, width, junk=-1):
    """Rows with pages of their own for `have` tokens, in no order; `junk` behind them."""
    order = rng.sample(range(pages), sum(T.pages_for(n, ps) for n in have))
    table, at = [], 0
    for n in have:
        k = T.pages_for(n, ps)
        table.append(order[at:at + k] + [junk] * (width - k))
        at += k
    return table


def check_update(A, table, have, want, pages, ps, into=None):
    t = ints(table) if into is None else into
    got, left = A.page_table_update(t, ints(have), ints(want), pages, ps)
    ref, seqlens, free = T.update(table, have, want, pages, ps)
    assert t.tolist() == ref and got.tolist() == seqlens and left.tolist() == [free] and got.dtype == left.dtype == torch.int32
    return ref, seqlens


def check_map(A, table, start, counts, total, ps):
    m = A.token_map(ints(table), ints(start), ints(counts), total, ps)
    ref = T.token_map(table, start, counts, total, ps)
    assert [m.row.tolist(), m.position.tolist(), m.slot.tolist(), m.first.tolist(), m.used.tolist()] == [*map(list, ref[:4]), [ref[4]]]
    assert [x.dtype for x in m] == [torch.int32, torch.int32, torch.int64, torch.int32, torch.int32]
    return m


@pytest.mark.parametrize("rows,longest,ps,slack", [
    (1, 1, 16, 0), (1, 40, 16, 5), (1, 300000, 16, 100), (3, 100, 32, 0), (16, 500, 16, 3), (63, 2000, 64, 40), (64, 900, 16, -7), (65, 3000, 16, -400), (257, 700, 128, 9),
    (1500, 90, 16, -20), (5000, 40, 16, 1000),
])
def test_rows_that_grow_shrink_begin_and_end(A, rows, longest, ps, slack):
    print(f"case rows={rows} longest={longest} page={ps} slack={slack}", flush=True)
    rng = random.Random(rows * 7 + longest)
    have = [rng.choice((0, rng.randint(1, longest), rng.randint(1, longest))) for _ in range(rows)]
    width = T.pages_for(longest + 70, ps) + 1
    pages = sum(T.pages_for(n, ps) for n in have) + max(1, slack) + (rows if slack > 0 else 0)
    table = tables_of(rng, have, ps, pages, width)
    for step in range(4):
        want = [rng.choice((0, n, n + 1, n + 1, n + rng.randint(0, 60), rng.randint(0, longest))) for n in have]
        table, have = check_update(A, table, have, want, pages, ps)
        check_map(A, table, have, [rng.randint(0, 3) for _ in have], 2 * rows, ps)
    alive = [p for row, n in zip(table, have) for p in row[:T.pages_for(n, ps)]]
    assert len(set(alive)) == len(alive) and all(0 <= p < pages for p in alive)


@pytest.mark.parametrize("have,want,free", [
    ([0, 0, 0], [48, 48, 16], 3),            # the first takes all, the others get none
    ([0, 0, 0], [64, 16, 16], 3),            # the first does not fit: none behind it gets any
    ([0, 16, 0], [64, 16, 16], 3),           # but rows that want none are not touched
    ([0, 16, 0], [64, 0, 64], 3),            # a page that comes back in this call goes out in it
    ([16, 0], [17, 32], 2),
    ([0], [0], 1),
    ([5], [16], 0),                          # room left in its page, none in the pool
    ([5], [17], 0),
    ([-3, -1], [-5, 16], 1),                 # lengths below 0 are 0
])
def test_too_few_pages(A, have, want, free):
    pages = sum(T.pages_for(n, 16) for n in have) + free
    table = tables_of(random.Random(1), have, 16, max(pages, 1), 6)
    check_update(A, table, have, want, max(pages, 1), 16)


def test_rows_longer_than_the_table(A):
    """A row that wants more than its table holds gets none, and nobody else suffers; numbers next to the ends of int32."""
    check_update(A, [[3, -1], [0, -1], [1, 2]], [16, 1, 32], [33, 17, 32], 7, 16)
    big = 2 ** 31 - 1
    check_update(A, [[3, -1], [0, -1], [1, 2]], [16, 1, big], [big, 17, 16], 7, 16)
    check_update(A, [[3, 5], [0, -1]], [big, 1], [-2 ** 31, 32], 7, 16)


def test_shared_pages_and_entries_that_name_none(A):
    """A common prefix is free when the last of its rows has ended; -1 and numbers behind the pool among kept entries are nobody's page; what stands behind a row's pages stays."""
    table = [[4, 7, 1], [4, 7, 2], [4, 9, -5]]
    table, have = check_update(A, table, [40, 40, 20], [0, 41, 20], 8, 16)[0], [0, 41, 20]
    assert table[0] == [-1, -1, -1]
    table = check_update(A, table, have, [48, 0, 20], 8, 16)[0]
    check_update(A, table, [48, 0, 20], [0, 0, 0], 8, 16)
    check_update(A, [[77, 78, 79], [80, 81, 82]], [0, 0], [20, 0], 4, 16)


@pytest.mark.parametrize("pages", [31, 32, 33, 2047, 2048, 2049, 1 << 19, (1 << 19) + 1, (1 << 20) + 4097])
def test_pools_of_any_size(A, pages):
    """Around the words, groups and parts that the pool is looked at in; more free pages than one part has."""
    print(f"case pages={pages}", flush=True)
    rng = random.Random(pages)
    n = min(pages - 3, 700000)
    kept = sorted(rng.sample(range(pages), 3))
    table = torch.full((3, n + 5), -1, dtype=torch.int32)
    table[0, :3] = torch.tensor(kept[::-1], dtype=torch.int32)
    have, want = [48, 0, 0], [16 * (n // 2), 16 * (n - n // 2), 16]
    t = table.to(DEV)
    got, left = A.page_table_update(t, ints(have), ints(want), pages, 16)
    free = [p for p in range(pages) if p not in kept]
    first, second = n // 2 - 3, n - n // 2
    over = first + second + 1 > pages - 3
    assert got.tolist() == ([want[0], want[1], 0] if over else want) and left.tolist() == [pages - 3 - first - second - (0 if over else 1)]
    t = t.cpu()
    assert t[0, :3].tolist() == kept[::-1] and t[0, 3:3 + first].tolist() == free[:first] and t[1, :second].tolist() == free[first:first + second]
    assert int((t[0, 3 + first:] != -1).sum()) == int((t[1, second:] != -1).sum()) == 0


def test_most_rows(A):
    n = 16384
    have, want = [0] * n, [16] * n
    t = torch.full((n, 2), -1, dtype=torch.int32, device=DEV)
    got, left = A.page_table_update(t, ints(have), ints(want), n - 5, 16)
    assert got.tolist() == [16] * (n - 5) + [0] * 5 and left.tolist() == [0] and t[:, 0].tolist() == list(range(n - 5)) + [-1] * 5
    check_map(A, t.tolist(), have, [1] * n, n, 16)
    with pytest.raises(RuntimeError):
        A.page_table_update(torch.full((n + 1, 2), -1, dtype=torch.int32, device=DEV), ints([0] * (n + 1)), ints([1] * (n + 1)), 5, 16)


def test_strided_tables_and_lists(A):
    """Rows of a wider table, with a stride that is no multiple of anything; lists, 64-bit numbers and numbers of the host."""
    rng = random.Random(3)
    have, want, ps = [40, 0, 17], [60, 33, 0], 16
    table = tables_of(rng, have, ps, 20, 5)
    wide = torch.full((3, 7), 99, dtype=torch.int32, device=DEV)
    wide[:, 1:6] = ints(table)
    check_update(A, table, have, want, 20, ps, into=wide[:, 1:6])
    assert wide[:, 0].tolist() == wide[:, 6].tolist() == [99] * 3
    ref = T.update(table, have, want, 20, ps)
    for h, w in ((have, want), (ints(have, torch.int64), ints(want, torch.int64)), (torch.tensor(have), torch.tensor(want)), (ints([x for n in have for x in (n, 9)])[::2], ints(want, torch.int16))):
        t = ints(table)
        got, left = A.page_table_update(t, h, w, 20, ps)
        assert (t.tolist(), got.tolist(), left.tolist()) == (ref[0], ref[1], [ref[2]])
        m = A.token_map(ints(table, torch.int64).t().contiguous().t(), h, [2, 1, 3], 9, ps)
        assert m.slot.tolist() == T.token_map(table, have, [2, 1, 3], 9, ps)[2]


@pytest.mark.parametrize("rows,longest,ps", [(1, 1, 16), (1, 5000, 16), (2, 1025, 64), (40, 700, 32), (300, 9, 16), (3000, 3, 16)])
def test_token_map(A, rows, longest, ps):
    rng = random.Random(rows + longest)
    counts = [rng.choice((0, rng.randint(0, longest), rng.randint(0, longest))) for _ in range(rows)]
    start = [rng.randint(0, 100) for _ in range(rows)]
    width = T.pages_for(longest + 90, ps)
    table = [[rng.choice((-1, rng.randint(0, 1 << 20), 2 ** 31 - 1)) for _ in range(width)] for _ in range(rows)]
    for total in (sum(counts), sum(counts) + 37, max(0, sum(counts) - 3), 0, 1):
        check_map(A, table, start, counts, total, ps)


def test_token_map_next_to_the_ends(A):
    """Positions in front of 0 and behind the table, counts below 0 and of 2^31 - 1."""
    check_map(A, [[5, 6]], [-3], [6], 10, 16)
    check_map(A, [[5, 6], [7, 8]], [30, 0], [9, 4], 20, 16)
    check_map(A, [[5, 6], [7, 8]], [0, 3], [-4, 4], 6, 16)
    big = 2 ** 31 - 1
    m = A.token_map(ints([[5, 6], [7, 8], [1, 2]]), ints([0, 3, big]), ints([2, big, big]), 40, 16)
    assert m.row.tolist() == [0, 0] + [1] * 38 and m.used.tolist() == [40] and m.slot.tolist()[2] == 7 * 16 + 3 and m.slot.tolist()[31:] == [-1] * 9
    m = A.token_map(ints([[5, 6]]), ints([big - 1]), ints([5]), 5, 16)
    assert m.slot.tolist() == [-1] * 5


@pytest.mark.parametrize("dtype,storage", [(BF16, BF16), (BF16, E4M3), (FP32, FP32), (FP32, E4M3)], ids=["bf16", "bf16-e4m3", "fp32", "fp32-e4m3"])
@pytest.mark.parametrize("counts,g,ps", [([1], 1, 16), ([5, 0, 40, 1], 8, 16), ([300, 7], 3, 64)])
def test_tokens_by_slots_are_tokens_by_rows(A, dtype, storage, counts, g, ps):
    """The same bits in the same places as paged_cache_write's, and no other place touched; slots of no page are dropped."""
    gen = torch.Generator().manual_seed(sum(counts) + g)
    rng = random.Random(5)
    start = [rng.randint(0, 50) for _ in counts]
    have = [s + n for s, n in zip(start, counts)]
    pages = sum(T.pages_for(n, ps) for n in have) + 2
    table = ints(tables_of(rng, have, ps, pages, max(T.pages_for(n, ps) for n in have)))
    total = sum(counts) + 3
    k, v = (torch.randn(total, g, 64, generator=gen).to(dtype).to(DEV) for _ in range(2))
    one, other = A.paged_cache(pages, g, ps, storage), A.paged_cache(pages, g, ps, storage)
    m = A.token_map(table, start, counts, total, ps)
    A.paged_cache_write_tokens(one, k, v, m.slot)
    longest = max(counts)
    padded = [torch.zeros(len(counts), g, longest, 64, dtype=dtype, device=DEV) for _ in range(2)]
    at = 0
    for b, n in enumerate(counts):
        for x, y in zip(padded, (k, v)):
            x[b, :, :n] = y[at:at + n].transpose(0, 1)
        at += n
    A.paged_cache_write(other, *padded, table, start, counts)
    for x, y in zip(one, other):
        assert x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    # as strided tensors, of the other integers; slots behind the pool and far away are nobody's
    third = A.paged_cache(pages, g, ps, storage)
    wide = torch.cat([k.transpose(0, 1), v.transpose(0, 1)]).contiguous()
    A.paged_cache_write_tokens(third, wide[:g].transpose(0, 1), wide[g:].transpose(0, 1), m.slot.int().tolist())
    A.paged_cache_write_tokens(third, k[:4].contiguous(), v[:4].contiguous(), ints([-1, pages * ps, 2 ** 40, -2 ** 50], torch.int64))
    for x, y in zip(third, other):
        assert x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    A.paged_cache_write_tokens(third, k[:0], v[:0], m.slot[:0])
    last = A.paged_cache(pages, g, ps, storage)
    if dtype == BF16:
        A.paged_cache_write_tokens(last, k.float().half(), v.float().half(), m.slot)
        A.paged_cache_write_tokens(one, k.float().half().to(BF16), v.float().half().to(BF16), m.slot)
        for x, y in zip(last, one):
            assert x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_a_step_captured_and_replayed(A):
    """Tables, map and write in one graph that follows the lengths; eager steps between the replays, two graphs of the same tables."""
    ps, pages, rows = 16, 40, 4
    gen = torch.Generator().manual_seed(2)
    table = torch.full((rows, 12), -1, dtype=torch.int32, device=DEV)
    have, want, cache = ints([0] * rows), ints([0] * rows), A.paged_cache(pages, 2, ps)
    k, v = (torch.randn(64, 2, 64, generator=gen).to(BF16).to(DEV) for _ in range(2))

    def step():
        got, left = A.page_table_update(table, have, want, pages, ps)
        m = A.token_map(table, have, got - have, 64, ps)
        A.paged_cache_write_tokens(cache, k, v, m.slot)
        return got, left, m

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(stream):
        step()
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                out = step()
            graphs.append((g, out))
    torch.cuda.current_stream().wait_stream(stream)
    rng, ref, lens = random.Random(4), [[-1] * 12 for _ in range(rows)], [0] * rows
    for i in range(8):
        new = [rng.choice((0, n + 1, min(n + rng.randint(0, 14), 150))) for n in lens]
        have.copy_(ints(lens))
        want.copy_(ints(new))
        g, (got, left, m) = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        ref, seqlens, free = T.update(ref, lens, new, pages, ps)
        assert table.tolist() == ref and got.tolist() == seqlens and left.tolist() == [free], i
        rm = T.token_map(ref, lens, [a - b for a, b in zip(seqlens, lens)], 64, ps)
        assert m.slot.tolist() == rm[2] and m.used.tolist() == [rm[4]]
        for t, s in enumerate(rm[2]):
            if s >= 0:
                assert torch.equal(cache.k[s // ps, :, s % ps], k[t])
        lens = seqlens
        want.copy_(have)
        have.copy_(ints(lens))          # eager: nothing changes
        got2, left2 = A.page_table_update(table, ints(lens), ints(lens), pages, ps)
        assert got2.tolist() == lens and left2.tolist() == [free] and table.tolist() == ref


def test_compiled(A):
    table, have, want = ints([[-1] * 4, [3, -1, -1, -1]]), ints([0, 10]), ints([20, 40])

    def f(t, h, w):
        got, left = A.page_table_update(t, h, w, 9, 16)
        m = A.token_map(t, h, got - h, 60, 16)
        return got, left, m.slot, m.first, m.used

    t = table.clone()
    want_out, want_table = f(t, have, want), t
    t = table.clone()
    got_out = torch.compile(f, backend="aot_eager", fullgraph=True)(t, have, want)
    assert torch.equal(t, want_table) and all(torch.equal(x, y) for x, y in zip(want_out, got_out))


def test_packed_prompts_through_the_adapter(A):
    """hip_flash_attention(paged=) with a TokenMap: rows that begin with the call, back to back, padding behind them: each row's attention is its own, its keys
    and values are in its pages."""
    class Layer:
        layer_idx, sliding_window, sinks = 0, None, None

    gen = torch.Generator().manual_seed(6)
    lens, ps, h, g, pad = [37, 1, 150, 64], 16, 8, 2, 5
    total = sum(lens) + pad
    q, k, v = (torch.randn(1, n, total, 64, generator=gen).to(BF16).to(DEV) for n in (h, g, g))
    for window in (None, 20):
        layer = Layer()
        layer.sinks, layer.sliding_window = torch.randn(h, generator=gen).to(BF16).to(DEV), window
        table = torch.full((4, 12), -1, dtype=torch.int32, device=DEV)
        cache = A.paged_cache(40, g, ps)
        seqlens, _ = A.page_table_update(table, [0] * 4, lens, 40, ps)
        tokens = A.token_map(table, [0] * 4, seqlens, total, ps)
        state = A.PagedState([cache], table, None, seqlens, tokens=tokens)
        out, _ = A.hip_flash_attention(layer, q, k, v, None, 0.125, paged=state)
        kk, vv = A.paged_cache_read(cache, table, seqlens, max(lens))
        at = 0
        for b, n in enumerate(lens):
            assert torch.equal(kk[b, :, :n], k[0, :, at:at + n]) and torch.equal(vv[b, :, :n], v[0, :, at:at + n])
            alone = A.attention(q[:, :, at:at + n], k[:, :, at:at + n], v[:, :, at:at + n], layer.sinks, 0.125, window, None)
            # (tiles lie differently in a packed row: within the roundings of bfloat16 results and weights, two of 2^-8 each of values below the largest |v|)
            assert float((out[0, at:at + n].float() - alone[0].float()).abs().max()) <= 2 * 2.0 ** -8 * 2 * float(v.float().abs().max())
            at += n
        assert float(out[0, at:].float().abs().max()) == 0.0
        with pytest.raises(RuntimeError, match="start must be None"):
            A.hip_flash_attention(layer, q, k, v, None, 0.125, paged=state._replace(start=seqlens))


def test_refusals(A):
    t, n = torch.full((2, 4), -1, dtype=torch.int32, device=DEV), ints([0, 0])
    cache, k = A.paged_cache(4, 2, 16), torch.zeros(3, 2, 64, dtype=BF16, device=DEV)
    slots = ints([0, 1, 2], torch.int64)
    for call, what in (
        (lambda: A.page_table_update(t.long(), n, n, 4, 16), "int32"),
        (lambda: A.page_table_update(t.t().contiguous().t(), n, n, 4, 16), "contiguous rows"),
        (lambda: A.page_table_update(t[:1].expand(2, 4), n, n, 4, 16), "pages|page table"),
        (lambda: A.page_table_update(t, n[:1], n, 4, 16), "one integer per row"),
        (lambda: A.page_table_update(t, n.float(), n, 4, 16), "one integer per row"),
        (lambda: A.page_table_update(t, n, n, 4, 24), "power of two"),
        (lambda: A.page_table_update(t, n, n, 0, 16), "pages|page"),
        (lambda: A.page_table_update(t, n, n, 2 ** 30 + 1, 16), "pages|page"),
        (lambda: A.page_table_update(t, n, n, 2 ** 31, 16), "too long"),
        (lambda: A.token_map(t, n, n, -1, 16), "total"),
        (lambda: A.token_map(t, n, n, 2 ** 30 + 1, 16), "total"),
        (lambda: A.token_map(t.float(), n, n, 4, 16), "integers"),
        (lambda: A.token_map(t, n, n, 4, 8), "power of two"),
        (lambda: A.paged_cache_write_tokens(cache, k, k, slots[:2]), "one integer per token"),
        (lambda: A.paged_cache_write_tokens(cache, k, k, slots.float()), "one integer per token"),
        (lambda: A.paged_cache_write_tokens(cache, k[:, :1], k[:, :1], slots), "must be"),
        (lambda: A.paged_cache_write_tokens(cache, k[None], k[None], slots), "must both be"),
        (lambda: A.paged_cache_write_tokens(cache, k, k.float(), slots), "one type"),
        (lambda: A.paged_cache_write_tokens(cache, k.cpu(), k, slots), "GPU"),
        (lambda: A.paged_cache_write_tokens(cache, k.clone().requires_grad_(), k, slots), "no gradient"),
    ):
        with pytest.raises(RuntimeError, match=what):
            call()


@pytest.mark.parametrize("rows,width,pages", [(128, 256, 3000), (129, 256, 3000), (32, 257, 9000), (33, 257, 9000), (33, 1025, 1 << 19), (33, 1025, (1 << 19) + 1), (700, 40, 40000), (5, 20000, 100000)])
def test_one_launch_or_two(A, rows, width, pages):
    """Tables on both sides of what decides whether a launch of its own sets the bits, and how many lanes read a run; as many new pages as are given out together, and more."""
    print(f"case rows={rows} width={width} pages={pages}", flush=True)
    rng = random.Random(rows + width)
    longest = min(16 * width, 16 * (pages // rows) // 2)
    have = [rng.choice((0, rng.randint(1, longest))) for _ in range(rows)]
    table = tables_of(rng, have, 16, pages, width)
    for new in (0, 40, 900):
        want = [min(n + rng.randint(0, new), 16 * width) if rng.random() < 0.9 else 0 for n in have]
        table, have = check_update(A, table, have, want, pages, 16)


def test_two_updates_at_once(A):
    """Tables of their own on two streams, with scratch of their own: what they give alone."""
    rng = random.Random(8)
    have = [rng.randint(1, 3000) for _ in range(300)]
    want = [n + rng.randint(0, 40) for n in have]
    pages = sum(T.pages_for(n, 16) for n in want) + 50
    table = tables_of(rng, have, 16, pages, 200)
    ref = T.update(table, have, want, pages, 16)
    tables = [ints(table) for _ in range(8)]
    h, w = ints(have), ints(want)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    out = []
    for i, t in enumerate(tables):
        with torch.cuda.stream(streams[i % 2]):
            out.append(A.page_table_update(t, h, w, pages, 16))
    torch.cuda.synchronize()
    for t, (got, left) in zip(tables, out):
        assert t.tolist() == ref[0] and got.tolist() == ref[1] and left.tolist() == [ref[2]]


@pytest.mark.parametrize("rows", [5, 700, 5000])
@pytest.mark.parametrize("onto", ["have", "want"])
def test_lengths_replaced_where_they_are(A, rows, onto):
    """Through the C interface: seqlens is have or want itself."""
    import ctypes

    from oregon_gpt_oss_patching_amd import _lib
    print(f"case rows={rows} onto={onto}", flush=True)
    rng, ps, width = random.Random(rows), 16, 12
    have = [rng.randint(0, 100) for _ in range(rows)]
    want = [rng.choice((0, n, n + 1, n + 40, 200)) for n in have]
    pages = sum(T.pages_for(n, ps) for n in have) + rows // 3
    table = tables_of(rng, have, ps, pages, width)
    t, h, w, left = ints(table), ints(have), ints(want), ints([0])
    p = _lib.TableParams()
    p.struct_size = ctypes.sizeof(p)
    p.B, p.table_width, p.page_size, p.pages, p.table_stride = rows, width, ps, pages, width
    p.page_table, p.have, p.want, p.left = t.data_ptr(), h.data_ptr(), w.data_ptr(), left.data_ptr()
    p.seqlens = {"have": h, "want": w}[onto].data_ptr()
    need = _lib.load().gptoss_attn_table_workspace_bytes(ctypes.byref(p))
    scratch = torch.empty(max(need, 4) // 4, dtype=torch.int32, device=DEV)
    p.scratch, p.scratch_bytes = scratch.data_ptr(), need
    assert _lib.load().gptoss_attn_page_table_update(ctypes.byref(p), torch.cuda.current_stream().cuda_stream) == 0
    ref, seqlens, free = T.update(table, have, want, pages, ps)
    assert t.tolist() == ref and {"have": h, "want": w}[onto].tolist() == seqlens and left.tolist() == [free]


@pytest.mark.parametrize("rows,longest,spare", [(70, 16384, 500), (40, 30000, -900), (300, 4000, 20), (1, 600000, 5)])
@pytest.mark.parametrize("pool", [0, 700001])
def test_many_new_pages(A, rows, longest, spare, pool):
    """More pages given out than one workgroup has threads, in pools that are looked at in one part and in two."""
    print(f"case rows={rows} longest={longest} spare={spare} pool={pool}", flush=True)
    rng, ps = random.Random(rows + longest), 16
    have = [rng.choice((0, 0, rng.randint(1, longest // 2))) for _ in range(rows)]
    want = [rng.choice((0, longest, rng.randint(longest // 2, longest))) if rows > 1 else longest for _ in range(rows)]
    kept, grown = sum(T.pages_for(min(a, b), ps) for a, b in zip(have, want)), sum(T.pages_for(b, ps) for b in want)
    pages = max(grown + spare, sum(T.pages_for(a, ps) for a in have), kept + 1)
    if pool:                                          # all but as many are one row's, which stays
        held = pool - pages
        t = [x + [-1] * (held + 1) for x in tables_of(rng, have, ps, pages, longest // ps + 1)]
        move = rng.randint(0, pages)                  # (the others lie on both sides of it)
        t = [[y if y < move else y + held for y in x] for x in t]
        t.append(list(range(move, move + held)) + [-1] * (len(t[0]) - held))
        have, want, pages = [*have, held * ps], [*want, held * ps], pool
    else:
        t = tables_of(rng, have, ps, pages, longest // ps + 1)
    check_update(A, t, have, want, pages, ps)


@pytest.mark.parametrize("rows", [255, 256, 257, 2048, 2049])
def test_token_map_of_many_rows(A, rows):
    """On both sides of the rows that one round of sums and the smaller kernel take, with tokens that fill workgroups and do not."""
    print(f"case rows={rows}", flush=True)
    rng, ps = random.Random(rows), 16
    start = [rng.randint(0, 90) for _ in range(rows)]
    counts = [rng.choice((0, 1, 1, 1, 40)) for _ in range(rows)]
    have = [a + b for a, b in zip(start, counts)]
    table = tables_of(rng, have, ps, sum(T.pages_for(n, ps) for n in have) + 3, 10)
    for total in (sum(counts), sum(counts) - 1, sum(counts) // 256 * 256, sum(counts) + 300):
        check_map(A, table, start, counts, total, ps)


def test_two_launches_captured(A):
    """A table large enough for a launch of its own for the bits, captured twice, replayed in turn with eager updates of another table between."""
    ps, rows, width = 16, 300, 64
    rng = random.Random(77)
    lens = [rng.randint(0, 600) for _ in range(rows)]
    pages = sum(T.pages_for(n, ps) for n in lens) + 200
    ref = tables_of(rng, lens, ps, pages, width)
    table, have, want = ints(ref), ints(lens), ints(lens)
    other = tables_of(rng, lens, ps, pages, width)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(stream):
        A.page_table_update(table, have, want, pages, ps)
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                out = A.page_table_update(table, have, want, pages, ps)
            graphs.append((g, out))
    torch.cuda.current_stream().wait_stream(stream)
    for i in range(6):
        new = [rng.choice((0, n, n + 1, min(n + rng.randint(0, 60), ps * width))) for n in lens]
        have.copy_(ints(lens))
        want.copy_(ints(new))
        g, (got, left) = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        ref, lens, free = T.update(ref, lens, new, pages, ps)
        assert table.tolist() == ref and got.tolist() == lens and left.tolist() == [free], i
        check_update(A, other, [0] * rows, [rng.randint(0, 90) for _ in lens], pages, ps)


def test_a_number_left_out_is_refused(A):
    """None where a whole number belongs (as a window or max_len it means that there is none)."""
    table, n = ints([[0, 1], [2, -1]]), ints([20, 5])
    cache = A.paged_cache(4, 2, 16)
    for call in (lambda: A.token_map(table, n, n, None, 16), lambda: A.token_map(table, n, n, 50, None), lambda: A.page_table_update(table, n, n, None, 16),
                 lambda: A.page_table_update(table, n, n, 4, None), lambda: A.paged_cache_read(cache, table, n, None)):
        with pytest.raises(TypeError):
            call()
    assert table.tolist() == [[0, 1], [2, -1]]
    q = torch.randn(2, 4, 1, 64, device=DEV, dtype=BF16)
    assert torch.equal(A.paged_attention(q, cache, table, n, None, 0.125, None, None, None), A.paged_attention(q, cache, table, n, None, 0.125, 0, None, 0))


@pytest.mark.parametrize("storage", [BF16, E4M3, torch.float4_e2m1fn_x2], ids=["bf16", "e4m3", "e2m1"])
def test_rows_that_share_whole_pages_grow_apart(A, storage):
    """Two rows over one prefix of whole pages, a third over a prefix whose last page, not full, it has copied: all grow by update, map and write, then the first ends.
    Each reads back the prefix as it was and its own tokens."""
    ps, g, pages, gen = 16, 2, 24, torch.Generator().manual_seed(17)
    cache, prefix = A.paged_cache(pages, g, ps, storage), 40
    table, zero = torch.full((3, 6), -1, dtype=torch.int32, device=DEV), ints([0])
    first, _ = A.page_table_update(table[:1], zero, ints([prefix]), pages, ps)
    common = torch.randn(2, prefix, g, 64, generator=gen).to(BF16).to(DEV)
    at = A.token_map(table[:1], zero, first, prefix, ps)
    A.paged_cache_write_tokens(cache, common[0], common[1], at.slot)
    # rows 1 and 2 begin with row 0's two full pages; row 2 has the 8 tokens behind them in a page of its own
    table[1:, :2] = table[0, :2]
    have = ints([prefix, 32, 32])
    have, _ = A.page_table_update(table, have, ints([prefix, 32, prefix]), pages, ps)
    own = table[2, 2].item()
    assert own not in table[0].tolist()
    for pool in cache:
        if pool is not None:
            pool = pool.view(torch.uint8) if pool.element_size() == 1 else pool
            pool[own] = pool[table[0, 2].long()]
    lens = [40, 32, 40]
    rows = [common[:, :n] for n in lens]
    for want in ([53, 61, 40], [54, 90, 71], [0, 91, 96]):
        counts = [max(0, w - n) for n, w in zip(lens, want)]
        got, _ = A.page_table_update(table, have, ints(want), pages, ps)
        assert got.tolist() == want
        new = torch.randn(2, sum(counts), g, 64, generator=gen).to(BF16).to(DEV)
        tokens = A.token_map(table, have, ints(counts), sum(counts) + 1, ps)
        A.paged_cache_write_tokens(cache, torch.cat((new[0], new[0, :1])), torch.cat((new[1], new[1, :1])), tokens.slot)
        pieces = list(new.split(counts, 1))
        rows = [torch.cat((r, p), 1) if w else r[:, :0] for r, p, w in zip(rows, pieces, want)]
        have, lens = got, want
        k, v = A.paged_cache_read(cache, table, have, 96)
        for b, n in enumerate(lens):
            for read, x in ((k, rows[b][0]), (v, rows[b][1])):
                # (what a cache of its own makes of the same tokens)
                alone = A.paged_cache(6, g, ps, storage)
                A.paged_cache_write_tokens(alone, x, x, torch.arange(n, device=DEV))
                want_b = A.paged_cache_read(alone, torch.arange(6, dtype=torch.int32, device=DEV)[None], ints([n]), 96)[0][0]
                assert torch.equal(read[b], want_b), (b, n)
