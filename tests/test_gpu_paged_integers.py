"""GPU tests of page tables, lengths and positions in 64 bits: what int32 does not hold is no page, in front of every position or behind each, as its size says."""
import pytest
import torch

from test_gpu_paged import BF16, DEV, E4M3, SCALE, A, make  # noqa: F401

pytestmark = pytest.mark.gpu
FAR = (2 ** 31, 2 ** 32, 2 ** 32 + 1, 2 ** 40 + 2, 2 ** 62, -2 ** 31 - 1, -2 ** 32, -2 ** 32 + 1, -2 ** 62)


def long(*x):
    return torch.tensor(x, dtype=torch.int64, device=DEV)


@pytest.mark.parametrize("storage", [BF16, E4M3])
@pytest.mark.parametrize("entry", FAR)
def test_entries(A, storage, entry):  # noqa: F811
    """Such an entry names no page, like -1: its keys are not seen, its rows are 0, what is written there is dropped."""
    cache, table, n, q, sinks, k, v = make(A, 61, [40, 33], 8, 2, 1, 16, BF16, storage)
    wide, none = table.long(), table.clone()
    wide[0, 1], none[0, 1] = entry, -1
    q, sinks, k = q.to(DEV), sinks.to(DEV), k.to(DEV)
    for x, y in zip(A.paged_attention_forward(q, cache, wide, n, sinks, SCALE), A.paged_attention_forward(q, cache, none, n, sinks, SCALE)):
        assert torch.equal(x, y)
    for x, y in zip(A.paged_cache_read(cache, wide, n, 40), A.paged_cache_read(cache, none, n, 40)):
        assert torch.equal(x, y)
    written = [A.PagedCache(*(None if t is None else t.clone() for t in cache)) for _ in range(2)]
    for c, t in zip(written, (wide, none)):
        A.paged_cache_write(c, -k, -k, t, [0, 0], n)
    for x, y in zip(*written):
        assert x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("storage", [BF16, E4M3])
@pytest.mark.parametrize("far", FAR)
def test_lengths_and_positions(A, storage, far):  # noqa: F811
    """Lengths beyond the table are the table's end, below 0 there is no token; positions beyond either end do not exist."""
    cache, table, n, q, sinks, k, v = make(A, 62, [48, 33], 8, 2, 1, 16, BF16, storage)
    q, sinks, k = q.to(DEV), sinks.to(DEV), k.to(DEV)
    end = table.shape[1] * 16 if far > 0 else 0
    near = A.paged_attention_forward(q, cache, table, torch.tensor([end, 33], dtype=torch.int32, device=DEV), sinks, SCALE)
    for x, y in zip(A.paged_attention_forward(q, cache, table, long(far, 33), sinks, SCALE), near):
        assert torch.equal(x, y)
    near = A.paged_cache_read(cache, table, torch.tensor([end, 33], dtype=torch.int32, device=DEV), 50)
    for x, y in zip(A.paged_cache_read(cache, table, long(far, 33), 50), near):
        assert torch.equal(x, y)
    # positions: no query, no row, nothing written
    o, lse = A.paged_attention_forward(q, cache, table, n, sinks, SCALE, None, long(far, 32))
    assert not o[0].any() and torch.equal(lse[0, :, 0], sinks.float()) and bool(o[1].any())
    assert not A.paged_cache_read(cache, table, n, 5, long(far, 0))[0][0].any()
    before = [None if t is None else t.clone() for t in cache]
    A.paged_cache_write(cache, k, k, table, long(far, 2 ** 40))
    for x, y in zip(cache, before):
        assert x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    # how many tokens are written: all of them, or none
    other = A.PagedCache(*(None if t is None else t.clone() for t in cache))
    A.paged_cache_write(cache, -k, -k, table, [0, 0], long(far, 0))
    A.paged_cache_write(other, -k, -k, table, [0, 0], torch.tensor([48 if far > 0 else 0, 0], dtype=torch.int32, device=DEV))
    for x, y in zip(cache, other):
        assert x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_a_graph_follows_them(A):  # noqa: F811
    """Tables, lengths and positions in 64 bits are narrowed inside a captured call: replays follow what they hold then."""
    cache, table, n, q, sinks, k, v = make(A, 63, [400, 90], 8, 2, 1, 16, BF16, E4M3)
    q, sinks = q.to(DEV), sinks.to(DEV)
    wide, lens, start = table.long(), n.long(), n.long() - 1

    def call(*x):
        return (*A.paged_attention_forward(q, cache, x[0], x[1], sinks, SCALE, None, x[2]), *A.paged_cache_read(cache, x[0], x[1], 30, x[2]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(wide, lens, start)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(wide, lens, start)
    for a, b, first, entry in ((400, 90, 380, 2 ** 40), (2 ** 33, 5, 399, -1), (100, -2 ** 35, 2 ** 32 + 7, 1), (350, 90, 10, 2 ** 32)):
        lens.copy_(torch.tensor([a, b]))
        start.copy_(torch.tensor([first, b - 1]))
        wide[0, 3] = entry
        graph.replay()
        got = [x.clone() for x in out]
        fit = lambda x: x.clamp(-2 ** 31, 2 ** 31 - 1).to(torch.int32)
        want = call(fit(wide), fit(lens), fit(start))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)), (a, b, first, entry)
