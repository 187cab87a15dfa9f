"""GPU tests of the rotary positions: results and gradients within bounds that follow from the roundings (oracle/rotary_ref.py), against complex
multiplications in 64 bits."""
import pytest
import torch

from oracle import rotary_ref as R

pytestmark = pytest.mark.gpu
DEV, BF16, FP32 = "cuda", torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def A():
    import oregon_gpt_oss_patching_amd as A_
    from oregon_gpt_oss_patching_amd import _lib
    _lib.load()
    return A_


def within(got, x, z, dtype, interleaved=False, angles=True):
    want = R.turn(x.detach().cpu(), z, interleaved)
    over = (got.detach().cpu().double() - want).abs() - R.bound(x.detach().cpu(), z, want, dtype, interleaved, angles)
    assert got.dtype == x.dtype and got.shape == x.shape
    assert bool((over <= 0).all()), (float(over.max()), [int(i) for i in torch.nonzero(over == over.max())[0]])
    turned = 2 * z.shape[-1]
    assert torch.equal(got[..., turned:], x[..., turned:])


CASES = [
    # B, H, G, S, D, R: a token, odd lengths, one head, heads of other widths turned in part, pairs that are no multiple of anything
    (1, 64, 8, 1, 64, 64),
    (2, 64, 8, 333, 64, 64),
    (3, 1, 1, 7, 64, 64),
    (1, 3, 5, 65, 64, 32),
    (2, 8, 2, 129, 80, 32),
    (1, 7, 1, 31, 96, 20),
    (2, 5, 3, 17, 64, 6),
    (1, 2, 2, 9, 7, 2),
    (1, 9, 1, 50, 256, 256),
    (40, 64, 8, 1, 64, 64),
    (1, 64, 8, 2500, 64, 64),        # several heads a thread
]


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("b,h,g,s,d,r", CASES)
def test_results_and_gradients(A, b, h, g, s, d, r, interleaved, dtype):
    print(f"case B={b} H={h} G={g} S={s} D={d} R={r} interleaved={interleaved} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(7 * b + s + d)
    rope = A.rotary_frequencies(r, 150000.0, factor=32.0, original_length=4096, interleaved=interleaved)
    positions = torch.randint(0, 1 << 17, (b, s), generator=gen)
    q = torch.randn(b, s, h, d, generator=gen).to(dtype).to(DEV).transpose(1, 2).requires_grad_()
    k = torch.randn(b, s, g, d, generator=gen).to(dtype).to(DEV).transpose(1, 2).requires_grad_()
    gq, gk = (torch.randn(x.shape, generator=gen).to(dtype).to(DEV) for x in (q, k))
    z = R.of_positions(positions, rope.frequencies.cpu(), rope.scale)
    at = positions.to(DEV)
    oq, ok = A.rotary(q, k, at, rope)
    for got, x in ((oq, q), (ok, k)):
        within(got, x, z, dtype, interleaved)
    dq, dk = torch.autograd.grad((oq, ok), (q, k), (gq, gk))
    for got, x in ((dq, gq), (dk, gk)):
        within(got, x, z.conj(), dtype, interleaved)
    # the same bits without a gradient, from int32 positions, and again
    with torch.no_grad():
        for p in (at, at.int(), at.clone()):
            assert all(torch.equal(x, y) for x, y in zip(A.rotary(q, k, p, rope), (oq, ok)))


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("tables", [BF16, FP32, torch.float16], ids=["bf16-tables", "fp32-tables", "fp16-tables"])
@pytest.mark.parametrize("rows", [1, 3])
def test_tables(A, rows, tables, dtype):
    gen = torch.Generator().manual_seed(rows)
    q, k = torch.randn(3, 8, 77, 64, generator=gen).to(dtype).to(DEV).requires_grad_(), torch.randn(3, 2, 77, 64, generator=gen).to(dtype).to(DEV).requires_grad_()
    cos, sin = (torch.randn(rows, 77, 32, generator=gen).to(tables) for _ in range(2))
    z = R.of_tables(cos, sin)
    for interleaved in (False, True):
        oq, ok = A.rotary_tables(q, k, cos.to(DEV), sin.to(DEV), interleaved)
        dq, dk = torch.autograd.grad((oq, ok), (q, k), (q.detach(), k.detach()))
        for got, x, by in ((oq, q, z), (ok, k, z), (dq, q, z.conj()), (dk, k, z.conj())):
            within(got, x, by, dtype, interleaved, angles=False)


def test_model_adapter(A):
    gen = torch.Generator().manual_seed(5)
    q, k = torch.randn(2, 8, 33, 64, generator=gen).to(BF16).to(DEV), torch.randn(2, 2, 33, 64, generator=gen).to(BF16).to(DEV)
    cos, sin = (torch.randn(2, 33, 32, generator=gen).to(BF16).to(DEV) for _ in range(2))
    want = A.rotary_tables(q, k, cos, sin)
    got = A.hip_rotary_pos_emb(q, k, cos, sin)
    other = A.hip_rotary_pos_emb(q.transpose(1, 2), k.transpose(1, 2), cos, sin, unsqueeze_dim=2)
    for x, y, t in zip(want, got, other):
        assert torch.equal(x, y) and torch.equal(x, t.transpose(1, 2))


def test_far_and_negative_positions(A):
    """Angles stay right where float32 has none of their bits left; up to positions of 2^40 the 64-bit product is off by 2^-12 of a turn at most, so
    these are held against the exact product of integers and a frequency that is a fraction of a turn."""
    rope = A.Rotary(torch.tensor([torch.pi / 8], dtype=torch.float64, device=DEV))
    x = torch.tensor([[[[1.0, 0.0]]]], device=DEV)
    for p in (0, 1, -1, 5, -3, 2 ** 31 + 3, -(2 ** 31) - 9, 2 ** 33 + 7):
        got = A.rotary(x, x, torch.tensor([[p]], device=DEV), rope)[0].cpu().double().flatten()
        angle = torch.tensor((p % 16) * torch.pi / 8, dtype=torch.float64)
        # pi / 8 is off by 2^-54: 2^33 times that, and the products' own 2^-53, come to 2^-19 of an eighth of a turn
        assert abs(float(got[0] - torch.cos(angle))) < 2.0 ** -18 and abs(float(got[1] - torch.sin(angle))) < 2.0 ** -18, p
    positions = torch.randint(-(1 << 20), 1 << 20, (2, 50), generator=torch.Generator().manual_seed(1))
    rope = A.rotary_frequencies(64, 150000.0)
    q = torch.randn(2, 4, 50, 64, generator=torch.Generator().manual_seed(2)).to(DEV)
    within(A.rotary(q, q, positions.to(DEV), rope)[0], q, R.of_positions(positions, rope.frequencies.cpu()), FP32)


def test_layouts(A):
    """Any strides: contiguous heads, a slice of a joint projection, broadcast rows and heads, rows on odd addresses, a last dimension that is not
    contiguous, positions of one row for all and with strides; results lie as (B, S, heads, D)."""
    gen = torch.Generator().manual_seed(3)
    rope = A.rotary_frequencies(64, 10000.0)
    qkv = torch.randn(2, 9, 12 * 64 + 1, generator=gen).to(BF16).to(DEV)
    joint = qkv[..., :768].unflatten(-1, (12, 64)).transpose(1, 2)
    odd = qkv[..., 1:].unflatten(-1, (12, 64)).transpose(1, 2)
    cases = [(joint[:, :8], joint[:, 8:10]), (joint[:, :8].contiguous(), joint[:, 8:10].contiguous()), (odd[:, :8], odd[:, 8:10]),
             (joint[:1, :8].expand(2, -1, -1, -1), joint[:, 8:9].expand(-1, 2, -1, -1)), (joint[:, :8].transpose(2, 3).contiguous().transpose(2, 3), joint[:, 8:10])]
    wide = torch.randint(0, 5000, (2, 18), generator=gen)
    for positions in (wide[:, ::2], wide[:1, 1::2], wide[0, :9], wide[:, ::2].to(torch.int16), wide[:, :9].tolist()):
        p = torch.as_tensor(positions).reshape(-1, 9)
        z = R.of_positions(p.expand(2, 9), rope.frequencies.cpu())
        for q, k in cases:
            oq, ok = A.rotary(q, k, positions if isinstance(positions, list) else positions.to(DEV), rope)
            within(oq, q, z, BF16)
            within(ok, k, z, BF16)
            assert oq.transpose(1, 2).is_contiguous() and ok.transpose(1, 2).is_contiguous()
    # positions of the host, frequencies in float32
    q, k = cases[0]
    rope32 = A.Rotary(rope.frequencies.float())
    within(A.rotary(q, k, wide[:, ::2], rope32)[0], q, R.of_positions(wide[:, ::2], rope32.frequencies.cpu()), BF16)


def test_float16_and_no_tokens(A):
    rope = A.rotary_frequencies(64, 10000.0)
    q = torch.randn(1, 4, 5, 64, generator=torch.Generator().manual_seed(4)).half().to(DEV)
    got = A.rotary(q, q, torch.arange(5, device=DEV), rope)[0]
    want = A.rotary(q.float(), q.float(), torch.arange(5, device=DEV), rope)[0]
    assert torch.equal(got, want.half())
    for shape in ((0, 4, 5, 64), (2, 4, 0, 64)):
        x = torch.empty(shape, device=DEV)
        out = A.rotary(x, x, torch.empty(shape[0], shape[2], dtype=torch.int64, device=DEV), rope)
        assert out[0].shape == out[1].shape == shape


def test_not_finite_numbers_stay_with_their_pairs(A):
    """A NaN or an infinity reaches its own pair and no other number."""
    rope = A.rotary_frequencies(64, 10000.0)
    q = torch.randn(1, 4, 6, 64, generator=torch.Generator().manual_seed(8)).to(DEV)
    at = torch.arange(1, 7, device=DEV)
    clean = A.rotary(q, q, at, rope)[0]
    for bad in (float("nan"), float("inf")):
        x = q.clone()
        x[0, 2, 3, 5] = bad
        got = A.rotary(x, x, at, rope)[0]
        hit = torch.zeros_like(q, dtype=torch.bool)
        hit[0, 2, 3, 5] = hit[0, 2, 3, 37] = True
        assert torch.equal(torch.isfinite(got), ~hit) and torch.equal(got[~hit], clean[~hit])


def test_one_gradient_of_two(A):
    """Only the keys', or only of the queries; shared and broadcast leaves add up."""
    rope = A.rotary_frequencies(64, 10000.0)
    gen = torch.Generator().manual_seed(9)
    at, z = torch.arange(11, device=DEV), R.of_positions(torch.arange(11)[None], rope.frequencies.cpu())
    q, k = torch.randn(2, 4, 11, 64, generator=gen).to(DEV), torch.randn(2, 1, 11, 64, generator=gen).to(DEV).requires_grad_()
    g = torch.randn(2, 1, 11, 64, generator=gen).to(DEV)
    (dk,) = torch.autograd.grad(A.rotary(q, k, at, rope)[1], k, g)
    within(dk, g, z.conj(), FP32)
    one = torch.randn(1, 1, 11, 64, generator=gen).to(DEV).requires_grad_()
    oq, ok = A.rotary(one.expand(2, 4, -1, -1), one.expand(2, -1, -1, -1), at, rope)
    gq = torch.randn(2, 4, 11, 64, generator=gen).to(DEV)
    (d,) = torch.autograd.grad((oq, ok), one, (gq, g))
    total = (gq.double().sum((0, 1)) + g.double().sum((0, 1)))[None, None].cpu()
    want = R.turn(total, z.conj())
    # ten gradients, each off by 8.1 u (a1 + a2), and their sum, ten roundings of at most 10 sqrt(2) times the largest: under 10 (16.2 + 14.2) u of it
    assert float((d.cpu().double() - want).abs().max()) < 10 * 31 * 2.0 ** -24 * max(float(gq.abs().max()), float(g.abs().max()))


def test_one_tensor_of_two_with_a_gradient(A):
    """The other's result has none: it can go into a cache while gradients are on, and the one gradient is what it is beside the other."""
    rope = A.rotary_frequencies(64, 10000.0)
    gen = torch.Generator().manual_seed(29)
    at, z = torch.arange(16, device=DEV), R.of_positions(torch.arange(16)[None], rope.frequencies.cpu())
    q, k = torch.randn(1, 4, 16, 64, generator=gen).to(BF16).to(DEV).requires_grad_(), torch.randn(1, 2, 16, 64, generator=gen).to(BF16).to(DEV)
    g = torch.randn(1, 4, 16, 64, generator=gen).to(BF16).to(DEV)
    for call in (A.rotary, torch.compile(A.rotary, backend="aot_eager", fullgraph=True)):
        oq, ok = call(q, k, at, rope)
        assert oq.requires_grad and not ok.requires_grad
        within(ok, k, z, BF16)
        (d,) = torch.autograd.grad(oq, q, g)
        within(d, g, z.conj(), BF16)
    cache = A.paged_cache(1, 2, 16)
    A.paged_cache_write(cache, ok, k, torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV))
    assert torch.equal(cache.k[0], ok[0]) and torch.equal(cache.v[0], k[0])


def test_second_derivative_and_differences(A):
    rope = A.rotary_frequencies(8, 100.0, attention_factor=1.3, interleaved=True)
    gen = torch.Generator().manual_seed(10)
    at = torch.arange(3, device=DEV)
    q, k = torch.randn(1, 2, 3, 8, generator=gen).to(DEV).requires_grad_(), torch.randn(1, 1, 3, 8, generator=gen).to(DEV).requires_grad_()

    def f(q, k):
        a, b = A.rotary(q, k, at, rope)
        return (a ** 2).sum() * 0.5 + (a * b).sum()

    g = torch.autograd.grad(f(q, k), q, create_graph=True)[0]
    # the turn is linear and keeps lengths but for 1.3: the gradient is 1.69 (q + k), its derivative along v 1.69 v
    assert float((g - 1.69 * (q + k)).detach().abs().max()) < 1e-5
    v = torch.randn(1, 2, 3, 8, generator=gen).to(DEV)
    (gg,) = torch.autograd.grad(g, q, v)
    assert float((gg - 1.69 * v).abs().max()) < 1e-5
    with torch.no_grad():
        e = 2.0 ** -6
        slope = (f(q + e * v, k).double() - f(q - e * v, k).double()) / (2 * e)      # (quadratic: exact but for the roundings, 2^-24 of sums below 2^7, over 2^-5)
    assert abs(float(slope - (g.detach().double() * v.double()).sum())) < 2e-3


def test_captured_and_replayed(A):
    """A captured step follows its positions; another stream than the tensors' own; the eager results in between."""
    rope = A.rotary_frequencies(64, 150000.0, factor=32.0, original_length=4096)
    gen = torch.Generator().manual_seed(11)
    q, k = torch.randn(4, 8, 1, 64, generator=gen).to(BF16).to(DEV), torch.randn(4, 2, 1, 64, generator=gen).to(BF16).to(DEV)
    at = torch.zeros(4, 1, dtype=torch.int32, device=DEV)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        A.rotary(q, k, at, rope)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = A.rotary(q, k, at, rope)
    torch.cuda.current_stream().wait_stream(stream)
    for step in range(4):
        at.fill_(1000 * step + 7)
        graph.replay()
        torch.cuda.synchronize()
        want = A.rotary(q, k, at, rope)
        assert all(torch.equal(x, y) for x, y in zip(out, want)), step


def test_compiled(A):
    rope = A.rotary_frequencies(64, 10000.0)
    q, k = torch.randn(1, 8, 20, 64, device=DEV, dtype=BF16).requires_grad_(), torch.randn(1, 2, 20, 64, device=DEV, dtype=BF16).requires_grad_()
    at = torch.arange(20, device=DEV)

    def f(q, k):
        a, b = A.rotary(q, k, at, rope)
        return a * 2, b

    want = f(q, k)
    got = torch.compile(f, backend="aot_eager", fullgraph=True)(q, k)
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    for x, y in zip(torch.autograd.grad(want, (q, k), (gq, gk)), torch.autograd.grad(got, (q, k), (gq, gk))):
        assert torch.equal(x, y)


def test_refusals(A):
    rope = A.rotary_frequencies(64, 10000.0)
    q, k, at = torch.randn(2, 4, 5, 64, device=DEV), torch.randn(2, 2, 5, 64, device=DEV), torch.arange(5, device=DEV)
    cos = torch.ones(2, 5, 32, device=DEV)
    for call, what in (
        (lambda: A.rotary(q, k[:1], at, rope), "must be"),
        (lambda: A.rotary(q, k[:, :, :4], at, rope), "must be"),
        (lambda: A.rotary(q, k.to(BF16), at, rope), "dtypes"),
        (lambda: A.rotary(q.double(), k.double(), at, rope), "dtypes"),
        (lambda: A.rotary(q, k.cpu(), at, rope), "on cpu"),
        (lambda: A.rotary(q, k, at[:4], rope), "positions"),
        (lambda: A.rotary(q, k, at.expand(3, 5), rope), "positions"),
        (lambda: A.rotary(q, k, at.float(), rope), "integers"),
        (lambda: A.rotary(q, k, at, A.rotary_frequencies(66)), "do not fit"),
        (lambda: A.rotary(q, k, at, A.Rotary(rope.frequencies[:0])), "do not fit"),
        (lambda: A.rotary(q, k, at, A.Rotary(rope.frequencies.clone().requires_grad_())), "no gradient"),
        (lambda: A.rotary_tables(q, k, cos, cos[:, :, :31]), "cos and sin"),
        (lambda: A.rotary_tables(q, k, cos[:, :4], cos[:, :4]), "cos"),
        (lambda: A.rotary_tables(q, k, cos.clone().requires_grad_(), cos), "no gradient"),
        (lambda: A.hip_rotary_pos_emb(q, k, cos, cos, 0), "unsqueeze_dim"),
        (lambda: A.rotary(torch.randn(1, 1, 1, 320, device=DEV), torch.randn(1, 1, 1, 320, device=DEV), at[:1], rope), "do not fit"),
        (lambda: torch.vmap(lambda x: A.rotary(x, x, at, rope)[0])(q[None]), "vmapped"),
    ):
        with pytest.raises(RuntimeError, match=what):
            call()


def test_patched_layer(A):
    """A model's layers with the embedding swapped are those with transformers' in the same precision: float32, where both round alike."""
    transformers = pytest.importorskip("transformers")
    from oregon_gpt_oss_patching_amd.patching import patch_flash_attention, unpatch_flash_attention
    from transformers.models.gpt_oss import modeling_gpt_oss as M
    config = transformers.GptOssConfig(vocab_size=64, hidden_size=128, intermediate_size=64, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                                       num_local_experts=2, num_experts_per_tok=1, layer_types=["sliding_attention", "full_attention"], sliding_window=8,
                                       attn_implementation="eager", use_cache=False)
    torch.manual_seed(0)
    with torch.device(DEV):
        model = transformers.GptOssForCausalLM(config).float()
    ids = torch.randint(0, 64, (2, 21), generator=torch.Generator().manual_seed(1)).to(DEV)
    found, before = [], M.apply_rotary_pos_emb
    try:
        for ours in (False, True):
            patch_flash_attention(rotary=ours)
            assert (M.apply_rotary_pos_emb is A.hip_rotary_pos_emb) == ours
            loss = model(ids, labels=ids).loss
            model.zero_grad()
            loss.backward()
            found.append([loss.detach()] + [p.grad.clone() for n, p in model.named_parameters() if "_proj.weight" in n and "experts" not in n])
    finally:
        unpatch_flash_attention()
    assert M.apply_rotary_pos_emb is before and len(found[0]) == 9
    for x, y in zip(*found):
        assert float((x - y).norm()) <= 1e-4 * float(x.norm())


def test_both_directions_captured(A):
    """The call and its way back (what a gradient goes through) in one graph, replayed with other positions between eager calls."""
    rope = A.rotary_frequencies(64, 150000.0, factor=32.0, original_length=4096)
    gen = torch.Generator().manual_seed(12)
    q, k, gq, gk = (torch.randn(2, n, 70, 64, generator=gen).to(BF16).to(DEV) for n in (8, 2, 8, 2))
    at = torch.arange(70, device=DEV).expand(2, 70).clone()

    def both():
        out = A.rotary(q, k, at, rope)
        return (*out, *torch.ops.gptoss_attn.rotary(gq, gk, at, rope.frequencies, None, None, rope.scale, False, True))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = both()
    for step in range(3):
        at += 977 * step
        for t in outs:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        x, y = q.clone().requires_grad_(), k.clone().requires_grad_()
        a, b = A.rotary(x, y, at, rope)
        want = (a, b, *torch.autograd.grad((a, b), (x, y), (gq, gk)))
        assert all(torch.equal(s, t) for s, t in zip(outs, want)), step


def test_transforms_and_changed_positions_are_refused(A):
    rope = A.rotary_frequencies(64, 10000.0)
    q, at = torch.randn(1, 2, 3, 64, device=DEV), torch.arange(3, device=DEV)
    for call in (lambda: torch.func.grad(lambda a: (A.rotary(a, q, at, rope)[0] ** 2).sum())(q), lambda: torch.func.jvp(lambda a: A.rotary(a, q, at, rope)[0], (q,), (q,)),
                 lambda: torch.vmap(lambda a: A.rotary(a, a, at, rope)[0])(q[None])):
        with pytest.raises(RuntimeError):
            call()
    x = q.clone().requires_grad_()
    out = A.rotary(x, q, at, rope)[0]
    at += 1                                    # the gradient would be turned by other angles
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(out.sum(), x)


def test_a_recorded_gradient_that_would_leave_its_graph_is_refused(A):
    """A leaf with an eager result alive, and a tensor of an eager call: their autograd nodes belong to another stream than the one that records.  The forward call
    raises, in front of any launch; what else is recorded stays whole, and without a gradient wanted the same tensors are taken."""
    rope = A.rotary_frequencies(64, 10000.0)
    gen = torch.Generator().manual_seed(21)
    at = torch.arange(9, device=DEV)
    x, k = torch.randn(1, 4, 9, 64, generator=gen).to(DEV).requires_grad_(), torch.randn(1, 2, 9, 64, generator=gen).to(DEV)
    alive = A.rotary(x, k, at, rope)
    product = k.clone().requires_grad_() * 2
    other = torch.randn(1, 4, 9, 64, generator=gen).to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        with pytest.raises(RuntimeError, match="gradient of q .* recorded"):
            A.rotary(x, k, at, rope)
        with pytest.raises(RuntimeError, match="gradient of k .* recorded"):
            A.rotary(other, product, at, rope)
        with pytest.raises(RuntimeError, match="gradient of q .* recorded"):
            A.rotary_tables(x, k, torch.ones(1, 9, 32, device=DEV), torch.ones(1, 9, 32, device=DEV))
        with torch.no_grad():
            out = A.rotary(x, product, at, rope)
    for step in range(3):
        at += step
        graph.replay()
        torch.cuda.synchronize()
        with torch.no_grad():
            assert all(torch.equal(a, b) for a, b in zip(out, A.rotary(x, product, at, rope))), step
    # eager, they have their gradients
    (d,) = torch.autograd.grad(A.rotary(x, k, torch.arange(9, device=DEV), rope)[0], x, other)
    within(d, other, R.of_positions(torch.arange(9)[None], rope.frequencies.cpu()).conj(), FP32)
    assert alive[0].requires_grad


def test_a_training_step_recorded(A):
    """Call and gradients by the engine in one graph, of leaves without an eager result, replayed with other inputs, positions and gradients between eager steps of other leaves."""
    rope = A.rotary_frequencies(64, 150000.0, factor=32.0, original_length=4096)
    gen = torch.Generator().manual_seed(22)

    def numbers():
        return [torch.randn(2, n, 33, 64, generator=gen).to(BF16).to(DEV) for n in (8, 2, 8, 2)]

    at = torch.arange(33, device=DEV).expand(2, 33).clone()

    def step(q, k, gq, gk):
        out = A.rotary(q, k, at, rope)
        return (*out, *torch.autograd.grad(out, (q, k), (gq, gk)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q, k, gq, gk = numbers()
        step(q.requires_grad_(), k.requires_grad_(), gq, gk)
    side.synchronize()
    q, k, gq, gk = numbers()
    q.requires_grad_(), k.requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step(q, k, gq, gk)
    for i in range(4):
        with torch.no_grad():
            for t, new in zip((q, k, gq, gk), numbers()):
                t.copy_(new)
        at += 311 * i
        for t in out:
            t.detach().fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        want = step(q.detach().clone().requires_grad_(), k.detach().clone().requires_grad_(), gq, gk)
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def _c_call(q, k, qo, ko, positions, frequencies, scale, interleaved, inverse, stride_of_one=None):
    """The C interface on tensors (B, heads, S, D) as they lie; `stride_of_one`: what is said of the tokens' stride where a row has one token."""
    import ctypes

    from oregon_gpt_oss_patching_amd import _lib
    p = _lib.RotaryParams()
    p.struct_size = ctypes.sizeof(p)
    p.dtype = _lib.DTYPE_FP32 if q.dtype == FP32 else _lib.DTYPE_BF16
    p.B, p.H, p.S, p.D = q.shape
    p.G, p.R, p.position_bytes = k.shape[1], 2 * frequencies.numel(), positions.element_size()
    p.interleaved, p.inverse, p.scale = interleaved, inverse, scale
    p.positions, p.frequencies = positions.data_ptr(), frequencies.data_ptr()
    p.position_stride_b, p.position_stride_s = positions.stride()
    for name, t in (("q", q), ("k", k), ("q_out", qo), ("k_out", ko)):
        assert t.stride(3) == 1
        setattr(p, name, t.data_ptr())
        s = getattr(p, name + "_stride")
        s.b, s.h, s.s = t.stride(0), t.stride(1), t.stride(2) if stride_of_one is None else stride_of_one
    rc = _lib.load().gptoss_attn_rotary(ctypes.byref(p), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == 0, rc


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("b,h,g,s,d,r", [(5, 7, 3, 1, 64, 64), (1, 1, 1, 1, 64, 32), (2, 7, 3, 33, 80, 32), (3, 3, 2, 17, 66, 6), (1, 13, 5, 2500, 64, 64), (2, 13, 5, 3000, 64, 48)])
def test_in_place_through_the_c_interface(A, b, h, g, s, d, r, interleaved, dtype):
    """q and k themselves as results, tokens or heads outermost, both directions: the bits of results of their own."""
    print(f"case B={b} H={h} G={g} S={s} D={d} R={r} interleaved={interleaved} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(b + s)
    rope = A.rotary_frequencies(r, 150000.0, attention_factor=1.25, interleaved=interleaved)
    positions = torch.randint(0, 9000, (b, s), generator=gen).to(DEV)
    for tokens_outermost in (True, False):
        def numbers(n):
            x = torch.randn(b, s, n, d, generator=gen).to(dtype).to(DEV)
            return x.transpose(1, 2) if tokens_outermost else x.transpose(1, 2).contiguous()
        q, k = numbers(h), numbers(g)
        want = A.rotary(q, k, positions, rope)
        back = torch.ops.gptoss_attn.rotary(*want, positions, rope.frequencies, None, None, rope.scale, interleaved, True)
        for inverse, expect in ((False, want), (True, back)):
            _c_call(q, k, q, k, positions, rope.frequencies, rope.scale, interleaved, inverse)
            assert torch.equal(q, expect[0]) and torch.equal(k, expect[1]), (tokens_outermost, inverse)


@pytest.mark.parametrize("stride", [0, 64, 4096, 1 << 30])
def test_rows_of_one_token_whatever_their_stride(A, stride):
    """Of one token a row, what is said of the way to the next one is not looked at."""
    rope = A.rotary_frequencies(64, 150000.0)
    gen = torch.Generator().manual_seed(31)
    positions = torch.randint(0, 9000, (300, 1), generator=gen).to(DEV)
    for transposed in (True, False):
        q, k = (torch.randn(300, n, 1, 64, generator=gen).to(BF16).to(DEV) for n in (64, 8))
        if transposed:                             # heads far apart, rows next to each other
            q, k = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k))
        want = A.rotary(q, k, positions, rope)
        out = [torch.full_like(x, float("nan")) for x in (q, k)]
        _c_call(q, k, *out, positions, rope.frequencies, rope.scale, False, False, stride)
        assert all(torch.equal(x, y) for x, y in zip(out, want))
        for got, x in zip(want, (q, k)):
            within(got, x, R.of_positions(positions.cpu(), rope.frequencies.cpu()), BF16)


def test_queries_of_a_stream_that_has_joined_the_recording(A):
    """A graph over two streams: q is computed on one and turned on the other, with a gradient wanted."""
    rope = A.rotary_frequencies(64, 10000.0)
    gen = torch.Generator().manual_seed(23)
    at = torch.arange(9, device=DEV)
    x, k = (torch.randn(1, n, 9, 64, generator=gen).to(DEV) for n in (4, 2))
    with torch.no_grad():
        A.rotary(x * 2, k, at, rope)
    leaf = x.clone().requires_grad_()
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        other.wait_stream(side)
        with torch.cuda.stream(other):
            q = leaf * 2
        side.wait_stream(other)
        out = A.rotary(q, k, at, rope)
    for step in range(3):
        at += step
        graph.replay()
        torch.cuda.synchronize()
        assert out[0].requires_grad and all(torch.equal(a, b) for a, b in zip(out, A.rotary(x * 2, k, at, rope))), step
