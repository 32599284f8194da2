"""joyomni_ops.prefix: the 4-bit projections, the rotary append and attention over a shared prefix run together, a
prompt and then single tokens, against the same layer in 64 bits over the weights that the 4 bits stand for.

The layer in 64 bits rounds where the layer does (projections to bf16, rotated keys to bf16, the attention's
result to bf16, activations to 4 bits).  Its codes may differ from the layer's where a bf16 rounding fell the
other way, a relative 2^-8 in front of a quantiser whose own step is up to 1/4: a code flips for a share 2^-8 / (1/8)
of the elements at most, by a step of a third of the value, so the outputs agree within sqrt(1/32) / 3 = 6 % of
their norm, and the bound is that.
"""
import pytest
import torch

from oracle import prefix as ref

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def linear64(x, w, fmt):
    codes, scale, row = ref.fp4_quantise(x, fmt)
    return ref.fp4_product(ref.fp4_values(codes, scale, fmt), row, w[0], w[1]).to(BF)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("b,h,hk,d,hidden,p", [(3, 4, 2, 64, 256, 500), (2, 2, 2, 128, 160, 77)])
def test_layer(jo, dev, fmt, b, h, hk, d, hidden, p):
    from joyomni_ops import prefix, rope

    g = torch.Generator(device=dev)
    g.manual_seed(b)
    rnd = lambda *s: torch.randn(s, generator=g, device=dev)
    w1, w2 = rnd((h + 2 * hk) * d, hidden) / hidden ** 0.5, rnd(hidden, h * d) / (h * d) ** 0.5
    layer = prefix.PrefixAttention(prefix.quantize_linear_fp4(w1, None, fmt), prefix.quantize_linear_fp4(w2, None, fmt),
                                   h, hk, d)
    held = []
    for w in (w1, w2):
        codes, scale, row = ref.fp4_quantise(w, fmt)
        held.append((ref.fp4_values(codes, scale, fmt), row))
    cos, sin = rope.rotary_tables(p + 40, d, scaling="yarn", factor=4.0, device=dev)
    cache = prefix.PrefixCache.allocate(rnd(p, hk, d).to(BF), rnd(p, hk, d).to(BF), b, 40)
    for x in (cache.k_own, cache.v_own):
        x.fill_(float("nan"))
    lens = [0] * b
    own = [[torch.zeros(b, 40, hk, d, dtype=BF, device=dev) for _ in range(2)]][0]
    for n, counts in ((20, [20, 7, 13][:b]), (1, [1] * b), (4, [4, 0, 3][:b])):
        x = rnd(b, n, hidden).to(BF)
        y = prefix.step(layer, x, cache, cos, sin, torch.tensor(counts, device=dev, dtype=torch.int32))
        qkv = linear64(x.view(b * n, hidden), held[0], fmt).view(b, n, h + 2 * hk, d)
        o = torch.zeros(b, n, h, d, device=dev, dtype=BF)
        for r in range(b):
            c = counts[r]
            part = qkv[r, n - c:]
            at = p + lens[r] + torch.arange(c, device=dev)
            q = ref.rotary(part[:, :h], cos, sin, at, False).to(BF)
            own[0][r, lens[r]:lens[r] + c] = ref.rotary(part[:, h:h + hk], cos, sin, at, False).to(BF)
            own[1][r, lens[r]:lens[r] + c] = part[:, h + hk:]
            lens[r] += c
            if c:
                o[r, n - c:] = ref.shared_prefix_attention(q[None], cache.k_prefix, cache.v_prefix, own[0][r:r + 1], own[1][r:r + 1],
                                                           [lens[r]])[0][0].to(BF)
        assert cache.lens.tolist() == lens
        want = linear64(o.view(b * n, h * d), held[1], fmt).view(b, n, hidden)
        for r in range(b):
            if counts[r]:
                got, exact = y[r, n - counts[r]:].double(), want[r, n - counts[r]:].double()
                assert (got - exact).norm() <= 0.06 * exact.norm()
    with pytest.raises(ValueError):
        prefix.step(layer, rnd(b, 16, hidden).to(BF), cache, cos, sin)


def test_step_in_a_graph(jo, dev):
    from joyomni_ops import prefix, rope

    g = torch.Generator(device=dev)
    g.manual_seed(1)
    rnd = lambda *s: torch.randn(s, generator=g, device=dev)
    layer = prefix.PrefixAttention(prefix.quantize_linear_fp4(rnd(384, 128)), prefix.quantize_linear_fp4(rnd(128, 128)), 2, 2, 64)
    cos, sin = rope.rotary_tables(200, 64, device=dev)
    kp, vp = rnd(100, 2, 64).to(BF), rnd(100, 2, 64).to(BF)
    eager, graphed = (prefix.PrefixCache.allocate(kp, vp, 4, 50) for _ in range(2))
    x = [rnd(4, 1, 128).to(BF) for _ in range(6)]
    want = [prefix.step(layer, v, eager, cos, sin) for v in x]
    held = x[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        prefix.step(layer, held, graphed, cos, sin)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = prefix.step(layer, held, graphed, cos, sin)
    for i in range(1, 6):
        held.copy_(x[i])
        graph.replay()
        assert torch.equal(y, want[i])


def test_replay_beyond_the_cache_leaves_the_next_request_alone(jo, dev):
    from joyomni_ops import prefix, rope

    g = torch.Generator(device=dev)
    g.manual_seed(2)
    rnd = lambda *s: torch.randn(s, generator=g, device=dev)
    layer = prefix.PrefixAttention(prefix.quantize_linear_fp4(rnd(384, 128)), prefix.quantize_linear_fp4(rnd(128, 128)),
                                   2, 2, 64)
    cos, sin = rope.rotary_tables(200, 64, device=dev)
    cache = prefix.PrefixCache.allocate(rnd(100, 2, 64).to(BF), rnd(100, 2, 64).to(BF), 3, 50)
    for x in (cache.k_own, cache.v_own):
        x.fill_(7)
    cache.lens[:] = torch.tensor([50, 3, 49], device=dev, dtype=torch.int32)  # the host does not know: filled is 0
    prefix.step(layer, rnd(3, 2, 128).to(BF), cache, cos, sin)
    for x in (cache.k_own, cache.v_own):
        changed = (x != 7).flatten(2).any(2)
        want = torch.zeros(3, 50, dtype=torch.bool, device=dev)
        want[1, 3:5], want[2, 49] = True, True
        assert torch.equal(changed, want)
