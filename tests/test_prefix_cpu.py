"""Host side of the attention layer whose requests share a long prefix: registration, shapes, tables, the oracle."""
import math

import pytest
import torch

from oracle import prefix as ref


def test_ops_registered_and_cuda_only(jo):
    for name in ("quant_fp4", "dequant_fp4", "fp4_scaled_mm", "fp4_linear", "rotary_embed", "rotary_embed_append",
                 "shared_prefix_attention"):
        assert hasattr(torch.ops.joyomni_ops, name) and name in jo.__all__
    with pytest.raises((NotImplementedError, RuntimeError)):
        jo.quant_fp4(torch.zeros(4, 64))
    with pytest.raises((NotImplementedError, RuntimeError)):
        jo.rotary_embed(torch.zeros(4, 1, 64), None, torch.zeros(4, 32), torch.zeros(4, 32), torch.zeros(4, dtype=torch.long))


def test_fake_shapes(jo):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty(130, 96, dtype=torch.bfloat16, device="cuda")
        q, block, row = jo.quant_fp4(x)
        assert q.shape == (130, 48) and block.shape == (2, 2, 32, 4, 4) and row.shape == (130, 1)
        assert block.dtype == torch.float8_e4m3fn
        q2, block2, none = jo.quant_fp4(x, "mxfp4")
        assert block2.shape == (2, 1, 32, 4, 4) and block2.dtype == torch.float8_e8m0fnu and none is None
        assert jo.dequant_fp4(q, block, row).shape == (130, 96)
        assert jo.fp4_scaled_mm(q, q, block, block, row, row, torch.float16).shape == (130, 130)
        assert jo.fp4_linear(x, q, block, row).dtype == torch.bfloat16
        h = torch.empty(5, 4, 64, dtype=torch.bfloat16, device="cuda")
        t = torch.empty(9, 32, device="cuda")
        at = torch.empty(5, dtype=torch.long, device="cuda")
        a, b = jo.rotary_embed(h, h[:, :2], t, t, at)
        assert a.shape == (5, 4, 64) and b.shape == (5, 2, 64)
        assert jo.rotary_embed_append(h, h, h, t, t, at, at, h, h).shape == (5, 4, 64)
        qq = torch.empty(2, 3, 4, 64, dtype=torch.bfloat16, device="cuda")
        kk = torch.empty(2, 7, 2, 64, dtype=torch.bfloat16, device="cuda")
        o, lse = jo.shared_prefix_attention(qq, kk[0], kk[0], kk, kk, torch.empty(2, dtype=torch.int32, device="cuda"))
        assert o.shape == qq.shape and lse.shape == (2, 4, 3) and lse.dtype == torch.float32


def test_rotary_tables():
    from joyomni_ops import rope

    cos, sin = rope.rotary_tables(100, 64)
    assert cos.shape == (100, 32) and cos.dtype == torch.float32
    full, _ = rope.rope_1d(64, torch.arange(100))
    assert (cos - full[:, ::2]).abs().max() < 1e-4  # fp32 angles there
    lin, _ = rope.rotary_tables(100, 64, scaling="linear", factor=4.0)
    assert torch.equal(lin[::4], cos[:25])
    base, one = rope.scaled_freqs(64)
    ntk, _ = rope.scaled_freqs(64, scaling="ntk", factor=8.0)
    assert one == 1.0 and ntk[0] == base[0] and abs(ntk[-1] * 8 / base[-1] - 1) < 1e-9
    yarn, scale = rope.scaled_freqs(64, scaling="yarn", factor=8.0, original=4096)
    turns = 4096 * base / (2 * math.pi)
    assert torch.equal(yarn[turns > 32], base[turns > 32]) and torch.allclose(yarn[turns < 1] * 8, base[turns < 1])
    assert ((yarn <= base) & (yarn >= base / 8)).all() and scale == 0.1 * math.log(8.0) + 1
    # a distant position keeps its phase
    far = torch.outer(torch.tensor([99999.0], dtype=torch.float64), base).cos().float()
    assert torch.equal(rope.rotary_tables(100000, 64)[0][-1:], far)
    for bad in (dict(dim=3), dict(dim=0), dict(dim=4, scaling="?"), dict(dim=4, factor=0.5), dict(dim=2, scaling="ntk", factor=2.0)):
        with pytest.raises(ValueError):
            rope.scaled_freqs(**bad)


def test_oracle_codes():
    codes = ref.e2m1_codes(torch.tensor([0.0, 0.25, 0.26, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.01, 100.0, -0.3, -0.1]).double())
    assert codes.tolist() == [0, 0, 1, 2, 2, 4, 4, 6, 6, 7, 7, 9, 0]


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_oracle_round_trip(fmt):
    x = torch.randn(130, 96, generator=torch.Generator().manual_seed(1))
    codes, scale, row = ref.fp4_quantise(x, fmt)
    v = ref.fp4_values(codes, scale, fmt) * (1 if row is None else row.double()[:, None])
    # a step is at most a third of the block's largest value, a block scale off by a sixteenth (nvfp4) or a half (mxfp4)
    top = x.view(130, -1, ref.BLOCK[fmt]).abs().amax(2).repeat_interleave(ref.BLOCK[fmt], 1)
    assert ((v - x).abs() <= top / 3).all()
    again = ref.fp4_untile(ref.fp4_tiles(scale), *scale.shape)
    assert torch.equal(again, scale) and torch.equal(ref.fp4_pack(codes) & 15, codes[:, 0::2])


def test_oracle_attention_is_softmax():
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(1, 5, 2, 8, generator=g) for _ in range(3))
    o, lse, _ = ref.shared_prefix_attention(q, k[0, :0], v[0, :0], k, v, [5], causal=True)
    x = torch.einsum("nhd,mhd->hnm", q[0], k[0]).double() / 8 ** 0.5
    x = x.masked_fill(torch.ones(5, 5).triu(1).bool(), -math.inf)
    assert torch.allclose(o[0], torch.einsum("hnm,mhd->nhd", x.softmax(-1), v[0].double()), atol=1e-6)
    assert torch.allclose(lse[0], x.logsumexp(-1), atol=1e-6)


@pytest.mark.parametrize("causal", [True, False])
def test_oracle_attention_by_request(causal):
    g = torch.Generator().manual_seed(3)
    q = torch.randn(5, 4, 6, 8, generator=g)
    kp, vp = (torch.randn(7, 2, 8, generator=g) for _ in range(2))
    ko, vo = (torch.randn(5, 9, 2, 8, generator=g) for _ in range(2))
    lens = [9, 2, 0, 4, 20]
    for r, n in enumerate(lens):
        ko[r, n:], vo[r, n:] = math.nan, math.inf
    for p in (7, 0):
        x = q, kp[:p], vp[:p], ko, vo, lens, causal
        for one, all_ in zip(ref.shared_prefix_attention(*x), ref.shared_prefix_attention_by_request(*x)):
            assert torch.allclose(one, all_, rtol=1e-12, atol=1e-12)


def test_rotary_derivatives(jo):
    """Forward and backward derivatives, alone and through torch.func, over a stand-in for the kernel."""
    import torch.autograd.forward_ad as fw

    g = torch.Generator().manual_seed(4)
    rnd = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)
    q, k, dq, dk = rnd(6, 3, 16), rnd(6, 1, 16), rnd(6, 3, 16), rnd(6, 1, 16)
    cos, sin, at = rnd(9, 6), rnd(9, 6), torch.arange(6) + 2
    f = lambda x: jo.rotary_embed(x, None, cos, sin, at)[0]
    both = lambda x, y: jo.rotary_embed(x, y, cos, sin, at)
    want, back = ref.rotary(dq, cos, sin, at, False), ref.rotary(dq, cos, sin, at, False, True)
    same = lambda x, y: torch.allclose(x, y, rtol=1e-12, atol=1e-12)

    def turn(q, k, cos, sin, positions, interleaved, inverse):
        assert q.stride(-1) == 1 and (k is None or k.stride(-1) == 1)
        r = lambda x: ref.rotary(x, cos, sin, positions, interleaved, inverse)
        return r(q), q.new_empty(0) if k is None else r(k)

    with torch.library._scoped_library("joyomni_ops", "IMPL") as lib:
        lib.impl("rotary_embed", turn, "CPU")
        for enabled in (True, False):
            with torch.set_grad_enabled(enabled), fw.dual_level():
                o, p = both(fw.make_dual(q, dq), fw.make_dual(k, dk))
                assert same(fw.unpack_dual(o).tangent, want)
                assert same(fw.unpack_dual(p).tangent, ref.rotary(dk, cos, sin, at, False))
                o, p = both(fw.make_dual(q, dq), k)
                assert same(fw.unpack_dual(o).tangent, want) and not fw.unpack_dual(p).tangent.any()
                assert same(fw.unpack_dual(f(fw.make_dual(q, dq))).tangent, want)
        assert same(torch.func.jvp(f, (q,), (dq,))[1], want)
        assert same(torch.func.grad(lambda x: (f(x) * dq).sum())(q), back)
        assert torch.func.grad(lambda x: f(x).sum())(q).shape == q.shape
        assert same(torch.func.jacfwd(f)(q), torch.func.jacrev(f)(q))
        assert same(torch.func.vmap(torch.func.grad(lambda x: (f(x) * dq).sum()))(rnd(4, 6, 3, 16))[1], back)
        assert same(torch.func.vmap(both)(rnd(2, 6, 3, 16), torch.stack((dk, k)))[1][0], ref.rotary(dk, cos, sin, at, False))
        a, b = q.clone().requires_grad_(), k.clone().requires_grad_()
        assert torch.autograd.gradcheck(both, (a, b), check_forward_ad=True)
        assert torch.autograd.gradgradcheck(f, (a,), check_fwd_over_rev=True)
        for x in (q, a):  # compiled, without and with a gradient
            o, _ = torch.compile(lambda y: both(y, k), backend="eager", fullgraph=True)(x)
            assert same(o, ref.rotary(q, cos, sin, at, False)) and o.requires_grad == x.requires_grad
        assert same(torch.autograd.grad(o, a, dq)[0], back)


def test_step_reckons_the_room_by_the_rows_that_come_in(jo, monkeypatch):
    from joyomni_ops import prefix

    def append(q, k, v, cos, sin, positions, slots, k_cache, v_cache, interleaved=False):
        live = slots >= 0
        k_cache[slots[live]], v_cache[slots[live]] = k[live], v[live]
        return q

    monkeypatch.setattr(jo, "rotary_embed_append", append)
    monkeypatch.setattr(jo, "shared_prefix_attention", lambda q, *a: (q, None))
    layer = prefix.PrefixAttention(lambda x: torch.ones(x.shape[0], 3 * 2 * 8), lambda x: x, 2, 2, 8)
    cache = prefix.PrefixCache.allocate(torch.zeros(5, 2, 8), torch.zeros(5, 2, 8), 3, 20)
    x = torch.zeros(3, 16, 16)
    for i in range(6):  # padded to 16 tokens, 3 at most are there
        assert prefix.step(layer, x, cache, None, None, torch.tensor([3, 0, 2], dtype=torch.int32), 3).shape == (3, 16, 16)
    assert cache.filled == 18 and cache.lens.tolist() == [18, 0, 12]
    prefix.step(layer, x[:, :2], cache, None, None)  # two more for each
    assert cache.filled == 20 and cache.lens.tolist() == [20, 2, 14]
    assert all((cache.k_own[r, :n] == 1).all() for r, n in enumerate((20, 2, 14)))
    with pytest.raises(ValueError):
        prefix.step(layer, x[:, :1], cache, None, None)
    for most in (-1, 3):
        with pytest.raises(ValueError):
            prefix.step(layer, x[:, :2], cache, None, None, None, most)
    prefix.step(layer, x[:, :2], cache, None, None, torch.zeros(3, dtype=torch.int32), 0)
    assert cache.filled == 20 and cache.lens.tolist() == [20, 2, 14]
