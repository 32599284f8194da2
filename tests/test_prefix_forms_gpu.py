"""The forms of the shared-prefix layer's kernels that large cases take, at the smallest sizes that reach them, against
the definitions in 64 bits (oracle/prefix.py).  Bounds: as in test_prefix_gpu.py.
"""
import math

import pytest
import torch

from oracle import prefix as ref
from test_prefix_gpu import BF, F16, F32, ROUND, check_product, check_quant, check_rotary, gen, inputs, normal, spoil, tables, within

pytestmark = pytest.mark.gpu


def check_attention(jo, q, kp, vp, ko, vo, lens, causal, scale=None):
    out, lse = jo.shared_prefix_attention(q, kp, vp, ko, vo, lens, causal, scale)
    want, wlse, mass = ref.shared_prefix_attention_by_request(q, kp, vp, ko, vo, lens, causal, scale)
    seen = [x for x in (vp, *(vo[r, :n] for r, n in enumerate(lens.clamp(0, vo.shape[1]).tolist()))) if x.numel()]
    top = max([x.double().abs().max().item() for x in seen] + [0.0])
    keys = kp.shape[0] + ko.shape[1]
    u = ROUND[q.dtype]
    within(out, want, u * want.abs() + (u + 2.0 ** -16) * mass + keys * 2.0 ** -24 * top, "out")
    k = [x for x in (kp, *(ko[r, :n] for r, n in enumerate(lens.clamp(0, ko.shape[1]).tolist()))) if x.numel()]
    size = (q.shape[-1] ** -0.5 if scale is None else scale) * q.double().norm(dim=-1).max() * max(
        [x.double().norm(dim=-1).max().item() for x in k] + [0.0])
    within(lse, wlse, 2.0 ** -20 * (1 + wlse.abs().nan_to_num(posinf=0.0) + size), "lse")
    assert torch.equal(torch.isneginf(lse), torch.isneginf(wlse))
    again = jo.shared_prefix_attention(q, kp, vp, ko, vo, lens, causal, scale)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1]), "two calls differ"
    return out, lse


def no_faults():
    from joyomni_ops import cabi

    torch.cuda.synchronize()
    assert cabi.device_fault_count() == 0


# Units of 256 rows: two streams share every key tile, and one tells the other what it found in an own value tile.
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,n,hk,g,p,s", [(64, 1, 4, 8, 12000, 60), (130, 1, 8, 1, 130, 60), (40, 40, 3, 1, 700, 60)])
def test_attention_of_units_with_idle_requests(jo, dev, d, b, n, hk, g, p, s):
    for dtype, live in ((BF, (0, 1, 15, 16, 30, 31)), (F16, (0, 3, 4, 5, 29)), (BF, (30, 31))):
        x = inputs(dev, b, n, hk, g, d, p, s, dtype, seed=b + d)
        x[5][:] = 0  # long runs of requests without a row of their own, between a few that have some
        for r in range(b):
            if r % 32 in live:
                x[5][r] = s - r % 7
        spoil(x[5], x[3], x[4])
        check_attention(jo, *x, True)
    no_faults()


# Every way in which walks of 256-row units are cut: none, all of them, only the last units'; requests that a unit
# straddles, and several units to a request; last row tiles of more and of fewer than 128 rows.
SHARED = [
    (2, 130, 40, 2, 0, 60), (40, 130, 2, 2, 0, 60), (2, 130, 40, 1, 150, 60),                  # whole
    (20, 7, 24, 1, 0, 60), (20, 3, 8, 8, 700, 60), (40, 40, 3, 1, 700, 60),                    # all in parts
    (1, 130, 40, 1, 130, 600), (5, 130, 3, 4, 130, 600), (1, 300, 8, 4, 130, 600),
    (40, 40, 24, 1, 0, 60), (100, 130, 3, 1, 130, 60), (2, 300, 16, 4, 130, 300), (5, 40, 40, 4, 130, 300),  # the last
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,d", [(BF, 128), (F16, 64)])
@pytest.mark.parametrize("b,n,hk,g,p,s", SHARED)
def test_attention_of_shared_units(jo, dev, causal, dtype, d, b, n, hk, g, p, s):
    x = inputs(dev, b, n, hk, g, d, p, s, dtype, seed=b + n + p)
    x[5][0] = s
    if b > 2:
        x[5][1], x[5][2] = 0, 1
    spoil(x[5], x[3], x[4])
    check_attention(jo, *x, causal)
    no_faults()


@pytest.mark.parametrize("dtype,d", [(F16, 128), (BF, 64)])
@pytest.mark.parametrize("b,n,hk,g,p,s", [(40, 40, 3, 1, 700, 60), (5, 130, 3, 4, 130, 600), (2, 300, 16, 4, 130, 300)])
def test_attention_of_shared_units_keeps_a_bad_value_to_the_rows_that_see_it(jo, dev, dtype, d, b, n, hk, g, p, s):
    q, kp, vp, ko, vo, lens = inputs(dev, b, n, hk, g, d, p, s, dtype, seed=3)
    lens[:] = s
    clean = jo.shared_prefix_attention(q, kp, vp, ko, vo, lens, True)
    at = s - n // 2  # of request 1; its queries from n - n // 2 on see it
    vo[1, at, 0, 5] = math.inf
    vo[1, at + 3, 1] = math.nan
    out, lse = jo.shared_prefix_attention(q, kp, vp, ko, vo, lens, True)
    first = n - n // 2
    sees = torch.zeros(b, n, hk * g, dtype=torch.bool, device=dev)
    sees[1, first:, :g], sees[1, first + 3:, g:2 * g] = True, True
    assert torch.equal(out[~sees], clean[0][~sees]) and torch.equal(lse, clean[1])
    assert not torch.isfinite(out[1, first:, :g, 5]).any() and torch.isnan(out[1, first + 3:, g:2 * g]).all()
    no_faults()


# More tiles than the GPU holds CTA pairs (74): the second accumulator, and the ring's state from tile to tile.
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("out", [BF, F16])
@pytest.mark.parametrize("m,n,k", [(2600, 2568, 288), (4000, 4008, 64), (2300, 2560, 2080), (5400, 3080, 32), (257, 20488, 1568)])
def test_product_of_several_tiles_per_pair(jo, dev, fmt, out, m, n, k):
    check_product(jo, dev, m, n, k, fmt, out, bias=m % 200 == 0)
    no_faults()


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("m,k", [(400, 12288), (250, 20480)])  # four and (16 bits) six runs per lane
def test_quant_of_long_rows(jo, dev, fmt, dtype, m, k):
    check_quant(jo, normal(gen(dev, k), dev, m, k).to(dtype), fmt)


# One key 26 bits above 43200 equal ones, which have 6.4e-4 of the weight between them.  Bound in fp16: every weight is
# rounded, a relative 2^-11 and an absolute 2^-32 of a sum of at least 1 (the kernel keeps weights up to 2^15).
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("n,hk,place", [(1, 2, 0), (256, 74, 0), (256, 74, 43199), (128, 74, 20000)])
def test_attention_weights_far_below_the_largest_keep_their_share(jo, dev, dtype, n, hk, place):
    p = 43200
    k, v = torch.zeros(p, hk, 64, device=dev, dtype=dtype), torch.ones(p, hk, 64, device=dev, dtype=dtype)
    k[place, :, 0], v[place] = 26 * math.log(2), 0
    q = torch.zeros(1, n, hk, 64, device=dev, dtype=dtype)
    q[..., 0] = 1
    own = torch.zeros(1, 8, hk, 64, device=dev, dtype=dtype)
    lens = torch.zeros(1, device=dev, dtype=torch.int32)
    out, lse = jo.shared_prefix_attention(q, k, v, own, own, lens, True, 1.0)
    want, wlse, mass = ref.shared_prefix_attention_by_request(q[:, :1], k, v, own, own, lens, True, 1.0)
    u = ROUND[dtype]
    within(out, want.expand_as(out), u * want.abs() + (u + 2.0 ** -16) * mass + p * 2.0 ** -32, "out")
    within(lse, wlse.expand_as(lse), 2.0 ** -20 * (1 + 2 * wlse.abs()), "lse")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("interleaved", [True, False])
def test_rotary_forward_derivative(jo, dev, dtype, interleaved):
    import torch.autograd.forward_ad as fw

    g = gen(dev, 11)
    q, k, dq, dk = (normal(g, dev, 6, h, 64).to(dtype) for h in (3, 1, 3, 1))
    cos, sin = tables(dev, 9, 48)
    at = torch.arange(6, device=dev)
    with fw.dual_level():
        out = jo.rotary_embed(fw.make_dual(q, dq), fw.make_dual(k, dk), cos, sin, at, interleaved)
        for o, x, t in zip(out, (q, k), (dq, dk)):
            value, tangent = fw.unpack_dual(o)
            check_rotary(value, x, cos, sin, at, interleaved)
            check_rotary(tangent, t, cos, sin, at, interleaved)
    f = lambda x: jo.rotary_embed(x, None, cos, sin, at, interleaved)[0]
    check_rotary(torch.func.jvp(f, (q,), (dq,))[1], dq, cos, sin, at, interleaved)
    check_rotary(torch.func.grad(lambda x: (f(x) * dq).sum())(q), dq, cos, sin, at, interleaved, inverse=True)


def test_longest_rows(jo, dev):
    from joyomni_ops import cabi

    room = cabi.lib().jo_fp4_linear_workspace
    for f, fmt in enumerate(("nvfp4", "mxfp4")):
        for dtype, most in ((BF, 98304), (F16, 98304), (F32, 65536)):
            check_quant(jo, normal(gen(dev, f), dev, 3, most).to(dtype), fmt)
            longer = torch.zeros(3, most + 32, device=dev, dtype=dtype)
            with pytest.raises(RuntimeError, match=f"at most {most}"):
                jo.quant_fp4(longer, fmt)
            assert jo.quant_fp4(longer[:0], fmt)[0].shape == (0, most // 2 + 16)
        assert room(20, 98304, f) > 0 and room(20, 98336, f) == -1 and room(2 ** 31, 64, f) == -1
        w = normal(gen(dev, 5), dev, 16, 98304).to(BF)
        for m in (1, 20):
            x = normal(gen(dev, m), dev, m, 98304).to(BF)
            a, b = jo.quant_fp4(x, fmt), jo.quant_fp4(w, fmt)
            assert torch.equal(jo.fp4_linear(x, *b), jo.fp4_scaled_mm(a[0], b[0], a[1], b[1], a[2], b[2], BF))
        # a block of 32 more than that
        tiles = b[1].new_zeros(1, 1537 if fmt == "nvfp4" else 769, 32, 4, 4)
        wide = torch.zeros(8, 49168, device=dev, dtype=torch.uint8), tiles, None if b[2] is None else b[2][:8]
        with pytest.raises(RuntimeError, match="at most 98304"):
            jo.fp4_linear(torch.zeros(1, 98336, device=dev, dtype=BF), *wide)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_one_row_with_any_row_stride(jo, dev, fmt):
    g = gen(dev, 12)
    x, w = normal(g, dev, 1, 64).to(BF), jo.quant_fp4(normal(g, dev, 8, 64), fmt)
    a = jo.quant_fp4(x, fmt)
    want = jo.fp4_scaled_mm(a[0], w[0], a[1], w[1], a[2], w[2], BF)
    turned = a[0].view(32, 1).clone().t()  # [1, 32], contiguous, row stride 1
    assert turned.stride() == (1, 1)
    assert torch.equal(jo.fp4_scaled_mm(turned, w[0], a[1], w[1], a[2], w[2], BF), want)
    assert torch.equal(jo.dequant_fp4(turned, *a[1:]), jo.dequant_fp4(*a))
    column = x.view(64, 1).clone().t()
    assert torch.equal(jo.fp4_linear(column, *w), want) and torch.equal(jo.quant_fp4(column, fmt)[0], a[0])
