"""The operators of an attention layer whose requests share a long prefix, against their definitions in 64 bits
(oracle/prefix.py): 4-bit rows and their product, the rotary embedding, attention over a shared prefix.

Bounds, derived from the arithmetic before anything ran.  u is the unit roundoff of the output type (2^-8 for
bf16, 2^-11 for fp16, 2^-24 for fp32: half a unit in the last place of 1).
  codes and scales   equal: the definition fixes every rounding
  product            u |d| + (K + 4) 2^-24 sum|a b| (fp32 sums in any order, then two scales and the bias)
  rotation           u |y| + 3 2^-24 (|x0| + |x1|) (two products and a sum in fp32)
  attention          u |o| + u m + 2^-16 m + n 2^-24 max|v|, m the softmax average of |v|: every weight is rounded
                     to the inputs' type (relative u; in fp16 at least 2^-25 absolute, of weights whose sum is at
                     least 1); the fp32 exponentials, whose arguments are off by some 2^-24 |score|, take 2^-16 m
  log-sum-exp        2^-20 (1 + |lse| + max|score|)
"""
import math

import pytest
import torch

from oracle import prefix as ref

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
ROUND = {BF: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}
TINY = {BF: 2.0 ** -133, F16: 2.0 ** -24, F32: 2.0 ** -149}


def gen(dev, seed):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def normal(g, dev, *shape):
    return torch.randn(shape, generator=g, device=dev)


def within(got, want, allowed, what=""):
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine), f"{what}: other places are finite"
    bad = ((got - want).abs() > allowed) & fine
    if bad.any():
        i = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {i}: {got[i].item()} for "
                             f"{want[i].item()}, allowed {allowed.expand_as(want)[i].item()}")


# ------------------------------------------------------------------ 4-bit rows
def check_quant(jo, x, fmt):
    q, block, row = jo.quant_fp4(x, fmt)
    codes, scale, rows = ref.fp4_quantise(x, fmt)
    m, k = x.shape
    want = ref.fp4_tiles(scale)
    assert block.shape == want.shape
    assert torch.equal(block.view(torch.uint8), want), "block scales"
    if fmt == "nvfp4":
        assert row.shape == (m, 1) and row.dtype == F32
        assert torch.equal(row.view(-1).nan_to_num(-1.0), rows.nan_to_num(-1.0)), "row scales"
    else:
        assert row is None
    got = torch.stack((q & 15, q >> 4), 2).view(m, k)
    got = torch.where(got == 8, 0, got)  # a zero's sign is not kept
    assert torch.equal(got, codes), f"{int((got != codes).sum())} codes differ"
    for dt in (BF, F16, F32):
        v = jo.dequant_fp4(q, block, row, dt)
        exact = ref.fp4_values(codes, scale, fmt)
        if row is not None:
            exact = (exact * rows.double()[:, None]).float()
        assert torch.equal(v.nan_to_num(7.0), exact.to(dt).nan_to_num(7.0)), f"values as {dt}"


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("m,k", [(1, 32), (3, 96), (127, 64), (128, 512), (129, 1056), (300, 160), (2, 12288), (1, 33024),
                                 (700, 2080)])
def test_quant_equals_definition(jo, dev, fmt, dtype, m, k):
    g = gen(dev, m + k)
    x = normal(g, dev, m, k) * torch.exp(2 * normal(g, dev, m, 1))
    check_quant(jo, x.to(dtype), fmt)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_quant_many_rows_takes_more_runs_per_lane(jo, dev, fmt):
    check_quant(jo, normal(gen(dev, 1), dev, 4000, 1568).to(BF), fmt)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_quant_edges(jo, dev, fmt):
    x = torch.zeros(9, 64, device=dev, dtype=F32)
    x[1, 5] = 1e-20
    x[2] = 1e-9 * torch.arange(64, device=dev)
    x[3] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 8, device=dev)  # every midpoint between codes
    x[4] = -x[3] * 2.0 ** -30
    x[5] = 3.3e38
    x[5, 1:] = torch.finfo(F32).tiny
    x[6, 0], x[6, 40] = 1e-42, -1e-45  # subnormal
    x[7, :16], x[7, 16:] = 1e-3, 1e3  # block scales far apart
    x[8] = torch.linspace(-448 * 6, 448 * 6, 64, device=dev)
    check_quant(jo, x, fmt)
    check_quant(jo, x.to(BF), fmt)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("dtype", [BF, F16, F32])
def test_quant_marks_rows_that_are_not_finite(jo, dev, fmt, dtype):
    x = normal(gen(dev, 3), dev, 5, 128).to(dtype)
    x[1, 17], x[3, 100] = math.nan, -math.inf
    check_quant(jo, x, fmt)
    v = jo.dequant_fp4(*jo.quant_fp4(x, fmt), F32)
    assert torch.isfinite(v[[0, 2, 4]]).all() and torch.isnan(v[1, 16:32]).all() and torch.isnan(v[3, 96:112]).all()


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("offset,stride", [(0, 200), (1, 193), (8, 208), (16, 192)])
def test_quant_strides_and_alignment(jo, dev, dtype, offset, stride):
    buf = normal(gen(dev, 4), dev, 40 * stride + 64).to(dtype)
    x = buf[offset:offset + 40 * stride].view(40, stride)[:, :160]
    for fmt in ("nvfp4", "mxfp4"):
        check_quant(jo, x, fmt)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_dequant_every_code_and_scale(jo, dev, fmt):
    block = ref.BLOCK[fmt]
    scale = torch.arange(256, device=dev, dtype=torch.uint8).view(256, 1).repeat(1, 32 // block)
    codes = (torch.arange(32, device=dev) % 16).to(torch.uint8).repeat(256, 1)
    q, tiles = ref.fp4_pack(codes), ref.fp4_tiles(scale)
    tiles = tiles.view(torch.float8_e4m3fn if fmt == "nvfp4" else torch.float8_e8m0fnu)
    row = torch.full((256, 1), 0.37, device=dev) if fmt == "nvfp4" else None
    exact = ref.fp4_values(codes, scale, fmt)
    if row is not None:
        exact = exact * row.double()
    for dt in (F32, BF):
        v, want = jo.dequant_fp4(q, tiles, row, dt), exact.float().to(dt)
        assert torch.equal(v.nan_to_num(7.0), want.nan_to_num(7.0))


# ------------------------------------------------------------------ product
def held(jo, w, fmt):
    q, block, row = jo.quant_fp4(w, fmt)
    codes, scale, rows = ref.fp4_quantise(w, fmt)
    return (q, block, row), (ref.fp4_values(codes, scale, fmt), rows)


def check_product(jo, dev, m, n, k, fmt, out, bias, seed=0):
    g = gen(dev, seed + m + n + k)
    a, ea = held(jo, normal(g, dev, m, k), fmt)
    b, eb = held(jo, normal(g, dev, n, k), fmt)
    add = normal(g, dev, n).to(out) if bias else None
    d = jo.fp4_scaled_mm(a[0], b[0], a[1], b[1], a[2], b[2], out, add)
    assert torch.equal(d, jo.fp4_scaled_mm(a[0], b[0], a[1], b[1], a[2], b[2], out, add)), "two calls differ"
    want = ref.fp4_product(ea[0], ea[1], eb[0], eb[1], add)
    sums = ref.fp4_product(ea[0].abs(), ea[1], eb[0].abs(), eb[1], None if add is None else add.abs())
    within(d, want, ROUND[out] * want.abs() + (k + 4) * 2.0 ** -24 * sums + TINY[out], f"{m}x{n}x{k}")


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("m", [1, 15, 17, 33, 64, 65, 129, 300])
@pytest.mark.parametrize("n,k", [(8, 32), (136, 96), (1000, 1056)])
def test_product(jo, dev, fmt, m, n, k):
    check_product(jo, dev, m, n, k, fmt, BF, bias=m % 2 == 0)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("m,n,k", [(700, 3080, 288), (257, 9472, 64), (2048, 1288, 2080), (5000, 520, 32), (513, 5000, 544)])
def test_product_on_cta_pairs(jo, dev, fmt, m, n, k):
    check_product(jo, dev, m, n, k, fmt, F16, bias=True)


@pytest.mark.parametrize("m,n,k", [(4, 264, 12288), (100, 128, 4128), (128, 256, 8192)])
def test_product_split_over_a_cluster(jo, dev, m, n, k):
    for fmt in ("nvfp4", "mxfp4"):
        check_product(jo, dev, m, n, k, fmt, BF, bias=True)


def test_product_operands_with_gaps_between_rows(jo, dev):
    g = gen(dev, 8)
    (q, block, row), _ = held(jo, normal(g, dev, 200, 320), "nvfp4")
    (p, pblock, prow), _ = held(jo, normal(g, dev, 72, 320), "nvfp4")
    wide, tall = torch.full((200, 208), 255, device=dev, dtype=torch.uint8), torch.full((72, 176), 255, device=dev, dtype=torch.uint8)
    wide[:, :160], tall[:, :160] = q, p
    want = jo.fp4_scaled_mm(q, p, block, pblock, row, prow, BF)
    assert torch.equal(jo.fp4_scaled_mm(wide[:, :160], tall[:, :160], block, pblock, row, prow, BF), want)


def test_product_keeps_a_bad_row_to_itself(jo, dev):
    g = gen(dev, 9)
    for fmt in ("nvfp4", "mxfp4"):
        for m, n in ((20, 136), (600, 4096)):
            x, w = normal(g, dev, m, 128).to(BF), normal(g, dev, n, 128).to(BF)
            x[m // 2, 3], w[n - 3, 70] = math.inf, math.nan
            d = jo.fp4_linear(x, *held(jo, w, fmt)[0])
            bad = torch.isnan(d)
            want = torch.zeros_like(bad)
            want[m // 2], want[:, n - 3] = True, True
            assert torch.equal(bad, want)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("m", [1, 70, 1500])
def test_linear_is_quantisation_and_product(jo, dev, dtype, fmt, m):
    g = gen(dev, 10)
    x, w = normal(g, dev, m, 352).to(dtype), held(jo, normal(g, dev, 520, 352), fmt)[0]
    add = normal(g, dev, 520).to(dtype)
    a = jo.quant_fp4(x, fmt)
    assert torch.equal(jo.fp4_linear(x, *w, add), jo.fp4_scaled_mm(a[0], w[0], a[1], w[1], a[2], w[2], dtype, add))


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("n,k", [(520, 32), (136, 288), (264, 2080), (1032, 4096), (9600, 3072), (72, 16384), (8, 20000), (3072, 12288),
                                 (20000, 1024)])
def test_linear_of_few_rows(jo, dev, dtype, fmt, n, k):
    g = gen(dev, n)
    w, add = held(jo, normal(g, dev, n, k), fmt)[0], normal(g, dev, n).to(dtype)
    for m in (1, 2, 3, 4, 5, 8, 9, 16):
        for shift in (0, 1, 8):  # rows on 32 bytes, on their elements, on 16 bytes
            x = normal(g, dev, m, k + 16 + shift).to(dtype)[:, shift:shift + k]
            if m > 2:  # the smallest values, a row of zeros, and rows with an infinity or a NaN
                x[0] *= 2.0 ** -14
                x[1] = 0
                x[2, k - 1] = math.nan if shift else math.inf
            a = jo.quant_fp4(x, fmt)
            want = jo.fp4_scaled_mm(a[0], w[0], a[1], w[1], a[2], w[2], dtype, add)
            torch.testing.assert_close(jo.fp4_linear(x, *w, add), want, rtol=0, atol=0, equal_nan=True)


def test_no_rows(jo, dev):
    x = torch.empty(0, 64, device=dev, dtype=BF)
    q, block, row = jo.quant_fp4(x)
    assert q.shape == (0, 32) and block.shape == (0, 1, 32, 4, 4) and row.shape == (0, 1)
    w = jo.quant_fp4(torch.ones(8, 64, device=dev))
    assert jo.fp4_linear(x, *w).shape == (0, 8) and jo.dequant_fp4(q, block, row).shape == (0, 64)


# ------------------------------------------------------------------ rotary
def tables(dev, p, r, seed=0):
    angle = normal(gen(dev, 100 + seed), dev, p, r // 2) * 3
    return angle.cos(), angle.sin()


def check_rotary(got, x, cos, sin, at, interleaved, inverse=False):
    want = ref.rotary(x, cos, sin, at, interleaved, inverse)
    big = ref.rotary(x.abs(), cos.abs(), -sin.abs(), at, interleaved).abs() + ref.rotary(x.abs(), cos.abs(), sin.abs(), at, interleaved).abs()
    within(got, want, ROUND[x.dtype] * want.abs() + 3 * 2.0 ** -24 * big + TINY[x.dtype])


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("t,hq,hk,d,r", [(1, 1, 1, 64, 64), (5, 8, 2, 128, 128), (33, 3, 1, 128, 64), (700, 24, 24, 128, 96),
                                         (9, 5, 5, 256, 256), (4, 2, 1, 80, 20), (3, 7, 1, 6, 2), (2, 4, 4, 72, 70)])
def test_rotary(jo, dev, interleaved, dtype, t, hq, hk, d, r):
    g = gen(dev, t + d)
    q, k = normal(g, dev, t, hq, d).to(dtype), normal(g, dev, t, hk, d).to(dtype)
    cos, sin = tables(dev, 50, r)
    at = torch.randint(0, 50, (t,), generator=g, device=dev)
    for index in (at, at.int()):
        qo, ko = jo.rotary_embed(q, k, cos, sin, index, interleaved)
        check_rotary(qo, q, cos, sin, at, interleaved)
        check_rotary(ko, k, cos, sin, at, interleaved)
    dq, dk = jo.rotary_embed_backward(q, k, cos, sin, at, interleaved)
    check_rotary(dq, q, cos, sin, at, interleaved, inverse=True)
    check_rotary(dk, k, cos, sin, at, interleaved, inverse=True)
    alone, none = jo.rotary_embed(q, None, cos, sin, at, interleaved)
    assert none is None and torch.equal(alone, qo)


@pytest.mark.parametrize("interleaved", [True, False])
def test_rotary_gradient(jo, dev, interleaved):
    g = gen(dev, 5)
    q, k = normal(g, dev, 6, 3, 16).requires_grad_(), normal(g, dev, 6, 1, 16).requires_grad_()
    cos, sin = tables(dev, 9, 12)
    at = torch.arange(6, device=dev)
    dq, dk = normal(g, dev, 6, 3, 16), normal(g, dev, 6, 1, 16)
    qo, ko = jo.rotary_embed(q, k, cos, sin, at, interleaved)
    gq, gk = torch.autograd.grad((qo, ko), (q, k), (dq, dk))
    check_rotary(gq, dq, cos, sin, at, interleaved, inverse=True)
    check_rotary(gk, dk, cos, sin, at, interleaved, inverse=True)
    # differences: the map is linear, so its directional derivative is a difference of any width
    e = normal(g, dev, 6, 3, 16)
    f = lambda x: jo.rotary_embed(x, None, cos, sin, at, interleaved)[0].double()
    slope = ((f(q.detach() + e) - f(q.detach() - e)) / 2 * dq.double()).sum()
    size = (e.double().abs() * gq.double().abs()).sum()
    assert abs((e.double() * gq.double()).sum() - slope) <= 2.0 ** -19 * (size + slope.abs() + 100)
    # only one of the two, and none
    gq2, = torch.autograd.grad(jo.rotary_embed(q, None, cos, sin, at, interleaved)[0], q, dq)
    assert torch.equal(gq2, gq)
    with torch.no_grad():
        assert not jo.rotary_embed(q, k, cos, sin, at, interleaved)[0].requires_grad


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rotary_gradient_of_broadcast_values(jo, dev, dtype):
    g = gen(dev, 7)
    q, k = (normal(g, dev, 6, h, 64).to(dtype).requires_grad_() for h in (3, 1))
    cos, sin = tables(dev, 9, 64)
    at = torch.arange(6, device=dev)
    qo, ko = jo.rotary_embed(q, k, cos, sin, at)
    (qo.sum() + ko.sum()).backward()  # one value for all elements
    check_rotary(q.grad, torch.ones_like(q), cos, sin, at, False, inverse=True)
    check_rotary(k.grad, torch.ones_like(k), cos, sin, at, False, inverse=True)
    q.grad = k.grad = None
    row = normal(g, dev, 64).to(dtype)
    qo, ko = jo.rotary_embed(q, k, cos, sin, at)
    torch.autograd.backward([qo], [row.expand(6, 3, 64)])  # one row for all heads; none for k
    check_rotary(q.grad, row.expand(6, 3, 64), cos, sin, at, False, inverse=True)
    assert not k.grad.any()
    # twice: the gradient of |dq|^2 with respect to the value that came in is twice its rotation there and back
    d = normal(g, dev, 6, 3, 64).to(dtype).requires_grad_()
    dq, = torch.autograd.grad(jo.rotary_embed(q, None, cos, sin, at)[0], q, d, create_graph=True)
    dd, = torch.autograd.grad(dq, d, dq.detach())
    check_rotary(dd, dq.detach(), cos, sin, at, False)


@pytest.mark.parametrize("interleaved", [True, False])
def test_rotary_strides_and_places_outside_the_tables(jo, dev, interleaved):
    g = gen(dev, 6)
    qkv = normal(g, dev, 20, 3 * 4 * 64).to(BF)  # q, k, v of a projection, as views of its rows
    q, k = (qkv[:, i * 256:(i + 1) * 256].view(20, 4, 64) for i in (0, 1))
    heads_first = normal(g, dev, 4, 20, 64).to(BF).transpose(0, 1)
    odd = normal(g, dev, 20, 4, 67).to(BF)[:, :, 3:]
    cos, sin = tables(dev, 30, 32)
    at = torch.arange(20, device=dev)
    for x in (q, k, heads_first, odd):
        check_rotary(jo.rotary_embed(x, k, cos, sin, at, interleaved)[0], x, cos, sin, at, interleaved)
    at[3], at[9], at[11] = -1, 30, 2 ** 40
    out = jo.rotary_embed(q, None, cos, sin, at, interleaved)[0]
    bad = torch.zeros(20, 4, 64, dtype=torch.bool, device=dev)
    bad[[3, 9, 11], :, :32] = True
    assert torch.equal(torch.isnan(out), bad) and torch.equal(out[..., 32:], q[..., 32:])


def test_rotary_in_place(dev):
    from joyomni_ops import cabi

    for interleaved in (0, 1):
        x = normal(gen(dev, 7), dev, 50, 6, 128).to(BF)
        cos, sin = tables(dev, 64, 96)
        at = torch.arange(50, device=dev)
        y = x.clone()
        cabi.call("jo_rotary_embed", y.data_ptr(), 768, 128, y.data_ptr(), 768, 128, None, 0, 0, None, 0, 0, cos.data_ptr(),
                  sin.data_ptr(), 64, at.data_ptr(), 64, 50, 6, 0, 128, 96, interleaved, 0, cabi.JO_BF16, cabi.stream())
        check_rotary(y, x, cos, sin, at, bool(interleaved))


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("t,hq,hk,d,r", [(1, 4, 1, 64, 64), (40, 6, 2, 128, 64), (300, 24, 24, 128, 128), (3, 2, 2, 40, 12)])
def test_append(jo, dev, interleaved, dtype, t, hq, hk, d, r):
    g = gen(dev, t)
    q, k, v = (normal(g, dev, t, h, d).to(dtype) for h in (hq, hk, hk))
    cache = normal(g, dev, 400, 2, hk, d).to(dtype)  # keys and values side by side
    before = cache.clone()
    cos, sin = tables(dev, 60, r)
    at = torch.randint(0, 60, (t,), generator=g, device=dev)
    slot = torch.randperm(400, generator=g, device=dev)[:t]
    slot[t // 2:t // 2 + 1], slot[t // 3:t // 3 + 1] = -1, 400  # padding tokens
    qo = jo.rotary_embed_append(q, k, v, cos, sin, at, slot, cache[:, 0], cache[:, 1], interleaved)
    check_rotary(qo, q, cos, sin, at, interleaved)
    live = (slot >= 0) & (slot < 400)
    rows = slot[live]
    check_rotary(cache[rows, 0], k[live], cos, sin, at[live], interleaved)
    assert torch.equal(cache[rows, 1], v[live])
    rest = torch.ones(400, dtype=torch.bool, device=dev)
    rest[rows] = False
    assert torch.equal(cache[rest], before[rest]), "a row that no token has was written"


# ------------------------------------------------------------------ attention
def inputs(dev, b, n, hk, g, d, p, s, dtype, seed):
    r = gen(dev, seed)
    q = normal(r, dev, b, n, hk * g, d).to(dtype)
    kp, vp = (normal(r, dev, p, hk, d).to(dtype) for _ in range(2))
    ko, vo = (normal(r, dev, b, s, hk, d).to(dtype) for _ in range(2))
    lens = torch.randint(0, s + 1, (b,), generator=r, device=dev, dtype=torch.int32)
    return q, kp, vp, ko, vo, lens


def spoil(lens, *own):
    for x in own:  # nothing beyond a request's rows may matter
        for r, length in enumerate(lens.clamp(0, x.shape[1]).tolist()):
            x[r, length:] = torch.tensor([math.nan, math.inf, -math.inf, 6e4], device=x.device)[: 1 + r % 4][-1]


def check_attention(jo, q, kp, vp, ko, vo, lens, causal, scale=None):
    out, lse = jo.shared_prefix_attention(q, kp, vp, ko, vo, lens, causal, scale)
    want, wlse, mass = ref.shared_prefix_attention(q, kp, vp, ko, vo, lens, causal, scale)
    used = [x[r, :max(int(length), 0)] for x in (vo,) for r, length in enumerate(lens)] + [vp]
    top = max([x.double().abs().max().item() for x in used if x.numel()] + [0.0])
    keys = kp.shape[0] + ko.shape[1]
    u = ROUND[q.dtype]
    within(out, want, u * want.abs() + (u + 2.0 ** -16) * mass + keys * 2.0 ** -24 * top + TINY[q.dtype], "out")
    size = (q.shape[-1] ** -0.5 if scale is None else scale) * q.double().norm(dim=-1).max() * max(
        [x.double().norm(dim=-1).max().item() for x in (kp, *(ko[r, :max(int(length), 0)] for r, length in enumerate(lens))) if x.numel()] + [0.0])
    within(lse, wlse, 2.0 ** -20 * (1 + wlse.abs().nan_to_num(posinf=0.0) + size), "lse")
    assert torch.equal(torch.isneginf(lse), torch.isneginf(wlse))
    return out, lse


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("b,n,hk,g,d,p,s", [
    (1, 1, 1, 1, 64, 1, 1),       # one key each
    (1, 1, 2, 4, 128, 300, 40),
    (3, 1, 2, 1, 64, 128, 128),   # whole tiles
    (5, 4, 1, 3, 128, 129, 257),  # one key past a tile
    (2, 130, 1, 1, 64, 127, 300),
    (40, 1, 2, 4, 128, 500, 90),  # a row tile of many requests
    (3, 50, 2, 3, 64, 260, 70),   # requests that straddle row tiles
    (70, 5, 1, 1, 64, 33, 20),
    (2, 300, 1, 2, 128, 200, 310),
    (4, 2, 3, 5, 64, 1000, 3),    # fewer rows than queries
    (3, 2, 1, 2, 64, 0, 60),      # no prefix
    (3, 2, 1, 2, 128, 150, 0),    # no own rows
])
def test_attention(jo, dev, causal, dtype, b, n, hk, g, d, p, s):
    x = inputs(dev, b, n, hk, g, d, p, s, dtype, seed=b + n + p)
    spoil(x[5], x[3], x[4])
    check_attention(jo, *x, causal)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,n,hk,g", [(1, 1, 1, 1), (4, 1, 3, 2), (2, 3, 1, 5), (1, 8, 2, 4), (1, 11, 1, 3), (3, 1, 24, 1)])
def test_attention_in_every_number_of_parts(jo, dev, d, b, n, hk, g):
    # up to 32 rows and more, walks of 4 to 40 tiles, and a request without rows of its own
    for p in (512, 700, 1024, 1281, 1500, 1793, 2100, 2305, 5000):
        x = inputs(dev, b, n, hk, g, d, p, 200, BF, p)
        x[-1][0] = 0
        spoil(x[-1], x[3], x[4])
        out, lse = check_attention(jo, *x, True)
        again = jo.shared_prefix_attention(*x, True)
        assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


def test_attention_parts_without_keys(jo, dev):
    # the walk is split for full caches, but its requests are short or empty: parts that see nothing
    for lens in ([0, 0], [1, 0], [0, 130], [2000, 3]):
        x = inputs(dev, 2, 1, 2, 2, 128, 0, 2000, F16, 1)
        x[-1][:] = torch.tensor(lens, device=dev, dtype=torch.int32)
        spoil(x[-1], x[3], x[4])
        check_attention(jo, *x, True)


@pytest.mark.parametrize("causal", [True, False])
def test_attention_of_nothing(jo, dev, causal):
    q, kp, vp, ko, vo, lens = inputs(dev, 4, 3, 2, 2, 64, 0, 50, BF, 1)
    lens[:] = torch.tensor([0, 1, -5, 70], device=dev, dtype=torch.int32)  # lengths are clamped to 0..50
    spoil(lens, ko, vo)
    out, lse = check_attention(jo, q, kp, vp, ko, vo, lens, causal)
    assert (out[0] == 0).all() and torch.isneginf(lse[0]).all() and (out[2] == 0).all()
    out, lse = jo.shared_prefix_attention(q, kp, vp, ko[:, :0], vo[:, :0], lens, causal)
    assert (out == 0).all() and torch.isneginf(lse).all()
    empty = jo.shared_prefix_attention(q[:0], kp, vp, ko[:0], vo[:0], lens[:0], causal)
    assert empty[0].shape == (0, 3, 4, 64) and empty[1].shape == (0, 4, 3)


@pytest.mark.parametrize("n,g", [(1, 4), (40, 2), (200, 1)])
def test_attention_keeps_a_bad_request_to_itself(jo, dev, n, g):
    q, kp, vp, ko, vo, lens = inputs(dev, 6, n, 2, g, 64, 200, 300, BF, 2)
    lens[:] = torch.tensor([300, 250, 290, 0, 300, 211], device=dev, dtype=torch.int32)
    clean = jo.shared_prefix_attention(q, kp, vp, ko, vo, lens, True)
    ko[1, 100], vo[2, 200], vo[4, 10, 1, 3] = math.nan, math.inf, math.nan
    out, lse = jo.shared_prefix_attention(q, kp, vp, ko, vo, lens, True)
    for r in (0, 3, 5):
        assert torch.equal(out[r], clean[0][r]) and torch.equal(lse[r], clean[1][r]), f"request {r} changed"
    for r, at in ((1, 100), (2, 200)):  # of these the queries that see the row, i >= at - (len - n)
        first = max(0, at - (int(lens[r]) - n))
        assert torch.equal(out[r, :first], clean[0][r, :first]) and not torch.isfinite(out[r, first:]).any()
    # the value's own head alone (row 10 is seen by all queries)
    assert torch.equal(out[4][:, :g], clean[0][4][:, :g]) and torch.isnan(out[4][:, g:, 3]).all()
    assert torch.isfinite(lse[[2, 4]]).all()


def test_attention_causal_hides_what_comes_later(jo, dev):
    for b, n in ((1, 20), (3, 150)):
        q, kp, vp, ko, vo, lens = inputs(dev, b, n, 1, 2, 64, 77, 400, F16, 3)
        lens[:] = 380
        clean = jo.shared_prefix_attention(q, kp, vp, ko, vo, lens, True)
        ko[:, 375], vo[:, 375] = math.nan, math.inf  # of the last n rows, row n - 5
        out, lse = jo.shared_prefix_attention(q, kp, vp, ko, vo, lens, True)
        assert torch.equal(out[:, :n - 5], clean[0][:, :n - 5]) and torch.equal(lse[:, :, :n - 5], clean[1][:, :, :n - 5])
        assert not torch.isfinite(out[:, n - 5:]).any()


@pytest.mark.parametrize("dtype", [BF, F16])
def test_attention_large_scores(jo, dev, dtype):
    x = list(inputs(dev, 2, 3, 1, 4, 128, 700, 200, dtype, 4))
    x[0] *= 30  # a softmax near its largest key; maxima that grow from tile to tile
    x[1] *= torch.linspace(0.1, 2, 700, device=dev)[:, None, None].to(dtype)
    check_attention(jo, *x, True)
    check_attention(jo, *x, False, scale=0.01)
    same = [x[0], x[1], torch.ones_like(x[2]), x[3], torch.ones_like(x[4]), x[5]]
    assert (jo.shared_prefix_attention(*same, True)[0].float() - 1).abs().max() <= 2 * ROUND[dtype]


def test_attention_strides(jo, dev):
    g = gen(dev, 5)
    b, n, hk, d, p, s = 3, 7, 2, 64, 150, 90
    qkv = normal(g, dev, b, n, 3, 4, d).to(BF)
    q = qkv[:, :, 0]                                                     # of a fused projection
    kp = normal(g, dev, hk, p, d).to(BF).transpose(0, 1)                 # heads first
    vp = normal(g, dev, p, 3, hk, d).to(BF)[:, 1]                        # rows with others between
    ko = normal(g, dev, s, b, hk, d).to(BF).transpose(0, 1)              # rows first
    vo = normal(g, dev, b, hk, s, d).to(BF).transpose(1, 2)
    lens = torch.tensor([90, 33, 7], device=dev, dtype=torch.int32)
    check_attention(jo, q, kp, vp, ko, vo, lens, True)


def test_attention_offsets_past_32_bits(jo, dev):
    p, step = 300, 2 ** 23  # 2.5e9 elements from the first row to the last
    kv = torch.empty(p * step + 64, device=dev, dtype=BF)
    k, v = kv.as_strided((p, 1, 64), (step, 64, 1)), kv.as_strided((p, 1, 64), (step, 64, 1), 4096)
    g = gen(dev, 6)
    k.copy_(normal(g, dev, p, 1, 64)), v.copy_(normal(g, dev, p, 1, 64))
    q, _, _, ko, vo, lens = inputs(dev, 2, 2, 1, 2, 64, 1, 20, BF, 7)
    check_attention(jo, q, k, v, ko, vo, lens, True)


def test_attention_is_the_same_every_time_and_on_other_streams(jo, dev):
    x = inputs(dev, 9, 3, 4, 3, 128, 3000, 500, BF, 8)
    first = jo.shared_prefix_attention(*x, True)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = jo.shared_prefix_attention(*x, True)
        w = jo.quant_fp4(torch.ones(64, 64, device=dev))
        y = jo.fp4_linear(torch.ones(3, 64, device=dev, dtype=BF), *w)
    side.synchronize()
    assert torch.equal(first[0], second[0]) and torch.equal(first[1], second[1])
    assert (y == 64).all()


def test_attention_of_many_units(jo, dev):
    # more row tiles than the GPU holds, the last ones split
    x = inputs(dev, 2, 700, 24, 1, 64, 300, 40, BF, 9)
    out, lse = jo.shared_prefix_attention(*x, False)
    want = jo.shared_prefix_attention(x[0][:1, 350:360], *x[1:3], x[3][:1], x[4][:1], x[5][:1], False)
    w, l, mass = ref.shared_prefix_attention(x[0][:1, 350:360], *x[1:3], x[3][:1], x[4][:1], x[5][:1], False)
    for o, s in ((out[:1, 350:360], lse[:1, :, 350:360]), want):
        within(o, w, ROUND[BF] * w.abs() + (ROUND[BF] + 2.0 ** -16) * mass + 340 * 2.0 ** -24 * 6, "out")
        within(s, l, 2.0 ** -20 * (1 + l.abs() + 64), "lse")


# ------------------------------------------------------------------ refusals
def test_refusals(jo, dev):
    x = torch.zeros(4, 64, device=dev, dtype=BF)
    w = jo.quant_fp4(torch.ones(8, 64, device=dev))
    mx = jo.quant_fp4(torch.ones(8, 64, device=dev), "mxfp4")
    cos, sin = tables(dev, 8, 64)
    q3 = torch.zeros(4, 2, 64, device=dev, dtype=BF)
    at = torch.zeros(4, device=dev, dtype=torch.long)
    q, kp, vp, ko, vo, lens = inputs(dev, 2, 1, 2, 2, 64, 16, 16, BF, 1)
    cases = [
        lambda: jo.quant_fp4(x, "int4"),
        lambda: jo.quant_fp4(x[:, :48].contiguous()[:, :40]),
        lambda: jo.quant_fp4(x.t()),
        lambda: jo.quant_fp4(x.to(torch.int32)),
        lambda: jo.quant_fp4(torch.zeros(4, 0, device=dev)),
        lambda: jo.dequant_fp4(w[0], w[1], None),
        lambda: jo.dequant_fp4(mx[0], mx[1], w[2]),
        lambda: jo.dequant_fp4(w[0], w[1][:, :, :16], w[2]),
        lambda: jo.fp4_scaled_mm(w[0], mx[0], w[1], mx[1], w[2], None, BF),
        lambda: jo.fp4_scaled_mm(w[0], w[0], w[1], w[1], w[2], w[2], F32),
        lambda: jo.fp4_scaled_mm(w[0], w[0][:4], w[1], w[1], w[2], w[2][:4], BF),
        lambda: jo.fp4_linear(x[:, :32], *w),
        lambda: jo.fp4_linear(x.float(), *w),
        lambda: jo.fp4_linear(x, *w, torch.zeros(8, device=dev)),
        lambda: jo.fp4_linear(x, *(t.cpu() for t in w)),
        lambda: jo.rotary_embed(q3, q3.float(), cos, sin, at),
        lambda: jo.rotary_embed(q3, None, cos, sin[:4], at),
        lambda: jo.rotary_embed(q3[..., :32], None, cos, sin, at),
        lambda: jo.rotary_embed(q3, None, cos, sin, at[:3]),
        lambda: jo.rotary_embed(q3, None, cos, sin, at.float()),
        lambda: jo.rotary_embed(torch.zeros(4, 2, 512, device=dev, dtype=BF), None, cos, sin, at),
        lambda: jo.rotary_embed_append(q3, q3, q3, cos, sin, at, at.int(), q3, q3),
        lambda: jo.rotary_embed_append(q3, q3, q3, cos, sin, at, at, q3[:, :1], q3[:, :1]),
        lambda: jo.shared_prefix_attention(q[:, :, :3], kp, vp, ko, vo, lens),
        lambda: jo.shared_prefix_attention(q[..., :32], kp[..., :32], vp[..., :32], ko[..., :32], vo[..., :32], lens),
        lambda: jo.shared_prefix_attention(q, kp, vp, ko, vo, lens.long()),
        lambda: jo.shared_prefix_attention(q, kp, vp.half(), ko, vo, lens),
        lambda: jo.shared_prefix_attention(q.float(), kp.float(), vp.float(), ko.float(), vo.float(), lens),
        lambda: jo.shared_prefix_attention(q, kp, vp, ko, vo, lens, True, 0.0),
        lambda: jo.shared_prefix_attention(q, kp, vp, ko, vo, lens, True, math.nan),
        lambda: jo.shared_prefix_attention(q, kp.cpu(), vp, ko, vo, lens),
        lambda: jo.shared_prefix_attention(q, torch.zeros(16, 2, 68, device=dev, dtype=BF)[..., :64], vp, ko, vo, lens),
    ]
    for i, call in enumerate(cases):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()
            pytest.fail(f"case {i} was accepted")
    torch.cuda.synchronize()


def test_c_abi_refusals(dev):
    from joyomni_ops import cabi

    t = torch.zeros(1 << 16, device=dev, dtype=torch.uint8)
    p, s = t.data_ptr(), cabi.stream()
    mm = lambda **o: cabi.status_of("jo_fp4_scaled_mm", *{**dict(
        d=p, ldd=64, a=p, lda=32, b=p, ldb=32, ba=p, bb=p, sa=None, sb=None, bias=None, m=4, n=64, k=64, f=0, dt=cabi.JO_BF16,
        st=s), **o}.values())
    assert mm(f=2) == cabi.JO_ERR_INVALID and mm(a=None) == cabi.JO_ERR_INVALID and mm(k=48) == cabi.JO_ERR_SHAPE
    assert mm(lda=40) == cabi.JO_ERR_ALIGN and mm(b=p + 8) == cabi.JO_ERR_ALIGN and mm(ldd=60) == cabi.JO_ERR_SHAPE
    assert mm(dt=cabi.JO_F32) == cabi.JO_ERR_DTYPE and mm(m=-1) == cabi.JO_ERR_SHAPE and mm(m=0) == cabi.JO_OK
    assert cabi.status_of("jo_quant_fp4", p, 32, p, None, p, 64, 4, 64, 0, cabi.JO_BF16, s) == cabi.JO_ERR_INVALID
    assert cabi.status_of("jo_quant_fp4", p, 32, p, p, p + 1, 64, 4, 64, 0, cabi.JO_BF16, s) == cabi.JO_ERR_ALIGN
    assert cabi.status_of("jo_quant_fp4", p, 32, p, p, p, 63, 4, 64, 0, cabi.JO_BF16, s) == cabi.JO_ERR_SHAPE
    assert cabi.lib().jo_fp4_scale_bytes(129, 96, 0) == 2 * 2 * 512 and cabi.lib().jo_fp4_scale_bytes(1, 32, 7) == -1
    assert cabi.lib().jo_shared_prefix_attention_workspace(1, 1, 3, 2, 64, 10, 10) == -1
    assert cabi.last_error()


def test_no_faults_recorded(dev):
    from joyomni_ops import cabi

    torch.cuda.synchronize()
    assert cabi.device_fault_count() == 0
