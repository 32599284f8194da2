"""Workloads of the 4-bit projections, the rotary embedding and the attention over a shared prefix.

The serving step these operators make up: a batch of requests (several edit prompts, or the guided and
the unguided branch of one) works on one long prefix that all of them share, such as the cached video
rows.  Its projections run in 4 bits (``quant_fp4``, ``fp4_scaled_mm``; ``dequant_fp4`` gives back what
the 4 bits stand for), its queries and keys are rotated (``rotary_embed`` in training and prefill,
``rotary_embed_append`` into the requests' own cache rows) and its queries attend over the shared prefix
and their own rows (``shared_prefix_attention``).

``run`` computes a case with plain torch operations in 32 bits, or, where ``own`` is true, by the calls a
user makes; ``exact`` computes it from the definitions in 64 bits.

Definitions
  4-bit rows, "nvfp4": x [M, K] in blocks of 16 along K.  r[m] = max(max|x[m, :]|, 1e-8) / 2688 in fp32,
    s[m, b] = e4m3((max|x[m, b, :]| / r[m]) / 6), code = e2m1(x / (s * r)) (0 where s is 0), each division
    and the product in fp32, every conversion to the nearest, ties to even.  Value: code * s * r.
  4-bit rows, "mxfp4": blocks of 32, s[m, b] = 2^clamp(floor(log2 max|x[m, b, :]|) - 2, -127, 127)
    (-127 for a zero block), code = e2m1(x / s), saturating at 6.  Value: code * s.
  packed: element 2i of a row in the low half of byte i, element 2i+1 in the high half.
  block scales: tiles of 128 rows x 4 blocks, [ceil(M/128), ceil(blocks/4), 32, 4, 4], where row m of a
    tile and block b of it sit at [m % 32, m // 32, b]; zero where there is no row or block.
  product: D[m, n] = (sum_k A[m, k] B[n, k]) * r_B[n] * r_A[m] (+ bias[n]), A and B being code * s.
  rotation: pairs (x0, x1) of the first R elements of a head become (x0 c - x1 s, x0 s + x1 c); a pair is
    (2i, 2i+1) where interleaved and (i, i + R/2) where not; the other elements stay.
  attention: query i of a request's Lq sees every prefix row and, of the request's len own rows, all of
    them or, causal, those up to len - Lq + i; a query that sees nothing gives 0 and -inf.
"""
import math
import os
import sys

import torch

own = False

_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "joyai-video-edit_b200")
_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BLOCK = {"nvfp4": 16, "mxfp4": 32}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _package():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    import joyomni_ops

    return joyomni_ops


# ------------------------------------------------------------------ cases
def listed():
    return [
        # the activations of one streamed chunk (3 x 45 x 80 tokens, 24 heads of 128) in front of a projection
        {"name": "quant_chunk", "kind": "quant", "fmt": "nvfp4", "dtype": "bf16", "M": 10800, "K": 3072},
        # the text rows of one of eight ranks in front of the MLP's down projection: a launch, hardly any bytes
        {"name": "quant_text_rows", "kind": "quant", "fmt": "mxfp4", "dtype": "f16", "M": 64, "K": 12288},
        # the chunk's QKV projection: the largest product
        {"name": "product_qkv", "kind": "product", "fmt": "nvfp4", "out": "bf16", "bias": False, "M": 10800, "N": 9216, "K": 3072},
        # the MLP's down projection on one of eight ranks: a ragged number of rows, long sums, a bias
        {"name": "product_down_rank", "kind": "product", "fmt": "mxfp4", "out": "f16", "bias": True, "M": 1350, "N": 3072, "K": 12288},
        # a layer applied to a single token: the weights are all there is to read
        {"name": "linear_token", "kind": "linear", "fmt": "nvfp4", "dtype": "bf16", "bias": True, "M": 1, "N": 9216, "K": 3072},
        # a training step of the chunk: rotation of q and k and its gradient, interleaved pairs, whole heads
        {"name": "rotary_train_chunk", "kind": "rotary", "dtype": "bf16", "T": 10800, "Hq": 24, "Hk": 24, "D": 128, "R": 128, "P": 16384, "interleaved": True, "stretch": 1.0},
        # a long context with shared key heads: half layout, half of each head rotated, positions stretched
        {"name": "rotary_long_partial", "kind": "rotary", "dtype": "f16", "T": 4099, "Hq": 32, "Hk": 8, "D": 128, "R": 64, "P": 131072, "interleaved": False, "stretch": 8.0},
        # one new token of each of 32 requests: rotate, put keys and values into their cache rows
        {"name": "append_tokens", "kind": "append", "dtype": "bf16", "T": 32, "Hq": 32, "Hk": 8, "D": 128, "R": 128, "P": 16384, "rows": 4096, "interleaved": False},
        # the rows of a text prompt for several requests at once, some of them padding
        {"name": "append_prompts", "kind": "append", "dtype": "f16", "T": 2043, "Hq": 24, "Hk": 24, "D": 128, "R": 96, "P": 16384, "rows": 8192, "interleaved": True},
        # one token of one request after a short prefix: latency
        {"name": "attend_token", "kind": "attend", "dtype": "f16", "B": 1, "Lq": 1, "Hk": 2, "G": 4, "D": 64, "P": 777, "S": 33, "causal": True},
        # a token for each of 32 requests that share a chunk of cached rows: the prefix is read once for all
        {"name": "attend_batch", "kind": "attend", "dtype": "bf16", "B": 32, "Lq": 1, "Hk": 8, "G": 4, "D": 128, "P": 10800, "S": 512, "causal": True},
        # the guided and the unguided branch over the same four cached chunks, a quarter of a frame each
        {"name": "attend_branches", "kind": "attend", "dtype": "bf16", "B": 2, "Lq": 900, "Hk": 24, "G": 1, "D": 128, "P": 43200, "S": 900, "causal": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _most(kind):
    return max(_cost(c) for c in listed() if c["kind"] == kind)


def _cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50)


def _drawn(rng):
    kind = rng.choice(("quant", "product", "linear", "rotary", "append", "attend", "attend"))
    half = rng.choice(("bf16", "f16"))
    if kind in ("quant", "product", "linear"):
        c = {"kind": kind, "fmt": rng.choice(("nvfp4", "mxfp4"))}
        k = 32 * _log(rng, 2, 384)
        if kind == "quant":
            return {**c, "dtype": rng.choice(("bf16", "f16", "f32")), "M": _log(rng, 1, 10800), "K": k}
        if kind == "product":
            return {**c, "out": half, "bias": rng.random() < 0.5, "M": _log(rng, 1, 10800), "N": 8 * _log(rng, 8, 1536), "K": k}
        return {**c, "dtype": half, "bias": rng.random() < 0.5, "M": _log(rng, 1, 512), "N": 8 * _log(rng, 8, 1536), "K": k}
    if kind in ("rotary", "append"):
        d = rng.choice((64, 128, 256))
        hk = rng.choice((1, 2, 4, 8, 24))
        r = rng.choice((d, d, d // 2, 3 * d // 4))
        c = {"kind": kind, "dtype": half, "T": _log(rng, 1, 10800 if kind == "rotary" else 4096)}
        c = {**c, "Hq": hk * rng.choice((1, 2, 3, 4)), "Hk": hk, "D": d, "R": r, "P": rng.choice((16384, 131072))}
        c["interleaved"] = rng.random() < 0.5
        if kind == "rotary":
            return {**c, "stretch": rng.choice((1.0, 4.0, 8.0))}
        return {**c, "rows": max(4096, c["T"] + rng.randrange(4096))}
    c = {"kind": "attend", "dtype": half, "B": _log(rng, 1, 64), "Lq": _log(rng, 1, 900), "Hk": rng.choice((1, 2, 4, 8, 24))}
    c = {**c, "G": rng.choice((1, 2, 3, 4, 6, 8)), "D": rng.choice((64, 128)), "P": _log(rng, 1, 43200)}
    return {**c, "S": _log(rng, 1, 2048), "causal": rng.random() < 0.5}


def draw(rng):
    while True:
        c = _drawn(rng)
        kind = "product" if c["kind"] == "linear" else c["kind"]
        if _cost(c) <= _most(kind) and (kind != "attend" or _scores(c) <= _scores(listed()[-1])):
            return c


def _scores(c):
    return c["B"] * c["Lq"] * c["Hk"] * c["G"] * (c["P"] + c["S"])


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return {**case, **_INPUTS[case["kind"]](case, g)}


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _activations(g, m, k, dtype):
    """Rows of differing size with a few channels that stand out, as in front of a projection."""
    x = _normal(g, m, k) * torch.exp(0.5 * _normal(g, m, 1))
    return (x * (1 + 15 * (torch.rand(k, generator=g, device="cuda") < 0.01))).to(dtype)


def _packed(g, rows, k, fmt):
    """A matrix held in 4 bits: packed codes, block scales in tiles, row scales (None for mxfp4)."""
    w = _normal(g, rows, k) / math.sqrt(k)
    codes, scale, row = _quantise(w, fmt)
    index = torch.searchsorted(torch.tensor(_E2M1, device="cuda"), codes.abs()).to(torch.uint8)
    index = index + 8 * torch.signbit(codes).to(torch.uint8)
    return index[:, 0::2] | (index[:, 1::2] << 4), _tiled(scale, fmt), row


def _tiled(scale, fmt):
    m, b = scale.shape
    t = scale.new_zeros(-(-m // 128) * 128, -(-b // 4) * 4)
    t[:m, :b] = scale
    t = t.view(-(-m // 128), 4, 32, -(-b // 4), 4).permute(0, 3, 2, 1, 4).contiguous()
    if fmt == "nvfp4":
        return t.to(torch.float8_e4m3fn)
    return torch.where(t > 0, torch.frexp(t).exponent - 1 + 127, 0).to(torch.uint8).view(torch.float8_e8m0fnu)


def _in_quant(c, g):
    return {"x": _activations(g, c["M"], c["K"], _DT[c["dtype"]])}


def _in_product(c, g):
    s = {"a": _packed(g, c["M"], c["K"], c["fmt"]), "b": _packed(g, c["N"], c["K"], c["fmt"])}
    s["add"] = _normal(g, c["N"]).to(_DT[c["out"]]) if c["bias"] else None
    return s


def _in_linear(c, g):
    s = {"x": _activations(g, c["M"], c["K"], _DT[c["dtype"]]), "b": _packed(g, c["N"], c["K"], c["fmt"])}
    s["add"] = _normal(g, c["N"]).to(_DT[c["dtype"]]) if c["bias"] else None
    return s


def _tables(c):
    freq = 10000.0 ** (-torch.arange(0, c["R"], 2, device="cuda", dtype=torch.float64) / c["R"])
    angle = torch.arange(c["P"], device="cuda", dtype=torch.float64)[:, None] / c.get("stretch", 1.0) * freq
    return {"cos": angle.cos().float(), "sin": angle.sin().float()}


def _in_rotary(c, g):
    dt, t, d = _DT[c["dtype"]], c["T"], c["D"]
    s = {"q": _normal(g, t, c["Hq"], d).to(dt), "k": _normal(g, t, c["Hk"], d).to(dt), **_tables(c)}
    s["dq"], s["dk"] = _normal(g, t, c["Hq"], d).to(dt), _normal(g, t, c["Hk"], d).to(dt)
    first = int(torch.randint(0, max(1, c["P"] - t), (1,), generator=g, device="cuda"))
    s["at"] = (torch.arange(t, device="cuda") + first) % c["P"]
    return s


def _in_append(c, g):
    dt, t, d = _DT[c["dtype"]], c["T"], c["D"]
    s = {"q": _normal(g, t, c["Hq"], d).to(dt), "k": _normal(g, t, c["Hk"], d).to(dt), **_tables(c)}
    s["v"] = _normal(g, t, c["Hk"], d).to(dt)
    s["k_cache"], s["v_cache"] = (_normal(g, c["rows"], c["Hk"], d).to(dt) for _ in range(2))
    s["at"] = torch.randint(0, c["P"], (t,), generator=g, device="cuda")
    slot = torch.randperm(c["rows"], generator=g, device="cuda")[:t]
    padding = torch.rand(t, generator=g, device="cuda") < (0.1 if t > 64 else 0.0)
    s["slot"] = torch.where(padding, -1, slot)
    return s


def _in_attend(c, g):
    dt, h, d = _DT[c["dtype"]], c["Hk"], c["D"]
    s = {"q": _normal(g, c["B"], c["Lq"], h * c["G"], d).to(dt)}
    for name in ("k", "v"):
        s[name + "_prefix"] = _normal(g, c["P"], h, d).to(dt)
        s[name + "_own"] = _normal(g, c["B"], c["S"], h, d).to(dt)
    lens = torch.randint(1, c["S"] + 1, (c["B"],), generator=g, device="cuda", dtype=torch.int32)
    lens[0] = c["S"]
    free = torch.arange(c["S"], device="cuda") >= lens[:, None]
    for name in ("k_own", "v_own"):  # cache rows that no request has written yet hold anything
        s[name].masked_fill_(free[:, :, None, None], math.nan)
    s["lens"] = lens
    return s


_INPUTS = {
    "quant": _in_quant,
    "product": _in_product,
    "linear": _in_linear,
    "rotary": _in_rotary,
    "append": _in_append,
    "attend": _in_attend,
}


# ------------------------------------------------------------------ plain forms
def run(state):
    return (_OWN if own else _PLAIN)[state["kind"]](state)


def _e2m1(y):
    """The nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with the sign of y, ties to the even code, saturating."""
    a = y.abs().clamp(max=6.0)
    v = torch.where(a < 2, torch.round(a * 2) * 0.5, torch.where(a < 4, torch.round(a), torch.round(a * 0.5) * 2))
    return torch.copysign(v, y)


def _quantise(x, fmt):
    """Codes' values [M, K], block scales [M, K / block] and row scales [M, 1] (None for mxfp4), in fp32."""
    m, k = x.shape
    x = x.float().view(m, -1, _BLOCK[fmt])
    top = x.abs().amax(2)
    if fmt == "nvfp4":
        most, six = torch.tensor([2688.0, 6.0], device="cuda")  # on the GPU: a number's division is a multiplication
        row = top.amax(1, keepdim=True).clamp(min=1e-8) / most
        scale = (top / row / six).to(torch.float8_e4m3fn).float()
        step = (scale * row)[:, :, None]
        codes = torch.where(scale[:, :, None] > 0, _e2m1(x / step), torch.copysign(torch.zeros_like(x), x))
    else:
        row = None
        power = torch.where(top > 0, torch.frexp(top).exponent - 3, -127).clamp(-127, 127)
        scale = torch.where(power > -127, (power + 127) << 23, 1 << 22).view(torch.float32)  # 2^power, bit by bit
        codes = _e2m1(x / scale[:, :, None])
    return codes.view(m, k), scale, row


def _values(codes, scale, fmt):
    return (codes.view(*scale.shape, _BLOCK[fmt]) * scale[:, :, None]).view(codes.shape)


def _unpacked(packed, tiles, fmt):
    """code * block scale [rows, K] in fp32 of a matrix held in 4 bits."""
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device="cuda")
    rows, k = packed.shape[0], 2 * packed.shape[1]
    codes = table[torch.stack((packed & 15, packed >> 4), 2).int()].view(rows, k)
    a, b = tiles.shape[:2]
    scale = tiles.float().permute(0, 3, 2, 1, 4).reshape(a * 128, b * 4)[:rows, : k // _BLOCK[fmt]]
    return _values(codes, scale, fmt)


def _product(a, ra, b, rb, add, dtype):
    d = a @ b.t()
    if rb is not None:
        d = d * rb.view(1, -1) * ra
    return (d if add is None else d + add.float()).to(dtype)


def _plain_quant(s):
    codes, scale, row = _quantise(s["x"], s["fmt"])
    v = _values(codes, scale, s["fmt"])
    return {"values": (v if row is None else v * row).to(s["x"].dtype)}


def _plain_product(s):
    (a, sa, ra), (b, sb, rb) = s["a"], s["b"]
    return _product(_unpacked(a, sa, s["fmt"]), ra, _unpacked(b, sb, s["fmt"]), rb, s["add"], _DT[s["out"]])


def _plain_linear(s):
    codes, scale, row = _quantise(s["x"], s["fmt"])
    b, sb, rb = s["b"]
    return _product(_values(codes, scale, s["fmt"]), row, _unpacked(b, sb, s["fmt"]), rb, s["add"], s["x"].dtype)


def _rotate(x, cos, sin, interleaved):
    r = 2 * cos.shape[-1]
    y = x.float().clone()
    if interleaved:
        x0, x1 = x[..., 0:r:2].float(), x[..., 1:r:2].float()
        y[..., 0:r:2], y[..., 1:r:2] = x0 * cos - x1 * sin, x0 * sin + x1 * cos
    else:
        x0, x1 = x[..., : r // 2].float(), x[..., r // 2 : r].float()
        y[..., : r // 2], y[..., r // 2 : r] = x0 * cos - x1 * sin, x0 * sin + x1 * cos
    return y.to(x.dtype)


def _plain_rotary(s):
    cos, sin, pairs = s["cos"][s["at"]][:, None], s["sin"][s["at"]][:, None], s["interleaved"]
    return {"q": _rotate(s["q"], cos, sin, pairs), "k": _rotate(s["k"], cos, sin, pairs),
            "dq": _rotate(s["dq"], cos, -sin, pairs), "dk": _rotate(s["dk"], cos, -sin, pairs)}


def _plain_append(s):
    cos, sin, pairs = s["cos"][s["at"]][:, None], s["sin"][s["at"]][:, None], s["interleaved"]
    used = s["slot"] >= 0
    rows = s["slot"][used]
    s["k_cache"][rows] = _rotate(s["k"], cos, sin, pairs)[used]
    s["v_cache"][rows] = s["v"][used]
    return {"q": _rotate(s["q"], cos, sin, pairs), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attend(s):
    b, lq, h, g, d, p, n = (s[x] for x in ("B", "Lq", "Hk", "G", "D", "P", "S"))
    q = s["q"].float().view(b, lq, h, g, d)
    row, lens = torch.arange(n, device="cuda"), s["lens"].long()
    live = (row < lens[:, None])[:, :, None, None]
    k_own, v_own = (torch.where(live, s[x].float(), 0.0).transpose(1, 2) for x in ("k_own", "v_own"))  # [B, Hk, S, D]
    last = lens[:, None] - lq + torch.arange(lq, device="cuda") if s["causal"] else (lens - 1)[:, None].expand(b, lq)
    seen = row <= last[:, :, None]  # [B, Lq, S]
    from_prefix = q.permute(2, 0, 1, 3, 4).reshape(h, b * lq * g, d) @ s["k_prefix"].float().permute(1, 2, 0)
    from_prefix = from_prefix.view(h, b, lq * g, p)
    from_own = q.permute(0, 2, 1, 3, 4).reshape(b, h, lq * g, d) @ k_own.transpose(2, 3)
    from_own = from_own.view(b, h, lq, g, n).masked_fill(~seen[:, None, :, None], -math.inf).view(b, h, lq * g, n)
    score = torch.cat((from_prefix, from_own.transpose(0, 1)), 3).mul_(1 / math.sqrt(d))
    del from_prefix, from_own
    top = score.amax(3, keepdim=True)
    weight = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = weight.sum(3, keepdim=True)
    o = (weight[..., :p].reshape(h, b * lq * g, p) @ s["v_prefix"].float().transpose(0, 1)).view(h, b, lq * g, d)
    o = o + weight[..., p:] @ v_own.transpose(0, 1)
    o = torch.where(total > 0, o / total, 0.0).view(h, b, lq, g, d).permute(1, 2, 0, 3, 4).reshape(b, lq, h * g, d)
    lse = (top + total.log()).view(h, b, lq, g).permute(1, 0, 3, 2).reshape(b, h * g, lq)
    return {"out": o.to(s["q"].dtype), "lse": lse}


_PLAIN = {
    "quant": _plain_quant,
    "product": _plain_product,
    "linear": _plain_linear,
    "rotary": _plain_rotary,
    "append": _plain_append,
    "attend": _plain_attend,
}


# ------------------------------------------------------------------ the calls a user makes
def _own_quant(s):
    jo = _package()
    q, scale, row = jo.quant_fp4(s["x"], s["fmt"])
    return {"values": jo.dequant_fp4(q, scale, row, s["x"].dtype)}


def _own_product(s):
    (a, sa, ra), (b, sb, rb) = s["a"], s["b"]
    return _package().fp4_scaled_mm(a, b, sa, sb, ra, rb, _DT[s["out"]], s["add"])


def _own_linear(s):
    b, sb, rb = s["b"]
    return _package().fp4_linear(s["x"], b, sb, rb, s["add"])


def _own_rotary(s):
    jo = _package()
    q, k = jo.rotary_embed(s["q"], s["k"], s["cos"], s["sin"], s["at"], s["interleaved"])
    dq, dk = jo.rotary_embed_backward(s["dq"], s["dk"], s["cos"], s["sin"], s["at"], s["interleaved"])
    return {"q": q, "k": k, "dq": dq, "dk": dk}


def _own_append(s):
    cache = s["k_cache"], s["v_cache"]
    q = _package().rotary_embed_append(
        s["q"], s["k"], s["v"], s["cos"], s["sin"], s["at"], s["slot"], *cache, s["interleaved"])
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_attend(s):
    o, lse = _package().shared_prefix_attention(
        s["q"], s["k_prefix"], s["v_prefix"], s["k_own"], s["v_own"], s["lens"], s["causal"])
    return {"out": o, "lse": lse}


_OWN = {
    "quant": _own_quant,
    "product": _own_product,
    "linear": _own_linear,
    "rotary": _own_rotary,
    "append": _own_append,
    "attend": _own_attend,
}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    if c["kind"] == "quant":
        n = c["M"] * c["K"] * (4 if c["dtype"] == "f32" else 2)
        return {"bytes": 2 * n, "flops": 2 * c["M"] * c["K"]}
    if c["kind"] in ("product", "linear"):
        bits = c["K"] * (0.5 + 1 / _BLOCK[c["fmt"]]) + (4 if c["fmt"] == "nvfp4" else 0)
        a = c["M"] * (bits if c["kind"] == "product" else 2 * c["K"])
        written = 2 * c["M"] * c["N"]
        return {"bytes": a + c["N"] * (bits + 2 * c["bias"]) + written, "flops": written * c["K"]}
    if c["kind"] == "rotary":
        rows = 2 * c["T"] * (c["Hq"] + c["Hk"]) * c["D"]
        return {"bytes": 4 * rows + c["T"] * (8 + 4 * c["R"]), "flops": 6 * c["T"] * (c["Hq"] + c["Hk"]) * c["R"]}
    if c["kind"] == "append":
        rows = 2 * c["T"] * (c["Hq"] + 2 * c["Hk"]) * c["D"]
        return {"bytes": 2 * rows + c["T"] * (16 + 4 * c["R"]), "flops": 3 * c["T"] * (c["Hq"] + c["Hk"]) * c["R"]}
    q = c["B"] * c["Lq"] * c["Hk"] * c["G"]
    seen = c["P"] + (c["S"] + 1) / 2  # lengths are spread evenly
    if c["causal"] and c["Lq"] < c["S"]:
        seen -= (c["Lq"] - 1) / 2
    kv = 4 * c["Hk"] * c["D"] * (c["P"] + c["B"] * (c["S"] + 1) / 2)
    return {"bytes": kv + 4 * q * c["D"] + 4 * q, "flops": 4 * q * c["D"] * max(c["P"], seen)}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    return _EXACT[case["kind"]](prepare(case, seed))


def _exact_codes(ratio):
    """e2m1 of a ratio by the midpoints between neighbours; at a midpoint the even code of the two."""
    a = ratio.abs()
    v = torch.zeros_like(a)
    for code in range(1, 8):
        middle = (_E2M1[code - 1] + _E2M1[code]) / 2
        up = a >= middle if code % 2 == 0 else a > middle
        v = torch.where(up, _E2M1[code], v)
    return torch.where(ratio < 0, -v, v)


def _exact_rows(x, fmt):
    """code * block scale and row scale in 64 bits; scales have the width in which they are held."""
    m, k = x.shape
    blocks = x.double().reshape(m, k // _BLOCK[fmt], _BLOCK[fmt])
    top = blocks.abs().max(2).values
    if fmt == "mxfp4":
        mantissa, _ = torch.frexp(top)
        scale = torch.where(top > 0, top / mantissa / 8, 0).clamp(min=2.0**-127)
        return (_exact_codes(blocks / scale[..., None]) * scale[..., None]).reshape(m, k), None
    most, six = torch.tensor([2688, 6], dtype=torch.float64, device="cuda")
    row = (torch.maximum(top.max(1).values, torch.full_like(top[:, 0], 1e-8).float().double()) / most).float().double()
    ratio = ((top / row[:, None]).float().double() / six).float()
    scale = ratio.to(torch.float8_e4m3fn).double()
    step = (scale * row[:, None]).float().double()
    codes = _exact_codes(torch.where(step[..., None] > 0, (blocks / step[..., None]).float().double(), 0.0))
    return (codes * scale[..., None]).reshape(m, k), row


def _exact_held(packed, tiles, fmt):
    rows, bytes_ = packed.shape
    nibble = torch.empty(rows, 2 * bytes_, dtype=torch.long, device="cuda")
    nibble[:, 0::2], nibble[:, 1::2] = (packed % 16).long(), (packed // 16).long()
    size = torch.tensor(_E2M1, dtype=torch.float64, device="cuda")[nibble % 8]
    m, b = torch.arange(rows, device="cuda")[:, None], torch.arange(2 * bytes_ // _BLOCK[fmt], device="cuda")[None]
    raw = tiles.view(torch.uint8)[m // 128, b // 4, m % 32, m % 128 // 32, b % 4]
    scale = raw.view(torch.float8_e4m3fn).double() if fmt == "nvfp4" else 2.0 ** (raw.double() - 127)
    return torch.where(nibble >= 8, -size, size) * scale.repeat_interleave(_BLOCK[fmt], 1)


def _exact_product(a, ra, b, rb, add):
    d = torch.matmul(a, b.transpose(0, 1))
    if ra is not None:
        d = d * ra.double().reshape(-1, 1) * rb.double().reshape(1, -1)
    return d if add is None else d + add.double()


def _exact_quant(s):
    v, row = _exact_rows(s["x"], s["fmt"])
    return {"values": v if row is None else v * row[:, None]}


def _exact_mm(s):
    (a, sa, ra), (b, sb, rb) = s["a"], s["b"]
    return _exact_product(_exact_held(a, sa, s["fmt"]), ra, _exact_held(b, sb, s["fmt"]), rb, s["add"])


def _exact_linear(s):
    a, ra = _exact_rows(s["x"], s["fmt"])
    b, sb, rb = s["b"]
    return _exact_product(a, ra, _exact_held(b, sb, s["fmt"]), rb, s["add"])


def _exact_turn(x, s, sign):
    """x * e^(i sign angle) on the complex numbers that the pairs are."""
    half = s["R"] // 2
    turn = torch.complex(s["cos"].double(), sign * s["sin"].double())[s["at"]].unsqueeze(1)
    part = x[..., : s["R"]].double()
    pairs = part.unflatten(-1, (half, 2)) if s["interleaved"] else part.unflatten(-1, (2, half)).transpose(-1, -2)
    out = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    out = out if s["interleaved"] else out.transpose(-1, -2)
    return torch.cat((out.flatten(-2), x[..., s["R"] :].double()), -1)


def _exact_rotary(s):
    turned = {x: _exact_turn(s[x], s, 1) for x in ("q", "k")}
    return {**turned, **{x: _exact_turn(s[x], s, -1) for x in ("dq", "dk")}}


def _exact_append(s):
    k_cache, v_cache, k = s["k_cache"].double(), s["v_cache"].double(), _exact_turn(s["k"], s, 1)
    t = torch.nonzero(s["slot"] >= 0).squeeze(1)
    k_cache.index_copy_(0, s["slot"][t], k[t])
    v_cache.index_copy_(0, s["slot"][t], s["v"][t].double())
    return {"q": _exact_turn(s["q"], s, 1), "k_cache": k_cache, "v_cache": v_cache}


def _exact_attend(s):
    """Request by request and key head by key head, over the rows that are there."""
    b, lq, h, g, d = (s[x] for x in ("B", "Lq", "Hk", "G", "D"))
    out = torch.zeros(b, lq, h * g, d, dtype=torch.float64, device="cuda")
    lse = torch.full((b, h * g, lq), -math.inf, dtype=torch.float64, device="cuda")
    lens = s["lens"].tolist()
    for j in range(h):
        pk, pv = s["k_prefix"][:, j].double(), s["v_prefix"][:, j].double()
        for r in range(b):
            k = torch.cat((pk, s["k_own"][r, : lens[r], j].double()))
            v = torch.cat((pv, s["v_own"][r, : lens[r], j].double()))
            x = torch.einsum("igd,nd->gin", s["q"][r, :, j * g : (j + 1) * g].double(), k) * d**-0.5
            if s["causal"]:
                n, i = torch.arange(k.shape[0], device="cuda"), torch.arange(lq, device="cuda")[:, None]
                x = torch.where((n < s["P"]) | (n - s["P"] <= lens[r] - lq + i), x, -math.inf)
            one = torch.logsumexp(x, 2)
            w = torch.where(torch.isfinite(one)[..., None], torch.exp(x - one[..., None]), 0.0)
            out[r, :, j * g : (j + 1) * g] = torch.einsum("gin,nd->igd", w, v)
            lse[r, j * g : (j + 1) * g] = one
    return {"out": out, "lse": lse}


_EXACT = {
    "quant": _exact_quant,
    "product": _exact_mm,
    "linear": _exact_linear,
    "rotary": _exact_rotary,
    "append": _exact_append,
    "attend": _exact_attend,
}
