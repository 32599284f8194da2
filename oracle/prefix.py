"""Restatement in 64 bits of the operators of an attention layer whose requests share a long prefix.

4-bit rows and their product, the rotary embedding and attention over a shared prefix, each written from
its definition (``include/joyomni_b200.h``) with torch operations on whatever device the inputs are.  Where
the definition itself rounds (scales that are held in 32 or 8 bits, quotients in fp32), so does this.
Test infrastructure only.
"""
from __future__ import annotations

import math

import torch

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BLOCK = {"nvfp4": 16, "mxfp4": 32}


def power_of_two(e: torch.Tensor) -> torch.Tensor:
    """2^e for integers -127..128, exactly (a GPU's pow is not)."""
    table = torch.tensor([2.0 ** i for i in range(-127, 129)], dtype=torch.float64, device=e.device)
    return table[e.long() + 127]


def e2m1_codes(ratio: torch.Tensor) -> torch.Tensor:
    """Code (0..7, + 8 for negative non-zero values) of the nearest e2m1 value, ties to the even code."""
    a = ratio.abs()
    code = torch.zeros(ratio.shape, dtype=torch.uint8, device=ratio.device)
    for c in range(1, 8):
        middle = (E2M1[c - 1] + E2M1[c]) / 2
        code[(a >= middle) if c % 2 == 0 else (a > middle)] = c
    return code + 8 * ((ratio < 0) & (code > 0)).to(torch.uint8)


def quotient32(x: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
    """RN32(x / y) of fp32 values held in 64 bits (the 53-bit quotient rounds to 24 bits as the exact one:
    a quotient of 24-bit numbers is no nearer than 2^-49 to a midpoint between them unless it is one)."""
    return (x / y).float().double()


def fp4_quantise(x: torch.Tensor, fmt: str):
    """(codes uint8 [M, K], block scale bytes uint8 [M, K / block], row scales fp32 [M] or None)."""
    m, k = x.shape
    b = x.double().view(m, -1, BLOCK[fmt])
    top = b.abs().amax(2)
    bad = ~torch.isfinite(b).all(2)
    if fmt == "mxfp4":
        power = torch.where(top > 0, torch.frexp(top.nan_to_num(posinf=1.0))[1] - 3, -127).clamp(-127, 127)
        step = power_of_two(power)
        codes = e2m1_codes((b / step[..., None]).clamp(-1e9, 1e9).nan_to_num(0.0))
        codes[bad] = 0
        return codes.view(m, k), torch.where(bad, 255, power + 127).to(torch.uint8), None
    bad_row = bad.any(1)
    row = quotient32(top.amax(1).nan_to_num(1.0, posinf=1.0).clamp(min=float(torch.tensor(1e-8))),
                     torch.tensor(2688.0, dtype=torch.float64, device=x.device))
    six = torch.tensor(6.0, dtype=torch.float64, device=x.device)
    scale = quotient32(quotient32(top.nan_to_num(0.0, posinf=0.0), row[:, None]), six).float().to(torch.float8_e4m3fn)
    step = (scale.double() * row[:, None]).float().double()
    codes = e2m1_codes(torch.where(step[..., None] > 0, quotient32(b.nan_to_num(0.0, 0.0, 0.0), step[..., None]), 0.0))
    codes[scale.double() == 0] = 0
    codes[bad_row] = 0
    scale = torch.where(bad_row[:, None], 0, scale.view(torch.uint8))
    return codes.view(m, k), scale, torch.where(bad_row, math.nan, row).float()


def fp4_pack(codes: torch.Tensor) -> torch.Tensor:
    return codes[:, 0::2] | (codes[:, 1::2] << 4)


def fp4_tiles(scale: torch.Tensor) -> torch.Tensor:
    """Scale bytes [M, blocks] as tiles [ceil(M/128), ceil(blocks/4), 32, 4, 4], zero where there is none."""
    m, b = scale.shape
    t = scale.new_zeros((m + 127) // 128 * 128, (b + 3) // 4 * 4)
    t[:m, :b] = scale
    return t.view(-1, 4, 32, t.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).contiguous()


def fp4_untile(tiles: torch.Tensor, rows: int, blocks: int) -> torch.Tensor:
    t = tiles.permute(0, 3, 2, 1, 4).reshape(tiles.shape[0] * 128, tiles.shape[1] * 4)
    return t[:rows, :blocks]


def fp4_scale_values(scale: torch.Tensor, fmt: str) -> torch.Tensor:
    if fmt == "nvfp4":
        return scale.view(torch.float8_e4m3fn).double()
    return torch.where(scale == 255, math.nan, power_of_two(scale.long() - 127))


def fp4_values(codes: torch.Tensor, scale: torch.Tensor, fmt: str) -> torch.Tensor:
    """code * block scale [M, K] in 64 bits."""
    size = torch.tensor(E2M1, dtype=torch.float64, device=codes.device)[(codes & 7).long()]
    v = torch.where(codes >= 8, -size, size)
    return v * fp4_scale_values(scale, fmt).repeat_interleave(BLOCK[fmt], 1)


def fp4_product(a: torch.Tensor, row_a, b: torch.Tensor, row_b, bias=None) -> torch.Tensor:
    """a [M, K], b [N, K]: fp4_values; row scales or None."""
    d = a @ b.t()
    if row_b is not None:
        d = d * row_b.double().view(1, -1)
    if row_a is not None:
        d = d * row_a.double().view(-1, 1)
    return d if bias is None else d + bias.double()


def rotary(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, interleaved: bool,
           inverse: bool = False) -> torch.Tensor:
    """Rotation of x [T, H, D] in 64 bits."""
    c, s = cos.double()[positions.long()][:, None], sin.double()[positions.long()][:, None]
    s = -s if inverse else s
    r = 2 * c.shape[-1]
    y = x.double().clone()
    first = slice(0, r, 2) if interleaved else slice(0, r // 2)
    second = slice(1, r, 2) if interleaved else slice(r // 2, r)
    x0, x1 = x[..., first].double(), x[..., second].double()
    y[..., first], y[..., second] = x0 * c - x1 * s, x0 * s + x1 * c
    return y


def shared_prefix_attention(q, k_prefix, v_prefix, k_own, v_own, lens, causal=True, scale=None):
    """(out [B, L, H, D], lse [B, H, L], mass [B, L, H, D]) in 64 bits, query by query; mass is the softmax
    average of |v|, which bounds what a relative error of the weights does to out."""
    b, n, h, d = q.shape
    hk = k_prefix.shape[1]
    g = h // hk
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(b, n, h, d, dtype=torch.float64, device=q.device)
    mass = torch.zeros_like(out)
    lse = torch.full((b, h, n), -math.inf, dtype=torch.float64, device=q.device)
    for r in range(b):
        length = min(max(int(lens[r]), 0), k_own.shape[1])
        for i in range(n):
            seen = length if not causal else min(length, max(0, length - n + i + 1))
            k = torch.cat((k_prefix, k_own[r, :seen])).double().repeat_interleave(g, 1)
            v = torch.cat((v_prefix, v_own[r, :seen])).double().repeat_interleave(g, 1)
            if k.shape[0] == 0:
                continue
            x = torch.einsum("hd,khd->hk", q[r, i].double(), k) * scale
            lse[r, :, i] = torch.logsumexp(x, 1)
            w = torch.softmax(x, 1)
            out[r, i] = torch.einsum("hk,khd->hd", w, v)
            mass[r, i] = torch.einsum("hk,khd->hd", w, v.abs())
    return out, lse, mass


def shared_prefix_attention_by_request(q, k_prefix, v_prefix, k_own, v_own, lens, causal=True, scale=None):
    """``shared_prefix_attention`` with a request's queries all at once, for sizes at which one by one takes too long."""
    b, n, h, d = q.shape
    hk, p = k_prefix.shape[1], k_prefix.shape[0]
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(b, n, hk, h // hk, d, dtype=torch.float64, device=q.device)
    mass = torch.zeros_like(out)
    lse = torch.full((b, hk, h // hk, n), -math.inf, dtype=torch.float64, device=q.device)
    i = torch.arange(n, device=q.device)[:, None]
    for r, length in enumerate(torch.as_tensor(lens).clamp(0, k_own.shape[1]).tolist()):
        k, v = (torch.cat((a, o[r, :length])).double() for a, o in ((k_prefix, k_own), (v_prefix, v_own)))
        if p + length == 0:
            continue
        x = torch.einsum("nhgd,khd->hgnk", q[r].double().view(n, hk, -1, d), k) * scale
        if causal:
            j = torch.arange(p + length, device=q.device) - p
            x = x.masked_fill((j >= 0) & (j > length - n + i), -math.inf)
        lse[r] = torch.logsumexp(x, 3)
        w = torch.exp(x - torch.where(torch.isneginf(lse[r]), 0.0, lse[r])[..., None])
        out[r], mass[r] = torch.einsum("hgnk,khd->nhgd", w, v), torch.einsum("hgnk,khd->nhgd", w, v.abs())
    return out.view(b, n, h, d), lse.view(b, h, n), mass.view(b, n, h, d)
