"""The forms of the shared-prefix layer's kernels that large cases take, at the smallest sizes that reach them, against
the definitions in 64 bits (oracle/prefix.py).  Bounds: as in test_prefix_gpu.py.
"""
import math

import pytest
import torch

from oracle import prefix as ref
from test_prefix_gpu import BF, F16, ROUND, inputs, spoil, within

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
