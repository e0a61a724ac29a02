"""GPU: how many bits the paged attention kernels keep, on inputs whose sums are
short or exact, so that the bounds are a few roundings and not a whole axis of
them.  u = 2^-24, half a step of float32."""

import math

import pytest
import torch

from test_gpu_paged import U, attend, make

pytestmark = pytest.mark.gpu


def fill(c, keys, values):
    """keys / values [N, hd] (the same in every sequence and kv head) into the pages."""
    ps = c["kp"].shape[1]
    c["kp"].zero_()
    c["vp"].zero_()
    for i, (a, b) in enumerate(zip(c["past"], c["new"])):
        at = torch.arange(a + b, device="cuda")
        page = c["table"][i][at // ps].long()
        c["kp"][page, at % ps] = keys[: a + b, None].to(c["kp"].dtype)
        c["vp"][page, at % ps] = values[: a + b, None].to(c["vp"].dtype)


def softmax64(c, scores, values):
    """Rows [T, H, hd] for scores [H, N] that do not depend on the token, and the weights behind them."""
    out, weights = [], []
    for a, b in zip(c["past"], c["new"]):
        for j in range(b):
            w = torch.softmax(scores[:, : a + j + 1].double(), -1)
            out.append(w @ values[: a + j + 1].double())
            weights.append(w)
    return torch.stack(out), weights


@pytest.mark.parametrize("outlier,kv", [(x, torch.float32) for x in (0.0, 1e3, -1e5, 1e20)] +
                         [(x, torch.float16) for x in (0.0, 1e3, 3e4, -1e5)])
@pytest.mark.parametrize("hd", [16, 64, 128])
@pytest.mark.parametrize("new", [1, 5])
def test_a_large_query_element_does_not_cost_the_others_their_bits(outlier, new, hd, kv):
    """One element of the query is far larger than the rest, and the keys are 0
    there.  A score is one product: its parts err by 4 u of it, the low part's
    product, the sum of the two, the scale and the exponent's subtraction by 2 u
    each: 12 u A.  FP16 pages: an element more than 2^17 below the largest errs
    by 2^-39 of the largest.  The values are unit vectors, so an output is one
    weight: 2 delta, the weight's parts 4 u, the sum of N <= hd weights and the
    quotient (N + 8) u."""
    n, H, N = 3, 8, hd
    c = make(n, H, 2, hd, 16, kv, [N - new] * n, [new] * n, seed=hd)
    g = torch.Generator().manual_seed(1)
    k1 = (torch.rand(N, generator=g) * 4 - 2).half().float()
    keys = torch.zeros(N, hd)
    keys[:, 1] = k1
    fill(c, keys.cuda(), torch.eye(N, hd).cuda())
    x = torch.linspace(1.1, 2.3, H)
    c["q"].zero_()
    c["q"][..., 0] = outlier
    c["q"][..., 1] = x.cuda()
    got = attend(c).double().cpu()
    scores = x.double()[:, None] * k1.double()[None] / math.sqrt(hd)
    want, _ = softmax64(c, scores, torch.eye(N, hd))
    A = float(scores.abs().max())
    delta = 12 * U * A
    if kv == torch.float16:
        delta += 2.0 ** -39 * abs(outlier) * 2 / math.sqrt(hd)
    err = ((got - want).abs() / want.clamp(min=1e-300)).masked_fill(want == 0, 0.0)
    assert not got[want == 0].any()
    assert float(err.max()) <= 2 * delta + (4 + N + 8) * U
