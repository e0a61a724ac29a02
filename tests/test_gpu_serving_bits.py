"""GPU: how many bits the paged attention kernels keep, on inputs whose sums are
short or exact, so that the bounds are a few roundings and not a whole axis of
them.  u = 2^-24, half a step of float32."""

import math

import pytest
import torch

from test_gpu_paged import U, attend, check, make

pytestmark = pytest.mark.gpu


def fill(c, keys, values):
    """keys / values [N, hd], those of a shared prefix first, into the pages of every sequence and kv head."""
    ps, P = c["kp"].shape[1], c["prefix"]
    c["kp"].zero_()
    c["vp"].zero_()
    parts = [(c["prefix_pages"], 0, P)] + [(row, P, a + b) for row, a, b in zip(c["table"], c["past"], c["new"])]
    for pages, first, count in parts:
        at = torch.arange(count, device="cuda")
        for pool, x in ((c["kp"], keys), (c["vp"], values)):
            pool[pages[at // ps].long(), at % ps] = x[first: first + count, None].to(pool.dtype)


def softmax64(c, scores, values):
    """Rows [T, H, hd] for scores [H, N] that do not depend on the token, and the weights behind them."""
    made, order = {}, []
    for a, b in zip(c["past"], c["new"]):
        for j in range(b):
            seen = c["prefix"] + a + j + 1
            if seen not in made:
                w = torch.softmax(scores[:, :seen].double(), -1)
                made[seen] = (w @ values[:seen].double(), w)
            order.append(seen)
    return torch.stack([made[s][0] for s in order]), [made[s][1] for s in order]


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


@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
@pytest.mark.parametrize("hd", [16, 64, 128])
@pytest.mark.parametrize("n,past,new,prefix", [(2, 4090, 1, 0), (1500, 200, 1, 0), (2, 4090, 5, 0), (2, 30, 1, 4000),
                                               (2, 30, 5, 4000)])
@pytest.mark.parametrize("above", [0, 6, 14, 17, 20, 22])
def test_many_small_weights_behind_a_sink(above, n, past, new, prefix, hd, kv):
    """The first key's weight is some 2^``above`` times those of the others, which are
    equal, and its value is 0: the output is what the small weights make of theirs.
    Relative to W = sum w |v|: 2 delta (as above); sums that a tensor core cuts, of up
    to 512 products before registers add them, 2 u each, and pieces of them, 1200 u;
    the sum of weights and the quotient, 300 u.  FP16 pages: a weight errs by 2^-37 of
    the largest."""
    H, N = 8, prefix + past + new
    c = make(n, H, 2, hd, 16, kv, [past] * n, [new] * n, seed=hd, prefix=prefix)
    g = torch.Generator().manual_seed(above)
    keys = torch.zeros(N, hd)
    keys[:, 1] = -0.3
    keys[0, 1] = above * math.log(2.0)
    keys = keys.half().float()
    values = torch.rand(N, hd, generator=g).half().float()
    values[0] = 0
    fill(c, keys.cuda(), values.cuda())
    c["q"].zero_()
    x = math.sqrt(hd) * torch.linspace(0.9, 1.0, H)
    c["q"][..., 1] = x.cuda()
    got = attend(c).double().cpu()
    scores = x.double()[:, None] * keys[None, :, 1].double() / math.sqrt(hd)
    want, weights = softmax64(c, scores, values)
    tols = {}
    for w in weights:
        if w.shape[1] not in tols:
            v = values[: w.shape[1]].abs().double()
            tols[w.shape[1]] = (2 * 12 * U * float(scores.abs().max()) + 1500 * U) * (w @ v)
            if kv == torch.float16:
                tols[w.shape[1]] += 2.0 ** -37 * w.amax(-1, keepdim=True) * v.sum(0)
    tol = torch.stack([tols[w.shape[1]] for w in weights])
    assert float(((got - want).abs() / tol).max()) <= 1.0


@pytest.mark.parametrize("new,prefix", [(1, 0), (40, 0), (1, 200), (40, 200)])
@pytest.mark.parametrize("hd", [16, 64, 128])
def test_large_float32_values_do_not_overflow(hd, new, prefix):
    """Values close to FP32's largest: every output is a mean of them, so it is finite."""
    c = make(3, 8, 2, hd, 16, torch.float32, [70, 3, 200], [new] * 3, seed=hd, prefix=prefix)
    c["vp"].clamp_(-1, 1).mul_(3.3e38)
    out = attend(c)
    assert bool(out.isfinite().all())
    check(c, out)


@pytest.mark.parametrize("hd", [16, 64, 128])
@pytest.mark.parametrize("value", [torch.finfo(torch.float32).min, 3.395e38, math.inf])
def test_a_later_value_of_any_size_stays_in_its_rows(value, hd):
    """Chunks over FP32 pages: rows that do not see a key do not meet its value, FP32's lowest among them."""
    c = make(2, 8, 2, hd, 16, torch.float32, [30, 0], [50, 20], seed=hd)
    want = attend(c)
    c["vp"][int(c["table"][0, 65 // 16]), 65 % 16] = value
    got = attend(c)
    assert torch.equal(got[:35], want[:35]) and torch.equal(got[50:], want[50:])
    if value == math.inf:
        assert not got[35:50].isfinite().any()
    else:
        c["q"] /= 64  # even weights: a mean with one such value
        got = attend(c)
        assert bool(got.isfinite().all())
        check(c, got)


@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
@pytest.mark.parametrize("H,KV,hd,ps", [(8, 4, 16, 16), (4, 4, 16, 8), (8, 2, 32, 2), (16, 2, 64, 16), (10, 2, 128, 32)])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_keys_that_are_not_finite(value, H, KV, hd, ps, kv):
    """Single tokens: an element of one kv head's keys that is not finite is no
    business of the other kv heads, and a score of -inf is a weight of 0."""
    lens = [5, 17, 64, 130, 400]
    c = make(len(lens), H, KV, hd, ps, kv, [x - 1 for x in lens], [1] * len(lens), seed=hd)
    struck = [(i, g, at) for i, x in enumerate(lens) for g, at in ((i % KV, x // 2), ((i + 1) % KV, x - 1))]
    for i, g, at in struck:
        c["kp"][int(c["table"][i, at // ps]), at % ps, g, (3 * i) % hd] = value
    got = attend(c).double()
    for i, x in enumerate(lens):
        page = c["table"][i, : -(-x // ps)].long()
        k, v = (pool[page].flatten(0, 1)[:x].double() for pool in (c["kp"], c["vp"]))
        q = c["q"][i].double().unflatten(0, (KV, H // KV))
        s = torch.einsum("grd,kgd->grk", q, k) / math.sqrt(hd)
        w = torch.softmax(s, -1)
        want = torch.einsum("grk,kgd->grd", w, v).flatten(0, 1)
        W = torch.einsum("grk,kgd->grd", w, v.abs()).flatten(0, 1)
        A = torch.einsum("grd,kgd->grk", q.abs(), torch.where(k.isfinite(), k.abs(), 0)).amax(-1).flatten() / math.sqrt(hd)
        tol = (2 * (hd + 16) * U * A[:, None] + (2 * x + 16) * U) * W
        finite = want.isfinite()
        assert torch.equal(got[i].isfinite(), finite), (i, value)
        assert bool(((got[i] - want).abs() <= tol)[finite].all())
    hit = {(i, g) for i, g, _ in struck}
    clean = torch.tensor([[(i, g) not in hit for g in range(KV)] for i in range(len(lens))]).repeat_interleave(H // KV, 1)
    assert bool(got[clean.cuda()].isfinite().all())


@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@pytest.mark.parametrize("new,prefix", [(1, 0), (5, 0), (1, 12), (5, 11)])
def test_every_operand_keeps_its_bits(new, prefix, hd, kv):
    """Scores of one product and outputs of one product, of operands with full
    significands: a query and a key of two (FP32 pages) parts err by 4 u each, the
    parts' products, their sum, the scale and the exponent by 4 u: 12 u A.  Outputs:
    2 delta, the parts of weight and value 8 u, the sum of N <= 16 weights and the
    quotient, and a join, 32 u.  Operands of 16 bits would miss it by 128 u."""
    N = 16
    c = make(3, 8, 2, hd, 16, kv, [N - prefix - new] * 3, [new] * 3, seed=hd, prefix=prefix)
    g = torch.Generator().manual_seed(2)
    keys = torch.zeros(N, hd)
    keys[:, 1] = torch.rand(N, generator=g) - 0.5
    values = torch.zeros(N, hd)
    values[range(N), range(N)] = torch.rand(N, generator=g) + 0.5
    keys, values = keys.to(kv).float(), values.to(kv).float()
    fill(c, keys.cuda(), values.cuda())
    x = math.sqrt(hd) * (torch.rand(8, generator=g) + 0.5)
    c["q"].zero_()
    c["q"][..., 1] = x.cuda()
    scores = x.double()[:, None] * keys[None, :, 1].double() / math.sqrt(hd)
    got = attend(c).double().cpu()
    want, _ = softmax64(c, scores, values)
    A = float(scores.abs().max())
    assert not got[want == 0].any()
    err = ((got - want).abs() / want.clamp(min=1e-300)).masked_fill(want == 0, 0.0)
    assert float(err.max()) <= (2 * 12 * A + 8 + 32) * U


def check_definition(c, out):
    """Every row against softmax over the keys that it sees: NaN and infinities where the
    definition has them; a head all of whose scores are -inf (0 / 0) is zero, like one without keys."""
    H, hd = c["q"].shape[1:]
    KV, ps, P = c["kp"].shape[2], c["kp"].shape[1], c["prefix"]
    t = 0
    for i, (a, b) in enumerate(zip(c["past"], c["new"])):
        at = torch.arange(a + b, device="cuda")
        pre = torch.arange(P, device="cuda")
        k, v = (torch.cat((pool[c["prefix_pages"][pre // ps].long(), pre % ps],
                           pool[c["table"][i, at // ps].long(), at % ps])).double() for pool in (c["kp"], c["vp"]))
        for j in range(b):
            N = P + a + j + 1
            q = c["q"][t].double().unflatten(0, (KV, H // KV))
            s = torch.einsum("grd,kgd->grk", q, k[:N]) / math.sqrt(hd)
            w = torch.softmax(s, -1)
            nothing = (s == -math.inf).all(-1).flatten()
            want = torch.einsum("grk,kgd->grd", w, v[:N]).flatten(0, 1)
            want[nothing] = 0.0
            finite = want.isfinite()
            plain = lambda x: torch.where(x.isfinite(), x.abs(), 0.0)
            W = torch.einsum("grk,kgd->grd", torch.nan_to_num(w, nan=0.0), plain(v[:N])).flatten(0, 1)
            A = torch.einsum("grd,kgd->grk", q.abs(), plain(k[:N])).amax(-1).flatten() / math.sqrt(hd)
            tol = (2 * (hd + 16) * U * A[:, None] + (2 * N + 16) * U) * W
            assert torch.equal(out[t].isfinite(), finite), (i, j)
            assert bool(((out[t].double() - want).abs() <= tol)[finite].all()), (i, j)
            t += 1


@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
@pytest.mark.parametrize("H,KV,hd,ps", [(8, 4, 16, 16), (16, 2, 64, 16), (10, 2, 128, 32)])
@pytest.mark.parametrize("new,prefix", [(1, 300), (20, 0), (20, 300)])
@pytest.mark.parametrize("where", ["keys", "values", "prefix keys", "prefix values"])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_what_is_not_finite_in_chunks_and_prefixes(value, where, new, prefix, H, KV, hd, ps, kv):
    """One element of one kv head's keys or values, in units that all rows see whole and in others."""
    if "prefix" in where and not prefix:
        where = where.split()[1]
    past = [0, 17, 140, 400]
    c = make(len(past), H, KV, hd, ps, kv, past, [new] * len(past), seed=hd, prefix=prefix)
    pool = c["kp" if "keys" in where else "vp"]
    if "prefix" in where:
        c["prefix_pages"] = c["prefix_pages"].clone()
        pool[int(c["prefix_pages"][131 // ps]), 131 % ps, KV - 1, 5] = value
    else:
        for i, a in enumerate(past):
            for at, g in ((a // 2, i % KV), (a + new - 1 - new // 3, (i + 1) % KV)):
                pool[int(c["table"][i, at // ps]), at % ps, g, (3 * i) % hd] = value
    check_definition(c, attend(c))
