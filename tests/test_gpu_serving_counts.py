"""GPU: every key counts once.  With queries of zero all weights are equal and
powers of two, and with unit vectors as values an output is a count of keys over
their number: sums of whole numbers, exact in float32 however they are split and
joined, so that a bound of three roundings (the reciprocal, the product, and one
in hand) sees one key lost or taken twice among tens of thousands.  And the
other way round: queries that pick one key each, at the seams of pages, units and
pieces."""

import pytest
import torch

from test_gpu_paged import U, attend, check, make

pytestmark = pytest.mark.gpu
KINDS = [torch.float32, torch.float16]


def bucket(keys, g, hd):
    return keys // (37 if g % 2 else 5) % hd


def count(c, **kw):
    """Attention with queries of zero over values that mark their keys, against the counts."""
    KV, hd, ps, P = c["kp"].shape[2], c["kp"].shape[3], c["kp"].shape[1], c["prefix"]
    H = c["q"].shape[1]
    c["q"].zero_()
    c["vp"].zero_()
    longest = P + max(a + b for a, b in zip(c["past"], c["new"]))
    keys = torch.arange(longest, device="cuda")
    marks = torch.stack([torch.nn.functional.one_hot(bucket(keys, g, hd), hd) for g in range(KV)], 1)  # [N, KV, hd]
    parts = [(c["prefix_pages"], 0, P)] + [(row, P, a + b) for row, a, b in zip(c["table"], c["past"], c["new"])]
    for pages, first, n in parts:
        at = torch.arange(n, device="cuda")
        c["vp"][pages[at // ps].long(), at % ps] = marks[first: first + n].to(c["vp"].dtype)
    upto = marks.cumsum(0).double()
    seen = torch.cat([torch.arange(P + a, P + a + b) for a, b in zip(c["past"], c["new"])]).cuda() + 1
    want = (upto[seen - 1] / seen[:, None, None]).repeat_interleave(H // KV, 1)
    got = attend(c, **kw).double()
    worst = ((got - want).abs() - 3 * U * want).max()
    assert worst <= 0, float(worst)


def lengths(n, most, seed):
    return torch.randint(0, most, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("H,KV,hd,ps", [(8, 4, 16, 16), (16, 8, 32, 8), (32, 4, 64, 1), (40, 2, 64, 16), (10, 2, 128, 64)])
@pytest.mark.parametrize("past", [[0], [19999], [7000, 11, 2332], [3] * 350 + [60000] + [3] * 350, lengths(2500, 90, 1),
                                  lengths(97, 3000, 2)], ids=["one", "long", "three", "long_among_many", "many", "ragged"])
def test_decode_counts(past, H, KV, hd, ps, kv):
    count(make(len(past), H, KV, hd, ps, kv, past, [1] * len(past), seed=3))


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("H,KV,hd,ps", [(8, 4, 16, 16), (6, 2, 32, 8), (32, 4, 64, 1), (10, 2, 128, 64), (40, 1, 128, 32)])
@pytest.mark.parametrize("past,new", [([0], [1]), ([0, 5, 0, 130, 64], [1, 3, 0, 70, 64]), ([0, 2500, 700], [1100, 333, 2]),
                                      ([30000], [40]), (lengths(300, 200, 4), lengths(300, 9, 5)), ([0] * 9, [257] * 9)])
def test_chunk_counts(past, new, H, KV, hd, ps, kv):
    c = make(len(past), H, KV, hd, ps, kv, past, new, seed=4)
    count(c, **({"ragged": True} if max(new) == 1 else {}))


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("H,KV,hd,ps", [(8, 4, 16, 16), (32, 4, 64, 16), (10, 2, 128, 64)])
@pytest.mark.parametrize("prefix", [1, 63, 128, 4999, 20001])
@pytest.mark.parametrize("past,new", [([0], [1]), ([0, 1, 30, 200, 7, 400], [1] * 6), (lengths(200, 90, 6), [1] * 200),
                                      ([0, 40, 200, 3], [5, 150, 33, 64])])
def test_prefix_counts(past, new, prefix, H, KV, hd, ps, kv):
    count(make(len(past), H, KV, hd, ps, kv, past, new, seed=5, prefix=prefix))


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("H,KV,hd,ps", [(4, 4, 16, 16), (8, 2, 64, 16), (4, 2, 128, 64)])
@pytest.mark.parametrize("new,prefix", [(1, 0), (1, 2048), (3, 0), (3, 2048)])
def test_one_key_each(new, prefix, H, KV, hd, ps, kv):
    """Sequences over the same pages, each of whose queries points at one key."""
    own = 4099 - prefix
    seams = [k + d for k in (16, 32, 64, 128, 1024, 2048, 2112, 4096) for d in (-1, 0)] + [0, 1, 4097, 4098]
    picks = sorted(set(seams + torch.randint(0, 4099, (200,), generator=torch.Generator().manual_seed(7)).tolist()))
    n = len(picks)
    c = make(1, H, KV, hd, ps, kv, [own - new], [new], seed=8, prefix=prefix)
    c["kp"].copy_(torch.where(c["kp"] < 0, -1.0, 1.0))
    c["table"], c["lens"] = c["table"].expand(n, -1), c["lens"].expand(n).contiguous()
    c["past"], c["new"] = [own - new] * n, [new] * n
    c["starts"] = torch.arange(n + 1, dtype=torch.int32, device="cuda") * new
    at = torch.arange(own, device="cuda")
    k = c["kp"][c["table"][0, at // ps].long(), at % ps]
    if prefix:
        at = torch.arange(prefix, device="cuda")
        k = torch.cat((c["kp"][c["prefix_pages"][at // ps].long(), at % ps], k))
    c["q"] = (k[torch.tensor(picks).cuda()].float() * (48 / hd ** 0.5)).repeat_interleave(H // KV, 1).repeat_interleave(new, 0)
    check(c, attend(c))
