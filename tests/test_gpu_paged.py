"""GPU: append to a paged cache, attention over its pages and behind a shared
prefix, against the definitions in 64 bits.

Append is exact: the rotation rounds each product before the add, as torch
does in float32, and the cache write rounds once.

Attention's bound per output element, u = 2^-24 (half a step of float32):

* a score is a dot product of hd products: its error is at most
  (hd + 8) u A + 4 u |s| with A = max_k sum_i |q_i k_i| / sqrt(hd) -- hd
  rounded adds, the roundings of the parts of q and k (each below 2^-22, 4 u,
  of their values), the scaling and the subtraction of the maximum;
* |s| <= A, so delta = (hd + 16) u A bounds it, and the exponential turns it
  into a relative error of delta of each weight, plus 4 u of its own;
* the sums over N keys of weights and of weighted values err by at most N u
  each, relative to the sums of absolute values, and rounding the parts of
  a weight adds 4 u;
* an output is the ratio of the two: |error| <= (2 delta + (2 N + 16) u) W
  with W = sum_k w_k |v_k|.
"""

import math

import pytest
import torch

from conftest import small_model_files
from q6w_b200 import Q6WError, ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def make(n, H, KV, hd, ps, kv, past, new, seed=0, prefix=0, layout="slots", stale=1.0):
    """A pool, tables and a step's tensors; lists ``past`` and ``new`` of n counts."""
    g = torch.Generator().manual_seed(seed)
    lens = [a + b for a, b in zip(past, new)]
    pages = [-(-x // ps) for x in lens]
    np_ = -(-prefix // ps)
    total = sum(pages) + np_ + 2
    ids = torch.randperm(total, generator=g).int()
    width = max(pages + [1]) + 1
    table = torch.full((n, width), -7, dtype=torch.int32)
    at = np_
    for i in range(n):
        table[i, : pages[i]] = ids[at: at + pages[i]]
        at += pages[i]
    shape = (total, ps, KV, hd) if layout == "slots" else (total, KV, ps, hd)
    kp, vp = (torch.randn(shape, generator=g).mul_(stale).to(kv).cuda() for _ in range(2))
    if layout != "slots":  # pages stored head by head
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    T = sum(new)
    starts = [0]
    for b in new:
        starts.append(starts[-1] + b)
    return {"q": torch.randn(T, H, hd, generator=g).cuda() * 1.5, "kp": kp, "vp": vp, "table": table.cuda(),
            "lens": torch.tensor(lens, dtype=torch.int32).cuda(),
            "starts": torch.tensor(starts, dtype=torch.int32).cuda(), "prefix_pages": ids[:np_].cuda(),
            "prefix": prefix, "past": past, "new": new}


def gathered(c, i, length):
    ps = c["kp"].shape[1]
    at = c["table"][i, : -(-length // ps)].long()
    out = []
    for pool, pre in ((c["kp"], c["prefix"]), (c["vp"], c["prefix"])):
        own = pool[at].flatten(0, 1)[:length]
        first = pool[c["prefix_pages"].long()].flatten(0, 1)[:pre]
        out.append(torch.cat((first, own)).double())
    return out


def check(c, out, rows=None):
    """Every row of ``out`` against the definition in 64 bits."""
    H, hd = c["q"].shape[1:]
    KV = c["kp"].shape[2]
    t = 0
    worst = 0.0
    for i, (a, b) in enumerate(zip(c["past"], c["new"])):
        k, v = gathered(c, i, a + b)
        q = c["q"][t: t + b].double().unflatten(1, (KV, H // KV))
        N = k.shape[0]
        if b and N:
            s = torch.einsum("tgrd,kgd->tgrk", q, k) / math.sqrt(hd)
            hidden = torch.arange(N, device=s.device)[None] > torch.arange(b, device=s.device)[:, None] + N - b
            s = s.masked_fill(hidden[:, None, None], -math.inf)
            w = torch.softmax(s, -1)
            want = torch.einsum("tgrk,kgd->tgrd", w, v).flatten(1, 2)
            W = torch.einsum("tgrk,kgd->tgrd", w, v.abs()).flatten(1, 2)
            A = (torch.einsum("tgrd,kgd->tgrk", q.abs(), k.abs()) / math.sqrt(hd)).amax(-1).flatten(1, 2)
            tol = (2 * (hd + 16) * U * A[..., None] + (2 * N + 16) * U) * W
            err = (out[t: t + b].double() - want).abs()
            assert not torch.isnan(err).any(), i
            worst = max(worst, float((err / tol).max()))
        elif b:
            assert not out[t: t + b].any()
        t += b
    assert worst <= 1.0, worst


def attend(c, **kw):
    ragged = any(b != 1 for b in c["new"]) or kw.pop("ragged", False)
    args = (c["table"], c["lens"], c["starts"] if ragged else None)
    if c["prefix"] or kw.pop("as_prefix", False):
        return ops.shared_prefix_attention(c["q"], c["kp"], c["vp"], c["prefix_pages"], c["prefix"], *args, **kw)
    return ops.paged_attention(c["q"], c["kp"], c["vp"], *args, **kw)


# ---- append ---------------------------------------------------------------------


def tables(count, hd):
    from q6w_b200.model import rope_tables

    cos, sin = rope_tables(hd, count)
    return cos.cuda(), sin.cuda()


def rotated(x, c, s):
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)


def append_inputs(T, H, KV, hd, seed):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(T, (H + 2 * KV) * hd, generator=g).cuda()
    q = qkv[:, : H * hd].view(T, H, hd)
    k = qkv[:, H * hd: (H + KV) * hd].view(T, KV, hd)
    return q, k, qkv[:, (H + KV) * hd:].view(T, KV, hd)


def expected_pools(c, k, v, cos, sin, first=0):
    kp, vp = c["kp"].clone(), c["vp"].clone()
    ps = kp.shape[1]
    t = 0
    qpos = []
    for i, (a, b) in enumerate(zip(c["past"], c["new"])):
        for j in range(b):
            at = a + j
            if at >= 0:
                page = int(c["table"][i, at // ps])
                kp[page, at % ps] = rotated(k[t], cos[first + at], sin[first + at]).to(kp.dtype)
                vp[page, at % ps] = v[t].to(vp.dtype)
            qpos.append(at)
            t += 1
    return kp, vp, qpos


@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
@pytest.mark.parametrize("H,KV,hd,ps,layout", [(8, 4, 16, 16, "slots"), (4, 2, 32, 1, "heads"), (32, 4, 64, 8, "slots"),
                                               (5, 5, 128, 64, "heads"), (3, 1, 64, 128, "slots")])
def test_append_is_exact(H, KV, hd, ps, layout, kv):
    past = [0, 3, 17, 0, 64, 5]
    new = [1, 5, 0, 40, 1, 2]
    c = make(6, H, KV, hd, ps, kv, past, new, seed=hd + ps, layout=layout)
    cos, sin = tables(100, hd)
    q, k, v = append_inputs(sum(new), H, KV, hd, 1)
    kp, vp, pos = expected_pools(c, k, v, cos, sin, first=7)
    got = ops.paged_append(q, k, v, cos, sin, c["kp"], c["vp"], c["table"], c["lens"], c["starts"], first_position=7)
    assert torch.equal(c["kp"], kp) and torch.equal(c["vp"], vp)
    at = torch.tensor(pos).cuda() + 7
    assert torch.equal(got, rotated(q, cos[at][:, None], sin[at][:, None]))


def test_append_one_token_each_in_place_and_without_queries():
    c = make(9, 4, 2, 64, 16, torch.float32, [0, 1, 15, 16, 31, 2, 0, 40, 7], [1] * 9)
    cos, sin = tables(64, 64)
    q, k, v = append_inputs(9, 4, 2, 64, 2)
    q = q.contiguous()
    kp, vp, pos = expected_pools(c, k, v, cos, sin)
    want = rotated(q, cos[pos][:, None], sin[pos][:, None])
    assert ops.paged_append(None, k, v, cos, sin, c["kp"], c["vp"], c["table"], c["lens"]) is None
    assert torch.equal(c["kp"], kp) and torch.equal(c["vp"], vp)
    assert ops.paged_append(q, k, v, cos, sin, c["kp"], c["vp"], c["table"], c["lens"], out=q) is q
    assert torch.equal(q, want)


def test_append_many_sequences_finds_each_token():
    """Ragged counts with runs of empty sequences: the search for a token's sequence."""
    g = torch.Generator().manual_seed(5)
    n = 3000
    new = torch.randint(0, 4, (n,), generator=g)
    new[100:1200] = 0
    new[0] = 0
    past = torch.randint(0, 9, (n,), generator=g).tolist()
    c = make(n, 2, 1, 16, 8, torch.float32, past, new.tolist())
    cos, sin = tables(16, 16)
    q, k, v = append_inputs(int(new.sum()), 2, 1, 16, 3)
    kp, vp, pos = expected_pools(c, k, v, cos, sin)
    got = ops.paged_append(q, k, v, cos, sin, c["kp"], c["vp"], c["table"], c["lens"], c["starts"])
    assert torch.equal(c["kp"], kp) and torch.equal(c["vp"], vp)
    assert torch.equal(got, rotated(q, cos[pos][:, None], sin[pos][:, None]))


@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
def test_append_many_tokens(kv):
    """Enough narrow tokens that a thread takes several, across the ends of
    sequences, with empty sequences and padding at both ends and inside."""
    g = torch.Generator().manual_seed(8)
    n = 600
    new = torch.randint(0, 41, (n,), generator=g)
    new[50:60] = 0
    c = make(n, 8, 4, 16, 16, kv, torch.randint(0, 30, (n,), generator=g).tolist(), new.tolist())
    T = int(new.sum())
    assert T * 32 >= 148 * 2048
    c["past"][7] -= int(c["past"][7]) + 3  # the first three new tokens of sequence 7 are padding
    c["lens"][7] = c["past"][7] + int(new[7])
    cos, sin = tables(128, 16)
    q, k, v = append_inputs(T + 9, 8, 4, 16, 12)
    kp, vp, pos = expected_pools(c, k[4:], v[4:], cos, sin)
    c["starts"] += 4
    got = ops.paged_append(q, k, v, cos, sin, c["kp"], c["vp"], c["table"], c["lens"], c["starts"])
    assert torch.equal(c["kp"], kp) and torch.equal(c["vp"], vp)
    pos = torch.tensor(pos).cuda()
    want = rotated(q[4: T + 4], cos[pos.clamp(min=0)][:, None], sin[pos.clamp(min=0)][:, None]) * (pos >= 0)[:, None, None]
    assert torch.equal(got[4: T + 4], want) and not got[:4].any() and not got[T + 4:].any()


def test_append_padding_rows():
    """Tokens in front of the first sequence, behind the last, and in front of
    position 0 append nothing; their rows stay as they were or come back zero."""
    c = make(2, 2, 2, 16, 4, torch.float32, [2, 0], [3, 4])
    c["starts"] = torch.tensor([1, 4, 8], dtype=torch.int32).cuda()
    c["lens"][1] = 2  # four new tokens, two of them padding
    cos, sin = tables(16, 16)
    q, k, v = append_inputs(11, 2, 2, 16, 4)
    kp, vp = c["kp"].clone(), c["vp"].clone()
    pos = [None, 2, 3, 4, None, None, 0, 1, None, None, None]
    want = torch.zeros(11, 2, 16).cuda()
    for t, p in enumerate(pos):
        if p is not None:
            page = int(c["table"][0 if t < 4 else 1, p // 4])
            kp[page, p % 4] = rotated(k[t], cos[p], sin[p])
            vp[page, p % 4] = v[t]
            want[t] = rotated(q[t], cos[p], sin[p])
    args = (q, k, v, cos, sin, c["kp"], c["vp"], c["table"], c["lens"], c["starts"])
    assert torch.equal(ops.paged_append(*args), want)
    assert torch.equal(c["kp"], kp) and torch.equal(c["vp"], vp)
    out = torch.full_like(want, 9.0)
    ops.paged_append(*args, out=out)
    pad = torch.tensor([p is None for p in pos]).cuda()
    assert torch.equal(out[~pad], want[~pad]) and bool((out[pad] == 9).all())


def test_append_bad_pages_and_positions_are_flagged():
    c = make(4, 2, 1, 16, 4, torch.float32, [0, 5, 3, 2], [1, 1, 1, 1])
    cos, sin = tables(5, 16)  # sequence 1's position 5 is behind the table
    q, k, v = append_inputs(4, 2, 1, 16, 6)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    kp, vp = c["kp"].clone(), c["vp"].clone()
    c["table"][0, 0] = c["kp"].shape[0]
    c["table"][2, 0] = -1
    page = int(c["table"][3, 0])
    kp[page, 2] = rotated(k[3], cos[2], sin[2])
    vp[page, 2] = v[3]
    ops.paged_append(q, k, v, cos, sin, c["kp"], c["vp"], c["table"], c["lens"], status=status)
    assert torch.equal(c["kp"], kp) and torch.equal(c["vp"], vp)
    with pytest.raises(Q6WError):
        ops.check_status(status)
    ops.check_status(status)  # cleared
    c["lens"][:] = 10 ** 6  # beyond the page table
    ops.paged_append(q, k, v, cos, sin, c["kp"], c["vp"], c["table"], c["lens"], status=status)
    assert torch.equal(c["kp"], kp) and torch.equal(c["vp"], vp)
    with pytest.raises(Q6WError):
        ops.check_status(status)


# ---- attention ---------------------------------------------------------------------

LENS = [0, 1, 2, 15, 16, 17, 31, 33, 64, 100, 127, 128, 129, 300, 513]


@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
@pytest.mark.parametrize("hd,ps,layout", [(16, 16, "slots"), (32, 8, "heads"), (64, 1, "slots"), (64, 32, "heads"),
                                          (128, 64, "slots"), (128, 1024, "slots")])
@pytest.mark.parametrize("rep", [1, 2, 3, 8])
def test_decode(hd, ps, layout, rep, kv):
    KV = 2 if rep < 8 else 4
    c = make(len(LENS), KV * rep, KV, hd, ps, kv, [x - 1 for x in LENS], [1] * len(LENS), seed=rep, layout=layout)
    out = attend(c)
    assert not out[0].any()  # a length of 0: the token is padding
    for name in ("q", "past", "new", "table"):
        c[name] = c[name][1:]
    check(c, out[1:])


@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
@pytest.mark.parametrize("rep", [5, 6, 7, 12, 16, 20])
def test_decode_odd_groups(rep, kv):
    c = make(5, 2 * rep, 2, 64, 16, kv, [0, 6, 99, 250, 33], [1] * 5, seed=rep)
    check(c, attend(c))


@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
@pytest.mark.parametrize("n,H,KV,hd,length", [(1, 32, 4, 64, 20000), (2, 8, 4, 16, 9000), (1, 5, 1, 128, 12345),
                                              (3, 16, 8, 32, 7001)])
def test_decode_long(n, H, KV, hd, length, kv):
    """Few sequences over a long axis: split over the whole GPU and joined."""
    past = [length - 1, 12, length // 3][:n]
    c = make(n, H, KV, hd, 16, kv, past, [1] * n, seed=n)
    check(c, attend(c))


@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
@pytest.mark.parametrize("n,H,KV,hd", [(2500, 8, 4, 16), (700, 16, 2, 64), (300, 8, 8, 128)])
def test_decode_many(n, H, KV, hd, kv):
    g = torch.Generator().manual_seed(n)
    past = torch.randint(0, 90, (n,), generator=g).tolist()
    past[n // 2] = 3000  # one long among many short
    c = make(n, H, KV, hd, 16, kv, past, [1] * n, seed=n)
    check(c, attend(c))


RAGGED = [([0, 5, 0, 130, 64], [1, 3, 0, 70, 64]), ([0], [200]), ([300, 0, 1000], [129, 17, 1]), ([0] * 40, [3] * 40),
          ([2000], [4])]


@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
@pytest.mark.parametrize("H,KV,hd,ps", [(8, 4, 16, 16), (6, 2, 32, 8), (16, 2, 64, 1), (32, 4, 64, 16), (10, 2, 128, 64),
                                        (4, 4, 128, 128), (20, 1, 64, 512)])
@pytest.mark.parametrize("shape", range(len(RAGGED)))
def test_ragged(shape, H, KV, hd, ps, kv):
    past, new = RAGGED[shape]
    c = make(len(past), H, KV, hd, ps, kv, past, new, seed=shape, layout="heads" if ps == 8 else "slots")
    check(c, attend(c))


@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
@pytest.mark.parametrize("H,KV,hd", [(8, 2, 64), (8, 8, 128), (3, 1, 16)])
def test_ragged_long(H, KV, hd, kv):
    c = make(3, H, KV, hd, 32, kv, [0, 2500, 700], [1100, 333, 2], seed=hd)
    check(c, attend(c))


@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
@pytest.mark.parametrize("H,KV,hd,ps", [(8, 4, 16, 16), (12, 4, 32, 32), (32, 4, 64, 16), (10, 2, 128, 64), (1, 1, 64, 8)])
@pytest.mark.parametrize("prefix", [1, 16, 129, 1500])
def test_shared_prefix(prefix, H, KV, hd, ps, kv):
    past = [0, 1, 30, 200, 7, 63, 64, 65, 400]
    c = make(9, H, KV, hd, ps, kv, past, [1] * 9, seed=prefix, prefix=prefix)
    check(c, attend(c))


@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
@pytest.mark.parametrize("n,H,KV,hd,prefix", [(200, 32, 4, 64, 700), (77, 8, 4, 16, 2100), (130, 6, 2, 128, 333),
                                              (1, 32, 4, 64, 5000), (2, 8, 8, 128, 3001)])
def test_shared_prefix_batches(n, H, KV, hd, prefix, kv):
    past = [(i * 37) % 150 for i in range(n)]
    c = make(n, H, KV, hd, 16, kv, past, [1] * n, seed=n, prefix=prefix)
    check(c, attend(c))


@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
@pytest.mark.parametrize("H,KV,hd", [(8, 4, 16), (16, 2, 64), (6, 2, 128)])
def test_shared_prefix_ragged(H, KV, hd, kv):
    c = make(6, H, KV, hd, 16, kv, [0, 0, 40, 7, 200, 3], [5, 1, 0, 150, 33, 64], seed=hd, prefix=777)
    check(c, attend(c))


def test_prefix_with_empty_own_caches():
    """A token whose sequence holds nothing of its own (padding by length) sees the prefix alone."""
    c = make(3, 8, 2, 64, 16, torch.float32, [0, 0, 0], [1, 1, 1], prefix=100)
    c["lens"][1] = 0
    out = attend(c)
    k, v = (x[c["prefix_pages"].long()].flatten(0, 1)[:100].double() for x in (c["kp"], c["vp"]))
    q = c["q"][1].double().view(2, 4, 64)
    w = torch.softmax(torch.einsum("grd,kgd->grk", q, k) / 8, -1)
    want = torch.einsum("grk,kgd->grd", w, v).flatten(0, 1)
    assert (out[1].double() - want).abs().max() <= 300 * U * float(v.abs().max())


def test_prefix_of_no_length_is_paged_attention():
    c = make(5, 8, 2, 64, 16, torch.float16, [3, 80, 0, 17, 200], [1] * 5)
    assert torch.equal(attend(c), attend(c, as_prefix=True))


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf, 3e38])
@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("prefix", [0, 70])
def test_slots_behind_a_length_may_hold_anything(prefix, new, kv, value):
    past = [0, 5, 63, 90]
    c = make(4, 8, 2, 64, 16, kv, past, [new] * 4, prefix=prefix)
    want = attend(c)
    ps = 16
    used = torch.zeros(c["kp"].shape[:2], dtype=torch.bool)
    for i, a in enumerate(past):
        for p in range(a + new):
            used[int(c["table"][i, p // ps]), p % ps] = True
    for p in range(prefix):
        used[int(c["prefix_pages"][p // ps]), p % ps] = True
    for pool in (c["kp"], c["vp"]):
        pool[~used.cuda()] = value
    assert torch.equal(attend(c), want)


@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
def test_nan_of_a_later_token_stays_in_its_rows(kv):
    """Causal masking: a chunk's row does not meet a later token's key or value."""
    c = make(2, 8, 2, 64, 16, kv, [30, 0], [50, 20])
    want = attend(c)
    for at, pool in ((60, c["kp"]), (65, c["vp"])):
        pool[int(c["table"][0, at // 16]), at % 16] = math.nan
    got = attend(c)
    first = 60 - 30
    assert torch.equal(got[:first], want[:first]) and torch.equal(got[50:], want[50:])
    assert bool(got[first:50].isnan().all())


@pytest.mark.parametrize("new,prefix", [(1, 0), (1, 50), (20, 0), (20, 50)])
def test_bad_page_ids_give_nan_rows_and_a_status(new, prefix):
    c = make(3, 8, 2, 64, 16, torch.float32, [40, 40, 40], [new] * 3, prefix=prefix)
    want = attend(c)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    attend(c, status=status)
    ops.check_status(status)
    c["table"][1, 1] = c["kp"].shape[0] + 5
    got = attend(c, status=status)
    bad = slice(new, 2 * new)
    assert bool(got[bad].isnan().all())
    assert torch.equal(got[:new], want[:new]) and torch.equal(got[2 * new:], want[2 * new:])
    with pytest.raises(Q6WError):
        ops.check_status(status)
    ops.check_status(status)


def test_length_beyond_the_table_is_flagged():
    c = make(2, 4, 2, 32, 16, torch.float32, [40, 20], [1, 1])
    c["table"][1] = c["table"][0]
    c["table"][:, -1] = c["table"][:, 0]
    cap = c["table"].shape[1] * 16
    c["lens"][1] = cap + 100
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = attend(c, status=status)
    with pytest.raises(Q6WError):
        ops.check_status(status)
    c["lens"][1] = cap
    assert torch.equal(got, attend(c, status=status))
    ops.check_status(status)


def test_padding_inside_ragged_sequences():
    """More new tokens than a sequence's length: the first ones are padding (zero
    rows), the others as in a call that holds them alone."""
    for prefix in (0, 60):
        c = make(2, 8, 2, 64, 16, torch.float16, [0, 30], [90, 20], prefix=prefix)
        c["lens"][0] = 50  # 40 of the 90 are padding
        got = attend(c)
        d = dict(c, q=c["q"][40:].contiguous(), new=[50, 20], past=[0, 30])
        d["starts"] = torch.tensor([0, 50, 70], dtype=torch.int32).cuda()
        check(d, got[40:])
        if not prefix:
            assert not got[:40].any()
        else:  # they see the prefix alone
            k, v = (x[c["prefix_pages"].long()].flatten(0, 1)[:60].double() for x in (c["kp"], c["vp"]))
            w = torch.softmax(torch.einsum("tgrd,kgd->tgrk", c["q"][:40].double().unflatten(1, (2, 4)), k) / 8, -1)
            want = torch.einsum("tgrk,kgd->tgrd", w, v).flatten(1, 2)
            assert (got[:40].double() - want).abs().max() <= 300 * U * float(v.abs().max())


@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
def test_decode_one_long_among_many(kv):
    """A request that reaches over most of the GPU among many that fill a tile each."""
    past = [3] * 700
    past[350] = 60000
    c = make(700, 16, 2, 64, 16, kv, past, [1] * 700, seed=4)
    check(c, attend(c))


def test_rows_outside_the_sequences():
    c = make(2, 8, 4, 16, 16, torch.float32, [3, 30], [4, 10])
    want = attend(c)
    q = torch.full((20, 8, 16), math.nan, device="cuda")
    q[2:16] = c["q"]
    c["q"], c["starts"] = q, c["starts"] + 2
    got = attend(c)
    assert torch.equal(got[2:16], want) and not got[:2].any() and not got[16:].any()
    out = torch.full((20, 8, 16), 5.0, device="cuda")
    assert attend(c, out=out) is out
    assert torch.equal(out[2:16], want) and bool((out[:2] == 5).all()) and bool((out[16:] == 5).all())


def test_extreme_scores():
    """Scores of thousands, and heads of one group with maxima far apart."""
    c = make(3, 8, 2, 64, 16, torch.float32, [99, 500, 3], [1] * 3)
    c["q"] *= torch.tensor([1e-6, 0.1, 1.0, 10.0, 100.0, 1000.0, 1e-20, 0.0]).cuda()[None, :, None]
    check(c, attend(c))
    c["q"] = c["q"].repeat(30, 1, 1)[:70].contiguous()
    c["past"], c["new"] = [40, 480, 0], [60, 6, 4]
    c["lens"] = torch.tensor([100, 486, 4], dtype=torch.int32).cuda()
    c["starts"] = torch.tensor([0, 60, 66, 70], dtype=torch.int32).cuda()
    check(c, attend(c))


@pytest.mark.parametrize("scale", [1e-30, 1e-6, 1e4])
def test_values_of_any_size(scale):
    """FP32 pages keep FP32's range: tiny and large values, queries scaled the other way."""
    for new, prefix in ((1, 0), (40, 0), (1, 200)):
        c = make(3, 8, 2, 64, 16, torch.float32, [70, 3, 200], [new] * 3, prefix=prefix)
        c["vp"] *= scale
        c["kp"] *= scale
        c["q"] /= scale
        check(c, attend(c))


def test_one_large_value_does_not_cost_the_others_their_precision():
    c = make(2, 8, 2, 64, 16, torch.float32, [100, 0], [30, 90])
    c["vp"][int(c["table"][0, 0]), 3] *= 1e12
    c["kp"][int(c["table"][0, 0]), 3] = 0
    c["q"][:30] *= 40  # sharp rows: most give the large value a weight that vanishes
    check(c, attend(c))


def test_offsets_beyond_32_bits():
    ps, KV, hd = 1024, 8, 128
    pages = (1 << 31) // (ps * KV * hd) + 3  # the last page starts behind 2^31 elements
    kp, vp = (torch.zeros(pages, ps, KV, hd, dtype=torch.float16, device="cuda") for _ in range(2))
    c = make(2, 16, KV, hd, ps, torch.float16, [900, 40], [1, 1])
    for i in range(2):
        src = int(c["table"][i, 0])
        kp[pages - 1 - i], vp[pages - 1 - i] = c["kp"][src], c["vp"][src]
    want = attend(c)
    c["kp"], c["vp"] = kp, vp
    c["table"][:, 0] = torch.tensor([pages - 1, pages - 2], dtype=torch.int32)
    assert torch.equal(attend(c), want)
    cos, sin = tables(1024, hd)
    q, k, v = append_inputs(2, 16, KV, hd, 9)
    want_k, want_v, _ = (x if isinstance(x, list) else x[-2:] for x in expected_pools(c, k, v, cos, sin))
    ops.paged_append(q, k, v, cos, sin, kp, vp, c["table"], c["lens"])
    assert torch.equal(kp[-2:], want_k) and torch.equal(vp[-2:], want_v)


def test_layers_and_interleaved_pools():
    """A layer of a larger pool, keys and values side by side, a strided table."""
    c = make(4, 8, 2, 64, 16, torch.float16, [3, 80, 0, 17], [1, 30, 2, 5])
    want = attend(c)
    pages = c["kp"].shape[0]
    both = torch.zeros(3, pages, 2, 16, 2, 64, dtype=torch.float16, device="cuda")
    both[1, :, 0], both[1, :, 1] = c["kp"], c["vp"]
    c["kp"], c["vp"] = both[1, :, 0], both[1, :, 1]
    wide = torch.zeros(4, c["table"].shape[1] + 5, dtype=torch.int32, device="cuda")
    wide[:, : c["table"].shape[1]] = c["table"]
    c["table"] = wide[:, : c["table"].shape[1]]
    assert torch.equal(attend(c), want)


def test_strided_queries():
    c = make(4, 8, 2, 64, 16, torch.float32, [3, 80, 0, 17], [1, 30, 2, 5])
    want = attend(c)
    wide = torch.randn(38, 12 * 64, device="cuda")
    wide[:, : 8 * 64] = c["q"].flatten(1)
    c["q"] = wide[:, : 8 * 64].view(38, 8, 64)
    assert torch.equal(attend(c), want)


def test_nothing_to_do():
    c = make(2, 8, 2, 64, 16, torch.float32, [3, 8], [1, 1])
    q = torch.empty(0, 8, 64, device="cuda")
    starts = torch.zeros(3, dtype=torch.int32, device="cuda")
    assert ops.paged_attention(q, c["kp"], c["vp"], c["table"], c["lens"], starts).shape == (0, 8, 64)
    assert ops.paged_attention(q, c["kp"], c["vp"], c["table"][:0], c["lens"][:0]).shape == (0, 8, 64)
    q = torch.ones(3, 8, 64, device="cuda")
    assert not ops.paged_attention(q, c["kp"], c["vp"], c["table"], c["lens"], starts).any()
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert not ops.paged_attention(q, c["kp"], c["vp"], c["table"][:0], c["lens"][:0], none).any()


@pytest.mark.parametrize("new,prefix", [(1, 0), (1, 333), (60, 0), (60, 333)])
def test_same_inputs_same_bits(new, prefix):
    c = make(5, 16, 2, 64, 16, torch.float16, [40, 3000, 0, 7, 800], [new] * 5, prefix=prefix)
    want = attend(c)
    for _ in range(4):
        assert torch.equal(attend(c), want)


# ---- streams, graphs, devices --------------------------------------------------------


@pytest.mark.parametrize("new,prefix", [(1, 0), (1, 333), (60, 333)])
def test_streams_and_graphs(new, prefix):
    """Two calls at once on two streams, and captured graphs replayed together on new inputs."""
    cs = [make(4, 8, 2, 64, 16, torch.float32, [40, 900, 0, 7], [new] * 4, seed=s, prefix=prefix) for s in (1, 2)]
    want = [attend(c) for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for c, st in zip(cs, streams):
            with torch.cuda.stream(st):
                got.append(attend(c))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for c in cs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(attend(c))
        graphs.append(g)
    cs[0]["q"].copy_(cs[1]["q"])
    cs[0]["lens"] -= 0  # same buffers, new values: lengths may change between replays
    cs[0]["lens"][1] = 200 + new
    for g, st in zip(graphs, streams):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[1], want[1])
    assert torch.equal(outs[0], attend(cs[0]))


# ---- a run of them together ------------------------------------------------------------


@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
@pytest.mark.parametrize("prefix", [0, 24])
def test_model_step_from_ops_matches_the_cached_step(tmp_path_factory, kv, prefix):
    """A Q6W model served from one pool of pages with the operators -- ragged
    prompts as chunks, then tokens one by one, the first ``prefix`` tokens held
    once for all -- against the framework's own prefill and batched step."""
    import torch.nn.functional as F

    from q6w_b200.model import Q6WCudaTransformer

    args = {"dim": 128, "n_layers": 2, "n_heads": 8, "n_kv_heads": 4, "vocab_size": 512, "hidden_dim": 384,
            "multiple_of": 32, "norm_eps": 1e-5, "max_seq_len": 96, "dropout": 0.0}
    model = Q6WCudaTransformer.from_q6w(*small_model_files(tmp_path_factory, args, 5, "paged"), kv_dtype=kv)
    L, H, KV, hd, ps, n = 2, 8, 4, 16, 8, 5
    pool = torch.full((2, L, 64, ps, KV, hd), math.nan, dtype=kv, device="cuda")
    ids = torch.randperm(64, generator=torch.Generator().manual_seed(1)).int()
    first, table = ids[: prefix // ps].cuda(), ids[8: 8 + n * 8].view(n, 8).cuda()
    dq = {e: model.dimg.qmat(e) for e in model.image.tensors if not e.endswith("norm.weight")}
    embed = ops.dequantize_rows(*dq["tok_embeddings.weight"])

    def linear(x, name):
        return ops.q6w_linear(x, *dq[name])

    def forward(tokens, table, lengths, starts, shared):
        x = embed[tokens]
        for l in range(L):
            p = f"layers.{l}."
            h = ops.rmsnorm(x, model.dimg.fp32(p + "attention_norm.weight"), 1e-5)
            q, k, v = (linear(h, p + f"attention.w{c}.weight").view(len(tokens), -1, hd) for c in "qkv")
            kp, vp = pool[0, l], pool[1, l]
            q = ops.paged_append(q, k, v, model.freqs_cos, model.freqs_sin, kp, vp, table, lengths, starts,
                                 first_position=shared)
            if shared:
                o = ops.shared_prefix_attention(q, kp, vp, first, shared, table, lengths, starts)
            else:
                o = ops.paged_attention(q, kp, vp, table, lengths, starts)
            x = x + linear(o.flatten(1), p + "attention.wo.weight")
            h = ops.rmsnorm(x, model.dimg.fp32(p + "ffn_norm.weight"), 1e-5)
            up = F.silu(linear(h, p + "feed_forward.w1.weight")) * linear(h, p + "feed_forward.w3.weight")
            x = x + linear(up, p + "feed_forward.w2.weight")
        return linear(ops.rmsnorm(x, model.dimg.fp32("norm.weight"), 1e-5), "tok_embeddings.weight")

    g = torch.Generator().manual_seed(2)
    head = torch.randint(3, 512, (prefix,), generator=g).tolist()
    prompts = [torch.randint(3, 512, (c,), generator=g).tolist() for c in (1, 9, 30, 16, 5)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    if prefix:
        forward(torch.tensor(head).cuda(), first[None], i32([prefix]), i32([0, prefix]), 0)
    counts = [len(p) for p in prompts]
    lengths = i32(counts)
    starts = i32([0] + torch.tensor(counts).cumsum(0).tolist())
    logits = forward(torch.tensor(sum(prompts, [])).cuda(), table, lengths, starts, prefix)
    logits = logits[starts[1:].long() - 1]
    want, (kc, vc) = model.prefill_batch([head + p for p in prompts])
    assert (logits - want).abs().max() <= 4e-4
    tok = torch.randint(3, 512, (6, n), generator=g).cuda()
    for t in range(6):
        lengths = lengths + 1
        got = forward(tok[t], table, lengths, None, prefix)
        want, _ = model.forward_batch(tok[t].int(), lengths + (prefix - 1), kc, vc)
        assert (got - want).abs().max() <= 4e-4


# ---- refusals of the Python operators ------------------------------------------------------


def test_python_refusals():
    c = make(3, 8, 2, 64, 16, torch.float32, [3, 20, 8], [1, 1, 1])
    a = dict(queries=c["q"], key_pages=c["kp"], value_pages=c["vp"], page_table=c["table"], lengths=c["lens"])
    bad = [dict(queries=c["q"].half()), dict(queries=c["q"][:, :, :32]), dict(queries=c["q"].transpose(1, 2)),
           dict(queries=c["q"][:2]), dict(key_pages=c["kp"].half()), dict(key_pages=c["kp"].double()),
           dict(key_pages=c["kp"][:-1]), dict(value_pages=c["vp"].transpose(1, 2).contiguous().transpose(1, 2)),
           dict(page_table=c["table"].long()), dict(page_table=c["table"].t().contiguous().t()), dict(page_table=c["table"][0]),
           dict(lengths=c["lens"].long()), dict(lengths=c["lens"][:2]), dict(lengths=c["lens"].cpu()),
           dict(query_starts=c["starts"][:3]), dict(query_starts=c["starts"].long()),
           dict(status=torch.zeros(1, device="cuda")), dict(out=torch.empty(3, 8, 32, device="cuda")),
           dict(out=torch.empty(3, 8, 128, device="cuda")[:, :, ::2])]
    ops.paged_attention(**a)
    for kw in bad:
        with pytest.raises(ValueError):
            ops.paged_attention(**{**a, **kw})
    with pytest.raises(Q6WError):  # seven heads over two kv heads
        ops.paged_attention(**{**a, "queries": c["q"][:, :7].contiguous()})
    pages = torch.zeros(2, dtype=torch.int32, device="cuda")
    for length in (-1, 33):
        with pytest.raises(ValueError):
            ops.shared_prefix_attention(prefix_pages=pages, prefix_length=length, **a)
    cos, sin = tables(64, 64)
    q, k, v = append_inputs(3, 8, 2, 64, 1)
    b = dict(a, queries=q, keys=k, values=v, cos=cos, sin=sin)
    ops.paged_append(**b)
    for kw in (dict(keys=k[:, :1]), dict(keys=k[:2]), dict(values=v[:2]), dict(values=v.half()), dict(cos=cos[:, :16]),
               dict(sin=sin[:5]), dict(cos=cos.double(), sin=sin.double()), dict(queries=q[:2]), dict(out=q)):
        with pytest.raises(ValueError):
            ops.paged_append(**{**b, **kw})
