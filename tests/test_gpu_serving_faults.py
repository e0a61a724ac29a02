"""GPU: waits of the paged attention kernels that run out.  With the diagnostic
on, the first thread block waits for tiles that it never sees arrive: the call
has to end soon, mark what it could not compute as NaN -- also where the caller
gave no status word -- and leave everything else as it is."""

import time

import pytest
import torch

from q6w_b200 import Q6WError, _lib, ops
from test_gpu_paged import attend, make

pytestmark = pytest.mark.gpu
CYCLES = 2_000_000  # about a millisecond; a tile takes a microsecond


def stalled(c, **kw):
    lib = _lib.load()
    torch.cuda.synchronize()
    _lib.check(lib.q6w_selftest_paged_stall(CYCLES))
    try:
        t0 = time.perf_counter()
        out = attend(c, **kw)
        torch.cuda.synchronize()
        return out, time.perf_counter() - t0
    finally:
        _lib.check(lib.q6w_selftest_paged_stall(0))


def check_stalled(c, heads):
    """``heads``: (token, head) rows that surely meet the first block."""
    want = attend(c)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for kw in (dict(status=status), dict()):
        got, seconds = stalled(c, **kw)
        assert seconds < 1.0
        nan = got.isnan().any(-1)
        assert torch.equal(nan, got.isnan().all(-1))  # whole rows
        for t, h in heads:
            assert bool(nan[t, h]), (t, h)
        assert torch.equal(got[~nan], want[~nan])
        share = float(nan.float().mean())
    with pytest.raises(Q6WError, match="ran out of time"):
        ops.check_status(status)
    assert torch.equal(attend(c, status=status), want)
    ops.check_status(status)
    return share


@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
@pytest.mark.parametrize("H,KV,hd", [(8, 4, 16), (32, 4, 64), (8, 4, 128)])
def test_decode_wait_runs_out(H, KV, hd, kv):
    """Ragged requests: the first block holds the first ones, nobody else misses anything."""
    c = make(2400, H, KV, hd, 16, kv, [(i * 29) % 90 for i in range(2400)], [1] * 2400, seed=3)
    share = check_stalled(c, [(0, h) for h in range(H)])
    assert share < 0.02


@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
def test_decode_wait_runs_out_in_a_piece(kv):
    """One long request: the first block's piece spoils the heads of the first kv head alone."""
    c = make(1, 16, 4, 64, 16, kv, [9000], [1], seed=5)
    assert check_stalled(c, [(0, h) for h in range(4)]) == 0.25


@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
@pytest.mark.parametrize("H,KV,hd", [(8, 4, 16), (16, 4, 64), (8, 4, 128)])
def test_chunk_wait_runs_out(H, KV, hd, kv):
    """Short chunks: the first block holds several, and the later ones of its stretch become NaN too."""
    n = 700
    c = make(n, H, KV, hd, 16, kv, [(i * 29) % 90 for i in range(n)], [7] * n, seed=3)
    units = 64 if kv == torch.float32 else 128
    stretch = sum(max(1, -(-int(x) // units)) for x in c["lens"]) * KV // 148  # units of the first block
    share = check_stalled(c, [(t, h) for t in range(7 * (stretch // (2 * KV))) for h in range(H)])
    assert share < 0.02


@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
@pytest.mark.parametrize("hd,tokens", [(64, 64), (128, 32)])
def test_chunk_wait_runs_out_in_a_piece(hd, tokens, kv):
    """One long chunk: the first block's piece spoils its 256 (128) rows alone."""
    c = make(1, 8, 2, hd, 16, kv, [3000], [300], seed=6)
    share = check_stalled(c, [(t, h) for t in range(tokens) for h in range(4)])
    assert share == pytest.approx(tokens * 4 / (300 * 8))


@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
@pytest.mark.parametrize("new", [1, 5])
def test_prefix_wait_runs_out(new, kv):
    """The prefix's first block holds a piece of the first kv head's rows; the sequences' own first block others."""
    n = 60 // new
    c = make(n, 8, 2, 64, 16, kv, [40 * i for i in range(n)], [new] * n, seed=7, prefix=3000)
    share = check_stalled(c, [(t, h) for t in range(n * new) for h in range(4)])
    assert share < 0.75


@pytest.mark.parametrize("starts,bad", [([0, 4, 8, 12], False), ([2, 2, 5, 11], False), ([0, 8, 4, 12], True),
                                        ([0, 4, 8, 13], True), ([-1, 4, 8, 12], True), ([9, 4, 8, 12], True),
                                        ([0, 4, 1 << 30, 12], True), ([0, 4, 8, -5], True)])
@pytest.mark.parametrize("prefix", [0, 40])
def test_starts_that_cannot_be_are_flagged(starts, bad, prefix):
    """Kept inside the step's tokens by both calls, and reported."""
    c = make(3, 8, 2, 64, 16, torch.float32, [20, 3, 40], [4, 4, 4], prefix=prefix)
    c["starts"] = torch.tensor(starts, dtype=torch.int32).cuda()
    cos, sin = (torch.ones(100, 32, device="cuda") for _ in range(2))
    k = torch.randn(12, 2, 64, device="cuda")
    calls = [lambda st: ops.paged_append(c["q"], k, k, cos, sin, c["kp"], c["vp"], c["table"], c["lens"], c["starts"],
                                         status=st),
             lambda st: attend(c, status=st)]
    for call in calls:
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        call(status)
        if bad:
            with pytest.raises(Q6WError):
                ops.check_status(status)
        else:
            ops.check_status(status)
        call(None)


@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
@pytest.mark.parametrize("H,KV,hd,ps", [(8, 4, 16, 8), (8, 2, 64, 1), (8, 2, 64, 16), (10, 2, 128, 64)])
@pytest.mark.parametrize("new", [1, 20])
@pytest.mark.parametrize("at", [0, 24, 200, 349, 399])
def test_a_bad_page_anywhere_spoils_the_rows_that_meet_it(at, new, H, KV, hd, ps, kv):
    """In a unit that every row sees whole, in a later one, in the second tile of a unit, behind some rows' positions."""
    c = make(3, H, KV, hd, ps, kv, [400 - new] * 3, [new] * 3, seed=at)
    want = attend(c)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for bad in (-1, c["kp"].shape[0], 1 << 30):
        c["table"][1, at // ps] = bad
        got = attend(c, status=status)
        first = max(0, at // ps * ps - (400 - new))  # rows in front of the page's first position see nothing of it
        spoilt = slice(new + first, 2 * new)
        assert bool(got[spoilt].isnan().all())
        keep = torch.ones(3 * new, dtype=torch.bool)
        keep[spoilt] = False
        assert torch.equal(got[keep], want[keep])
        with pytest.raises(Q6WError):
            ops.check_status(status)


@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
@pytest.mark.parametrize("new", [1, 20])
@pytest.mark.parametrize("at", [0, 130, 299])
def test_a_bad_prefix_page_spoils_every_row(at, new, kv):
    c = make(3, 8, 2, 64, 16, kv, [40, 0, 300], [new] * 3, prefix=300)
    c["prefix_pages"][at // 16] = c["kp"].shape[0]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert bool(attend(c, status=status).isnan().all())
    with pytest.raises(Q6WError):
        ops.check_status(status)
