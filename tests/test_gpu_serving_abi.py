"""GPU: the paged attention calls as a C program makes them, and pools whose
pages lie behind 2^31 elements."""

import pytest
import torch

from q6w_b200 import _lib
from test_gpu_paged import attend, check, make

pytestmark = pytest.mark.gpu


def c_batch(c, ragged, status=0):
    kp, vp, table = c["kp"], c["vp"], c["table"]
    pages, ps, KV, hd = kp.shape
    sp, ss, sh, _ = kp.stride()
    return _lib.PAGED_BATCH.pack(kp.data_ptr(), vp.data_ptr(), int(kp.dtype == torch.float16), pages, ps, KV, hd, sp, ss, sh,
                                 table.shape[0], table.shape[1], table.data_ptr(), table.stride(0), c["lens"].data_ptr(),
                                 c["starts"].data_ptr() if ragged else 0, status)


@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
@pytest.mark.parametrize("new", [1, 30])
def test_paged_attention_entry(new, kv):
    """q6w_paged_attention itself, with a workspace that holds anything and no more bytes than it asks for."""
    lib = _lib.load()
    c = make(4, 8, 2, 64, 16, kv, [3, 80, 0, 517], [new] * 4)
    want = attend(c)
    T = 4 * new
    b = c_batch(c, new != 1)
    need = lib.q6w_paged_workspace_bytes(b, T, 8, 0)
    ws = torch.full((need + 4096,), 0xFF, dtype=torch.uint8, device="cuda")  # NaN, whatever is read
    out = torch.full((T + 2, 8, 64), 7.0, device="cuda")
    _lib.check(lib.q6w_paged_attention(b, T, 8, c["q"].data_ptr(), 512, out[1:].data_ptr(), 0, ws.data_ptr(), need,
                                       _lib.stream_handle()))
    assert torch.equal(out[1: T + 1], want)
    assert bool((out[[0, T + 1]] == 7).all()) and bool((ws[need:] == 0xFF).all())
    # once more, over what the call left in it
    _lib.check(lib.q6w_paged_attention(b, T, 8, c["q"].data_ptr(), 512, out[1:].data_ptr(), 0, ws.data_ptr(), need,
                                       _lib.stream_handle()))
    assert torch.equal(out[1: T + 1], want)


@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
@pytest.mark.parametrize("prefix", [0, 700])
def test_chunks_beyond_32_bits(prefix, kv):
    """Chunks and prefixes whose pages start behind 2^31 elements of the pool."""
    ps, KV, hd = 1024, 8, 64
    pages = (1 << 31) // (ps * KV * hd) + 4
    c = make(2, 16, KV, hd, ps, kv, [900, 40], [50, 300], prefix=prefix)
    want = attend(c)
    check(c, want)
    kp, vp = (torch.zeros(pages, ps, KV, hd, dtype=kv, device="cuda") for _ in range(2))
    moved = [c["table"][0, 0], c["table"][1, 0]] + ([c["prefix_pages"][0]] if prefix else [])
    for i, src in enumerate(moved):
        kp[pages - 1 - i], vp[pages - 1 - i] = c["kp"][int(src)], c["vp"][int(src)]
    c["kp"], c["vp"] = kp, vp
    c["table"][:, 0] = torch.tensor([pages - 1, pages - 2], dtype=torch.int32)
    if prefix:
        c["prefix_pages"][0] = pages - 3
    assert torch.equal(attend(c), want)


@pytest.mark.parametrize("kv", [torch.float32, torch.float16])
@pytest.mark.parametrize("prefix", [0, 90])
def test_a_mixed_step_in_two_calls(prefix, kv):
    """Single tokens and chunks of one step, each in a call of its own, into slices of one buffer."""
    from q6w_b200 import ops

    singles, chunks = 12, 3
    past, new = [i * 31 for i in range(singles)] + [0, 40, 333], [1] * singles + [70, 5, 128]
    c = make(singles + chunks, 8, 2, 64, 16, kv, past, new, seed=1, prefix=prefix)
    out = torch.full_like(c["q"], 7.0)
    for rows, toks, starts in ((slice(0, singles), slice(0, singles), None),
                               (slice(singles, None), slice(singles, None), c["starts"][singles:] - singles)):
        args = (c["table"][rows], c["lens"][rows], starts)
        if prefix:
            ops.shared_prefix_attention(c["q"][toks], c["kp"], c["vp"], c["prefix_pages"], prefix, *args, out=out[toks])
        else:
            ops.paged_attention(c["q"][toks], c["kp"], c["vp"], *args, out=out[toks])
    check(c, out)
    check(c, attend(c))
