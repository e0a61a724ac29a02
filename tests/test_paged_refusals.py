"""CPU: what the paged-cache calls refuse, answered by the host before any
kernel, and the sizes of their workspace."""

import ctypes

import pytest
import torch

from q6w_b200 import _lib, ops

P = 1 << 20  # a 16-byte aligned address that no refused call follows
FIELDS = ("k_pages", "v_pages", "kv_dtype", "n_pages", "page_size", "kv_heads", "head_dim", "page_stride", "slot_stride",
          "head_stride", "n_seqs", "max_pages", "page_table", "table_stride", "lengths", "query_starts", "status")
GOOD = dict(zip(FIELDS, (P, P, 0, 8, 16, 4, 64, 4096, 256, 64, 3, 4, P, 4, P, 0, 0)))


def batch(**kw):
    return _lib.PAGED_BATCH.pack(*{**GOOD, **kw}.values())


def append(b, T=3, H=8, q=P, ldq=512, k=P, ldk=256, v=P, ldv=256, cos=P, sin=P, rope=64, first=0, out=2 * P):
    return _lib.load().q6w_paged_append(b, T, H, q, ldq, k, ldk, v, ldv, cos, sin, rope, first, out, 1, None)


def attend(b, T=3, H=8, q=P, ldq=512, out=P, ws=P, n=1 << 40, prefix=None, P_len=0):
    lib = _lib.load()
    if prefix is None and P_len == 0:
        return lib.q6w_paged_attention(b, T, H, q, ldq, out, 1, ws, n, None)
    return lib.q6w_shared_prefix_attention(b, prefix, P_len, T, H, q, ldq, out, 1, ws, n, None)


def message():
    return _lib.load().q6w_last_error().decode()


def test_struct_matches_the_header():
    class Batch(ctypes.Structure):
        p, i, q = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64
        _fields_ = list(zip(FIELDS, (p, p, i, i, i, i, i, q, q, q, i, i, p, q, p, p, p)))

    b = Batch.from_buffer_copy(batch(n_seqs=77, query_starts=5, status=9))
    assert ctypes.sizeof(Batch) == _lib.PAGED_BATCH.size
    assert (b.n_seqs, b.query_starts, b.status, b.head_stride, b.max_pages) == (77, 5, 9, 64, 4)


SHAPES = [dict(kv_dtype=2), dict(head_dim=48), dict(head_dim=256), dict(page_size=0), dict(page_size=24),
          dict(page_size=2048), dict(kv_heads=0), dict(n_pages=-1), dict(n_seqs=-1), dict(max_pages=-1),
          dict(n_seqs=4), dict(max_pages=1 << 30), dict(slot_stride=1 << 26)]


@pytest.mark.parametrize("bad", SHAPES)
def test_bad_shapes(bad):
    assert append(batch(**bad)) == _lib.Q6W_ERR_ARG
    assert attend(batch(**bad)) == _lib.Q6W_ERR_ARG
    assert attend(batch(**bad), prefix=P, P_len=5) == _lib.Q6W_ERR_ARG
    assert message().startswith("q6w_shared_prefix_attention")


@pytest.mark.parametrize("bad", [dict(page_stride=4098), dict(slot_stride=258), dict(head_stride=66), dict(k_pages=P + 4),
                                 dict(v_pages=P + 8), dict(kv_dtype=1, head_stride=68)])
def test_bad_alignment(bad):
    assert append(batch(**bad)) == _lib.Q6W_ERR_ALIGN
    assert attend(batch(**bad)) == _lib.Q6W_ERR_ALIGN


@pytest.mark.parametrize("bad", [dict(k_pages=0), dict(v_pages=0), dict(page_table=0), dict(lengths=0)])
def test_null_pointers(bad):
    assert append(batch(**bad)) == _lib.Q6W_ERR_ARG
    assert attend(batch(**bad)) == _lib.Q6W_ERR_ARG


def test_append_arguments():
    b = batch()
    assert append(None) == _lib.Q6W_ERR_ARG
    for kw in (dict(k=None), dict(v=None), dict(cos=None), dict(sin=None), dict(q=None), dict(out=None), dict(H=-1),
               dict(rope=-1), dict(first=-1), dict(T=-1), dict(ldq=508), dict(ldk=252), dict(ldv=128),
               dict(T=2), dict(ldq=1024, out=P)):
        assert append(b, **kw) == _lib.Q6W_ERR_ARG, kw
    for kw in (dict(q=P + 4), dict(k=P + 8), dict(v=P + 4), dict(cos=P + 4), dict(out=P + 4), dict(ldq=514), dict(ldk=257)):
        assert append(b, **kw) == _lib.Q6W_ERR_ALIGN, kw
    assert append(batch(query_starts=P), T=0) == _lib.Q6W_OK  # nothing to do


def test_attention_arguments():
    b = batch()
    assert attend(None) == _lib.Q6W_ERR_ARG
    for kw in (dict(H=6), dict(H=0), dict(T=-1), dict(T=4), dict(q=None), dict(out=None), dict(ldq=508), dict(ws=None),
               dict(n=64), dict(P_len=5), dict(prefix=P, P_len=-1)):
        assert attend(b, **kw) == _lib.Q6W_ERR_ARG, kw
    for kw in (dict(q=P + 4), dict(out=P + 8), dict(ldq=514), dict(ws=P + 16)):
        assert attend(b, **kw) == _lib.Q6W_ERR_ALIGN, kw
    # a kv head's part of a page is too small for one copy
    small = dict(head_dim=16, head_stride=16, slot_stride=64, page_stride=64, page_size=1)
    assert attend(batch(**small)) == _lib.Q6W_ERR_ARG and "128 bytes" in message()
    assert attend(batch(query_starts=P), T=0) == _lib.Q6W_OK


def test_workspace_sizes():
    lib = _lib.load()
    size = lib.q6w_paged_workspace_bytes
    decode = size(batch(), 3, 8, 0)
    assert decode > 0 and size(batch(), 3, 8, 100) > decode
    assert size(batch(query_starts=P), 500, 8, 0) > 0
    assert size(batch(query_starts=P), 500, 8, 9000) > size(batch(query_starts=P), 500, 8, 0)
    for bad in (size(None, 3, 8, 0), size(batch(), 4, 8, 0), size(batch(), 3, 7, 0), size(batch(), 3, 8, -1),
                size(batch(head_dim=20), 3, 8, 0)):
        assert bad == 0


def test_python_ops_refuse_the_cpu():
    pool, table, lens = torch.zeros(2, 16, 2, 64), torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q, k = torch.zeros(1, 4, 64), torch.zeros(1, 2, 64)
    tab = torch.zeros(16, 32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_append(q, k, k, tab, tab, pool, pool, table, lens)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_attention(q, pool, pool, table, lens)
    with pytest.raises(ValueError):
        ops.shared_prefix_attention(q, pool, pool, table[0], 3, table, lens)


def test_rows_are_counted_in_32_bits():
    """2^24 tokens of 128 heads: the row numbers of the attention kernels would wrap."""
    many = batch(kv_heads=1, head_dim=16, slot_stride=16, page_stride=256, head_stride=16, query_starts=P)
    for kw in (dict(), dict(prefix=P, P_len=5)):
        assert attend(many, T=1 << 24, H=128, ldq=2048, **kw) == _lib.Q6W_ERR_ARG
        assert "32 bits" in message()
        # one head fewer passes this check and stops at the next one
        assert attend(many, T=1 << 24, H=127, ldq=2048, ws=None, **kw) == _lib.Q6W_ERR_ARG
        assert "workspace" in message()


def test_stall_diagnostic_arguments():
    stall = _lib.load().q6w_selftest_paged_stall
    assert stall(-1) == _lib.Q6W_ERR_ARG and stall((1 << 31) + 1) == _lib.Q6W_ERR_ARG
    assert stall(0) == _lib.Q6W_OK


def test_workspace_of_refused_calls_is_0():
    """What the attention calls refuse by shape has no workspace."""
    size = _lib.load().q6w_paged_workspace_bytes
    small = dict(head_dim=16, head_stride=16, slot_stride=64, page_stride=64)
    assert size(batch(**small, page_size=1), 3, 8, 0) == 0
    assert size(batch(**small, page_size=2), 3, 8, 0) > 0
    assert size(batch(**small, page_size=2, kv_dtype=1), 3, 8, 0) == 0
    many = dict(kv_heads=1, head_dim=16, slot_stride=16, page_stride=256, head_stride=16, query_starts=P)
    assert size(batch(**many), 1 << 24, 128, 0) == 0 < size(batch(**many), 1 << 24, 127, 0)


def test_check_status_refuses_the_cpu():
    with pytest.raises(ValueError, match="CUDA"):
        ops.check_status(torch.zeros(1, dtype=torch.int32))
