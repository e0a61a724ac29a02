"""Device codec and linear ops over the C ABI (torch tensors as plumbing).

These mirror the reference's codec functions (quantization/q6w_format.py)
with the work done by the sm_100a kernels: same names, same argument
meaning, same ValueError messages for malformed input.  Results are CUDA
tensors on ``device``.
"""

import json
import math
from pathlib import Path

import numpy as np
import torch

from . import _lib
from .format import HEADER, MAGIC, VERSION, Q6WImage


def _dev(device):
    d = torch.device(device)
    if d.type != "cuda":
        raise ValueError("q6w_b200 ops run on CUDA devices only")
    return d


def _bytes_to_device(data, device):
    buf = torch.frombuffer(bytearray(data), dtype=torch.uint8) if len(data) else torch.empty(0, dtype=torch.uint8)
    return buf.to(device, non_blocking=False)


def unpack_signed_int6(data, rows, columns, device="cuda"):
    """Decode packed Q6 bytes to int8 codes [rows, columns] on the GPU.

    Same contract as quantization/q6w_format.py:67-81 (the result is a CUDA
    int8 tensor instead of a numpy array).  ``data`` is bytes-like or a
    CUDA uint8 tensor.
    """
    if columns % 4:
        raise ValueError("Q6 row width must be divisible by four")
    expected = rows * columns * 6 // 8
    device = _dev(device)
    packed = data if isinstance(data, torch.Tensor) else _bytes_to_device(data, device)
    if packed.numel() != expected:
        raise ValueError(f"Packed Q6 length mismatch: expected {expected}, got {packed.numel()}")
    out = torch.empty((rows, columns), dtype=torch.int8, device=device)
    lib = _lib.load()
    with torch.cuda.device(device):
        _lib.check(lib.q6w_unpack(packed.data_ptr(), out.data_ptr(), rows, columns, _lib.stream_handle()), "q6w_unpack")
    return out


def dequantize_rows(packed, scales, rows, columns):
    """``float32(q) * scale[row]`` on the GPU (quantization/q6w_format.py:257-259)."""
    out = torch.empty((rows, columns), dtype=torch.float32, device=packed.device)
    lib = _lib.load()
    with torch.cuda.device(packed.device):
        _lib.check(lib.q6w_dequant(packed.data_ptr(), scales.data_ptr(), out.data_ptr(), rows, columns,
                                   _lib.stream_handle()), "q6w_dequant")
    return out


def quantize_rows(tensor, device="cuda"):
    """Row-wise int6 quantization + packing on the GPU: the device half of the
    Q6W writer (quantization/q6w_format.py:84-98 and 52-64).

    Codes and scales are bit-identical to the reference's ``quantize_rows``
    (same FP32 division and round-half-even); the codes come back already
    packed.  Returns (packed uint8 [rows*cols*3/4], scales float32 [rows],
    stats dict) with packed/scales on ``device``; the stats are summed in
    FP64 and agree with the reference's FP32 reductions to their rounding.
    """
    device = _dev(device)
    w = tensor.detach().to(device=device, dtype=torch.float32).contiguous()
    if w.ndim != 2:
        raise ValueError("Per-output-row quantization requires a matrix")
    rows, cols = w.shape
    if cols % 4:
        raise ValueError("Q6 rows must be 2D and have a width divisible by four")
    packed = torch.empty(rows * cols * 3 // 4, dtype=torch.uint8, device=device)
    scales = torch.empty(rows, dtype=torch.float32, device=device)
    row_err = torch.empty((max(rows, 1), 3), dtype=torch.float64, device=device)
    stats = torch.zeros(3, dtype=torch.float64, device=device)
    lib = _lib.load()
    with torch.cuda.device(device):
        _lib.check(lib.q6w_quantize_rows(w.data_ptr(), rows, cols, packed.data_ptr(), scales.data_ptr(),
                                         row_err.data_ptr(), stats.data_ptr(), _lib.stream_handle()),
                   "q6w_quantize_rows")
    st = stats.tolist()
    return packed, scales, {"max_abs_error": st[0], "mean_abs_error": st[1], "rmse": st[2]}


_LINEAR_WS = {}  # device index -> cached workspace of the tensor-core linear


def _linear_workspace(device, nbytes):
    buf = _LINEAR_WS.get(device.index)
    if buf is None or buf.numel() < nbytes:
        raw = torch.zeros(nbytes + 256, dtype=torch.uint8, device=device)
        off = (-raw.data_ptr()) % 256
        buf = raw[off: off + nbytes]
        _LINEAR_WS[device.index] = buf
    return buf


def linear_workspace_bytes(rows, columns, n):
    """Workspace the tensor-core linear needs for this shape (0: FP32 kernels)."""
    return int(_lib.load().q6w_linear_workspace_bytes(rows, columns, n))


def q6w_linear(x, packed, scales, rows, columns, tensor_cores=True):
    """``x @ dequant(W).T`` for x [..., columns] FP32 on the GPU -> [..., rows].

    The ``nn.Linear`` of the cached step (torch_benchmark.py:105-107, 121,
    123, 125).  Batches of 16 or more rows whose width is a multiple of 128
    run on the tcgen05 tensor cores (q6w_linear_ex, a cached workspace per
    device; agreement with FP64 within 1e-4 * sum|w x| per element); other
    shapes, and ``tensor_cores=False``, run the FP32 kernels (1e-5).
    """
    if x.dtype != torch.float32 or x.shape[-1] != columns:
        raise ValueError("x must be float32 with last dimension == columns")
    xs = x.reshape(-1, columns).contiguous()
    n = xs.shape[0]
    y = torch.empty((n, rows), dtype=torch.float32, device=x.device)
    lib = _lib.load()
    need = linear_workspace_bytes(rows, columns, n) if tensor_cores else 0
    with torch.cuda.device(x.device):
        if need:
            ws = _linear_workspace(x.device, need)
            _lib.check(lib.q6w_linear_ex(packed.data_ptr(), scales.data_ptr(), xs.data_ptr(), y.data_ptr(), rows,
                                         columns, n, ws.data_ptr(), ws.numel(), _lib.stream_handle()),
                       "q6w_linear_ex")
        else:
            _lib.check(lib.q6w_linear(packed.data_ptr(), scales.data_ptr(), xs.data_ptr(), y.data_ptr(), rows,
                                      columns, n, _lib.stream_handle()), "q6w_linear")
    return y.reshape(*x.shape[:-1], rows)


class DeviceImage:
    """A verified Q6W file uploaded unchanged to one GPU.

    The device blob is the file's bytes (64-byte aligned sections, the
    allocation itself 256-byte aligned), so every tensor is addressed in
    place: ``qmat(name)`` returns (packed view, scales view, rows, cols).
    """

    def __init__(self, image, device):
        self.image = image
        self.device = _dev(device)
        self.blob = _bytes_to_device(image.blob, self.device)

    def _view(self, offset, nbytes):
        return self.blob[offset: offset + nbytes]

    def qmat(self, name):
        e = self.image.tensors[name]
        rows, cols = e["shape"]
        packed = self._view(e["data_offset"], e["data_bytes"])
        scales = self._view(e["scale_offset"], e["scale_bytes"]).view(torch.float32)
        return packed, scales, rows, cols

    def fp32(self, name):
        e = self.image.tensors[name]
        return self._view(e["data_offset"], e["data_bytes"]).view(torch.float32).view(*e["shape"])


def load_dequantized_state(binary_path, manifest_path, checkpoint_state=None, device="cuda"):
    """Q6W file -> dict of dequantized FP32 CUDA tensors, plus the manifest.

    Same checks and result keys as quantization/q6w_format.py:230-268 (SHA,
    header, offsets; ``output.weight`` aliases ``tok_embeddings.weight``), with
    the unpack and dequantization done on the GPU.  ``checkpoint_state``, when
    given, supplies extra non-file tensors and is copied to ``device``.
    """
    image = Q6WImage(binary_path, manifest_path)
    dimg = DeviceImage(image, device)
    result = {}
    if checkpoint_state:
        result = {k: v.detach().to(device=dimg.device, dtype=torch.float32).clone() for k, v in checkpoint_state.items()}
    for name, e in image.tensors.items():
        if e["dtype"] == "signed_int6_twos_complement":
            packed, scales, rows, cols = dimg.qmat(name)
            result[name] = dequantize_rows(packed, scales, rows, cols)
        else:
            result[name] = dimg.fp32(name).clone()
    result["output.weight"] = result["tok_embeddings.weight"]
    return result, image.manifest


def linear_argmax(x, packed, scales, rows, columns, want_logits=False):
    """Fused ``x @ dequant(W).T`` + first-maximum argmax per row.

    Returns (argmax int32 [n], logits [n, rows] or None).
    """
    xs = x.reshape(-1, columns).contiguous()
    n = xs.shape[0]
    am = torch.empty(n, dtype=torch.int32, device=x.device)
    lg = torch.empty((n, rows), dtype=torch.float32, device=x.device) if want_logits else None
    scratch = torch.empty(max(1, n), dtype=torch.int64, device=x.device)
    lib = _lib.load()
    with torch.cuda.device(x.device):
        _lib.check(lib.q6w_linear_argmax(packed.data_ptr(), scales.data_ptr(), xs.data_ptr(),
                                         lg.data_ptr() if lg is not None else None, am.data_ptr(),
                                         scratch.data_ptr(), scratch.numel() * 8, rows, columns, n,
                                         _lib.stream_handle()), "q6w_linear_argmax")
    return am, lg


def sample(logits, history, history_len, rng_state, temperature, top_p=0.9, repetition_penalty=1.0,
           no_repeat_ngram_size=0, stop_ids=(), min_new_tokens=0, stop_token_bias=0.0, stop_token_bias_after=None):
    """The reference's per-step sampling (torch_benchmark.py:272-285) on rows
    of logits, on the GPU: repetition penalty and n-gram blocking over each
    row's ``history`` (its first ``history_len`` tokens; history_len is also
    the decode index), stop-id masking / bias, then temperature / top-p
    sampling from each row's XorShift64 state.

    logits [n, V] float32; history [n, H] int32; history_len [n] int32;
    rng_state [n] int64 (the generator states, advanced in place).  Returns
    int32 tokens [n].
    """
    n, V = logits.shape
    lg = logits.contiguous()
    hist = history.to(torch.int32).contiguous()
    hl = history_len.to(torch.int32).contiguous()
    if rng_state.dtype != torch.int64 or not rng_state.is_contiguous():
        raise ValueError("rng_state must be a contiguous int64 tensor")
    out = torch.empty(n, dtype=torch.int32, device=logits.device)
    stop = sorted(set(int(t) for t in stop_ids))
    arr = (_lib.c_int32 * max(1, len(stop)))(*stop) if stop else None
    bias_after = min_new_tokens if stop_token_bias_after is None else stop_token_bias_after
    sa = _lib.SampleArgs(float(temperature), float(top_p), float(repetition_penalty), int(no_repeat_ngram_size),
                         float(stop_token_bias), int(bias_after), None)
    lib = _lib.load()
    with torch.cuda.device(logits.device):
        _lib.check(lib.q6w_sample(lg.data_ptr(), V, n, V, hist.data_ptr() if hist.numel() else None,
                                  hist.shape[1] if hist.dim() == 2 else 0, hl.data_ptr(), rng_state.data_ptr(), sa,
                                  arr, len(stop), int(min_new_tokens), out.data_ptr(), _lib.stream_handle()),
                   "q6w_sample")
    return out


def rmsnorm(x, weight, eps):
    """Row-wise RMSNorm of x [..., length] (torch_benchmark.py:22-24)."""
    xs = x.reshape(-1, x.shape[-1]).contiguous()
    out = torch.empty_like(xs)
    lib = _lib.load()
    with torch.cuda.device(x.device):
        _lib.check(lib.q6w_rmsnorm(xs.data_ptr(), weight.data_ptr(), out.data_ptr(), xs.shape[0], xs.shape[1],
                                   float(eps), _lib.stream_handle()), "q6w_rmsnorm")
    return out.view_as(x)


def gqa_attention(queries, keys, values, lengths, groups_per_kv):
    """Decode attention over per-sequence caches.

    queries [n, heads, hd]; keys/values [n, max_len, kv_heads, hd] (any
    sequence stride); lengths int32 [n] on the device.  Returns [n, heads, hd].
    """
    n, H, hd = queries.shape
    _, max_len, kv, _ = keys.shape
    q = queries.contiguous()
    out = torch.empty_like(q)
    if keys.stride()[1:] != (kv * hd, hd, 1) or values.stride() != keys.stride():
        raise ValueError("keys/values must be [n, max_len, kv_heads, head_dim] with contiguous rows")
    lib = _lib.load()
    with torch.cuda.device(q.device):
        _lib.check(lib.q6w_gqa_attention(q.data_ptr(), keys.data_ptr(), values.data_ptr(), out.data_ptr(),
                                         lengths.to(torch.int32).contiguous().data_ptr(), n, kv, groups_per_kv, hd,
                                         max_len, keys.stride(0), _lib.stream_handle()), "q6w_gqa_attention")
    return out


# ---- serving from a paged cache -------------------------------------------------

_I32, _F32, _F16 = torch.int32, torch.float32, torch.float16
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # (a build without CUDA has none)


def _int32(name, t, dev, dim):
    """Address of an int32 tensor with contiguous rows on device ``dev``."""
    if t.dtype is not _I32 or t.get_device() != dev or t.dim() != dim or (t.stride(-1) != 1 and t.shape[-1] > 1):
        raise ValueError(f"{name} must be an int32 tensor of {dim} dimension(s) on cuda:{dev} with contiguous rows")
    return t.data_ptr()


def _token_rows(name, t, heads, hd, dev):
    """(tokens, heads, token stride) of t [T, heads, hd] FP32: heads contiguous, tokens at any stride."""
    if t.dtype is not _F32 or t.get_device() != dev or t.dim() != 3:
        raise ValueError(f"{name} must be float32 [tokens, heads, {hd}] on cuda:{dev}")
    T, H, d = t.shape
    st, sh, sd = t.stride()
    if d != hd or (heads is not None and H != heads):
        raise ValueError(f"{name} must be float32 [tokens, heads, {hd}] on cuda:{dev}")
    if T and (sd != 1 or (sh != hd and H > 1)):
        raise ValueError(f"the heads of a token of {name} must be contiguous")
    return T, H, st if T > 1 else H * hd


def _paged_batch(key_pages, value_pages, page_table, lengths, query_starts, status, n_tokens):
    """(q6w_paged_batch as bytes, device index, kv_heads, head_dim)."""
    dev = key_pages.get_device()
    if dev < 0:
        raise ValueError("q6w_b200 ops run on CUDA devices only")
    dtype = key_pages.dtype
    if (dtype is not _F32 and dtype is not _F16) or value_pages.dtype is not dtype or value_pages.get_device() != dev:
        raise ValueError("key_pages and value_pages must both be float32 or float16 on one device")
    strides = key_pages.stride()
    if len(strides) != 4 or value_pages.shape != key_pages.shape or value_pages.stride() != strides:
        raise ValueError("key_pages and value_pages must be [pages, page_size, kv_heads, head_dim] with equal strides")
    pages, page_size, kv_heads, hd = key_pages.shape
    sp, ss, sh, sd = strides
    if sd != 1:
        raise ValueError("the last dimension of the pages must be contiguous")
    table = _int32("page_table", page_table, dev, 2)
    n, width = page_table.shape
    lens = _int32("lengths", lengths, dev, 1)
    if lengths.shape[0] != n:
        raise ValueError(f"lengths must have one entry for each of the {n} rows of page_table")
    starts = flags = 0
    if query_starts is not None:
        starts = _int32("query_starts", query_starts, dev, 1)
        if query_starts.shape[0] != n + 1:
            raise ValueError(f"query_starts must have {n + 1} entries")
    elif n_tokens != n:
        raise ValueError(f"{n_tokens} tokens of {n} sequences need query_starts")
    if status is not None:
        flags = _int32("status", status, dev, 1)
        if status.shape[0] < 1:
            raise ValueError("status must have an entry")
    return _lib.PAGED_BATCH.pack(key_pages.data_ptr(), value_pages.data_ptr(), 0 if dtype is _F32 else 1, pages, page_size,
                                 kv_heads, hd, sp, ss, sh, n, width, table, page_table.stride(0), lens, starts,
                                 flags), dev, kv_heads, hd


def _on_device(dev, call, *args):
    """``call(*args, stream)`` with device ``dev`` and its current stream."""
    if torch._C._cuda_getDevice() == dev:
        return call(*args, _raw_stream(dev))
    with torch.cuda.device(dev):
        return call(*args, _raw_stream(dev))


def _rows_out(out, queries, T, H, hd, dev):
    if out is None:
        return queries.new_empty((T, H, hd))
    if out.shape != queries.shape or out.dtype is not _F32 or out.get_device() != dev or not out.is_contiguous():
        raise ValueError("out must be contiguous float32 of the queries' shape")
    return out


def paged_append(queries, keys, values, cos, sin, key_pages, value_pages, page_table, lengths, query_starts=None,
                 first_position=0, status=None, out=None):
    """Rotate a step's queries and keys (RoPE) and append its keys and values
    to the pages of their sequences, in one pass.

    queries [T, heads, hd] (or None), keys and values [T, kv_heads, hd]
    float32, tokens at any stride (parts of one QKV output, say); cos and sin
    [positions, hd / 2] (``Q6WCudaTransformer.freqs_cos`` / ``freqs_sin``).
    key_pages and value_pages [pages, page_size, kv_heads, hd] float32 or
    float16, page_size a power of two; page_table int32 [n, max_pages];
    lengths int32 [n], each sequence's tokens including this step's;
    query_starts int32 [n + 1], the step's tokens of every sequence (None:
    one token each).  ``first_position`` is added to a token's position for
    the rotation (the length of a shared prefix).  Returns the rotated
    queries, in ``out`` if given (which may be ``queries``); tokens that no
    sequence holds append nothing, their rows come back zero (in ``out``: as
    they were).

    ``status``: int32 [1] on the device, zeroed once; bit 0 is set when a
    length, page id or position is out of range or ``query_starts`` descends
    or leaves [0, T] (``check_status``).
    """
    T = keys.shape[0]
    batch, dev, kv_heads, hd = _paged_batch(key_pages, value_pages, page_table, lengths, query_starts, status, T)
    ldk = _token_rows("keys", keys, kv_heads, hd, dev)[2]
    Tv, _, ldv = _token_rows("values", values, kv_heads, hd, dev)
    H = ldq = 0
    q = rot = None
    Tq = T
    zero = out is None
    if queries is not None:
        Tq, H, ldq = _token_rows("queries", queries, None, hd, dev)
        out = _rows_out(out, queries, Tq, H, hd, dev)
        q, rot = queries.data_ptr(), out.data_ptr()
    if Tv != T or Tq != T:
        raise ValueError("queries, keys and values must have the same number of tokens")
    positions = cos.shape
    if (cos.dtype is not _F32 or sin.dtype is not _F32 or cos.get_device() != dev or sin.get_device() != dev
            or len(positions) != 2 or positions[1] * 2 != hd or sin.shape != positions or not cos.is_contiguous()
            or not sin.is_contiguous()):
        raise ValueError(f"cos and sin must be contiguous float32 [positions, {hd // 2}] on cuda:{dev}")
    lib = _lib.load()
    _lib.check(_on_device(dev, lib.q6w_paged_append, batch, T, H, q, ldq, keys.data_ptr(), ldk, values.data_ptr(), ldv,
                          cos.data_ptr(), sin.data_ptr(), positions[0], int(first_position), rot, zero),
               "q6w_paged_append")
    return out if queries is not None else None


def paged_attention(queries, key_pages, value_pages, page_table, lengths, query_starts=None, status=None, out=None):
    """Causal grouped-query attention of a step's tokens over paged caches:
    ``gqa_attention`` for one token a sequence, and the attention of prompts
    or chunks of prompts for more (``query_starts``).

    queries [T, heads, hd] float32 (rotated; tokens at any stride), the
    other arguments as ``paged_append`` takes them, after it has run: a token
    sees its sequence's positions up to its own.  Returns [T, heads, hd];
    a token without a visible key gives zeros, and so do rows of tokens that
    no sequence holds (in ``out``, if given, they stay as they were; ``out``
    must not overlap ``queries``).

    Single tokens are fastest without ``query_starts``, in a call of their
    own: with it every sequence takes tiles of 128 or 256 rows (tokens times
    heads of a kv head).
    """
    return _paged_attention(queries, key_pages, value_pages, None, 0, page_table, lengths, query_starts, status, out)


def shared_prefix_attention(queries, key_pages, value_pages, prefix_pages, prefix_length, page_table, lengths,
                            query_starts=None, status=None, out=None):
    """``paged_attention`` of a batch whose sequences all continue one prefix:
    every token also sees the ``prefix_length`` tokens in pages
    ``prefix_pages`` (int32, on the device) of the same pool, which are read
    once for the whole batch.  page_table and lengths describe the sequences'
    own tokens (a length may be 0); their positions start at prefix_length
    (``paged_append(..., first_position=prefix_length)``).
    """
    pages = _int32("prefix_pages", prefix_pages, key_pages.get_device(), 1)
    if prefix_length < 0 or prefix_length > prefix_pages.shape[0] * key_pages.shape[1]:
        raise ValueError("prefix_length is more than prefix_pages hold")
    return _paged_attention(queries, key_pages, value_pages, pages, int(prefix_length), page_table, lengths,
                            query_starts, status, out)


def _paged_attention(queries, key_pages, value_pages, prefix_pages, prefix_length, page_table, lengths, query_starts,
                     status, out):
    batch, dev, _, hd = _paged_batch(key_pages, value_pages, page_table, lengths, query_starts, status, queries.shape[0])
    T, H, ldq = _token_rows("queries", queries, None, hd, dev)
    zero = out is None
    out = _rows_out(out, queries, T, H, hd, dev)
    lib = _lib.load()
    need = lib.q6w_paged_workspace_bytes(batch, T, H, prefix_length)
    ws = key_pages.new_empty(need, dtype=torch.uint8)  # (stream-ordered: a call's own, released as it returns)
    _lib.check(_on_device(dev, lib.q6w_shared_prefix_attention, batch, prefix_pages, prefix_length, T, H,
                          queries.data_ptr(), ldq, out.data_ptr(), zero, ws.data_ptr(), need), "paged attention")
    return out


def check_status(status):
    """Synchronise and raise Q6WError if a paged call set ``status`` (then clear it)."""
    dev = status.get_device()
    if dev < 0 or status.dtype is not _I32 or status.numel() < 1:
        raise ValueError("status must be an int32 tensor on a CUDA device")
    _lib.check(_on_device(dev, _lib.load().q6w_workspace_status, status.data_ptr()), "paged cache")
