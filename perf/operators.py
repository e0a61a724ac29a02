"""Measured cases of the paged-cache serving operators.

Three operators that serve many requests from one pool of cache pages:

* ``append``  -- rotate the new tokens' queries and keys (RoPE) and write their
  keys and values into the pages of their sequences;
* ``attend``  -- causal grouped-query attention of the new tokens over the paged
  caches, one token a sequence (decode) or several (a prompt, a chunk of one);
* ``prefix``  -- the same for a batch whose sequences all continue one cached
  prefix, which is kept in the pool once.

Each case is run in two forms: in elementary torch operations (``own`` false)
and through the framework's operators (``own`` true).  ``exact`` evaluates the
definition in 64 bits, sequence by sequence.
"""

import math
import sys
from pathlib import Path

import torch

own = False

_OPS = None


def _ops():
    """The framework's operators (imported on first use)."""
    global _OPS
    if _OPS is None:
        pkg = str(Path(__file__).resolve().parents[1] / "tinyllm-pynq-z2_b200")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from q6w_b200 import ops

        _OPS = ops
    return _OPS


# ---- cases -------------------------------------------------------------------
#
# n sequences; sequence i holds past_i cached tokens before the call and gets
# new_i tokens in it, both spread evenly over [min_past, max_past] and
# [min_new, max_new].  prefix: tokens of the shared prefix (operator "prefix";
# past then counts a sequence's own tokens).  kv: the storage type of the pages.


def _case(name, op, n, heads, kv_heads, head_dim, kv, page, past, new, prefix=0):
    return {"name": name, "op": op, "n": n, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "kv": kv,
            "page": page, "min_past": past[0], "max_past": past[1], "min_new": new[0], "max_new": new[1],
            "prefix": prefix}


def listed():
    return [
        # one decode step of one request of the 1.1B-shape model: latency
        _case("append_step_1b_b1", "append", 1, 32, 4, 64, "float32", 16, (255, 255), (1, 1)),
        # the ragged prompts of the tiny model's batched prefill
        _case("append_prompts_tiny", "append", 2048, 8, 4, 16, "float32", 16, (0, 0), (8, 256)),
        # ragged chunks of prompts behind earlier chunks, FP16 pages, wide heads
        _case("append_chunks_f16", "append", 64, 32, 8, 128, "float16", 64, (0, 2048), (1, 511)),
        # decode of one long request: the key axis has to be split
        _case("decode_long_b1", "attend", 1, 32, 4, 64, "float32", 16, (32767, 32767), (1, 1)),
        # the tiny model's 8192 concurrent requests of 20 + 128 tokens
        _case("decode_tiny_8192", "attend", 8192, 8, 4, 16, "float32", 16, (19, 146), (1, 1)),
        # 64 ragged requests of the 1.1B shape, FP16 pages
        _case("decode_ragged_f16", "attend", 64, 32, 4, 64, "float16", 16, (127, 16383), (1, 1)),
        # odd batch, five query heads a KV head, 128-wide heads
        _case("decode_odd_groups", "attend", 37, 20, 4, 128, "float32", 32, (0, 4999), (1, 1)),
        # chunked prefill of a few requests
        _case("chunk_prefill", "attend", 8, 32, 4, 64, "float32", 16, (0, 1500), (201, 597)),
        # long prompts behind long contexts, FP16 pages
        _case("prefill_long_f16", "attend", 2, 32, 8, 128, "float16", 64, (2048, 6144), (2048, 2048)),
        # a few requests behind one system prompt
        _case("prefix_8", "prefix", 8, 32, 4, 64, "float32", 16, (0, 127), (1, 1), 2048),
        # a large batch behind one long prompt
        _case("prefix_1024", "prefix", 1024, 32, 4, 64, "float32", 16, (19, 147), (1, 1), 4096),
        # a document behind which many short answers are written, FP16 pages
        _case("prefix_256_f16", "prefix", 256, 32, 8, 128, "float16", 64, (0, 511), (1, 1), 16384),
    ]


def _logint(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999))))))


def _time_like(case):
    w = work(case)
    return w["bytes"] / 6e12 + w["flops"] / 2e14


def _plain_elements(c):
    """Elements of the largest tensors that the plain form makes: scores, gathered pages."""
    longest = c["max_past"] + c["max_new"]
    scores = c["n"] * c["heads"] * c["max_new"] * (longest + c["prefix"])
    return max(scores, 2 * c["n"] * longest * c["kv_heads"] * c["head_dim"])


def draw(rng):
    most = max(_time_like(c) for c in listed())
    while True:
        op = rng.choice(["append", "attend", "attend", "prefix"])
        n = _logint(rng, 1, 8192 if op != "prefix" else 2048)
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16])
        head_dim = rng.choice([16, 32, 64, 128])
        page = rng.choice([8, 16, 32, 64, 128])
        long = _logint(rng, 1, 32768)
        past = (min(long, rng.choice([0, 1, long // 3, long])), long)
        many = op != "prefix" and rng.random() < 0.5
        new = (1, _logint(rng, 2, 2048)) if many else (1, 1)
        prefix = _logint(rng, 17, 32768) if op == "prefix" else 0
        c = _case("", op, n, heads, kv_heads, head_dim, rng.choice(["float32", "float16"]), page, past, new, prefix)
        del c["name"]
        small = op == "append" and _pool_elements(c) <= 1 << 29 and _tokens(c) * heads * head_dim <= 1 << 28
        if (small or (op != "append" and _plain_elements(c) <= 1 << 30)) and _time_like(c) <= most:
            return c


# ---- shapes of a case ----------------------------------------------------------


def _spread(lo, hi, n):
    return [hi] if n == 1 else [lo + (i * (hi - lo)) // (n - 1) for i in range(n)]


def _counts(case):
    """(past, new) of every sequence, in a fixed pairing that mixes short and long."""
    n = case["n"]
    past = _spread(case["min_past"], case["max_past"], n)
    new = _spread(case["min_new"], case["max_new"], n)
    step = next(s for s in (7, 11, 13, 17, 19, 23) if math.gcd(s, n) == 1 or s == 23)
    return [(past[i], new[(i * step) % n]) for i in range(n)]


def _tokens(case):
    return sum(b for _, b in _counts(case))


def _pages_of(case):
    return [-(-(a + b) // case["page"]) for a, b in _counts(case)]


def _pool_pages(case):
    return sum(_pages_of(case)) + -(-case["prefix"] // case["page"]) + 3


def _pool_elements(case):
    return _pool_pages(case) * case["page"] * case["kv_heads"] * case["head_dim"]


def work(case):
    """Bytes and operations of the operator itself: every input read once, every output written once."""
    H, KV, hd = case["heads"], case["kv_heads"], case["head_dim"]
    es = 2 if case["kv"] == "float16" else 4
    counts = _counts(case)
    T = _tokens(case)
    ids = 4 * sum(_pages_of(case)) + 4 * case["n"]
    row = KV * hd * es * 2  # a token's key and value in the pages
    if case["op"] == "append":
        positions = len({p for a, b in counts for p in (a, a + b - 1)})
        return {"bytes": 4 * T * hd * (2 * H + 2 * KV) + T * row + 4 * positions * hd + ids, "flops": 3 * T * (H + KV) * hd}
    cached = sum(a + b for a, b in counts) + case["prefix"]
    seen = sum(a * b + b * (b + 1) // 2 for a, b in counts) + T * case["prefix"]
    return {"bytes": cached * row + 8 * T * H * hd + ids, "flops": 4 * seen * H * hd}


# ---- inputs --------------------------------------------------------------------


def prepare(case, seed):
    """What a serving program holds before the call: the pool of pages with the
    earlier tokens in it, the page tables, the step's lengths and the output of
    the fused QKV projection (append) or the rotated queries (attend, prefix)."""
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(int(seed))
    host = torch.Generator().manual_seed(int(seed))
    H, KV, hd, ps, n = case["heads"], case["kv_heads"], case["head_dim"], case["page"], case["n"]
    counts = _counts(case)
    order = torch.randperm(n, generator=host).tolist()
    counts = [counts[i] for i in order]
    new = torch.tensor([b for _, b in counts])
    lengths = torch.tensor([a + b for a, b in counts])
    T = int(new.sum())
    pages = (lengths + ps - 1) // ps
    width = int(pages.max())
    n_pages = _pool_pages(case)
    ids = torch.randperm(n_pages, generator=host).int()
    table = torch.full((n, width), -1, dtype=torch.int32)
    held = torch.arange(width)[None, :] < pages[:, None]
    table[held] = ids[: int(pages.sum())]
    dtype = getattr(torch, case["kv"])
    shape = (n_pages, ps, KV, hd)
    s = {"op": case["op"], "longest": int(lengths.max()), "most_new": int(new.max()), "prefix_length": case["prefix"],
         "key_pages": torch.randn(shape, generator=g, device=dev, dtype=dtype),
         "value_pages": torch.randn(shape, generator=g, device=dev, dtype=dtype),
         "page_table": table.to(dev), "lengths": lengths.int().to(dev)}
    starts = torch.zeros(n + 1, dtype=torch.int32)
    starts[1:] = new.cumsum(0)
    # one token a sequence needs no starts: query i belongs to sequence i
    s["query_starts"] = None if case["max_new"] == 1 else starts.to(dev)
    if case["op"] == "append":
        qkv = torch.randn(T, (H + 2 * KV) * hd, generator=g, device=dev)
        s["queries"] = qkv[:, : H * hd].view(T, H, hd)
        s["keys"] = qkv[:, H * hd: (H + KV) * hd].view(T, KV, hd)
        s["values"] = qkv[:, (H + KV) * hd:].view(T, KV, hd)
        inv = 1.0 / (10000.0 ** (torch.arange(0, hd, 2).float() / hd))
        ang = torch.outer(torch.arange(s["longest"]).float(), inv)
        s["cos"], s["sin"] = ang.cos().to(dev), ang.sin().to(dev)
    else:
        # rotated queries; some heads attend sharply, some evenly
        sharp = torch.linspace(0.25, 2.0, H, device=dev)[None, :, None]
        s["queries"] = torch.randn(T, H, hd, generator=g, device=dev) * sharp
        used = int(pages.sum())
        s["prefix_pages"] = ids[used: used + -(-case["prefix"] // ps)].to(dev)
    return s


# ---- one pass --------------------------------------------------------------------


def run(state):
    s = state
    if s["op"] == "append":
        if own:
            q = _ops().paged_append(s["queries"], s["keys"], s["values"], s["cos"], s["sin"], s["key_pages"],
                                    s["value_pages"], s["page_table"], s["lengths"], s["query_starts"])
        else:
            q = _plain_append(s)
        return {"queries": q, "key_pages": s["key_pages"], "value_pages": s["value_pages"]}
    if s["op"] == "attend":
        if own:
            return _ops().paged_attention(s["queries"], s["key_pages"], s["value_pages"], s["page_table"],
                                          s["lengths"], s["query_starts"])
        return _plain_attention(s)
    if own:
        return _ops().shared_prefix_attention(s["queries"], s["key_pages"], s["value_pages"], s["prefix_pages"],
                                              s["prefix_length"], s["page_table"], s["lengths"], s["query_starts"])
    return _plain_attention(s)


def _token_places(s):
    """(sequence, position) of every new token."""
    T, n, dev = s["queries"].shape[0], s["lengths"].shape[0], s["lengths"].device
    if s["query_starts"] is None:
        return torch.arange(n, device=dev), s["lengths"].long() - 1
    starts = s["query_starts"].long()
    new = starts[1:] - starts[:-1]
    seq = torch.repeat_interleave(torch.arange(n, device=dev), new, output_size=T)
    return seq, s["lengths"].long()[seq] - new[seq] + torch.arange(T, device=dev) - starts[seq]


def _rotated(x, c, sn):
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * c - b * sn, a * sn + b * c), dim=-1).flatten(-2)


def _plain_append(s):
    seq, pos = _token_places(s)
    ps = s["key_pages"].shape[1]
    page, slot = s["page_table"][seq, pos // ps].long(), pos % ps
    c, sn = s["cos"][pos][:, None, :], s["sin"][pos][:, None, :]
    s["key_pages"][page, slot] = _rotated(s["keys"], c, sn).to(s["key_pages"].dtype)
    s["value_pages"][page, slot] = s["values"].to(s["value_pages"].dtype)
    return _rotated(s["queries"], c, sn)


def _plain_attention(s):
    """Softmax attention in FP32 over the gathered pages, every sequence padded to the longest."""
    q = s["queries"]
    T, H, hd = q.shape
    KV, n, M, L = s["key_pages"].shape[2], s["lengths"].shape[0], s["most_new"], s["longest"]
    table = s["page_table"].clamp(min=0).long()
    k = s["key_pages"][table].flatten(1, 2)[:, :L].float().permute(0, 2, 3, 1)    # [n, KV, hd, L]
    v = s["value_pages"][table].flatten(1, 2)[:, :L].float().permute(0, 2, 1, 3)  # [n, KV, L, hd]
    seq, pos = _token_places(s)
    at = torch.zeros_like(seq) if s["query_starts"] is None else torch.arange(T, device=q.device) - s["query_starts"].long()[seq]
    rows = torch.zeros(n, M, H, hd, device=q.device)
    rows[seq, at] = q
    last = torch.full((n, M), -1, device=q.device)
    last[seq, at] = pos
    rows = rows.view(n, M, KV, H // KV, hd).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [n, KV, M * rep, hd]
    score = torch.matmul(rows, k).div_(math.sqrt(hd)).view(n, KV, M, H // KV, L)
    hidden = torch.arange(L, device=q.device)[None, None, :] > last[:, :, None]
    score.masked_fill_(hidden[:, None, :, None, :], -math.inf)
    m = score.amax(-1, keepdim=True)
    if s["prefix_length"]:
        P = s["prefix_length"]
        pages = s["prefix_pages"].long()
        pk = s["key_pages"][pages].flatten(0, 1)[:P].float().permute(1, 2, 0)     # [KV, hd, P]
        pv = s["value_pages"][pages].flatten(0, 1)[:P].float().permute(1, 0, 2)   # [KV, P, hd]
        every = rows.permute(1, 0, 2, 3).flatten(1, 2)                            # [KV, n * M * rep, hd]
        first = torch.matmul(every, pk).div_(math.sqrt(hd)).view(KV, n, M, H // KV, P).permute(1, 0, 2, 3, 4)
        m = torch.maximum(m, first.amax(-1, keepdim=True))
    m = m.clamp(min=torch.finfo(torch.float32).min)
    p = score.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.flatten(2, 3), v).view(n, KV, M, H // KV, hd)
    if s["prefix_length"]:
        p = first.sub_(m).exp_()
        total = total + p.sum(-1, keepdim=True)
        own_rows = p.permute(1, 0, 2, 3, 4).flatten(1, 3)
        out = out + torch.matmul(own_rows, pv).view(KV, n, M, H // KV, hd).permute(1, 0, 2, 3, 4)
    out = (out / total).permute(0, 2, 1, 3, 4).flatten(2, 3)                      # [n, M, H, hd]
    return out[seq, at]


# ---- the definition in 64 bits -----------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    lengths = s["lengths"].tolist()
    table = s["page_table"].cpu()
    n, ps = case["n"], case["page"]
    starts = list(range(n + 1)) if s["query_starts"] is None else s["query_starts"].tolist()
    q = s["queries"].double()
    T, H, hd = q.shape
    if case["op"] == "append":
        kp, vp = s["key_pages"].double(), s["value_pages"].double()
        place = torch.empty(T, 3, dtype=torch.long)
        for i in range(n):
            pos = torch.arange(lengths[i] - (starts[i + 1] - starts[i]), lengths[i])
            place[starts[i]: starts[i + 1]] = torch.stack((table[i][pos // ps].long(), pos % ps, pos), 1)
        page, slot, pos = place.to(q.device).unbind(1)
        # a pair of dimensions is a complex number, turned by the table's angle
        turn = torch.complex(s["cos"].double(), s["sin"].double())[pos][:, None, :]
        spin = lambda x: torch.view_as_real(torch.view_as_complex(x.double().unflatten(-1, (-1, 2)).contiguous()) * turn).flatten(-2)
        kp.index_put_((page, slot), spin(s["keys"]))
        vp.index_put_((page, slot), s["values"].double())
        return {"queries": spin(q), "key_pages": kp, "value_pages": vp}
    if 4 * sum((b - a) * x for a, b, x in zip(starts, starts[1:], lengths)) * H * hd + n * 2e8 > 4e12:
        return None
    KV = case["kv_heads"]
    out = torch.empty(T, H, hd, dtype=torch.float64, device=q.device)
    def rows_of(pages, count):
        at = pages[: -(-count // ps)].to(q.device).long()
        return [x[at].flatten(0, 1)[:count].double().transpose(0, 1) for x in (s["key_pages"], s["value_pages"])]
    pk, pv = rows_of(s["prefix_pages"], case["prefix"])
    for i in range(n):
        a, b, L = starts[i], starts[i + 1], lengths[i]
        k, v = rows_of(table[i], L)
        k, v = (torch.cat(x, 1) if case["prefix"] else x[1] for x in ((pk, k), (pv, v)))
        sc = torch.einsum("tgrd,gkd->gtrk", q[a:b].unflatten(1, (KV, H // KV)), k) / math.sqrt(hd)
        ahead = torch.arange(k.shape[1], device=q.device)[None, :] > torch.arange(b - a, device=q.device)[:, None] + (case["prefix"] + L - (b - a))
        w = torch.softmax(sc.masked_fill(ahead[None, :, None, :], -math.inf), -1)
        out[a:b] = torch.einsum("gtrk,gkd->tgrd", w, v).flatten(1, 2)
    return out
