"""Attention over a key-value cache and what keeps that cache, as cases that can be timed on one GPU.

Four operators of a program that serves a decoder: attention of a prompt (causal, with an optional window of recent
tokens and a few first tokens that stay visible), attention of one new token per sequence over a paged cache, storing
new keys and values in the cache's pages, and copying pages (a forked sequence, a compacted cache).

* ``q``, ``k``, ``v`` are [batch, tokens, heads, head_dim]; query head h reads key-value head h // (heads // kv_heads).
  The queries are the last tokens of the sequence: query t stands at position tokens_k - tokens_q + t.
* The token at position j is visible from position i if j <= i and (no window, or j > i - window, or j < sinks) and j
  lies before the sequence's length.  A row that sees nothing is zero.
* A cache is [pages, 2, kv_heads, page_size, head_dim], keys at 0 and values at 1; the token at position j of sequence s
  lies in page ``page_table[s, j // page_size]`` at place ``j % page_size``.

``own`` says which form ``run`` takes: elementary torch operations, or the library's operators.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
MOST_PROMPT = 16384 * 16384 // 2 * 8 * 128  # visible pairs x heads x head_dim of the largest listed prompt
MOST_CACHE = 1 << 29                         # values of the largest cache
MOST_READ = 64 * 2560 * 8 * 128              # tokens x kv_heads x head_dim that one decode step may read
MOST_APPEND = 2 * 4096 * 8 * 128
MOST_COPY = 4000 * 2 * 8 * 16 * 128


def listed() -> list:
    return [
        # a short prompt of one user on one rank of eight: a few heads, nothing to fill the chip with
        _prompt(1, 77, 77, 8, 1, 128, 0, 0, False, "fp16", "prompt-short"),
        # prompts of a batch, sliding window with sinks, the heads of a 4096-wide block on one GPU
        _prompt(2, 4096, 4096, 32, 8, 128, 1024, 4, False, "bf16", "prompt-window"),
        # a long document, everything visible, one rank of eight (64 query and 8 key-value heads in all); the largest
        _prompt(1, 16384, 16384, 8, 1, 128, 0, 0, False, "fp16", "prompt-long"),
        # the next piece of prompts whose beginning has been read before; ragged batch, odd length, narrow heads
        _prompt(3, 500, 5003, 12, 4, 64, 2048, 16, True, "bf16", "prompt-chunk-ragged"),
        # chat with one user: one sequence, latency only
        _decode(1, 900, 900, 32, 8, 128, 16, 0, 0, "bf16", "decode-one"),
        # a serving batch of ragged sequences, the heads of a 4096-wide block
        _decode(64, 1, 4999, 32, 8, 128, 64, 0, 0, "bf16", "decode-batch"),
        # two very long sequences on one rank of eight: one key-value head, all work along the length
        _decode(2, 100003, 131072, 8, 1, 128, 64, 0, 0, "fp16", "decode-long"),
        # windowed decoding with sinks in a batch whose slots are partly empty; pages that end inside any tile
        _decode(48, 0, 30000, 16, 2, 64, 24, 4096, 4, "bf16", "decode-window"),
        # a decode step stores one token of each sequence
        _append(64, 1, 2000, 8, 128, 64, False, "bf16", "append-decode"),
        # a batch of prompts, padded to the longest, goes into the cache
        _append(2, 4096, 0, 8, 128, 64, True, "bf16", "append-prompts"),
        # forking eight sequences copies the last, partly filled page of each
        _copy(8, 8, 128, 64, "bf16", "copy-fork"),
        # compacting a cache moves thousands of small pages
        _copy(4000, 8, 128, 16, "fp16", "copy-compact"),
    ]


def _named(case: dict, name: str) -> dict:
    return dict(case, name=name) if name else case


def _prompt(batch, sq, sk, heads, kv, dim, window, sinks, ragged, dtype, name="") -> dict:
    return _named({"kind": "prompt", "batch": batch, "sq": sq, "sk": sk, "heads": heads, "kv": kv, "dim": dim,
                   "window": window, "sinks": sinks, "ragged": ragged, "dtype": dtype}, name)


def _decode(seqs, shortest, longest, heads, kv, dim, page, window, sinks, dtype, name="") -> dict:
    return _named({"kind": "decode", "seqs": seqs, "shortest": shortest, "longest": longest, "heads": heads, "kv": kv,
                   "dim": dim, "page": page, "window": window, "sinks": sinks, "dtype": dtype}, name)


def _append(seqs, tokens, before, kv, dim, page, ragged, dtype, name="") -> dict:
    return _named({"kind": "append", "seqs": seqs, "tokens": tokens, "before": before, "kv": kv, "dim": dim, "page": page,
                   "ragged": ragged, "dtype": dtype}, name)


def _copy(moves, kv, dim, page, dtype, name="") -> dict:
    return _named({"kind": "copy", "moves": moves, "kv": kv, "dim": dim, "page": page, "dtype": dtype}, name)


def _log(rng, lo: int, hi: int) -> int:
    """A whole number of [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999))))))


# query and key-value heads: whole models and ranks of two to eight; groups of 1 to 16, not only powers of two
HEADS = [(32, 8), (64, 8), (8, 1), (16, 2), (4, 4), (12, 4), (20, 4), (14, 2), (16, 1)]
PAGES = [8, 16, 24, 32, 50, 64, 128]


def draw(rng) -> dict:
    kind = rng.choice(["prompt", "prompt", "decode", "decode", "append", "copy"])
    dtype = rng.choice(sorted(DTYPES))
    dim = rng.choice([64, 128, 128])
    heads, kv = rng.choice(HEADS)
    page = rng.choice(PAGES)
    window = rng.choice([0, _log(rng, 16, 4096)])
    sinks = rng.choice([0, _log(rng, 1, 64)]) if window else 0
    while kind == "prompt":
        batch, sq, before = rng.choice([1, 1, 2, 3, 5]), _log(rng, 1, 16384), rng.choice([0, 0, _log(rng, 1, 8192)])
        c = _prompt(batch, sq, sq + before, heads, kv, dim, window, sinks, batch > 1 and rng.random() < 0.5, dtype)
        # (the plain form works on all pairs, also on those a window hides)
        if batch * sq * (before + sq // 2) * heads * dim <= MOST_PROMPT:
            return c
    while kind == "decode":
        seqs, longest = _log(rng, 1, 256), _log(rng, 16, 131072)
        shortest = rng.choice([0, 1, longest // 3, longest])
        width = -(-longest // page) * page
        read = min(longest, window + sinks) if window else (shortest + longest) // 2
        if seqs * width * kv * dim * 2 <= MOST_CACHE and seqs * read * kv * dim <= MOST_READ:
            return _decode(seqs, shortest, longest, heads, kv, dim, page, window, sinks, dtype)
    while kind == "append":
        seqs, tokens, before = _log(rng, 1, 256), rng.choice([1, _log(rng, 2, 8192)]), rng.choice([0, _log(rng, 1, 4096)])
        if (seqs * tokens * kv * dim <= MOST_APPEND
                and seqs * (-(-(before + tokens) // page) + 1) * page * kv * dim * 2 <= MOST_CACHE):
            return _append(seqs, tokens, before, kv, dim, page, rng.random() < 0.5, dtype)
    while True:
        moves = _log(rng, 1, 4000)
        if moves * 2 * kv * page * dim <= MOST_COPY:
            return _copy(moves, kv, dim, page, dtype)


# ---------------------------------------------------------------------------
def _spread(lo: int, hi: int, n: int, seed: int) -> list:
    """n lengths from lo to hi, evenly, in an order that the seed gives."""
    if n == 1:
        return [hi]
    g = torch.Generator().manual_seed(seed)
    steps = [lo + (hi - lo) * i // (n - 1) for i in range(n)]
    return [steps[i] for i in torch.randperm(n, generator=g).tolist()]


def _prompt_lengths(case: dict, seed: int) -> list:
    sk, sq = case["sk"], case["sq"]
    # a padded batch: the shortest has half of the new tokens
    return _spread(sk - sq // 2, sk, case["batch"], seed) if case["ragged"] else [sk] * case["batch"]


def _inputs(case: dict, seed: int) -> dict:
    dt, dim, kv = DTYPES[case["dtype"]], case["dim"], case["kv"]
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.empty(shape, dtype=dt, device="cuda").normal_(generator=gen)

    kind = case["kind"]
    if kind == "prompt":
        batch, sq, sk, heads = case["batch"], case["sq"], case["sk"], case["heads"]
        # the new tokens' queries, keys and values lie side by side, as the QKV projection stores them
        qkv = normal(batch, sq, heads + 2 * kv, dim)
        q, k, v = qkv.split([heads, kv, kv], dim=2)
        if sk > sq:  # keys and values of the earlier tokens stand in front of the new ones
            k, v = (torch.cat([normal(batch, sk - sq, kv, dim), x], dim=1) for x in (k, v))
        lengths = torch.tensor(_prompt_lengths(case, seed), dtype=torch.int32, device="cuda") if case["ragged"] else None
        return {"q": q, "k": k, "v": v, "lengths": lengths}
    page = case["page"]
    if kind == "copy":
        moves = case["moves"]
        pages = 2 * moves + 3
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        return {"cache": normal(pages, 2, kv, page, dim), "moves": torch.stack([order[:moves], order[moves:2 * moves]], 1)}
    seqs = case["seqs"]
    if kind == "decode":
        lengths = _spread(case["shortest"], case["longest"], seqs, seed)
        width = -(-case["longest"] // page)
    else:
        # where each sequence's new tokens begin, and how many it has
        starts = _spread(case["before"] // 2, case["before"], seqs, seed)
        counts = _spread((case["tokens"] + 1) // 2, case["tokens"], seqs, seed + 1) if case["ragged"] else None
        lengths = [s + case["tokens"] for s in starts]
        width = -(-(case["before"] + case["tokens"]) // page)
    used = [-(-n // page) for n in lengths]
    # pages in no order, as after many sequences have come and gone; some belong to nobody
    order = torch.randperm(sum(used) + 5, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((seqs, width), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(used):
        table[s, :n] = order[at:at + n]
        at += n
    t = {"cache": normal(sum(used) + 5, 2, kv, page, dim), "table": table.cuda()}
    if kind == "decode":
        t["q"] = normal(seqs, case["heads"] + 2 * kv, dim)[:, :case["heads"]]
        t["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        return t
    new = normal(seqs, case["tokens"], 2 * kv, dim)
    t["k"], t["v"] = new[:, :, :kv], new[:, :, kv:]
    t["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    t["counts"] = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    return t


def prepare(case: dict, seed: int) -> dict:
    return dict(_inputs(case, seed), kind=case["kind"], window=case.get("window", 0), sinks=case.get("sinks", 0))


def run(s: dict):
    kind = s["kind"]
    if own:
        from flashoverlap_b200 import ops

        if kind == "prompt":
            return ops.prompt_attention(s["q"], s["k"], s["v"], window=s["window"], sinks=s["sinks"], lengths=s["lengths"])
        if kind == "decode":
            return ops.paged_attention(s["q"], s["cache"], s["table"], s["lengths"], window=s["window"], sinks=s["sinks"])
        if kind == "append":
            ops.cache_append(s["k"], s["v"], s["cache"], s["table"], s["starts"], counts=s["counts"])
        else:
            ops.copy_pages(s["cache"], s["moves"])
        return s["cache"]
    if kind == "prompt":
        return _plain_prompt(s["q"], s["k"], s["v"], s["window"], s["sinks"], s["lengths"])
    if kind == "decode":
        return _plain_decode(s["q"], s["cache"], s["table"], s["lengths"], s["window"], s["sinks"])
    if kind == "append":
        return _plain_append(s["k"], s["v"], s["cache"], s["table"], s["starts"], s["counts"])
    src, dst = s["moves"].to(s["cache"].device, torch.long).unbind(1)
    s["cache"][dst] = s["cache"][src]
    return s["cache"]


# ---- the operators in elementary operations, fp32 inside ---------------------
def _weights(scores, visible):
    """exp(score - row's largest) of the visible places and its sum; both zero where nothing is visible."""
    scores = torch.where(visible, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    return p, p.sum(-1, keepdim=True)


def _plain_prompt(q, k, v, window, sinks, lengths):
    batch, sq, heads, dim = q.shape
    sk, group = k.shape[1], heads // k.shape[2]
    out = torch.empty((batch, sq, heads, dim), dtype=q.dtype, device=q.device)
    j = torch.arange(sk, device=q.device)
    rows = max(1, min(sq, (1 << 27) // sk))  # scores of 512 MB at a time
    for b in range(batch):
        for t in range(0, sq, rows):
            i = sk - sq + torch.arange(t, min(sq, t + rows), device=q.device)[:, None]
            see = j <= i
            if window:
                see = see & ((j > i - window) | (j < sinks))
            if lengths is not None:
                see = see & (j < lengths[b]) & (i < lengths[b])
            for h in range(heads):
                scores = q[b, t:t + rows, h].float() @ k[b, :, h // group].float().t() / math.sqrt(dim)
                p, total = _weights(scores, see)
                o = p @ v[b, :, h // group].float()
                out[b, t:t + rows, h] = torch.where(total > 0, o / total, torch.zeros_like(o)).to(q.dtype)
    return out


def _plain_decode(q, cache, table, lengths, window, sinks):
    seqs, heads, dim = q.shape
    kv, page = cache.shape[2], cache.shape[3]
    group = heads // kv
    pages = table.clamp(min=0).long()
    j = torch.arange(table.shape[1] * page, device=q.device)
    n = lengths[:, None].long()
    see = j < n
    if window:
        see = see & ((j >= n - window) | (j < sinks))
    out = torch.empty((seqs, heads, dim), dtype=q.dtype, device=q.device)
    for h in range(kv):
        keys, values = (cache[pages, i, h].float().reshape(seqs, -1, dim) for i in (0, 1))
        mine = q[:, h * group:(h + 1) * group].float()
        p, total = _weights(mine @ keys.transpose(1, 2) / math.sqrt(dim), see[:, None])
        o = p @ values
        out[:, h * group:(h + 1) * group] = torch.where(total > 0, o / total, torch.zeros_like(o)).to(q.dtype)
    return out


def _plain_append(k, v, cache, table, starts, counts):
    seqs, tokens = k.shape[:2]
    page = cache.shape[3]
    i = torch.arange(tokens, device=k.device).expand(seqs, tokens)
    at = starts[:, None].long() + i
    rows = table.long().gather(1, at // page)
    places = at % page
    if counts is not None:  # tokens behind a sequence's count are padding: write back what their place holds
        keep = (i < counts[:, None])[:, :, None, None]
        k = torch.where(keep, k, cache[rows, 0, :, places])
        v = torch.where(keep, v, cache[rows, 1, :, places])
    cache[rows, 0, :, places] = k
    cache[rows, 1, :, places] = v
    return cache


# ---- the same from the definition, in 64 bits --------------------------------
def exact(case: dict, seed: int):
    if case["kind"] in ("append", "copy"):
        return None  # nothing is computed
    t = _inputs(case, seed)
    window, sinks, group = case["window"], case["sinks"], case["heads"] // case["kv"]

    def attend(q, keys, values, first, length):
        """Rows of q at positions first, first + 1, ... over the first `length` tokens."""
        out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
        for lo in range(0, min(q.shape[0], max(0, length - first)), 2048):
            hi = min(lo + 2048, q.shape[0], length - first)
            i = torch.arange(first + lo, first + hi, device="cuda").unsqueeze(1)
            j = torch.arange(length, device="cuda").unsqueeze(0)
            hidden = j > i
            if window:
                hidden |= (i - j >= window) & (j >= sinks)
            s = torch.einsum("id,jd->ij", q[lo:hi].double(), keys[:length].double()).mul_(case["dim"] ** -0.5)
            out[lo:hi] = s.masked_fill_(hidden, -math.inf).softmax(1) @ values[:length].double()
        return out

    if case["kind"] == "prompt":
        lengths = _prompt_lengths(case, seed)
        out = torch.empty(t["q"].shape, dtype=torch.float64, device="cuda")
        for b in range(case["batch"]):
            for h in range(case["heads"]):
                out[b, :, h] = attend(t["q"][b, :, h], t["k"][b, :, h // group], t["v"][b, :, h // group],
                                      case["sk"] - case["sq"], lengths[b])
        return out
    out = torch.zeros(t["q"].shape, dtype=torch.float64, device="cuda")
    for s, length in enumerate(t["lengths"].tolist()):
        if length == 0:
            continue
        mine = t["cache"][t["table"][s, :-(-length // case["page"])].long()]
        for h in range(case["heads"]):
            keys, values = (mine[:, i, h // group].reshape(-1, case["dim"]) for i in (0, 1))
            out[s, h] = attend(t["q"][s, h][None], keys, values, length - 1, length)[0]
    return out


def _seen(i: int, window: int, sinks: int) -> int:
    """Visible tokens from position i."""
    return i + 1 if not window else min(i + 1, window + min(sinks, max(0, i + 1 - window)))


def work(case: dict) -> dict:
    kind, kv, dim = case["kind"], case["kv"], case["dim"]
    if kind == "copy":
        return {"bytes": 2 * case["moves"] * 2 * kv * case["page"] * dim * 2, "flops": 0}
    if kind == "append":
        counts = (_spread((case["tokens"] + 1) // 2, case["tokens"], case["seqs"], 1) if case["ragged"]
                  else [case["tokens"]] * case["seqs"])
        return {"bytes": 2 * sum(counts) * 2 * kv * dim * 2, "flops": 0}
    heads, window, sinks = case["heads"], case["window"], case["sinks"]
    if kind == "decode":
        seen = sum(_seen(n - 1, window, sinks) for n in _spread(case["shortest"], case["longest"], case["seqs"], 1) if n)
        return {"bytes": 2 * (2 * seen * kv * dim + 2 * case["seqs"] * heads * dim), "flops": 4 * seen * heads * dim}
    first = case["sk"] - case["sq"]
    pairs = sum(sum(_seen(i, window, sinks) for i in range(first, n)) for n in _prompt_lengths(case, 1))
    tokens = case["batch"] * (2 * case["sq"] * heads + 2 * case["sk"] * kv)
    return {"bytes": 2 * tokens * dim, "flops": 4 * pairs * heads * dim}
