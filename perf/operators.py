"""Serving from a paged key/value cache, as cases that can be timed and checked.

Kinds of case, each one operator:

  append    the rotary embedding of new tokens, their keys and values written into pages
  decode    attention of one new token per sequence over its pages
  prompt    attention of prompt chunks over their pages, causal, with an optional sliding
            window beside a few first tokens that stay visible
  resample  sequences given up and others forked into their place: pages freed, shared, copied
  compact   the pages in use moved to the lowest page numbers
  logprobs  log probabilities of given tokens, the entropy and the top alternatives

With `own` false, `run` computes the plain form in elementary torch operations; with `own` true
it makes the package's calls. Lengths follow from the case alone (`work` counts them), values,
tokens and the order of pages from the seed.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------ cases --
def listed():
    return [
        # a decode step of 16 sequences of a 1B model (16 heads): rotation and cache write
        dict(name="append_16seq", kind="append", dtype="bf16", tokens=16, seqs=16, heads=16,
             kv_heads=16, hd=128, page=16, context=1024, norm=False),
        # prompts of a grouped-query model with per-head norms, ragged, up to 2048 tokens each
        dict(name="append_prompts_qknorm", kind="append", dtype="bf16", tokens=2048, seqs=6,
             heads=32, kv_heads=8, hd=128, page=64, context=0, norm=True),
        # one user, one new token, a short odd context: latency
        dict(name="decode_1seq_717", kind="decode", dtype="fp16", seqs=1, longest=717, heads=16,
             kv_heads=16, hd=64, page=16, window=0, sinks=0),
        # long documents in one batch with short ones: the long one sets the pace
        dict(name="decode_ragged_60k", kind="decode", dtype="bf16", seqs=4, longest=60001,
             heads=32, kv_heads=8, hd=128, page=64, window=0, sinks=0),
        # endless chats: 64 sequences, a window of 1024 tokens and 4 first tokens
        dict(name="decode_window_64seq", kind="decode", dtype="bf16", seqs=64, longest=16000,
             heads=16, kv_heads=16, hd=128, page=16, window=1024, sinks=4),
        # short ragged prompts of a 60M model (8 heads of 64, fp32)
        dict(name="prompt_60m_fp32", kind="prompt", dtype="fp32", seqs=5, tokens=129, context=0,
             heads=8, kv_heads=8, hd=64, page=16, window=0, sinks=0),
        # a whole prompt of 4096 tokens through a 1B model's heads
        dict(name="prompt_4096", kind="prompt", dtype="bf16", seqs=1, tokens=4096, context=0,
             heads=16, kv_heads=16, hd=128, page=64, window=0, sinks=0),
        # the next 512 tokens of long inputs, a sliding window of 2048 and 4 first tokens
        dict(name="prompt_chunk_window", kind="prompt", dtype="fp16", seqs=6, tokens=512,
             context=8000, heads=32, kv_heads=8, hd=128, page=16, window=2048, sinks=4),
        # 32 candidates with a common prompt: half are dropped, the others forked in their place
        dict(name="resample_32seq", kind="resample", dtype="bf16", layers=16, seqs=32,
             longest=1500, heads=16, hd=128, page=16),
        # a scattered cache of a grouped-query model made contiguous: a quarter of it moves
        dict(name="compact_4096pages", kind="compact", dtype="bf16", layers=8, seqs=64,
             pages=4096, live=2048, moves=1024, heads=8, hd=128, page=16),
        # one decode step of 16 sequences: the sampled token and its alternatives
        dict(name="logprobs_16seq", kind="logprobs", dtype="bf16", rows=16, vocab=32000, top=8,
             masked=False),
        # a prompt scored: 2000 tokens, fp32 logits, five alternatives each
        dict(name="logprobs_prompt", kind="logprobs", dtype="fp32", rows=2000, vocab=32000, top=5,
             masked=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _window(rng, longest):
    if rng.random() < 0.5:
        return 0, 0
    return _log_int(rng, 16, max(17, longest)), rng.choice([0, 1, 4, 4, 50])


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        for k in ("bytes", "flops"):
            most[c["kind"], k] = max(most.get((c["kind"], k), 0), w[k])
    while True:
        c = _draw(rng)
        w = work(c)
        # fp32 products run at a sixteenth of the 16-bit rate
        slow = 16 if c["dtype"] == "fp32" and c["kind"] == "prompt" else 1
        if all(w[k] * (slow if k == "flops" else 1) <= most[c["kind"], k]
               for k in ("bytes", "flops")) and _held(c) <= 2.2e9:
            return c


def _held(c):
    """Elements that a form without tiles holds at once (the gathered keys, a prompt's scores)."""
    if c["kind"] == "decode":
        return c["seqs"] * c["longest"] * c["kv_heads"] * c["hd"]
    if c["kind"] == "prompt":
        reach = c["tokens"] + c["context"]
        return c["seqs"] * reach * max(2.5 * c["tokens"] * c["heads"], c["kv_heads"] * c["hd"])
    return 0


def _draw(rng):
    kind = rng.choice(["append", "decode", "decode", "decode", "prompt", "prompt", "prompt",
                       "resample", "compact", "logprobs", "logprobs"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    hd = rng.choice([64, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8, 16])
    heads = kv * rng.choice([1, 1, 2, 3, 4, 7, 8])
    page = rng.choice([16, 16, 32, 64, 128, 256])
    if kind == "append":
        seqs = _log_int(rng, 1, 64)
        return dict(kind=kind, dtype=dtype, tokens=_log_int(rng, 1, 2048), seqs=seqs, heads=heads,
                    kv_heads=kv, hd=hd, page=page, context=rng.choice([0, _log_int(rng, 1, 5000)]),
                    norm=rng.random() < 0.3)
    if kind == "decode":
        longest = _log_int(rng, 1, 60000)
        w, s = _window(rng, longest)
        return dict(kind=kind, dtype=dtype, seqs=_log_int(rng, 1, 128), longest=longest,
                    heads=heads, kv_heads=kv, hd=hd, page=page, window=w, sinks=s)
    if kind == "prompt":
        tokens = _log_int(rng, 1, 4096)
        context = rng.choice([0, 0, _log_int(rng, 1, 8000)])
        w, s = _window(rng, tokens + context)
        return dict(kind=kind, dtype=dtype, seqs=_log_int(rng, 1, 8), tokens=tokens,
                    context=context, heads=heads, kv_heads=kv, hd=hd, page=page, window=w, sinks=s)
    if kind == "resample":
        return dict(kind=kind, dtype=dtype, layers=_log_int(rng, 1, 16), seqs=_log_int(rng, 2, 64),
                    longest=_log_int(rng, 1, 3000), heads=kv, hd=hd, page=page)
    if kind == "compact":
        pages = _log_int(rng, 16, 16384)
        live = max(1, int(pages * rng.uniform(0.05, 0.95)))
        return dict(kind=kind, dtype=dtype, layers=_log_int(rng, 1, 16), seqs=_log_int(rng, 1, 64),
                    pages=pages, live=live, moves=int(min(live, pages - live) * rng.random()),
                    heads=kv, hd=hd, page=page)
    return dict(kind=kind, dtype=dtype, rows=_log_int(rng, 1, 2000), vocab=_log_int(rng, 100, 160000),
                top=rng.choice([0, 1, 5, 8, 20]), masked=rng.random() < 0.3)


def _spread(longest, n, least=1):
    """n lengths up to `longest` (the first), most of them well below it."""
    return [max(least, int(longest * (1 - 0.618034 * i % 1) ** 2)) for i in range(n)]


def _chunks(c):
    """(cached tokens, new tokens) of each prompt of the case."""
    t = _spread(c["tokens"], c["seqs"])
    return list(zip(_spread(c["context"], c["seqs"], 0), t))


def _split(total, n):
    """`total` tokens over n sequences, raggedly (some may get none)."""
    cut = [round(total * (i / n) ** 1.5) for i in range(n + 1)]
    return [b - a for a, b in zip(cut, cut[1:])]


def _visible(length, window, sinks):
    """How many of the first `length` positions the last of them sees."""
    return length if window == 0 else min(length, window + min(sinks, max(0, length - window)))


def work(c):
    e, kind = BYTES[c["dtype"]], c["kind"]
    if kind == "append":
        row = (c["heads"] + 2 * c["kv_heads"]) * c["hd"]
        return {"bytes": c["tokens"] * (2.0 * e * row + 4 * c["hd"] + 8),
                "flops": 6.0 * c["tokens"] * (c["heads"] + c["kv_heads"]) * c["hd"]}
    if kind == "decode":
        seen = sum(_visible(n, c["window"], c["sinks"]) for n in _spread(c["longest"], c["seqs"]))
        return {"bytes": e * c["hd"] * (2.0 * seen * c["kv_heads"] + 2 * c["seqs"] * c["heads"])
                + 4.0 * c["seqs"] * (1 + c["longest"] / c["page"]),
                "flops": 4.0 * seen * c["heads"] * c["hd"]}
    if kind == "prompt":
        w, s = c["window"], c["sinks"]
        pairs = seen = tokens = 0
        for ctx, t in _chunks(c):
            pairs += sum(_visible(p + 1, w, s) for p in range(ctx, ctx + t))
            first = max(0, ctx + 1 - w) if w else 0  # the first position the window reaches
            seen += ctx + t - first + min(s if w else 0, first)
            tokens += t
        return {"bytes": e * c["hd"] * (2.0 * seen * c["kv_heads"] + 2 * tokens * c["heads"]),
                "flops": 4.0 * pairs * c["heads"] * c["hd"]}
    if kind == "resample":
        lens, n = _spread(c["longest"], c["seqs"]), c["seqs"] // 2
        copied = sum(lens[i] % c["page"] for i in range(n))
        cols = -(-c["longest"] // c["page"])
        return {"bytes": 4.0 * copied * c["layers"] * c["heads"] * c["hd"] * e
                + 8.0 * (c["seqs"] * cols + _pool_pages(c)), "flops": 0.0}
    if kind == "compact":
        page = c["layers"] * c["heads"] * c["page"] * c["hd"] * e
        return {"bytes": 4.0 * c["moves"] * page + 8.0 * (c["pages"] + c["live"]), "flops": 0.0}
    return {"bytes": c["rows"] * (c["vocab"] * float(e) + 16 + 12 * c["top"]),
            "flops": 5.0 * c["rows"] * c["vocab"]}


# ----------------------------------------------------------------- inputs --
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _table(g, lens, page):
    """A page table for sequences of these lengths, pages in the seed's order, and the pages of
    the pool: one eighth more than are in use."""
    used = [-(-n // page) for n in lens]
    pages = sum(used) + sum(used) // 8 + 1
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.full((len(lens), max(1, max(used))), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(used):
        table[i, :n] = order[at: at + n]
        at += n
    return table, pages


def _angles(c, positions):
    """cos and sin of the rotary embedding up to the last position, [positions, hd / 2] fp32."""
    inv = 500000.0 ** -(torch.arange(0, c["hd"], 2, device="cuda", dtype=torch.float64) / c["hd"])
    a = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * inv
    return a.cos().float(), a.sin().float()


def _pool_pages(c):
    """Pages of a resample case's pool: the common prompt's, each sequence's own, and room."""
    lens, page = _spread(c["longest"], c["seqs"]), c["page"]
    whole = min(lens) // page // 2
    return whole + sum(-(-n // page) - whole for n in lens) + c["seqs"]


def prepare(case, seed):
    c, g, dt, kind = case, _gen(seed), DTYPES[case["dtype"]], case["kind"]
    s = {"case": c}
    if kind == "append":
        counts = _split(c["tokens"], c["seqs"])
        starts = _spread(c["context"], c["seqs"], 0)
        s["table"], pages = _table(g, [a + n for a, n in zip(starts, counts)], c["page"])
        s["seqs"] = _ints([i for i, n in enumerate(counts) for _ in range(n)])
        s["positions"] = _ints([a + j for a, n in zip(starts, counts) for j in range(n)])
        for name, heads in (("q", c["heads"]), ("k", c["kv_heads"]), ("v", c["kv_heads"])):
            s[name] = _randn(g, c["tokens"], heads, c["hd"], dtype=dt)
        s["cos"], s["sin"] = _angles(c, max(a + n for a, n in zip(starts, counts)) + 1)
        for name in ("q_norm", "k_norm"):
            s[name] = (1 + _randn(g, c["hd"], scale=0.1)).to(dt) if c["norm"] else None
        for name in ("k_pool", "v_pool"):
            s[name] = _randn(g, pages, c["kv_heads"], c["page"], c["hd"], dtype=dt)
    elif kind in ("decode", "prompt"):
        if kind == "decode":
            lens, tokens = _spread(c["longest"], c["seqs"]), c["seqs"]
        else:
            chunks = _chunks(c)
            lens, tokens = [a + t for a, t in chunks], sum(t for _, t in chunks)
            cu = [0]
            for _, t in chunks:
                cu.append(cu[-1] + t)
            s["cu"], s["max_tokens"] = _ints(cu), max(t for _, t in chunks)
        s["table"], pages = _table(g, lens, c["page"])
        s["lengths"], s["max_length"] = _ints(lens), max(lens)
        # queries twice as long as keys: some tokens stand out, as in a trained model
        s["q"] = _randn(g, tokens, c["heads"], c["hd"], dtype=dt, scale=2.0)
        for name in ("k_pool", "v_pool"):
            s[name] = _randn(g, pages, c["kv_heads"], c["page"], c["hd"], dtype=dt)
    elif kind == "resample":
        lens, page, n = _spread(c["longest"], c["seqs"]), c["page"], c["seqs"] // 2
        pages, whole = _pool_pages(c), min(lens) // page // 2
        order = torch.randperm(pages, generator=g, device="cuda").int()
        s["table"] = torch.full((c["seqs"], -(-max(lens) // page)), -1, dtype=torch.int32,
                                device="cuda")
        at = whole
        for i, length in enumerate(lens):
            used = -(-length // page)
            s["table"][i, :whole] = order[:whole]
            s["table"][i, whole:used] = order[at: at + used - whole]
            at += used - whole
        s["refs"] = torch.zeros(pages, dtype=torch.int32, device="cuda")
        s["refs"][order[whole:at].long()] = 1
        s["refs"][order[:whole].long()] = c["seqs"]
        s["lengths"] = _ints(lens)
        # the first half of the sequences goes on twice, the second half is given up
        s["src"] = torch.arange(n, dtype=torch.int32, device="cuda")
        perm = torch.randperm(c["seqs"] - n, generator=g, device="cuda")[:n]
        s["dst"] = (n + perm).int()
    elif kind == "compact":
        live, moves, pages = c["live"], c["moves"], c["pages"]
        low = torch.randperm(live, generator=g, device="cuda")[: live - moves]
        high = live + torch.randperm(pages - live, generator=g, device="cuda")[:moves]
        ids = torch.cat([low, high])[torch.randperm(live, generator=g, device="cuda")].int()
        cols = -(-live // c["seqs"])
        s["table"] = torch.full((c["seqs"] * cols,), -1, dtype=torch.int32, device="cuda")
        s["table"][:live] = ids
        s["table"] = s["table"].view(c["seqs"], cols)
        s["refs"] = torch.zeros(pages, dtype=torch.int32, device="cuda")
        s["refs"][ids.long()] = 1
    else:
        # a language model's logits: most tokens far below the few likely ones
        s["logits"] = _randn(g, c["rows"], c["vocab"], scale=3.0).to(dt)
        if c["masked"]:  # a grammar forbids a third of the tokens
            s["logits"].masked_fill_(torch.rand(c["vocab"], generator=g, device="cuda") < 0.33,
                                     -math.inf)
        s["tokens"] = torch.randint(0, c["vocab"], (c["rows"],), generator=g, device="cuda")
    if kind in ("resample", "compact"):
        pages = s["refs"].numel()
        for name in ("k_pool", "v_pool"):
            s[name] = torch.empty(c["layers"], pages, c["heads"], c["page"], c["hd"], dtype=dt,
                                  device="cuda").normal_(generator=g)
    return s


# ------------------------------------------------------------- plain forms --
def _rotate(x, w, cos, sin):
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.float()
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_append(s):
    pos, page = s["positions"].long(), s["case"]["page"]
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    at = s["table"][s["seqs"].long(), pos // page].long()
    s["k_pool"][at, :, pos % page] = _rotate(s["k"], s["k_norm"], cos, sin).to(s["k"].dtype)
    s["v_pool"][at, :, pos % page] = s["v"]
    return _rotate(s["q"], s["q_norm"], cos, sin).to(s["q"].dtype), s["k_pool"], s["v_pool"]


def _gathered(s, name):
    """The pool's pages in the order of the tables, fp32 [seqs, kv_heads, positions, hd]."""
    x = s[name][s["table"].clamp(min=0).long()].transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[4]).float()


def _plain_attention(s, q, pos):
    """q [seqs, heads, T, hd] fp32 at positions `pos` [seqs, T] (below 0: no token)."""
    c = s["case"]
    k, v = _gathered(s, "k_pool"), _gathered(s, "v_pool")
    n, heads, t, hd = q.shape
    q = q.reshape(n, c["kv_heads"], -1, hd)
    p = (q @ k.transpose(2, 3)).view(n, heads, t, -1) * hd ** -0.5
    j, pos = torch.arange(k.shape[2], device=q.device), pos[..., None]
    see = j <= pos
    if c["window"]:
        see = see & ((j > pos - c["window"]) | (j < c["sinks"]))
    p.masked_fill_(~see[:, None], -math.inf)
    p -= p.amax(-1, keepdim=True).clamp(min=torch.finfo(p.dtype).min)
    p.exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.view(n, c["kv_heads"], -1, k.shape[2]) @ v).view(n, heads, t, hd)
    return torch.where(total > 0, o / total, 0.0)


def _plain_decode(s):
    q = s["q"].float()[:, :, None]
    return _plain_attention(s, q, s["lengths"][:, None] - 1)[:, :, 0].to(s["q"].dtype)


def _plain_prompt(s):
    cu, most = s["cu"].long(), s["max_tokens"]
    count = cu[1:] - cu[:-1]
    off = torch.arange(most, device=cu.device)
    pos = torch.where(off < count[:, None], (s["lengths"] - count)[:, None] + off, -1)
    q = s["q"].float()[(cu[:-1, None] + off).clamp(max=s["q"].shape[0] - 1)].transpose(1, 2)
    o = _plain_attention(s, q, pos).transpose(1, 2)
    t = torch.arange(s["q"].shape[0], device=cu.device)
    row = torch.searchsorted(cu[1:], t, right=True)
    return o[row, t - cu[row]].to(s["q"].dtype)


def _plain_free(table, lengths, refs, seqs):
    gone = torch.zeros_like(lengths, dtype=torch.bool)
    gone[seqs.long()] = True
    held = torch.where(gone[:, None] & (table >= 0), table, refs.numel()).long().view(-1)
    less = torch.zeros(refs.numel() + 1, dtype=refs.dtype, device=refs.device)
    less.index_add_(0, held, torch.ones_like(held, dtype=refs.dtype))
    return (table.masked_fill(gone[:, None], -1), lengths.masked_fill(gone, 0), refs - less[:-1])


def _plain_fork(s, table, lengths, refs):
    page, src, dst = s["case"]["page"], s["src"].long(), s["dst"].long()
    whole, part = lengths[src].long() // page, lengths[src].long() % page
    need = part > 0
    free = torch.argsort((refs != 0).int(), stable=True)
    rank = need.long().cumsum(0) - 1
    ok = (lengths[dst] == 0) & (~need | (rank < (refs == 0).sum()))
    take = ok & need
    fresh = free[rank.clamp(0, refs.numel() - 1)]
    col = torch.arange(table.shape[1], device=table.device)
    shared = torch.where(ok[:, None] & (col < whole[:, None]), table[src], -1)
    last = take[:, None] & (col == whole[:, None])
    rows = torch.where(last, fresh[:, None].int(), shared)
    new_table, new_lengths = table.clone(), lengths.clone()
    new_table[dst] = torch.where(ok[:, None], rows, table[dst])
    new_lengths[dst] = torch.where(ok, lengths[src], lengths[dst])
    more = torch.zeros(refs.numel() + 1, dtype=refs.dtype, device=refs.device)
    held = torch.where(rows >= 0, rows, refs.numel()).long().view(-1)
    more.index_add_(0, held, torch.ones_like(held, dtype=refs.dtype))
    i = take.nonzero()[:, 0]
    a, b = table[src[i], whole[i]].long(), fresh[i]
    mine = (torch.arange(page, device=a.device) < part[i, None])[:, None, :, None]
    for pool in (s["k_pool"], s["v_pool"]):
        pool[:, b] = torch.where(mine, pool[:, a], pool[:, b])
    return new_table, new_lengths, refs + more[:-1], ok


def _plain_resample(s):
    table, lengths, refs = _plain_free(s["table"], s["lengths"], s["refs"], s["dst"])
    return *_plain_fork(s, table, lengths, refs), s["k_pool"], s["v_pool"]


def _plain_compact(s):
    refs, table = s["refs"], s["table"]
    live = refs > 0
    n = live.sum()
    ids = torch.arange(refs.numel(), device=refs.device)
    holes, movers = (~live & (ids < n)).nonzero()[:, 0], (live & (ids >= n)).nonzero()[:, 0]
    to = ids.clone()
    to[movers] = holes
    new_refs = torch.zeros_like(refs)
    new_refs[to[live]] = refs[live]
    for pool in (s["k_pool"], s["v_pool"]):
        pool[:, holes] = pool[:, movers]
    new_table = torch.where(table >= 0, to[table.clamp(min=0).long()].int(), table)
    return new_table, new_refs, n.int(), s["k_pool"], s["v_pool"]


def _plain_logprobs(s):
    x, top = s["logits"].float(), s["case"]["top"]
    best = x.amax(-1, keepdim=True)
    d = (x - best).double()
    e = d.exp()
    total = e.sum(-1, keepdim=True)
    log_total = total.log()
    entropy = log_total[:, 0] - torch.where(e > 0, e * d, 0.0).sum(-1) / total[:, 0]
    given = (d.gather(1, s["tokens"][:, None]) - log_total)[:, 0]
    ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    return (given.float(), entropy.float(), ids, (d.gather(1, ids) - log_total).float())


_PLAIN = {"append": _plain_append, "decode": _plain_decode, "prompt": _plain_prompt,
          "resample": _plain_resample, "compact": _plain_compact, "logprobs": _plain_logprobs}


# --------------------------------------------------- the package's own calls --
def _package():
    at = str(Path(__file__).resolve().parent.parent / "s-salaad_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import ssalaad_amd

    return ssalaad_amd


def _own(s):
    sa, c, kind = _package(), s["case"], s["case"]["kind"]
    if kind == "append":
        q = sa.paged_append(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["k_pool"], s["v_pool"],
                            s["table"], s["seqs"], s["positions"], q_norm=s["q_norm"],
                            k_norm=s["k_norm"], eps=1e-6)
        return q, s["k_pool"], s["v_pool"]
    if kind == "decode":
        return sa.paged_decode_attention(s["q"], s["k_pool"], s["v_pool"], s["table"],
                                         s["lengths"], window=c["window"], sinks=c["sinks"],
                                         max_length=s["max_length"])
    if kind == "prompt":
        return sa.paged_prompt_attention(s["q"], s["k_pool"], s["v_pool"], s["table"],
                                         s["lengths"], s["cu"], window=c["window"],
                                         sinks=c["sinks"], max_tokens=s["max_tokens"],
                                         max_length=s["max_length"])
    if kind == "resample":
        table, lengths, refs = sa.free_pages(s["table"], s["lengths"], s["refs"], s["dst"])
        table, lengths, refs, ok = sa.fork_pages(table, lengths, refs, s["k_pool"], s["v_pool"],
                                                 s["src"], s["dst"])
        return table, lengths, refs, ok, s["k_pool"], s["v_pool"]
    if kind == "compact":
        table, refs, live = sa.compact_pages(s["table"], s["refs"], s["k_pool"], s["v_pool"])
        return table, refs, live, s["k_pool"], s["v_pool"]
    return tuple(sa.token_logprobs(s["logits"], s["tokens"], top=c["top"]))


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["kind"]](state)


# -------------------------------------------------------------------- exact --
def _exact_append(c, s):
    pos, rows = s["positions"].tolist(), s["seqs"].tolist()
    table = s["table"].tolist()
    half = c["hd"] // 2
    cos, sin = s["cos"].double()[pos], s["sin"].double()[pos]
    turn = torch.complex(cos, sin)[:, None]

    def turned(x, w):
        x = x.double()
        if w is not None:
            x = w.double() * x / ((x * x).sum(-1, keepdim=True) / c["hd"] + 1e-6).sqrt()
        z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * turn
        return torch.cat([z.real, z.imag], -1)

    kp, vp = s["k_pool"].double(), s["v_pool"].double()
    page = torch.tensor([table[r][p // c["page"]] for r, p in zip(rows, pos)], device="cuda")
    slot = torch.tensor([p % c["page"] for p in pos], device="cuda")
    flat = (page * c["kv_heads"])[:, None] + torch.arange(c["kv_heads"], device="cuda")
    flat = (flat * c["page"] + slot[:, None]).view(-1)
    kp.view(-1, c["hd"]).index_copy_(0, flat, turned(s["k"], s["k_norm"]).reshape(-1, c["hd"]))
    vp.view(-1, c["hd"]).index_copy_(0, flat, s["v"].double().reshape(-1, c["hd"]))
    return turned(s["q"], s["q_norm"]), kp, vp


def _exact_rows(c, s, seq, length, q, first):
    """Attention of tokens at positions first, first + 1, … of one sequence, in 64 bits."""
    at = torch.arange(length, device="cuda")
    page, slot = s["table"][seq].long()[at // c["page"]], at % c["page"]
    group, out = c["heads"] // c["kv_heads"], []
    pos = first + torch.arange(q.shape[0], device="cuda")[:, None]
    hidden = at[None] > pos
    if c["window"]:
        hidden |= (at[None] <= pos - c["window"]) & (at[None] >= c["sinks"])
    for h in range(c["heads"]):
        k, v = (s[x][page, h // group, slot].double() for x in ("k_pool", "v_pool"))
        a = torch.mm(q[:, h].double(), k.t()) / math.sqrt(c["hd"])
        out.append(torch.mm(torch.softmax(a.masked_fill(hidden, -math.inf), -1), v))
    return torch.stack(out, 1)


def _exact_decode(c, s):
    return torch.cat([_exact_rows(c, s, i, n, s["q"][i: i + 1], n - 1)
                      for i, n in enumerate(s["lengths"].tolist())])


def _exact_prompt(c, s):
    cu, out = s["cu"].tolist(), []
    for i, n in enumerate(s["lengths"].tolist()):
        t = cu[i + 1] - cu[i]
        for a in range(0, t, 1024):
            b = min(t, a + 1024)
            out.append(_exact_rows(c, s, i, n, s["q"][cu[i] + a: cu[i] + b], n - t + a))
    return torch.cat(out)


def _exact_resample(c, s):
    page = c["page"]
    table, lens, refs = (s[x].tolist() for x in ("table", "lengths", "refs"))
    for d in s["dst"].tolist():
        for p in table[d]:
            if p >= 0:
                refs[p] -= 1
        table[d], lens[d] = [-1] * len(table[d]), 0
    ok = []
    for a, d in zip(s["src"].tolist(), s["dst"].tolist()):
        whole, part = divmod(lens[a], page)
        fresh = next((p for p, n in enumerate(refs) if n == 0), None) if part else -1
        ok.append(fresh is not None and lens[d] == 0)
        if not ok[-1]:
            continue
        for j in range(whole):
            refs[table[a][j]] += 1
            table[d][j] = table[a][j]
        if part:
            refs[fresh], table[d][whole] = 1, fresh
            for pool in (s["k_pool"], s["v_pool"]):
                pool[:, fresh, :, :part].copy_(pool[:, table[a][whole], :, :part])
        lens[d] = lens[a]
    return (_ints(table), _ints(lens), _ints(refs), torch.tensor(ok, device="cuda"), s["k_pool"],
            s["v_pool"])


def _exact_compact(c, s):
    refs, table = s["refs"].tolist(), s["table"].tolist()
    live = sum(n > 0 for n in refs)
    holes = [p for p in range(live) if refs[p] == 0]
    movers = [p for p in range(live, len(refs)) if refs[p] > 0]
    to = dict(zip(movers, holes))
    for a, b in to.items():
        refs[b], refs[a] = refs[a], 0
        for pool in (s["k_pool"], s["v_pool"]):
            pool[:, b].copy_(pool[:, a])
    table = [[to.get(p, p) for p in row] for row in table]
    return _ints(table), _ints(refs), _ints([live])[0], s["k_pool"], s["v_pool"]


def _exact_logprobs(c, s):
    outs = []
    for x, t in zip(s["logits"].split(256), s["tokens"].split(256)):
        lp = torch.log_softmax(x.double(), -1)
        p = lp.exp()
        ids = torch.argsort(-x.double(), dim=-1, stable=True)[:, : c["top"]]
        outs.append((torch.take_along_dim(lp, t[:, None], 1)[:, 0], -torch.xlogy(p, p).sum(-1),
                     ids, torch.take_along_dim(lp, ids, 1)))
    return tuple(torch.cat(v) for v in zip(*outs))


def exact(case, seed):
    """The operator's definition in 64 bits (page numbers and copies in host integers)."""
    return globals()["_exact_" + case["kind"]](case, prepare(case, seed))
