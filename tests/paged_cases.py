"""Inputs and float64 definitions for the paged-cache tests (CPU only).

Every definition is written out per token in float64 on the CPU. `u(dtype)` is
the largest relative error of one rounding to the dtype.
"""

from __future__ import annotations

import math

import torch

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
F32 = 2.0 ** -24


def u(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def pages_of(lens, page, gen, spare=3, cols=None):
    """(table, pages): a table over pages in a random order, -1 past each length."""
    used = [-(-n // page) for n in lens]
    pages = sum(used) + spare
    order = torch.randperm(pages, generator=gen).int()
    table = torch.full((len(lens), cols or max(1, max(used, default=1))), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(used):
        table[i, :n] = order[at: at + n]
        at += n
    return table, pages


def seen(p: int, n: int, window: int, sinks: int) -> list[int]:
    """Positions a token at p sees among n."""
    return [j for j in range(min(p + 1, n)) if not window or j > p - window or j < sinks]


def attention(q, k_pool, v_pool, table, owners, positions, page, window=0, sinks=0, scale=None,
              lengths=None):
    """(out, tol) in float64: the softmax average of each token's visible
    positions, and a bound of a kernel's error built from its roundings:
    scores in fp32 (a sum of head_dim products), their exponentials, the
    weights rounded to the pools' type (none in fp32; fp16 weights also lose
    what lies below half its smallest step), fp32 sums, and one rounding of the
    result."""
    dt = q.dtype
    hd, heads, kv = q.shape[2], q.shape[1], k_pool.shape[1]
    scale = hd ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64)
    tol = torch.zeros_like(out)
    low = u(dt) if dt != torch.float32 else 0.0
    for t in range(q.shape[0]):
        s, p = int(owners[t]), int(positions[t])
        if s < 0 or p < 0:
            continue
        row = table[s].tolist()
        n = len(row) * page if lengths is None else int(lengths[s])
        js = [j for j in seen(p, n, window, sinks) if 0 <= row[j // page] < k_pool.shape[0]]
        if not js:
            continue
        pg = torch.tensor([row[j // page] for j in js])
        sl = torch.tensor([j % page for j in js])
        k = k_pool[pg, :, sl].double().repeat_interleave(heads // kv, 1)  # [n, heads, hd]
        v = v_pool[pg, :, sl].double().repeat_interleave(heads // kv, 1)
        x = torch.einsum("hd,nhd->hn", q[t].double(), k) * scale
        w = torch.softmax(x, -1)
        out[t] = torch.einsum("hn,nhd->hd", w, v)
        size = torch.einsum("hn,nhd->hd", w, v.abs())
        mag = torch.einsum("hd,nhd->hn", q[t].double().abs(), k.abs()).amax(-1) * abs(scale)
        score = 2 * F32 * ((hd + 8) * mag + x.abs().amax(-1))  # of an exponent, both ends
        n_err = F32 * (len(js) + 64)
        tol[t] = (low + score + n_err)[:, None] * size * 1.01 + u(dt) * out[t].abs() * 1.01
        if dt == torch.float16:
            tol[t] += len(js) * 2.0 ** -25 * v.abs().amax(0)
        tol[t] += torch.finfo(dt).tiny
    return out, tol


def attention_parts(q, k_pool, v_pool, table, owners, positions, page):
    """(out, size, spread, other) in float64: the softmax average of what each token
    sees, Σ p |v|, Σ p |v − out|, and the bound of a kernel's error from its fp32
    scores, exponentials and sums and the rounding of its result."""
    dt, hd, heads, kv = q.dtype, q.shape[2], q.shape[1], k_pool.shape[1]
    out, size, spread, other = (torch.zeros(q.shape, dtype=torch.float64) for _ in range(4))
    for t in range(q.shape[0]):
        row, p = table[owners[t]].long(), int(positions[t])
        at = torch.arange(p + 1)
        k, v = (x[row[at // page], :, at % page].double().repeat_interleave(heads // kv, 1)
                for x in (k_pool, v_pool))
        x = (q[t].double() * k).sum(-1).t() * hd ** -0.5
        w = torch.softmax(x, -1).t()[..., None]
        out[t], size[t] = (w * v).sum(0), (w * v.abs()).sum(0)
        spread[t] = (w * (v - out[t]).abs()).sum(0)
        mag = (q[t].double().abs() * k.abs()).sum(-1).amax(0) * hd ** -0.5
        score = 2 * F32 * ((hd + 8) * mag + x.abs().amax(-1))
        other[t] = (score + F32 * (p + 65))[:, None] * size[t] * 1.01 + u(dt) * out[t].abs() * 1.01
    return out, size, spread, other + torch.finfo(dt).tiny


def rotated(x, norm, eps, cos, sin, pos):
    """(x', tol) of paged_append for x [tokens, heads, hd]."""
    dt, hd = x.dtype, x.shape[-1]
    y = x.double()
    slack = 4 * F32
    if norm is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * norm.double()
        slack += (hd + 16) * F32
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    a, b = y.chunk(2, -1)
    out = torch.cat([a * c - b * s, b * c + a * s], -1)
    size = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()], -1)
    return out, u(dt) * out.abs() * 1.01 + slack * size + torch.finfo(dt).tiny


def logprobs(x, tokens, top):
    """(logprob, entropy, ids, top logprobs) in float64 and the bounds of the two
    scalars: exponentials of differences d rounded to fp32 (2|d| + 4 roundings
    each), 64-bit sums, one rounding at the end."""
    x = x.double()
    d = x - x.amax(-1, keepdim=True)
    e = d.exp()
    S = e.sum(-1)
    p = e / S[:, None]
    dd = torch.where(p > 0, d, 0.0)
    lp = d - S.log()[:, None]
    ent = S.log() - (p * dd).sum(-1)
    ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    mean = (p * dd.abs()).sum(-1)
    s_err = F32 * (2 * mean + 4)
    given = lp.gather(1, tokens[:, None].clamp(0, x.shape[1] - 1))[:, 0]
    tol_lp = (s_err[:, None] + F32 * (d.abs() + 2 * lp.abs()) + 1e-30)
    tol_ent = F32 * ((p * (2 * dd.square() + 5 * dd.abs())).sum(-1) + 2 * ent.abs()) + s_err * (
        1 + mean) + 1e-30
    return given, ent, ids, lp, tol_lp, tol_ent


def angles(n, hd):
    inv = 10000.0 ** -(torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    a = torch.arange(n, dtype=torch.float64)[:, None] * inv
    return a.cos().float(), a.sin().float()


def cache(pages, kv, page, hd, dtype, gen, layers=None):
    shape = (pages, kv, page, hd) if layers is None else (layers, pages, kv, page, hd)
    return (torch.randn(*shape, generator=gen).to(dtype), torch.randn(*shape, generator=gen).to(dtype))


def chunk_rows(counts, lens):
    """(owners, positions) of the tokens of chunks at the sequences' ends."""
    owners = [s for s, c in enumerate(counts) for _ in range(c)]
    positions = [n - c + j for c, n in zip(counts, lens) for j in range(c)]
    return owners, positions


def spread(rng_max, n):
    return [max(1, math.floor(rng_max * (i + 1) / n)) for i in range(n)]
