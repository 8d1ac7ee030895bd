"""The paged cache's operators on the GPU against their float64 definitions
(tests/paged_cases.py), which also give the error bounds."""

from __future__ import annotations

import pytest
import torch

import paged_cases as pc

pytestmark = pytest.mark.gpu

DT = pc.DTYPES


def _close(got, want, tol, what=""):
    got = got.double().cpu()
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), float(((got - want).abs() / tol).max()))


def _attend(dev, dtype, heads, kv, hd, page, lens, counts=None, window=0, sinks=0, seed=0,
            scale=None, max_tokens="given", max_length="given", poison=False, q=None):
    """Run decode (counts None) or prompt attention and check every output."""
    import ssalaad_amd as sa

    g = torch.Generator().manual_seed(seed)
    table, pages = pc.pages_of(lens, page, g)
    kp, vp = pc.cache(pages, kv, page, hd, dtype, g)
    n = len(lens) if counts is None else sum(counts)
    q = (2 * torch.randn(n, heads, hd, generator=g)).to(dtype) if q is None else q
    owners, pos = pc.chunk_rows([1] * len(lens) if counts is None else counts, lens)
    want, tol = pc.attention(q, kp, vp, table, owners, pos, page, window, sinks, scale, lens)
    kd, vd = kp.clone(), vp.clone()
    if poison:  # what no token of a sequence sees holds anything
        keep = torch.zeros(pages, page, dtype=torch.bool)
        for s, p in zip(owners, pos):
            for j in pc.seen(p, lens[s], window, sinks):
                keep[table[s, j // page], j % page] = True
        for x, junk in ((kd, float("nan")), (vd, float("inf"))):
            x.masked_fill_(~keep[:, None, :, None], junk)
    d = [t.to(dev) for t in (q, kd, vd, table, torch.tensor(lens, dtype=torch.int32))]
    kw = dict(window=window, sinks=sinks, scale=scale)
    if max_length != "given":
        kw["max_length"] = max_length
    else:
        kw["max_length"] = max(lens)
    if counts is None:
        out = sa.paged_decode_attention(*d, **kw)
    else:
        cu = torch.tensor([0] + counts).cumsum(0).int().to(dev)
        kw["max_tokens"] = max(counts) if max_tokens == "given" else max_tokens
        out = sa.paged_prompt_attention(*d, cu, **kw)
    assert out.dtype == dtype and out.shape == q.shape
    _close(out, want, tol, (lens, counts, window, sinks))
    return out


# ----------------------------------------------------------------- decode --
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("heads,kv", [(4, 4), (7, 1), (6, 2), (40, 2)])
@pytest.mark.parametrize("page", [16, 64])
def test_decode_matches_the_definition(dt, hd, heads, kv, page, gpu_device):
    _attend(gpu_device, DT[dt], heads, kv, hd, page, [1, 2, 0, 15, 16, 17, 129, 300], seed=hd + page)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (33, 50), (100, 0), (100, 70),
                                          (1000, 4)])
@pytest.mark.parametrize("page", [16, 128])
def test_decode_window_and_sinks(dt, window, sinks, page, gpu_device):
    _attend(gpu_device, DT[dt], 6, 2, 64, page, [0, 1, 31, 64, 100, 101, 257, 700], window=window,
            sinks=sinks, poison=True, seed=window + sinks)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("page", [16, 32, 256, 1024])
def test_decode_long_ragged(dt, page, gpu_device):
    _attend(gpu_device, DT[dt], 8, 2, 128, page, [5003, 1, 1024, 4097], poison=True, seed=page)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("counts", [None, [2, 1, 3]])  # one token each; chunks of few rows
def test_few_rows_lose_no_digits_of_their_weights(dt, hd, counts, gpu_device):
    """Outputs as close as one rounding: a weight in two numbers of the type is off by
    its u squared, or by half the least step of the 256-fold fp16 ones."""
    import ssalaad_amd as sa

    dev, dtype, g = gpu_device, DT[dt], torch.Generator().manual_seed(hd)
    lens = [717, 40, 3]
    table, pages = pc.pages_of(lens, 16, g)
    kp, vp = pc.cache(pages, 2, 16, hd, dtype, g)
    owners, pos = pc.chunk_rows(counts or [1, 1, 1], lens)
    q = (2 * torch.randn(len(owners), 4, hd, generator=g)).to(dtype)
    want, size, _, other = pc.attention_parts(q, kp, vp, table, owners, pos, 16)
    d = [t.to(dev) for t in (q, kp, vp, table, torch.tensor(lens, dtype=torch.int32))]
    if counts is None:
        got = sa.paged_decode_attention(*d)
    else:
        cu = torch.tensor([0] + counts).cumsum(0).int().to(dev)
        got = sa.paged_prompt_attention(*d, cu, max_tokens=3, max_length=717)
    tol = 1.01 * pc.u(dtype) ** 2 * size + other
    if dt == "f16":
        tol = tol + 717 * 2.0 ** -33 * vp.double().abs().max()
    _close(got, want, tol)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("infinity", [False, True])
def test_a_rows_sum_is_of_its_rounded_weights(dt, hd, infinity, gpu_device):
    """Many rows: a weight's rounding moves the result by its distance from its value,
    not by the value, also in rows taken anew beside an infinity of the last token."""
    import ssalaad_amd as sa

    dev, dtype, g = gpu_device, DT[dt], torch.Generator().manual_seed(hd)
    lens, counts = [230], [90]
    table, pages = pc.pages_of(lens, 16, g)
    kp, vp = pc.cache(pages, 1, 16, hd, dtype, g)
    vp = vp + 8  # values far from zero beside their spread
    q = (2 * torch.randn(90, 8, hd, generator=g)).to(dtype)
    owners, pos = pc.chunk_rows(counts, lens)
    want, _, spread, other = pc.attention_parts(q, kp, vp, table, owners, pos, 16)
    vd = vp.clone()
    if infinity:
        vd[table[0, 229 // 16], 0, 229 % 16, ::7] = float("inf")
    d = [t.to(dev) for t in (q, kp, vd, table, torch.tensor(lens, dtype=torch.int32))]
    got = sa.paged_prompt_attention(*d, torch.tensor([0, 90], dtype=torch.int32, device=dev))
    tol = 1.01 * pc.u(dtype) * spread + other
    if dt == "f16":  # 16-fold weights below half their least step
        tol = tol + 2 * 230 * 2.0 ** -29 * vp.double().abs().max()
    n = 89 if infinity else 90
    _close(got[:n], want[:n], tol[:n])


@pytest.mark.parametrize("bound", [1, 100, None])
def test_decode_bound_shapes_only_the_launch(bound, gpu_device):
    _attend(gpu_device, torch.bfloat16, 8, 8, 64, 16, [2000, 3], max_length=bound)
    _attend(gpu_device, torch.bfloat16, 8, 8, 64, 16, [2000, 300], counts=[40, 300],
            max_length=bound, max_tokens=bound)


# ----------------------------------------------------------------- prompt --
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("heads,kv", [(2, 2), (7, 1), (6, 2), (8, 1)])
def test_prompt_matches_the_definition(dt, hd, heads, kv, gpu_device):
    _attend(gpu_device, DT[dt], heads, kv, hd, 16, [1, 17, 70, 140], counts=[1, 17, 70, 140],
            seed=hd)
    _attend(gpu_device, DT[dt], heads, kv, hd, 64, [33, 200, 7, 131], counts=[2, 70, 0, 131],
            seed=hd + 1)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (16, 4), (40, 50), (100, 0), (64, 130)])
def test_prompt_window_and_sinks(dt, window, sinks, gpu_device):
    _attend(gpu_device, DT[dt], 4, 2, 64, 16, [150, 40, 333], counts=[150, 9, 65], window=window,
            sinks=sinks, poison=True, seed=window)
    _attend(gpu_device, DT[dt], 3, 1, 128, 32, [500], counts=[33], window=window, sinks=sinks,
            poison=True, seed=window)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [64, 65, 130, 200])
def test_prompts_of_many_sequences(dt, n, gpu_device):
    """More sequences than a wave has lanes, some without tokens; the rows of one of
    them take the kernel for many rows."""
    counts = pc.spread(9, n)
    for i in (0, 5, 63, n - 2):
        counts[i] = 0
    counts[n // 2], counts[n - 1] = 140, 75
    lens = [c + i % 7 if i % 3 else c for i, c in enumerate(counts)]
    heads, kv = (8, 1) if dt != "f32" else (32, 1)
    _attend(gpu_device, DT[dt], heads, kv, 64, 16, lens, counts=counts, poison=n == 65, seed=n)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("counts,lens", [([1], [3000]), ([5, 1], [2500, 1]), ([130], [1500]),
                                         ([300, 1, 2], [300, 900, 2])])
def test_prompt_few_rows_over_long_contexts(dt, counts, lens, gpu_device):
    _attend(gpu_device, DT[dt], 4, 1, 128, 16, lens, counts=counts, poison=True, seed=len(lens))
    _attend(gpu_device, DT[dt], 2, 2, 256, 64, lens, counts=counts, window=700, sinks=5, seed=3)


def test_prompt_of_one_token_each_equals_decode(gpu_device):
    import ssalaad_amd as sa

    g = torch.Generator().manual_seed(1)
    lens = [1, 40, 333]
    table, pages = pc.pages_of(lens, 16, g)
    kp, vp = (t.to(gpu_device) for t in pc.cache(pages, 2, 16, 64, torch.float32, g))
    q = torch.randn(3, 4, 64, generator=g).to(gpu_device)
    L = torch.tensor(lens, dtype=torch.int32, device=gpu_device)
    cu = torch.arange(4, dtype=torch.int32, device=gpu_device)
    a = sa.paged_decode_attention(q, kp, vp, table.to(gpu_device), L)
    b = sa.paged_prompt_attention(q, kp, vp, table.to(gpu_device), L, cu)
    torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-6)


def test_prompt_rows_that_see_nothing_and_tokens_past_the_last(gpu_device):
    """A chunk longer than its sequence's length, tokens past cu's end, a
    length beyond the table."""
    import ssalaad_amd as sa

    g = torch.Generator().manual_seed(2)
    dev = gpu_device
    for dtype in DT.values():
        table, pages = pc.pages_of([64, 32], 16, g)
        kp, vp = pc.cache(pages, 2, 16, 64, dtype, g)
        q = torch.randn(50, 4, 64, generator=g).to(dtype)
        lens, cu = [3, 1000], [0, 5, 45]  # 1000 is cut at 4 columns of 16
        out = sa.paged_prompt_attention(q.to(dev), kp.to(dev), vp.to(dev), table.to(dev),
                                        torch.tensor(lens, dtype=torch.int32, device=dev),
                                        torch.tensor(cu, dtype=torch.int32, device=dev))
        owners = [0] * 5 + [1] * 40 + [-1] * 5
        pos = [-2, -1, 0, 1, 2] + list(range(24, 64)) + [-1] * 5
        want, tol = pc.attention(q, kp, vp, table, owners, pos, 16, lengths=[3, 64])
        _close(out, want, tol)
        assert (out[:2] == 0).all() and (out[45:] == 0).all()


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tokens", [1, 10, 100, 600])  # few rows of a head, and many
def test_tokens_without_sequences_are_zeros(dt, tokens, gpu_device):
    import ssalaad_amd as sa

    dev = gpu_device
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)  # noqa: E731
    pool = torch.ones(3, 1, 16, 64, dtype=DT[dt], device=dev)
    q = torch.ones(tokens, 8, 64, dtype=DT[dt], device=dev)
    out = sa.paged_prompt_attention(q, pool, pool, i32(0, 4), i32(0), i32(1))
    assert out.shape == q.shape and not out.any()


def test_missing_pages_are_not_seen(gpu_device):
    import ssalaad_amd as sa

    g = torch.Generator().manual_seed(3)
    dev = gpu_device
    for dtype in DT.values():
        table, pages = pc.pages_of([200, 90], 16, g)
        table[0, 3], table[0, 7], table[1, 0], table[1, 5] = -1, pages, 2 ** 31 - 1, -(2 ** 31)
        kp, vp = pc.cache(pages, 2, 16, 128, dtype, g)
        d = [kp.to(dev), vp.to(dev), table.to(dev)]
        L = torch.tensor([200, 90], dtype=torch.int32, device=dev)
        q = torch.randn(2, 4, 128, generator=g).to(dtype)
        want, tol = pc.attention(q, kp, vp, table, [0, 1], [199, 89], 16)
        _close(sa.paged_decode_attention(q.to(dev), *d, L), want, tol)
        q = torch.randn(110, 4, 128, generator=g).to(dtype)
        owners, pos = pc.chunk_rows([20, 90], [200, 90])
        want, tol = pc.attention(q, kp, vp, table, owners, pos, 16)
        cu = torch.tensor([0, 20, 110], dtype=torch.int32, device=dev)
        _close(sa.paged_prompt_attention(q.to(dev), *d, L, cu), want, tol)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("heads,kv,counts,lens,window,sinks,bad", [
    (2, 1, [70], [70], 0, 0, [40, 69]),              # one row tile of each kernel
    (2, 1, [600], [600], 0, 0, [3, 300, 599]),       # many
    (4, 2, [9, 1], [2000, 300], 0, 0, [1995, 299]),  # few rows, contexts in parts
    (6, 2, [150, 40], [500, 900], 100, 3, [420, 870]),
    (1, 1, [330], [1200], 0, 0, [1000, 1190])])
def test_a_chunks_rows_see_no_later_infinity(dt, hd, heads, kv, counts, lens, window, sinks, bad,
                                             gpu_device):
    """NaN and infinities among the values of a chunk's later tokens, and before its
    later tokens' windows: rows that do not see them stay as they are."""
    import ssalaad_amd as sa

    g = torch.Generator().manual_seed(8)
    dtype = DT[dt]
    table, pages = pc.pages_of(lens, 16, g)
    kp, vp = pc.cache(pages, kv, 16, hd, dtype, g)
    for s, n in enumerate(lens):
        for j in bad:
            if j < n:
                at = vp[table[s, j // 16], 0, j % 16]
                at[3], at[hd // 2 + 1], at[hd - 1] = float("nan"), -float("inf"), float("inf")
    q = torch.randn(sum(counts), heads, hd, generator=g).to(dtype)
    owners, pos = pc.chunk_rows(counts, lens)
    want, tol = pc.attention(q, kp, vp, table, owners, pos, 16, window, sinks, None, lens)
    cu = torch.tensor([0] + counts).cumsum(0).int()
    d = [t.to(gpu_device) for t in (q, kp, vp, table, torch.tensor(lens, dtype=torch.int32), cu)]
    got = sa.paged_prompt_attention(*d, window=window, sinks=sinks, max_tokens=max(counts),
                                    max_length=max(lens)).double().cpu()
    fine = torch.isfinite(want)
    assert fine.any() and not fine.all()
    assert torch.equal(torch.isfinite(got), fine) and torch.equal(got.isnan(), want.isnan())
    assert ((got - want).abs() <= tol)[fine].all()
    assert torch.equal(got[~fine].sign().nan_to_num(), want[~fine].sign().nan_to_num())


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_attention_extreme_scores(dt, gpu_device):
    """Scores far apart and all far below zero: the running maximum carries them."""
    import ssalaad_amd as sa

    g = torch.Generator().manual_seed(4)
    dev, dtype = gpu_device, DT[dt]
    table, pages = pc.pages_of([300], 16, g)
    kp, vp = pc.cache(pages, 1, 16, 64, dtype, g)
    kp[..., 0] = torch.linspace(-1, 1, pages * 16).view(pages, 1, 16).to(dtype) - 4
    q = torch.zeros(1, 2, 64, dtype=dtype)
    q[0, 0, 0], q[0, 1, 0] = 1000.0, -1000.0
    want, tol = pc.attention(q, kp, vp, table, [0], [299], 16)
    L = torch.tensor([300], dtype=torch.int32, device=dev)
    d = [q.to(dev), kp.to(dev), vp.to(dev), table.to(dev), L]
    _close(sa.paged_decode_attention(*d), want, tol)
    cu = torch.tensor([0, 1], dtype=torch.int32, device=dev)
    _close(sa.paged_prompt_attention(*d, cu), want, tol)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("bits", [19, 20, 24, 25, 26, 27, 28, 31, 40, 100])
def test_attention_scores_of_any_size(dt, hd, sign, bits, gpu_device):
    """Scores of a single exact product, about 2^bits and 2^(bits - 7) apart: a row is
    the mean of the values at its largest ones. Few rows, many, one token each, and
    rows taken anew beside an infinity that only the last token sees."""
    import ssalaad_amd as sa

    dev, dtype, g = gpu_device, DT[dt], torch.Generator().manual_seed(bits)
    tokens = 560 if dt == "f32" else 100  # of 8 heads: many rows
    lens = [tokens + 70]
    table, pages = pc.pages_of(lens, 16, g)
    kp, vp = pc.cache(pages, 1, 16, hd, dtype, g)
    level = 1024 + 8 * torch.randint(0, 8, (pages, 1, 16), generator=g)
    kp[..., 0] = level.to(dtype)
    q = torch.zeros(tokens, 8, hd, dtype=dtype)
    q[..., 0] = sign * 1024
    at = torch.arange(lens[0])
    page = table[0].long()[at // 16]
    x = (sign * level[page, 0, at % 16]).double()
    v = vp[page, 0, at % 16].double()
    want, size = torch.empty(tokens, hd).double(), torch.empty(tokens, hd).double()
    for t in range(tokens):
        top = x[: 71 + t] == x[: 71 + t].max()
        want[t], size[t] = v[: 71 + t][top].mean(0), v[: 71 + t][top].abs().mean(0)
    # the weights' rounding (equal, if not all to 1), fp32 sums, the output's rounding
    tol = (2 * pc.u(dtype) + pc.F32 * (lens[0] + 64)) * size + pc.u(dtype) * want.abs()
    tol = 1.01 * tol + (lens[0] * 2.0 ** -25 * v.abs().amax(0) if dt == "f16" else 0) + 1e-30
    L = torch.tensor(lens, dtype=torch.int32, device=dev)
    kd, vd, td = kp.to(dev), vp.to(dev), table.to(dev)
    kw = dict(scale=2.0 ** (bits - 20))

    def close(out, rows, what):
        _close(out.cpu().double().amin(1), want[rows], tol[rows], what)
        _close(out.cpu().double().amax(1), want[rows], tol[rows], what)

    for n in (tokens, 3):
        cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
        out = sa.paged_prompt_attention(q[-n:].to(dev), kd, vd, td, L, cu, **kw)
        close(out, slice(tokens - n, tokens), (n, "prompt"))
        vd[table[0, -1].item(), 0, (lens[0] - 1) % 16, 5] = float("inf")
        out = sa.paged_prompt_attention(q[-n:].to(dev), kd, vd, td, L, cu, **kw)
        close(out[:-1], slice(tokens - n, tokens - 1), (n, "prompt beside an infinity"))
        vd.copy_(vp)
    close(sa.paged_decode_attention(q[-1:].to(dev), kd, vd, td, L, **kw),
          slice(tokens - 1, tokens), "decode")


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("scale", [0.0, 1e-44, 1e-46, -1e-46, 5e-324])
def test_attention_of_a_vanishing_scale(dt, scale, gpu_device):
    """Means of what is seen, in every kernel: few rows, many, one token each."""
    _attend(gpu_device, DT[dt], 4, 2, 64, 16, [300, 1, 0], scale=scale)
    _attend(gpu_device, DT[dt], 4, 2, 64, 16, [90, 30], counts=[40, 30], scale=scale)
    _attend(gpu_device, DT[dt], 8, 1, 64, 16, [700], counts=[560 if dt == "f32" else 100],
            window=50, sinks=3, scale=scale)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_attention_strides(dt, gpu_device):
    """q as a view of a fused projection, pools interleaved, a wider table."""
    import ssalaad_amd as sa

    g = torch.Generator().manual_seed(5)
    dev, dtype = gpu_device, DT[dt]
    lens, counts = [100, 61], [30, 61]
    table, pages = pc.pages_of(lens, 32, g)
    kp, vp = pc.cache(pages, 2, 32, 128, dtype, g)
    both = torch.empty(pages, 2, 2, 34, 128, dtype=dtype, device=dev)[:, :, :, 1:33]
    both[:, 0], both[:, 1] = kp.to(dev), vp.to(dev)
    wide = torch.full((2, 9), -1, dtype=torch.int32, device=dev)
    wide[:, 2: 2 + table.shape[1]] = table.to(dev)
    tv = wide[:, 2: 2 + table.shape[1]]
    L = torch.tensor(lens, dtype=torch.int32, device=dev)
    qkv = torch.randn(91, 8, 128, generator=g).to(dtype)
    q, qd = qkv[:, ::2], qkv.to(dev)[:, ::2]  # every second of 8 heads
    assert not qd.is_contiguous()
    owners, pos = pc.chunk_rows(counts, lens)
    want, tol = pc.attention(q, kp, vp, table, owners, pos, 32)
    cu = torch.tensor([0, 30, 91], dtype=torch.int32, device=dev)
    _close(sa.paged_prompt_attention(qd, both[:, 0], both[:, 1], tv, L, cu), want, tol)
    want, tol = pc.attention(q[:2], kp, vp, table, [0, 1], [99, 60], 32)
    _close(sa.paged_decode_attention(qd[:2], both[:, 0], both[:, 1], tv, L), want, tol)
    odd = torch.empty(2 * 4 * 128 + 1, dtype=dtype, device=dev)[1:].view(2, 4, 128)
    odd.copy_(qd[:2])  # misaligned rows
    _close(sa.paged_decode_attention(odd, both[:, 0], both[:, 1], tv, L), want, tol)


def test_offsets_beyond_32_bits(gpu_device):
    """Pages whose elements and bytes lie past 2^31 and 2^32."""
    import ssalaad_amd as sa

    dev, g = gpu_device, torch.Generator().manual_seed(6)
    kv, page, hd = 2, 64, 128
    pages = (1 << 32) // (kv * page * hd) + 9  # 2^32 elements and a little
    kp = torch.empty(pages, kv, page, hd, dtype=torch.bfloat16, device=dev)
    vp = torch.empty_like(kp)
    ids = [pages - 1, 0, pages // 2 + 1, pages - 7]
    small = pc.cache(4, kv, page, hd, torch.bfloat16, g)
    for i, p in enumerate(ids):
        kp[p], vp[p] = small[0][i].to(dev), small[1][i].to(dev)
    table = torch.tensor([ids], dtype=torch.int32)
    local = torch.arange(4, dtype=torch.int32)[None]
    L = torch.tensor([250], dtype=torch.int32, device=dev)
    q = torch.randn(40, 4, hd, generator=g).to(torch.bfloat16)
    owners, pos = pc.chunk_rows([40], [250])
    want, tol = pc.attention(q, *small, local, owners, pos, page)
    cu = torch.tensor([0, 40], dtype=torch.int32, device=dev)
    _close(sa.paged_prompt_attention(q.to(dev), kp, vp, table.to(dev), L, cu), want, tol)
    _close(sa.paged_decode_attention(q[-1:].to(dev), kp, vp, table.to(dev), L), want[-1:], tol[-1:])
    cos, sin = (t.to(dev) for t in pc.angles(256, hd))
    k = torch.randn(1, kv, hd, generator=g).to(torch.bfloat16)
    sa.paged_append(q[:1].to(dev), k.to(dev), k.to(dev), cos, sin, kp, vp, table.to(dev),
                    torch.zeros(1, dtype=torch.int32, device=dev),
                    torch.tensor([255], dtype=torch.int32, device=dev))
    assert torch.equal(vp[pages - 7, :, 63].cpu(), k[0])
    refs = torch.zeros(pages, dtype=torch.int32, device=dev)
    refs[table[0].long()] = 1
    t2, l2, r2, ok = sa.fork_pages(torch.cat([table, torch.full((1, 4), -1).int()]).to(dev),
                                   torch.tensor([250, 0], dtype=torch.int32, device=dev), refs, kp,
                                   vp, torch.tensor([0], dtype=torch.int32, device=dev),
                                   torch.tensor([1], dtype=torch.int32, device=dev))
    assert ok.all() and t2[1].tolist() == [*ids[:3], 1]
    assert torch.equal(kp[1, :, :58], kp[pages - 7, :, :58])
    t3, r3, live = sa.compact_pages(t2, r2, kp, vp)
    assert int(live) == 5 and int(r3[:5].min()) > 0 and int(r3[5:].abs().max()) == 0
    out = sa.paged_decode_attention(q[-1:].to(dev).repeat(2, 1, 1), kp, vp, t3,
                                    torch.tensor([250, 250], dtype=torch.int32, device=dev))
    # position 255 was written after the first check, but lies past the length
    _close(out, want[-1:].repeat(2, 1, 1), tol[-1:].repeat(2, 1, 1))


# ----------------------------------------------------------------- append --
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("heads,kv,page", [(4, 4, 16), (7, 1, 32), (6, 2, 128)])
def test_append_matches_the_definition(dt, hd, norm, heads, kv, page, gpu_device):
    import ssalaad_amd as sa

    dev, dtype = gpu_device, DT[dt]
    g = torch.Generator().manual_seed(hd + heads)
    lens, counts = [1, 50, 0, 133], [1, 7, 0, 133]
    table, pages = pc.pages_of(lens, page, g)
    kp, vp = pc.cache(pages, kv, page, hd, dtype, g)
    owners, pos = pc.chunk_rows(counts, lens)
    n = len(owners)
    qkv = torch.randn(n, heads + 2 * kv, hd, generator=g).to(dtype)
    q, k, v = qkv.split([heads, kv, kv], 1)
    qn = (1 + 0.1 * torch.randn(hd, generator=g)).to(dtype) if norm else None
    kn = (1 + 0.1 * torch.randn(hd, generator=g)).to(dtype) if norm else None
    cos, sin = pc.angles(140, hd)
    qkv_d = qkv.to(dev)
    qd, kd, vd = qkv_d.split([heads, kv, kv], 1)  # views
    kpd, vpd = kp.to(dev), vp.to(dev)
    ids = torch.tensor(owners, dtype=torch.int32, device=dev)
    ps = torch.tensor(pos, dtype=torch.int32, device=dev)
    out = sa.paged_append(qd, kd, vd, cos.to(dev), sin.to(dev), kpd, vpd, table.to(dev), ids, ps,
                          q_norm=None if qn is None else qn.to(dev),
                          k_norm=None if kn is None else kn.to(dev), eps=1e-5)
    _close(out, *pc.rotated(q, qn, 1e-5, cos, sin, pos))
    wk, tk = pc.rotated(k, kn, 1e-5, cos, sin, pos)
    pg = torch.tensor([int(table[s, p // page]) for s, p in zip(owners, pos)])
    sl = torch.tensor([p % page for p in pos])
    _close(kpd.cpu()[pg, :, sl], wk, tk)
    assert torch.equal(vpd.cpu()[pg, :, sl], v)
    rest = torch.ones(pages, page, dtype=torch.bool)
    rest[pg, sl] = False
    for a, b in ((kpd, kp), (vpd, vp)):  # nothing else changed
        assert torch.equal(a.cpu().transpose(1, 2)[rest], b.transpose(1, 2)[rest])


def test_append_passes_over_bad_places(gpu_device):
    import ssalaad_amd as sa

    dev, g = gpu_device, torch.Generator().manual_seed(7)
    table = torch.tensor([[0, -1, 5], [1, 2, 3]], dtype=torch.int32)
    kp, vp = pc.cache(4, 2, 16, 64, torch.float32, g)
    q, k, v = (torch.randn(9, h, 64, generator=g) for h in (4, 2, 2))
    seqs = [0, 0, 0, -1, 2, 1, 1, 1, 1]
    pos = [3, 17, 40, 1, 1, -1, 48, 100, 47]  # good: 0 and 8
    cos, sin = pc.angles(60, 64)
    kd, vd = kp.to(dev), vp.to(dev)
    out = sa.paged_append(q.to(dev), k.to(dev), v.to(dev), cos.to(dev), sin.to(dev), kd, vd,
                          table.to(dev), torch.tensor(seqs, dtype=torch.int32, device=dev),
                          torch.tensor(pos, dtype=torch.int32, device=dev))
    want, tol = pc.rotated(q, None, 0, cos, sin, [p if 0 <= p < 60 else 0 for p in pos])
    for t, p in enumerate(pos):
        if not 0 <= p < 60:
            want[t] = 0
    _close(out, want, tol)
    vp[0, :, 3], vp[3, :, 15] = v[0], v[8]
    assert torch.equal(vd.cpu(), vp)


# ------------------------------------------------------------------ pages --
def _state(seed, seqs=6, page=16, pages=40, cols=5):
    g = torch.Generator().manual_seed(seed)
    table = torch.full((seqs, cols), -1, dtype=torch.int32)
    lens, refs = [], [0] * pages
    order = torch.randperm(pages, generator=g).tolist()
    for s in range(seqs):
        n = int(torch.randint(0, cols * page + 1, (1,), generator=g))
        lens.append(n)
        for c in range(-(-n // page)):
            p = int(table[s - 1, c]) if s and c == 0 and table[s - 1, 0] >= 0 else order.pop()
            table[s, c] = p
            refs[p] += 1
    return table, torch.tensor(lens, dtype=torch.int32), torch.tensor(refs, dtype=torch.int32), g


@pytest.mark.parametrize("seed", range(4))
def test_free_takes_references_back(seed, gpu_device):
    import ssalaad_amd as sa

    table, lens, refs, _ = _state(seed)
    gone = [[], [0], [3, 1, 3, -1, 99], list(range(6))][seed]
    before = [t.to(gpu_device) for t in (table, lens, refs)]
    got = sa.free_pages(*before, torch.tensor(gone, dtype=torch.int32, device=gpu_device))
    for t, b in zip((table, lens, refs), before):
        assert torch.equal(b.cpu(), t)  # the given state stays
    for s in set(x for x in gone if 0 <= x < 6):
        for p in table[s].tolist():
            if p >= 0:
                refs[p] -= 1
        table[s], lens[s] = -1, 0
    for a, b in zip(got, (table, lens, refs)):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("seqs,cols,pages", [
    (1, 1, 1), (4096, 1, 4096), (32, 128, 4095), (1024, 4, 4097), (4097, 1, 300), (3, 0, 5), (0, 4, 7)])
def test_free_at_the_edge_of_a_small_state(seqs, cols, pages, gpu_device):
    import ssalaad_amd as sa

    g = torch.Generator().manual_seed(6)
    wide = torch.randint(-2, pages + 2, (seqs, cols + 3), generator=g).int()
    lens = torch.randint(0, 400, (seqs,), generator=g).int()
    refs = torch.randint(5, 9, (pages,), generator=g).int()
    gone = torch.randint(-1, seqs + 1, (2 * seqs // 3 + 1,), generator=g).int()
    got = sa.free_pages(wide.to(gpu_device)[:, :cols], *(t.to(gpu_device) for t in (lens, refs, gone)))
    table = wide[:, :cols].clone()
    rows = gone[(gone >= 0) & (gone < seqs)].long().unique()
    held = table[rows]
    held = held[(held >= 0) & (held < pages)].long()
    refs.index_add_(0, held, torch.full(held.shape, -1, dtype=torch.int32))
    table[rows], lens[rows] = -1, 0
    for a, b in zip(got, (table, lens, refs)):
        assert torch.equal(a.cpu(), b)


def test_free_of_a_large_state(gpu_device):
    import ssalaad_amd as sa

    g = torch.Generator().manual_seed(5)
    seqs, cols, pages = 5000, 30, 90000
    table = torch.randint(-3, pages + 2, (seqs, cols), generator=g).int()
    lens = torch.randint(0, 400, (seqs,), generator=g).int()
    refs = torch.randint(5, 9, (pages,), generator=g).int()
    gone = torch.randint(-1, seqs + 1, (700,), generator=g).int()
    got = sa.free_pages(*(t.to(gpu_device) for t in (table, lens, refs, gone)))
    rows = gone[(gone >= 0) & (gone < seqs)].long().unique()
    held = table[rows]
    held = held[(held >= 0) & (held < pages)].long()
    refs.index_add_(0, held, torch.full(held.shape, -1, dtype=torch.int32))
    table[rows], lens[rows] = -1, 0
    for a, b in zip(got, (table, lens, refs)):
        assert torch.equal(a.cpu(), b)


def _fork(table, lens, refs, pools, src, dst, page):
    """The definition, in host integers."""
    t, n, r, ok = table.clone(), lens.clone(), refs.clone(), []
    P = refs.numel()
    S, cols = table.shape
    for i, (a, d) in enumerate(zip(src, dst)):
        good = 0 <= a < S and 0 <= d < S and int(lens[d]) == 0 and d not in dst[:i]
        good = good and 0 <= int(lens[a]) <= cols * page
        if good:
            whole, part = divmod(int(lens[a]), page)
            need = whole + (part > 0)
            good = all(0 <= int(p) < P for p in table[a, :need])
        fresh = -1
        if good and part:
            free = [p for p in range(P) if int(r[p]) == 0 and int(refs[p]) == 0]
            good = bool(free)
            fresh = free[0] if good else -1
        ok.append(good)
        if not good:
            continue
        t[d] = -1
        for c in range(whole):
            t[d, c] = table[a, c]
            r[int(table[a, c])] += 1
        if part:
            t[d, whole] = fresh
            r[fresh] = 1
            for x in pools:
                x[:, fresh, :, :part] = x[:, int(table[a, whole]), :, :part]
        n[d] = lens[a]
    return t, n, r, torch.tensor(ok, dtype=torch.bool)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("seed,pages", [(0, 40), (1, 40), (2, 33), (3, 26)])
def test_fork_shares_and_copies(dt, seed, pages, gpu_device):
    import ssalaad_amd as sa

    dev, page = gpu_device, 16
    table, lens, refs, g = _state(seed, pages=pages)
    extra = torch.full((6, 5), -1, dtype=torch.int32)
    table, lens = torch.cat([table, extra]), torch.cat([lens, torch.zeros(6, dtype=torch.int32)])
    src = [0, 1, 2, 2, 9, 3, -1, 4, 5, 12, 5]
    dst = [6, 7, 8, 6, 9, 0, 10, 99, 10, 11, 11]
    kp, vp = pc.cache(pages, 2, page, 64, DT[dt], g, layers=3)
    kd, vd = kp.to(dev), vp.to(dev)
    ints = [torch.tensor(x, dtype=torch.int32, device=dev) for x in (src, dst)]
    got = sa.fork_pages(table.to(dev), lens.to(dev), refs.to(dev), kd, vd, *ints)
    want = _fork(table, lens, refs, (kp, vp), src, dst, page)
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)
    assert torch.equal(kd.cpu(), kp) and torch.equal(vd.cpu(), vp)


def test_fork_of_missing_pages_and_one_layer(gpu_device):
    import ssalaad_amd as sa

    dev, g = gpu_device, torch.Generator().manual_seed(9)
    table = torch.tensor([[3, -1], [0, 7], [-1, -1], [-1, -1]], dtype=torch.int32)
    lens = torch.tensor([20, 16, 0, 0], dtype=torch.int32)
    refs = torch.tensor([1, 0, 0, 1], dtype=torch.int32)
    kp, vp = pc.cache(4, 1, 16, 128, torch.bfloat16, g)
    kd, vd = kp.to(dev), vp.to(dev)
    got = sa.fork_pages(table.to(dev), lens.to(dev), refs.to(dev), kd, vd,
                        torch.tensor([0, 1], dtype=torch.int32, device=dev),
                        torch.tensor([2, 3], dtype=torch.int32, device=dev))
    assert got[3].tolist() == [False, True]  # a whole page only, nothing copied
    assert got[0].tolist() == [[3, -1], [0, 7], [-1, -1], [0, -1]]
    assert got[2].tolist() == [2, 0, 0, 1] and got[1].tolist() == [20, 16, 0, 16]
    assert torch.equal(kd.cpu(), kp) and torch.equal(vd.cpu(), vp)


def test_a_fork_gives_back_what_its_row_held(gpu_device):
    """An empty sequence whose row names pages (reserved for it, say): the counts stay
    those of the entries."""
    import ssalaad_amd as sa

    dev, g = gpu_device, torch.Generator().manual_seed(14)
    table = torch.tensor([[3, 5, -1], [1, 9, 0], [2, -1, 3], [-1, -1, -1]], dtype=torch.int32)
    lens = torch.tensor([20, 0, 0, 0], dtype=torch.int32)
    refs = torch.tensor([1, 1, 1, 2, 0, 1, 0], dtype=torch.int32)
    kp, vp = (t.to(dev) for t in pc.cache(7, 1, 16, 64, torch.bfloat16, g, layers=2))
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    t, n, r, ok = sa.fork_pages(table.to(dev), lens.to(dev), refs.to(dev), kp, vp, i32(0, 0, 0),
                                i32(1, 2, 1))
    assert ok.tolist() == [True, True, False] and n.tolist() == [20, 20, 20, 0]
    assert t.tolist() == [[3, 5, -1], [3, 4, -1], [3, 6, -1], [-1, -1, -1]]
    held = t[t >= 0].long().cpu()
    assert torch.equal(r.cpu().long(), torch.bincount(held, minlength=7))


def test_many_forks_and_pages(gpu_device):
    """More forks and pages than one workgroup holds at a time, and more forks
    than free pages."""
    import ssalaad_amd as sa

    dev, n, page = gpu_device, 2500, 16
    g = torch.Generator().manual_seed(13)
    pages = 9000
    order = torch.randperm(pages, generator=g).int()
    table = torch.full((2 * n, 1), -1, dtype=torch.int32)
    table[:n, 0] = order[:n]
    lens = torch.zeros(2 * n, dtype=torch.int32)
    lens[:n] = torch.randint(0, 17, (n,), generator=g).int()
    table[:n][lens[:n] == 0] = -1
    refs = torch.zeros(pages, dtype=torch.int32)
    refs[table[table >= 0].long()] = 1
    refs[order[n: pages - 1200].long()] = 1  # others hold these: too few are free
    kp, vp = pc.cache(pages, 1, page, 64, torch.bfloat16, g, layers=1)
    src = torch.randperm(n, generator=g)
    dst = n + torch.randperm(n, generator=g)
    kd, vd = kp.to(dev), vp.to(dev)
    got = sa.fork_pages(table.to(dev), lens.to(dev), refs.to(dev), kd, vd, src.int().to(dev),
                        dst.int().to(dev))
    part = lens[src].long() % page
    need = part > 0
    free = (refs == 0).nonzero()[:, 0]
    rank = need.long().cumsum(0) - 1
    ok = ~need | (rank < free.numel())
    assert need.sum() > free.numel() > 1024
    t, ln, r = table.clone(), lens.clone(), refs.clone()
    i = (ok & need).nonzero()[:, 0]
    fresh = free[rank[i]]
    t[dst[i], 0] = fresh.int()
    r[fresh] = 1
    whole = (ok & ~need & (lens[src] > 0)).nonzero()[:, 0]
    t[dst[whole], 0] = table[src[whole], 0]
    r[table[src[whole], 0].long()] += 1
    ln[dst[ok]] = lens[src[ok]]
    for a, b in zip(got, (t, ln, r, ok)):
        assert torch.equal(a.cpu(), b)
    keep = torch.arange(page) < part[i, None]
    for a, b in ((kd, kp), (vd, vp)):
        b[0, fresh] = torch.where(keep[:, None, :, None], b[0, table[src[i], 0].long()], b[0, fresh])
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("pages", [1, 5, 64, 1023, 2500])
@pytest.mark.parametrize("share", [0.0, 0.1, 0.6, 1.0])
def test_compact_moves_the_pages_in_use_down(pages, share, gpu_device):
    import ssalaad_amd as sa

    dev, g = gpu_device, torch.Generator().manual_seed(pages)
    live = torch.rand(pages, generator=g) < share
    refs = torch.where(live, torch.randint(1, 4, (pages,), generator=g), 0).int()
    ids = live.nonzero()[:, 0].int()
    table = torch.full((3, pages + 1), -1, dtype=torch.int32)
    for s in range(3):
        table[s, : ids.numel()] = ids[torch.randperm(ids.numel(), generator=g)]
    table[2, -1] = pages + 5  # left as it is
    kp, vp = pc.cache(pages, 2, 16, 64, torch.float16, g, layers=2)
    kd, vd = kp.to(dev), vp.to(dev)
    t, r, n = sa.compact_pages(table.to(dev), refs.to(dev), kd, vd)
    L = int(live.sum())
    holes = [p for p in range(L) if not live[p]]
    movers = [p for p in range(L, pages) if live[p]]
    to = list(range(pages))
    for a, b in zip(movers, holes):
        to[a] = b
        refs[b], refs[a] = refs[a].clone(), 0
        kp[:, b], vp[:, b] = kp[:, a], vp[:, a]
    want = torch.tensor([[to[p] if 0 <= p < pages else p for p in row] for row in table.tolist()])
    assert int(n) == L and n.shape == ()
    assert torch.equal(t.cpu(), want.int()) and torch.equal(r.cpu(), refs)
    assert torch.equal(kd.cpu(), kp) and torch.equal(vd.cpu(), vp)


# --------------------------------------------------------------- logprobs --
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 7, 7), (5, 100, 20), (2, 1000, 64),
                                            (17, 4097, 8), (1, 160000, 20), (4, 32003, 0)])
def test_logprobs_match_the_definition(dt, rows, vocab, top, gpu_device):
    import ssalaad_amd as sa

    g = torch.Generator().manual_seed(vocab)
    x = (3 * torch.randn(rows, vocab, generator=g)).to(DT[dt])
    if vocab > 50:  # a forbidden third, and a row with one likely token
        x[0, torch.rand(vocab, generator=g) < 0.33] = float("-inf")
        x[-1, vocab // 2] = 40
    tok = torch.randint(0, vocab, (rows,), generator=g)
    tok[-1] = vocab // 2
    wide = torch.full((rows, vocab + 5), 99.0, dtype=DT[dt], device=gpu_device)
    wide[:, 2: vocab + 2] = x.to(gpu_device)
    given, ent, ids, lp, tol_lp, tol_ent = pc.logprobs(x, tok, top)
    for view in (x.to(gpu_device), wide[:, 2: vocab + 2]):  # a strided, unaligned view too
        got = sa.token_logprobs(view, tok.to(gpu_device), top=top)
        assert torch.equal(got.top_ids.cpu(), ids)
        t = tol_lp.gather(1, tok[:, None])[:, 0]
        same = given.isinf()
        assert torch.equal(got.logprobs.cpu()[same].double(), given[same])
        _close(got.logprobs.cpu()[~same], given[~same], t[~same])
        _close(got.entropy, ent, tol_ent)
        want = lp.gather(1, ids)
        fin = want.isfinite()
        assert torch.equal(got.top_logprobs.cpu()[~fin].double(), want[~fin])
        _close(got.top_logprobs.cpu()[fin], want[fin], tol_lp.gather(1, ids)[fin])


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab", [64, 5000, 100000])
def test_logprobs_ties_go_to_the_lowest_index(dt, vocab, gpu_device):
    import ssalaad_amd as sa

    g = torch.Generator().manual_seed(vocab)
    rows = [torch.zeros(vocab), torch.randint(0, 3, (vocab,), generator=g).float(),
            torch.full((vocab,), -1e4), torch.where(torch.arange(vocab) % 2 == 1, 0.0, -0.0),
            torch.where(torch.arange(vocab) == vocab - 1, 1.0, float("-inf")),
            -torch.arange(vocab).div(7, rounding_mode="floor").float().clamp(max=100),
            torch.arange(vocab).div(7, rounding_mode="floor").float().clamp(max=100)]
    x = torch.stack(rows).to(DT[dt])
    want = torch.sort(x.double() + 0.0, dim=-1, descending=True, stable=True).indices[:, :20]
    got = sa.token_logprobs(x.to(gpu_device), torch.zeros(7, dtype=torch.int64, device=gpu_device),
                            top=20)
    assert torch.equal(got.top_ids.cpu(), want)


def test_logprobs_of_broken_rows(gpu_device):
    import ssalaad_amd as sa

    inf, nan = float("inf"), float("nan")
    x = torch.randn(6, 500, generator=torch.Generator().manual_seed(1))
    x[0] = -inf
    x[1, 400] = inf
    x[2, 3] = nan
    x[3, 7] = -inf
    tok = torch.tensor([5, 400, 0, 7, -1, 500])
    for dt in DT.values():
        got = sa.token_logprobs(x.to(dt).to(gpu_device), tok.to(gpu_device), top=4)
        assert got.logprobs[:3].isnan().all() and got.entropy[:3].isnan().all()
        assert got.top_logprobs[:3].isnan().all()
        assert got.top_ids[0].tolist() == [0, 1, 2, 3] and int(got.top_ids[1, 0]) == 400
        assert int(got.top_ids[2, 0]) == 3
        assert float(got.logprobs[3]) == -inf and got.logprobs[4:].isnan().all()
        assert got.entropy[3:].isfinite().all() and got.top_logprobs[3:].isfinite().all()


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab,top", [(1, 1), (5, 5), (64, 64), (700, 20)])
def test_logprobs_order_a_row_of_nans(dt, vocab, top, gpu_device):
    """NaN first, also in the first place, each index once, the whole row asked for."""
    import ssalaad_amd as sa

    x = torch.randn(4, vocab, generator=torch.Generator().manual_seed(vocab))
    x[0, 0] = float("nan")
    x[1, ::2] = float("nan")
    x[2] = float("nan")
    x[3, 0], x[3, -1] = float("inf"), float("nan")
    x = x.to(DT[dt])
    order = torch.where(x.isnan(), float("inf"), x.double().clamp(max=1e300))
    want = torch.sort(order, dim=-1, descending=True, stable=True).indices[:, :top]
    got = sa.token_logprobs(x.to(gpu_device), torch.zeros(4, dtype=torch.int64, device=gpu_device),
                            top=top)
    assert torch.equal(got.top_ids.cpu(), want)
    assert got.logprobs.isnan().all() and got.entropy.isnan().all()
    assert got.top_logprobs.isnan().all()


def test_logprobs_keep_the_digits_of_a_certain_token(gpu_device):
    """One token with almost all the mass: log p near zero, to fp32 relative accuracy."""
    import ssalaad_amd as sa

    x = torch.zeros(1, 30000)
    x[0, 12345] = 25.0
    given, ent, *_ = pc.logprobs(x, torch.tensor([12345]), 0)
    got = sa.token_logprobs(x.to(gpu_device), torch.tensor([12345], device=gpu_device))
    # every small term carries the same exponent, 25: 2·25 + 4 roundings
    assert abs(float(got.logprobs[0]) / float(given[0]) - 1) <= 56 * pc.F32
    assert abs(float(got.entropy[0]) / float(ent[0]) - 1) <= 60 * pc.F32


# --------------------------------------------------------- streams, graphs --
def test_a_captured_step_replays(gpu_device):
    """Append, attention, fork and scores in one graph, replayed between eager
    work; every replay equals the eager result."""
    import ssalaad_amd as sa

    dev, g = gpu_device, torch.Generator().manual_seed(11)
    lens = [700, 33, 0]
    table, pages = pc.pages_of(lens, 16, g, spare=4, cols=60)
    kp, vp = (t.to(dev) for t in pc.cache(pages, 2, 16, 64, torch.bfloat16, g))
    q, k, v = (torch.randn(2, h, 64, generator=g).to(torch.bfloat16).to(dev) for h in (4, 2, 2))
    cos, sin = (t.to(dev) for t in pc.angles(800, 64))
    L = torch.tensor(lens, dtype=torch.int32, device=dev)
    tb = table.to(dev)
    refs = torch.zeros(pages, dtype=torch.int32)
    refs[table[table >= 0].long()] = 1
    refs = refs.to(dev)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    seqs, pos, src, dst, one = i32(0, 1), i32(699, 32), i32(0), i32(2), i32(0)
    cu = i32(0, 1, 2)
    logits = torch.randn(2, 1000, generator=g).to(dev)
    tok = torch.tensor([1, 2], device=dev)

    def step():
        r = sa.paged_append(q, k, v, cos, sin, kp, vp, tb, seqs, pos)
        a = sa.paged_decode_attention(r, kp, vp, tb[:2], L[:2], max_length=700)
        b = sa.paged_prompt_attention(r, kp, vp, tb[:2], L[:2], cu, max_length=700)
        t, n, rf, ok = sa.fork_pages(tb, L, refs, kp, vp, src, dst)
        t2, n2, rf2 = sa.free_pages(t, n, rf, one)
        t3, rf3, live = sa.compact_pages(t2, rf2, kp.clone(), vp.clone())
        return (r, a, b, t, n, rf, ok, t2, n2, rf2, t3, rf3, live,
                *sa.token_logprobs(logits, tok, top=3))

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        want = [t.clone() for t in step()]
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step()
    for i in range(4):
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), i
        eager = step()
        torch.cuda.synchronize()
        for a, b in zip(eager, want):
            assert torch.equal(a, b), i
        q.add_(0)  # eager work between the replays


def test_calls_of_several_threads(gpu_device):
    """Eight threads, a stream each, whose first calls of these kernels meet."""
    import threading

    import ssalaad_amd as sa

    dev, g = gpu_device, torch.Generator().manual_seed(15)
    table, pages = pc.pages_of([300], 16, g)
    td, L = table.to(dev), torch.tensor([300], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 90], dtype=torch.int32, device=dev)
    kinds = [(DT[dt], hd) for dt in ("f32", "bf16", "f16") for hd in (128, 256)]
    data = {k: tuple(t.to(dev) for t in (*pc.cache(pages, 1, 16, k[1], k[0], g),
                                         torch.randn(90, 8, k[1], generator=g).to(k[0])))
            for k in kinds}
    torch.cuda.synchronize()
    results, start = [None] * 8, threading.Barrier(8)

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream(dev)):
            start.wait()
            results[i] = [f for kp, vp, q in data.values()
                          for f in (sa.paged_prompt_attention(q, kp, vp, td, L, cu),
                                    sa.paged_decode_attention(q[:1], kp, vp, td, L))]
            torch.cuda.current_stream(dev).synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for r in results[1:]:
        for a, b in zip(r, results[0], strict=True):
            assert torch.equal(a, b)
    assert all(bool(a.isfinite().all()) and bool(a.any()) for a in results[0])


# ------------------------------------------------------------- call paths --
class _Nothing:
    """A compiled path that takes no call."""

    def __getattr__(self, name):
        return lambda *a: None


def test_the_compiled_and_the_python_path_issue_the_same_calls(gpu_device, monkeypatch):
    import ssalaad_amd as sa
    from ssalaad_amd import _lib

    dev = gpu_device

    def results():
        g = torch.Generator().manual_seed(12)
        lens, counts = [40, 17, 0], [9, 17, 0]
        table, pages = pc.pages_of(lens, 16, g, cols=4)
        kp, vp = (t.to(dev) for t in pc.cache(pages, 2, 16, 64, torch.bfloat16, g))
        q, k, v = (torch.randn(26, h, 64, generator=g).to(torch.bfloat16).to(dev) for h in (4, 2, 2))
        cos, sin = (t.to(dev) for t in pc.angles(64, 64))
        w = (1 + torch.randn(64, generator=g)).to(torch.bfloat16).to(dev)
        owners, pos = pc.chunk_rows(counts, lens)
        i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        tb, L = table.to(dev), i32(*lens)
        refs = torch.zeros(pages, dtype=torch.int32)
        refs[table[table >= 0].long()] = 1
        out = [sa.paged_append(q, k, v, cos, sin, kp, vp, tb, i32(*owners), i32(*pos), q_norm=w)]
        out.append(sa.paged_decode_attention(q[:3], kp, vp, tb, L, window=20, sinks=2, scale=0.2))
        out.append(sa.paged_prompt_attention(q, kp, vp, tb, L, i32(0, 9, 26, 26), max_tokens=17,
                                             max_length=40))
        out += sa.fork_pages(tb, L, refs.to(dev), kp, vp, i32(0), i32(2))
        out += sa.free_pages(*out[-4:-1], i32(1))
        out += sa.compact_pages(out[-3], out[-1], kp, vp)
        out += sa.token_logprobs(torch.randn(4, 99, generator=g).to(dev),
                                 torch.arange(4, device=dev), top=5)
        return [t.cpu() for t in (*out, kp, vp)]

    taken = results()
    monkeypatch.setattr(_lib, "tensorcall", _Nothing)
    for a, b in zip(taken, results(), strict=True):
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_the_compiled_path_takes_what_a_step_passes(gpu_device):
    from ssalaad_amd import _lib

    tc, dev = _lib.tensorcall(), gpu_device
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device=dev)  # noqa: E731
    i = lambda *s: z(*s, dtype=torch.int32)  # noqa: E731
    pool = z(9, 2, 16, 64)
    args = [z(3, 2, 64), pool, pool, i(3, 5), i(3), None, 0, 0, None, 1, None]
    assert torch.is_tensor(tc.attention(*args))
    assert torch.is_tensor(tc.attention(torch.nn.Parameter(args[0]), *args[1:]))
    for k, bad in ((0, z(3, 2, 128)[:, :, ::2]), (0, z(3, 3, 64)), (0, args[0].float()),
                   (1, z(9, 2, 17, 64)[:, :, 1:]), (3, i(3, 5).long()), (4, i(6)[::2]),
                   (6, -1), (7, 1.5), (8, "x"), (10, -1)):
        assert tc.attention(*args[:k], bad, *args[k + 1:]) is None, k
    big = z(9, 2, 16, 64, dtype=torch.int8)
    assert tc.attention(z(3, 2, 64, dtype=torch.int8), big, big, *args[3:]) is None
    # a page size without a kernel is the C ABI's refusal
    odd = z(9, 2, 24, 64)
    assert tc.attention(args[0], odd, odd, *args[3:]) == _lib.SSL_ERR_UNSUPPORTED
