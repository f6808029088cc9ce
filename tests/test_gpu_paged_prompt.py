"""Attention of several new tokens per sequence over a paged cache (bb_paged_prompt_attention), its form
of one token each, and the 4-bit pool (its append, its reading back, both attentions over it) against their formulas in
64 bits: types, head layouts, lengths from none to long ones, odd sizes and page sizes, strides, windows and
prefixes, capped scores and biases, pages that are not there, values that are not finite in places that a row does
not see, captured calls.

Tolerances count roundings. u = 2^-24 is half a step of f32. A sum of n terms is off by at most n·u of the terms'
absolute sum, and by independent roundings of about sqrt(n)·u of it: 8·sqrt(n)·u is allowed. A stored value of
type t is off by finfo(t).eps / 2 of itself. Weights that are rounded to 16 bits are off by half a step of that type.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

from bebelm_amd import BBError, _lib, kernels
from bebelm_amd.model import BF16, F16, F32, KV4, Context, PagedKv, RopePlan, kv4_bytes

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -25, BF16: 2.0 ** -134}   # half a step of the smallest values
INF, NAN = float("inf"), float("nan")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(seed, shape, dt, spread=1.0):
    return (spread * torch.randn(shape, generator=gen(seed))).to(TYPES[dt])


def half_step(dt):
    return torch.finfo(TYPES[dt]).eps / 2


def done(ctx):
    ctx.synchronize()
    torch.cuda.synchronize()


def on_gpu(*tensors):
    """Copies that are there when a call on another stream begins, to be held until it is done."""
    copies = [t.cuda() for t in tensors]
    torch.cuda.synchronize()
    return copies


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def close(got, want, tol, what):
    got, want = got.double().cpu(), want.double().cpu()
    tol = torch.as_tensor(tol, dtype=torch.float64).expand_as(want)
    off = (got - want).abs()
    bad = ~((off <= tol) | (got.isnan() & want.isnan()))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / tol).nan_to_num(1e9).max()):.3g} times"


# ---- the 4-bit cache in 64 bits -------------------------------------------------------------------
STEPS = torch.tensor([i * 2.0 ** -18 for i in range(32)] +
                     [(16 + i) * 2.0 ** (e - 4) for e in range(-13, 16) for i in range(16)], dtype=torch.float64)


def quantised(x):
    """(step, offset, codes) of blocks x [..., 32]: step NaN where an element is not finite."""
    x = x.double()
    odd = ~torch.isfinite(x).all(-1, keepdim=True)
    x = torch.where(odd, 0.0, x.clamp(-16384.0, 16384.0))
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    at = torch.maximum(torch.maximum(torch.searchsorted(15 * STEPS, (hi - lo).contiguous()),
                                     torch.searchsorted(63 * STEPS, hi.contiguous())),
                       torch.searchsorted(47 * STEPS, (-lo).contiguous()))
    d = STEPS[at]
    by = torch.where(d > 0, d, 1.0)
    z = torch.round(lo / by)
    code = (torch.round(x / by) - z).clamp(0, 15)
    return torch.where(odd, NAN, d), torch.where(odd, 0.0, z), torch.where(odd, 0.0, code)


def held(x):
    """What a 4-bit pool holds for x [..., head_dim], float64."""
    b = x.double().unflatten(-1, (-1, 32))
    d, z, code = quantised(b)
    return (d * (z + code)).flatten(-2)


def packed(x):
    """The bytes of rows x [..., head_dim]: (codes, heads) as a piece of the pool has them."""
    d, z, code = quantised(x.double().unflatten(-1, (-1, 32)))
    code = code.to(torch.uint8).flatten(-2)
    z = z.to(torch.int32)
    head = torch.where(d.isnan(), 0x7fc0, d.nan_to_num(0).half().view(torch.int16).to(torch.int32) | (z & 63) | (z < 0).int() * 0x8000)
    head = head.squeeze(-1).to(torch.int16)
    if head.shape[-1] % 2:
        head = torch.cat((head, torch.zeros_like(head[..., :1])), -1)
    return code[..., 0::2] | code[..., 1::2] << 4, head.contiguous().view(torch.uint8)


class Pool:
    """A pool, the page table of sequences of the given lengths, and what is at their positions (float64)."""

    def __init__(self, ctx, seed, lens, ct, page, kv, hd, order="phd", spare=2, extra=1, spread=1.0):
        g = gen(seed)
        need = [(max(n, 0) + page - 1) // page for n in lens]
        self.n_pages = sum(need) + spare
        ids = torch.randperm(self.n_pages, generator=g).int()
        self.table = torch.full((len(lens), max(need + [1]) + extra), 1 << 30, dtype=torch.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = ids[at:at + n]
            at += n
        self.page, self.lens_list, self.lens, self.ct, self.hd = page, lens, i32(lens), ct, hd
        shape = (self.n_pages, page, kv, hd)
        values = [spread * torch.randn(shape, generator=gen(seed + i)) for i in (1, 2)]
        if ct == KV4:
            self.values = [held(x) for x in values]
            size = kv4_bytes(page, hd)
            self.k, self.v = (torch.zeros(self.n_pages, kv, size, dtype=torch.uint8) for _ in range(2))
            for to, x in zip((self.k, self.v), values):
                codes, heads = packed(x.transpose(1, 2))
                to[..., :page * hd // 2] = codes.flatten(2)
                to[..., page * hd // 2:page * hd // 2 + heads[0, 0].numel()] = heads.flatten(2)
            if order == "hps":   # heads first
                self.k, self.v = (x.transpose(0, 1).contiguous().cuda().transpose(0, 1) for x in (self.k, self.v))
            else:
                self.k, self.v = self.k.cuda(), self.v.cuda()
            self.kv = PagedKv.four_bit(ctx, self.k, self.v, page, hd)
        else:
            dims = {"phd": "pshd", "hnd": "phsd", "hps": "hpsd"}[order]
            there = [dims.index(c) for c in "pshd"]
            self.values = [x.to(TYPES[ct]).double() for x in values]
            self.k, self.v = (x.to(TYPES[ct]).permute(*["pshd".index(c) for c in dims]).contiguous().cuda().permute(*there)
                              for x in values)
            self.kv = PagedKv(ctx, self.k, self.v)

    def where(self, s, n=None):
        j = torch.arange(self.lens_list[s] if n is None else n)
        return self.table[s][j // self.page].long(), j % self.page

    def history(self, s):
        p, r = self.where(s)
        return self.values[0][p, r], self.values[1][p, r]

    def put(self, which, s, j, value):
        """A value at position j of sequence s, all heads (of 4 bits: the whole row)."""
        p, r = int(self.table[s, j // self.page]), j % self.page
        self.values[which][p, r] = value
        pool = (self.k, self.v)[which]
        if self.ct == KV4:
            at = self.page * self.hd // 2 + r * 2 * ((self.hd // 32 + 1) // 2 * 2)
            pool[p, :, at:at + self.hd // 16] = i32([0x7fc0] * (self.hd // 32)).to(torch.int16).view(torch.uint8).cuda()
            self.values[which][p, r] = NAN
        else:
            pool[p, r] = value


# ---- the formulas in 64 bits -----------------------------------------------------------------------
def attention64(q, hist, index, scale, dt, ct, cap=0.0, slopes=None, window=0, prefix=0):
    """(out, lse, tolerance of out without its own rounding, of lse) of q [tokens, heads, hd] at the given indexes."""
    k, v = hist
    n, kv, hd = k.shape
    t, heads = q.shape[:2]
    g = heads // kv
    qk = q.double().reshape(t, kv, g, hd).permute(1, 0, 2, 3)                # [kv, t, g, hd]
    kt, vt = k.permute(1, 2, 0).contiguous()[:, None], v.permute(1, 0, 2).contiguous()[:, None]
    i, j = torch.as_tensor(index)[:, None], torch.arange(n)[None]
    seen = (j <= i) & ((i - j < window) if window else torch.ones(1, dtype=torch.bool)) | (j < prefix)
    seen = seen[None, :, None]                                               # [1, t, 1, n]
    x = (qk @ kt) * scale
    # a score: its sum over hd, the scale's and the logarithm base's products
    d = (8 * math.sqrt(hd) + 4) * U * abs(scale) * (qk.abs() @ kt.abs()) + 4 * U * x.abs()
    if cap:
        x = cap * torch.tanh(x / cap)
        d = d + 12 * U * x.abs()     # (the quotient: exponential, sums, reciprocal and product)
    if slopes is not None:
        far = slopes.double().view(kv, 1, g, 1) * (i - j).abs()[None, :, None]
        x = x - far
        d = d + 4 * U * far + U * x.abs()
    hidden = ~seen.expand_as(x)
    x = x.masked_fill(hidden, -INF)
    d = d.masked_fill(hidden, 0.0)
    lse = torch.logsumexp(x, -1) if n else torch.full((kv, t, g), -INF, dtype=torch.float64)
    p = torch.exp(x - torch.where(lse == -INF, 0.0, lse)[..., None])
    vs = torch.where(torch.isfinite(vt), vt, 0.0)
    out = p @ vs
    d = (d.amax(-1) if n else torch.zeros_like(lse)) + 4 * U
    sums = (8 * math.sqrt(max(n, 1)) + 16) * U
    # weights rounded to 16 bits
    w16 = 0.0
    if ct == BF16:
        w16 = {BF16: 2.0 ** -8, F16: 2.0 ** -16, F32: 0.0}[dt]
    elif ct in (F16, KV4):
        w16 = {BF16: 2.0 ** -11, F16: 2.0 ** -11, F32: 0.0}[dt]
    tol = (2 * d + 2 * sums + w16)[..., None] * (p @ vs.abs())
    if ct in (F16, KV4):
        tol = tol + 2.0 ** -33 * (seen.double() @ vs.abs())   # (what f16's range costs of each)
    # a value that is not finite: NaN for the rows that see it
    bad = (seen.double() @ (~torch.isfinite(vt)).double()) > 0
    out = torch.where(bad, NAN, out)
    back = lambda a: a.permute(1, 0, 2, *range(3, a.dim())).flatten(1, 2)
    return back(out), back(lse), back(tol), back(d + sums + 4 * U * lse.abs())


def run(ctx, pool, q, start=None, kv=None, fill=7.0, workspace=None, table=None, lens=None, **kw):
    out = torch.full(q.shape, fill, dtype=q.dtype, device="cuda")
    lse = torch.full(q.shape[:2], fill, device="cuda")
    kw = {a: b.cuda() if isinstance(b, torch.Tensor) else b for a, b in kw.items()}
    torch.cuda.synchronize()
    kernels.paged_prompt_attention(ctx, kv or pool.kv, (pool.table if table is None else table).cuda(),
                                   (pool.lens if lens is None else lens).cuda(), q.cuda(), out,
                                   seq_start=None if start is None else i32(start).cuda(), lse=lse, workspace=workspace, **kw)
    done(ctx)
    return out.cpu(), lse.cpu()


def check(ctx, pool, q, dt, bring, scale=None, cap=0.0, slopes=None, window=0, prefix=None, single=False, what="",
          padding=0, **kw):
    """The call on a batch whose sequences bring the given numbers of tokens, against the formulas."""
    start = [0] + np.cumsum(bring).tolist()
    out, lse = run(ctx, pool, q, None if single else start, scale=scale, cap=cap, slopes=slopes, window=window,
                   prefix=None if prefix is None else i32(prefix), **kw)
    by = scale if scale is not None else 1 / math.sqrt(pool.hd)
    for s, n in enumerate(bring):
        rows = slice(start[s], start[s + 1])
        if n == 0:
            continue
        length = pool.lens_list[s]
        index = torch.arange(length - n, length)
        want, wl, tol, tl = attention64(q[rows], pool.history(s), index, by, dt, pool.ct, cap, slopes, window,
                                        min(prefix[s], length) if prefix is not None else 0)
        close(out[rows], want, tol * (1 + half_step(dt)) + half_step(dt) * want.abs() + TINY[dt], f"{what} out of {s}")
        none = torch.isneginf(wl)
        assert torch.equal(torch.isneginf(lse[rows]), none), f"{what}: rows of {s} that see nothing"
        close(lse[rows][~none], wl[~none], (tl + U * wl.abs())[~none], f"{what} lse of {s}")
    if padding:
        assert bool((out[start[-1]:] == 7.0).all()) and bool((lse[start[-1]:] == 7.0).all()), "padding was written"
    return out, lse


SHAPES = [dict(), dict(cap=5.0), dict(slopes=True), dict(cap=3.0, slopes=True, window=9), dict(prefix=True),
          dict(window=20, prefix=True)]


def slopes_of(heads):
    return torch.exp2(-8.0 * torch.arange(1, heads + 1) / heads)


# ---- prompts ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("ct", [F32, F16, BF16, KV4])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_types(gpu_ctx, dt, ct, hd):
    bring, before = [17, 0, 1, 40, 90], [0, 9, 70, 33, 0]
    pool = Pool(gpu_ctx, 1, [a + b for a, b in zip(before, bring)], ct, 16, 2, hd)
    q = randn(5, (sum(bring) + 3, 8, hd), dt, 1.5)
    for i, kw in enumerate(SHAPES):
        print("types", dt, ct, hd, kw, flush=True)
        kw = dict(kw)
        if kw.get("slopes"):
            kw["slopes"] = slopes_of(8)
        if kw.get("prefix"):
            kw["prefix"] = [5, 3, 200, 50, 0]
        check(gpu_ctx, pool, q, dt, bring, padding=3, what=str(kw), **kw)


HEADS = [(1, 1, 8), (3, 3, 24), (5, 1, 96), (24, 1, 64), (12, 4, 80), (16, 16, 40), (33, 1, 128), (7, 7, 200), (2, 1, 256),
         (40, 8, 32), (130, 1, 64)]


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("dt,ct", [(F32, F32), (BF16, BF16), (F32, BF16), (F16, F16), (BF16, KV4), (F32, KV4)])
def test_heads(gpu_ctx, heads, dt, ct):
    nh, kv, hd = heads
    if ct == KV4 and hd % 32:
        hd = (hd + 31) // 32 * 32
    print("heads", heads, dt, ct, flush=True)
    for bring, before in (([1, 2, 5], [3, 0, 130]), ([37, 64], [0, 11]), ([9, 9, 9], [0, 300, 1])):
        pool = Pool(gpu_ctx, 3, [a + b for a, b in zip(before, bring)], ct, 16, kv, hd)
        q = randn(7, (sum(bring), nh, hd), dt)
        check(gpu_ctx, pool, q, dt, bring, what=str((bring, before)))


@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 33, 64, 100, 256])
@pytest.mark.parametrize("order", ["phd", "hnd", "hps"])
@pytest.mark.parametrize("ct", [BF16, F32, KV4])
def test_pages(gpu_ctx, page, order, ct):
    print("pages", page, order, ct, flush=True)
    bring, before = [65, 3, 130], [63, 200, 0]
    pool = Pool(gpu_ctx, 4, [a + b for a, b in zip(before, bring)], ct, page, 2, 64, order)
    q = randn(8, (sum(bring), 4, 64), BF16)
    check(gpu_ctx, pool, q, BF16, bring)
    check(gpu_ctx, pool, q, BF16, bring, window=40, prefix=[70, 0, 3])
    check(gpu_ctx, pool, q[:3], BF16, [1, 1, 1], single=True, cap=4.0)


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 63, 64, 65, 128, 500, 10_000, 1 << 40])
@pytest.mark.parametrize("ct", [F16, KV4])
def test_windows_and_prefixes(gpu_ctx, window, ct):
    print("window", window, ct, flush=True)
    bring, before = [150, 1, 7, 33, 2], [0, 600, 64, 128, 1500]
    lens = [a + b for a, b in zip(before, bring)]
    pool = Pool(gpu_ctx, 6, lens, ct, 16, 2, 128)
    q = randn(9, (sum(bring), 4, 128), F16)
    for prefix in (None, [0, 0, 0, 0, 0], [1, 64, 65, 10_000, 63], [150, 601, 1, 161, 1400]):
        check(gpu_ctx, pool, q, F16, bring, window=window, prefix=prefix, what=str(prefix))


@pytest.mark.parametrize("bring", [1, 3, 8, 9, 16, 17, 31, 32, 33])
@pytest.mark.parametrize("ct,hd", [(BF16, 128), (F32, 64), (F32, 256), (F16, 256), (KV4, 64)])
def test_few_tokens_over_a_long_cache(gpu_ctx, bring, ct, hd):
    """Positions in parts for several blocks, joined; lengths that leave parts without any."""
    print("few", bring, ct, hd, flush=True)
    lens = [bring + 3000, bring, bring + 257, bring + 1111]
    pool = Pool(gpu_ctx, 10, lens, ct, 16, 1, hd)
    dt = F32 if ct == F32 else BF16
    q = randn(11, (4 * bring, 4, hd), dt, 1.5)
    check(gpu_ctx, pool, q, dt, [bring] * 4)
    check(gpu_ctx, pool, q, dt, [bring] * 4, window=700, prefix=[100, 1, 0, 64], slopes=slopes_of(4))


def test_a_long_prompt(gpu_ctx):
    for ct, dt, hd in ((BF16, BF16, 128), (KV4, BF16, 64), (F32, F32, 64)):
        print("long", ct, dt, hd, flush=True)
        pool = Pool(gpu_ctx, 12, [1531], ct, 16, 1, hd)
        q = randn(13, (1400, 2, hd), dt, 1.5)
        check(gpu_ctx, pool, q, dt, [1400], prefix=[600])


def test_equal_calls_give_equal_bits(gpu_ctx):
    pool = Pool(gpu_ctx, 14, [900, 40, 2000], BF16, 16, 2, 64)
    q = randn(15, (50, 8, 64), F32)
    first = run(gpu_ctx, pool, q, [0, 20, 30, 50], cap=9.0)
    for _ in range(3):
        again = run(gpu_ctx, pool, q, [0, 20, 30, 50], cap=9.0)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_scale_and_extremes(gpu_ctx):
    """Negative and large scales, queries and keys of very different sizes, scores that differ by thousands, heads whose
    scores all are -inf."""
    pool = Pool(gpu_ctx, 16, [70], F16, 16, 1, 64, spread=4.0)
    q = randn(17, (70, 3, 64), F32, 3.0)
    q[:, 1] *= 1e-30
    q[:, 2] *= 1e4
    check(gpu_ctx, pool, q, F32, [70], scale=-0.25)
    check(gpu_ctx, pool, q, F32, [70], scale=3.0)
    check(gpu_ctx, pool, q, F32, [70], scale=1e-38)
    check(gpu_ctx, pool, q, F32, [70], scale=2.0, cap=1e-3)
    pool = Pool(gpu_ctx, 18, [20], F32, 16, 1, 64)
    pool.k.fill_(-INF)
    out, lse = run(gpu_ctx, pool, torch.ones(20, 2, 64), [0, 20])
    assert bool((out == 0).all()) and bool(torch.isneginf(lse).all())


# ---- what a row does not see ------------------------------------------------------------------------
@pytest.mark.parametrize("ct,dt", [(F32, F32), (F16, F16), (BF16, BF16), (BF16, F32), (KV4, F32), (F16, F32)])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_values_that_are_not_finite(gpu_ctx, ct, dt, hd):
    """In positions that some rows of a tile see and others do not: those that do get NaN (a key: in the whole row; a
    value: in its element), the others are as if it were not there."""
    print("not finite", ct, dt, hd, flush=True)
    lens, bring = [150, 90], [140, 5]
    for which, what in ((1, NAN), (1, INF), (1, -INF), (0, NAN)):
        pool = Pool(gpu_ctx, 20, lens, ct, 16, 1, hd)
        q = randn(21, (145, 4, hd), dt)
        for j in (60, 75, 140):
            pool.put(which, 0, j, what)
        pool.put(which, 1, 88, what)
        kw = dict(window=30, prefix=[3, 0])
        start = [0, 140, 145]
        out, lse = run(gpu_ctx, pool, q, start, **{**kw, "prefix": i32(kw["prefix"])})
        for s in range(2):
            rows = slice(start[s], start[s + 1])
            index = torch.arange(lens[s] - bring[s], lens[s])
            k, v = pool.history(s)
            if which == 1:
                want, wl, tol, tl = attention64(q[rows], (k, v), index, 1 / math.sqrt(hd), dt, ct, window=30,
                                                prefix=kw["prefix"][s])
                # (the value's element only: every element of these rows is bad)
                close(out[rows], want, tol * (1 + half_step(dt)) + half_step(dt) * want.abs().nan_to_num() + TINY[dt], f"{what}")
                close(lse[rows], wl, tl + U * wl.abs(), "lse")
            else:
                odd = ~torch.isfinite(k).all(-1).all(-1)
                j = torch.arange(lens[s])[None]
                seen = (j <= index[:, None]) & (index[:, None] - j < 30) | (j < kw["prefix"][s])
                bad = (seen & odd[None]).any(-1)
                want, _, tol, _ = attention64(q[rows], (torch.where(odd[:, None, None], 0.0, k), v), index,
                                              1 / math.sqrt(hd), dt, ct, window=30, prefix=kw["prefix"][s])
                assert bool(out[rows][bad].isnan().all()) and not bool(out[rows][~bad].isnan().any())
                close(out[rows][~bad], want[~bad],
                      (tol * (1 + half_step(dt)) + half_step(dt) * want.abs() + TINY[dt])[~bad], "rows without")


def test_one_element_that_is_not_finite(gpu_ctx):
    for ct in (F32, F16, BF16):
        pool = Pool(gpu_ctx, 22, [100], ct, 16, 2, 128)
        q = randn(23, (100, 4, 128), F32)
        p, r = int(pool.table[0, 70 // 16]), 70 % 16
        for x in (pool.v, pool.values[1]):
            x[p, r, 1, 77] = INF
        out, _ = check(gpu_ctx, pool, q, F32, [100])
        nan = out.isnan()
        assert int(nan.sum()) == 30 * 2 and bool(nan[70:, 2:, 77].all())


@pytest.mark.parametrize("ct", [F32, BF16, KV4])
def test_what_lies_behind_makes_no_difference(gpu_ctx, ct):
    """Positions past a length, pages past a sequence's, pages between a prefix and a window: all of it NaN or not there."""
    lens, bring = [100, 33, 64], [20, 33, 1]
    pool = Pool(gpu_ctx, 24, lens, ct, 16, 2, 64)
    q = randn(25, (54, 4, 64), F32)
    start = [0, 20, 53, 54]
    kw = dict(window=10, prefix=i32([4, 0, 20]), cap=6.0)
    first = run(gpu_ctx, pool, q, start, **kw)
    kept = [set(), set(), set()]
    for s, n in enumerate(lens):
        for j in range(n):
            lo = n - bring[s] - 10 + 1
            if j >= lo or j < int(kw["prefix"][s]):
                kept[s].add((int(pool.table[s, j // 16]), j % 16))
    everything = {(p, r) for p in range(pool.n_pages) for r in range(16)} - kept[0] - kept[1] - kept[2]
    for p, r in everything:
        for pool_ in (pool.k, pool.v):
            if ct == KV4:
                pool_[p, :, 16 * 32 + 4 * r:16 * 32 + 4 * r + 4] = i32([0x7fc07fc0]).view(torch.uint8).cuda()
                pool_[p, :, 32 * r:32 * r + 32] = 255
            else:
                pool_[p, r] = NAN
    table = pool.table.clone()
    for s, n in enumerate(lens):
        for e in range(table.shape[1]):
            if not any(int(table[s, e]) == p for p, _ in kept[s]):
                table[s, e] = [-1, 1 << 30, pool.n_pages, -(1 << 31)][(s + e) % 4]
    again = run(gpu_ctx, pool, q, start, table=table, **kw)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_empty_and_short_sequences(gpu_ctx):
    """Sequences without positions or tokens, tokens past what a sequence has, lengths past the table, missing pages."""
    for ct in (F32, KV4):
        pool = Pool(gpu_ctx, 26, [40, 0, 5, 64], ct, 16, 1, 64, extra=0)
        q = randn(27, (30, 2, 64), F32)
        start = [0, 10, 13, 21, 30]
        lens = i32([40, 0, 5, 1 << 30])     # the third is shorter than its 8 tokens
        table = pool.table.clone()
        table[0, 1] = -1                    # positions 16..31 are not there
        out, lse = run(gpu_ctx, pool, q, start, lens=lens, table=table)
        assert bool((out[10:13] == 0).all()) and bool(torch.isneginf(lse[10:13]).all())
        assert bool((out[13:16] == 0).all()) and bool(torch.isneginf(lse[13:16]).all())
        k, v = pool.history(0)
        keep = torch.tensor([j for j in range(40) if not 16 <= j < 32])
        for t in range(10):
            n = int((keep <= 30 + t).sum())
            want, wl, tol, tl = attention64(q[t:t + 1], (k[keep[:n]], v[keep[:n]]), [n - 1], 1 / 8, F32, ct)
            close(out[t:t + 1], want, tol + half_step(F32) * want.abs(), f"token {t}")
        for s, (a, b) in ((2, (16, 21)), (3, (21, 30))):   # (a length past the table counts as all of it)
            n = pool.lens_list[s]
            want, _, tol, _ = attention64(q[a:b], pool.history(s), torch.arange(n - (b - a), n), 1 / 8, F32, ct)
            close(out[a:b], want, tol + half_step(F32) * want.abs(), f"sequence {s}")


def test_starts_that_do_not_ascend(gpu_ctx):
    """On the device they are what they are: nothing outside of the arrays is touched."""
    pool = Pool(gpu_ctx, 28, [40, 50, 60], BF16, 16, 2, 64)
    q = randn(29, (20, 4, 64), BF16)
    for start in ([0, 30, 10, 20], [5, -7, 1 << 30, 3], [20, 10, 5, 0], [-(1 << 31), (1 << 31) - 1, 0, 20]):
        out, lse = run(gpu_ctx, pool, q, start)
        assert out.shape == q.shape
    check(gpu_ctx, pool, q, BF16, [5, 5, 10])


@pytest.mark.parametrize("ct", [F32, F16, BF16, KV4])
@pytest.mark.parametrize("page", [5, 16])
def test_single_tokens_behind_values_that_are_not_finite(gpu_ctx, page, ct):
    """Keys and values before the window (in the window's first rows of a tile too) make no difference."""
    lens = [1, 20, 21, 33, 50, 61, 200]
    for hd, dt in ((64, F16), (128, BF16), (256, F32)):
        pool = Pool(gpu_ctx, 95, lens, ct, page, 1, hd)
        q = randn(96, (len(lens), 2, hd), dt)
        for window in (1, 7, 20):
            for s, n in enumerate(lens):
                for j in range(max(0, n - window)):
                    pool.put(0, s, j, NAN)
                    pool.put(1, s, j, INF)
            out, lse = check(gpu_ctx, pool, q, dt, [1] * len(lens), window=window, single=True)
            assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(lse).all())
            pool = Pool(gpu_ctx, 95, lens, ct, page, 1, hd)


@pytest.mark.parametrize("ct", [F32, BF16, KV4])
def test_many_sequences(gpu_ctx, ct):
    """More sequences than a wave looks through at once, most of them with a token or two or none, a few with prompts."""
    r = np.random.RandomState(30)
    bring = [int(x) for x in r.choice([0, 1, 2, 3, 70], 200, p=[0.4, 0.3, 0.15, 0.13, 0.02])]
    bring[63:66] = [0, 0, 5]
    bring[-1] = 1
    lens = [n + int(r.choice([0, 1, 17, 300])) for n in bring]
    pool = Pool(gpu_ctx, 31, lens, ct, 16, 2, 64)
    q = randn(32, (sum(bring) + 3, 4, 64), F16)
    check(gpu_ctx, pool, q, F16, bring, window=100, prefix=[3] * 200, padding=3)


@pytest.mark.parametrize("ct", [F32, F16, BF16, KV4])
def test_queries_that_are_not_finite(gpu_ctx, ct):
    """They spoil their own rows, and no others of the same tile."""
    pool = Pool(gpu_ctx, 33, [200], ct, 16, 1, 64)
    for dt in (F32, BF16):
        q = randn(34, (90, 2, 64), dt)
        want, wl = run(gpu_ctx, pool, q, [0, 90])
        odd = [(0, 0), (3, 1), (40, 0), (89, 1)]
        for n, (t, h) in enumerate(odd):
            q[t, h, 7 * n] = (NAN, INF, -INF, NAN)[n]
        out, lse = run(gpu_ctx, pool, q, [0, 90])
        keep = torch.ones(90, 2, dtype=torch.bool)
        for t, h in odd:
            keep[t, h] = False
            assert bool(out[t, h].isnan().all()) and not bool(torch.isfinite(lse[t, h]))
        assert torch.equal(out[keep], want[keep]) and torch.equal(lse[keep], wl[keep])


def test_two_streams_at_once(gpu_ctx):
    """Calls of two contexts over one pool, each with its own stream, the same workspaces call after call."""
    pool = Pool(gpu_ctx, 35, [3000, 2500, 90], BF16, 16, 2, 64)
    plans = [([0, 5, 9, 29], dict(cap=4.0)), ([0, 1, 2, 92], dict(window=200))]
    queries = [randn(36 + i, (start[-1], 8, 64), BF16) for i, (start, _) in enumerate(plans)]
    want = [run(gpu_ctx, pool, x, start, **kw) for x, (start, kw) in zip(queries, plans)]
    streams = [torch.cuda.Stream() for _ in plans]
    ctxs, args = [], []
    table, lens = on_gpu(pool.table, pool.lens)
    for x, (start, kw), stream in zip(queries, plans, streams):
        ctx = Context(0)
        ctx.set_stream(stream.cuda_stream)
        ctxs.append(ctx)
        size = max(pool.kv.prompt_workspace(8, 3, start[-1]), 16)
        args.append((x.cuda(), torch.zeros(x.shape, dtype=x.dtype, device="cuda"), i32(start).cuda(),
                     torch.zeros(x.shape[:2], device="cuda"), torch.empty(size, dtype=torch.uint8, device="cuda"), kw))
    torch.cuda.synchronize()
    for _ in range(20):
        for ctx, (x, out, start, lse, ws, kw) in zip(ctxs, args):
            kernels.paged_prompt_attention(ctx, pool.kv, table, lens, x, out, seq_start=start, lse=lse, workspace=ws, **kw)
    torch.cuda.synchronize()
    for (x, out, start, lse, ws, kw), (a, b) in zip(args, want):
        assert torch.equal(out.cpu(), a) and torch.equal(lse.cpu(), b)
    for ctx in ctxs:
        ctx.close()


# ---- one token each ---------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("ct", [F32, F16, BF16, KV4])
@pytest.mark.parametrize("hd", [32, 64, 96, 128, 256])
def test_single_tokens(gpu_ctx, dt, ct, hd):
    lens = [1, 17, 0, 300, 64, 1000, 33]
    pool = Pool(gpu_ctx, 30, lens, ct, 16, 2, hd)
    q = randn(31, (7, 8, hd), dt, 1.5)
    bring = [min(n, 1) for n in lens]
    for kw in (dict(), dict(cap=4.0), dict(slopes=slopes_of(8)), dict(cap=4.0, slopes=slopes_of(8), window=50),
               dict(window=20, prefix=[3] * 7), dict(prefix=[9] * 7)):
        print("single", dt, ct, hd, list(kw), flush=True)
        want = {}
        out, lse = run(gpu_ctx, pool, q, None, **{a: i32(b) if a == "prefix" else b for a, b in kw.items()})
        for s, n in enumerate(lens):
            if n == 0:
                assert bool((out[s] == 0).all()) and bool(torch.isneginf(lse[s]).all())
                continue
            p = {**kw, "prefix": kw["prefix"][s]} if "prefix" in kw else kw
            want, wl, tol, tl = attention64(q[s:s + 1], pool.history(s), [n - 1], 1 / math.sqrt(hd), dt, ct, **p)
            close(out[s:s + 1], want, tol * (1 + half_step(dt)) + half_step(dt) * want.abs() + TINY[dt], f"out {s}")
            close(lse[s:s + 1], wl, tl + U * wl.abs(), f"lse {s}")


@pytest.mark.parametrize("page", [1, 5, 8, 13, 16, 24, 40, 256])
@pytest.mark.parametrize("hd", [32, 64, 128, 224, 256])
def test_single_tokens_on_4_bits(gpu_ctx, page, hd):
    """bb_paged_attention over a 4-bit pool, and the same with scores of every kind."""
    print("4 bits", page, hd, flush=True)
    lens = [1, 40, 0, 700, page, 3 * page + 1]
    for order, window in (("phd", 0), ("hps", 37)):
        pool = Pool(gpu_ctx, 32, lens, KV4, page, 2, hd, order)
        q = randn(33, (6, 6, hd), F32, 1.5)
        out, lse = torch.full(q.shape, 7.0, device="cuda"), torch.full((6, 6), 7.0, device="cuda")
        torch.cuda.synchronize()
        kernels.paged_attention(gpu_ctx, pool.kv, pool.table.cuda(), pool.lens.cuda(), q.cuda(), out, window=window, lse=lse)
        done(gpu_ctx)
        capped, capped_lse = run(gpu_ctx, pool, q, None, window=window, cap=2.0, slopes=slopes_of(6))
        for s, n in enumerate(lens):
            if n == 0:
                assert bool((out[s] == 0).all()) and bool(torch.isneginf(lse[s]).all())
                continue
            for o, z, kw in ((out, lse, {}), (capped, capped_lse, dict(cap=2.0, slopes=slopes_of(6)))):
                want, wl, tol, tl = attention64(q[s:s + 1], pool.history(s), [n - 1], 1 / math.sqrt(hd), F32, KV4,
                                                window=window, **kw)
                close(o[s:s + 1], want, tol + half_step(F32) * want.abs(), f"out {s}")
                close(z[s:s + 1], wl, tl + U * wl.abs(), f"lse {s}")


def test_distance_over_other_pages(gpu_ctx):
    """The bias counts positions, not the places of pages whose slots are in part empty."""
    for page in (12, 24, 30, 40):
        for ct in (F32, BF16, KV4):
            pool = Pool(gpu_ctx, 34, [1, 500, 77], ct, page, 1, 64)
            q = randn(35, (3, 4, 64), F32)
            check(gpu_ctx, pool, q, F32, [1, 1, 1], single=True, slopes=torch.tensor([0.5, 0.1, 0.01, 0.0]))
            check(gpu_ctx, pool, q, F32, [1, 1, 1], slopes=torch.tensor([0.5, 0.1, 0.01, 0.0]))


# ---- the 4-bit pool ---------------------------------------------------------------------------------
def blocks(seed, dt):
    """Blocks of every kind [n, 32]: normal ones, shifted ones, one sign, zeros, equal values, tiny and huge ones, ones whose
    elements lie on the borders between codes."""
    g = gen(seed)
    x = [torch.randn(200, 32, generator=g) * torch.exp2(torch.randint(-22, 14, (200, 1), generator=g).float()),
         torch.randn(60, 32, generator=g) + 8 * torch.randn(60, 1, generator=g),
         torch.rand(40, 32, generator=g) + 3, -torch.rand(40, 32, generator=g) - 1, torch.zeros(3, 32),
         torch.randn(20, 1, generator=g).expand(20, 32), torch.randn(20, 32, generator=g) * 1e5,
         torch.randn(10, 32, generator=g) * 1e-7, torch.zeros(1, 32) + 6e-8, torch.randn(5, 32, generator=g) * 2.0 ** -130]
    d = torch.exp2(torch.randint(-8, 4, (200, 1), generator=g).float()) * (16 + torch.randint(0, 16, (200, 1), generator=g)) / 16
    n = torch.randint(-8, 8, (200, 32), generator=g) + 0.5 * torch.randint(0, 2, (200, 32), generator=g)
    n[:, 0], n[:, 1] = -7.5, 7.5
    edge = n * d
    x += [edge, torch.nextafter(edge, torch.tensor(INF)), torch.nextafter(edge, torch.tensor(-INF))]
    return torch.cat(x).to(TYPES[dt])


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("hd", [32, 64, 96, 128, 160, 256])
def test_append_to_4_bits(gpu_ctx, dt, hd):
    """Every byte of the pool: the tokens' as the definition in 64 bits says, all others as they were."""
    print("append 4", dt, hd, flush=True)
    b = blocks(hd, dt)
    odd = b[:12].clone()
    odd[0, 3], odd[1, 31], odd[2, 0], odd[3] = NAN, INF, -INF, NAN
    b = torch.cat((b, odd))
    kv, page = 2, 16
    t = len(b) * 32 // (kv * hd)
    rows = b[:t * kv * hd // 32].reshape(t, kv, hd)
    k, v = rows, rows.flip(0).contiguous()
    bring = [t // 3, 0, t - t // 3]
    before = [5, 3, 30]
    pool = Pool(gpu_ctx, 40, [a + c for a, c in zip(before, bring)], KV4, page, kv, hd)
    want = [x.cpu().clone() for x in (pool.k, pool.v)]
    start = [0] + np.cumsum(bring).tolist()
    for w, x in zip(want, (k, v)):
        codes, heads = packed(x)
        for s, n in enumerate(bring):
            p, r = pool.where(s)
            for i in range(n):
                pg, at, token = int(p[before[s] + i]), int(r[before[s] + i]), start[s] + i
                w[pg, :, at * hd // 2:(at + 1) * hd // 2] = codes[token]
                h0 = page * hd // 2 + at * heads.shape[-1]
                w[pg, :, h0:h0 + hd // 16] = heads[token][:, :hd // 16]
    fused = torch.cat((k, v), 1).cuda()      # side by side for each token
    torch.cuda.synchronize()
    kernels.paged_append(gpu_ctx, pool.kv, pool.table.cuda(), pool.lens.cuda(), fused[:, :kv], fused[:, kv:],
                         seq_start=i32(start).cuda())
    done(gpu_ctx)
    for got, w, what in zip((pool.k, pool.v), want, ("keys", "values")):
        assert torch.equal(got.cpu(), w), what
    # and back, in every type
    for back in (F32, F16, BF16):
        kb, vb = (torch.full((t, kv, hd), 7.0, dtype=TYPES[back], device="cuda") for _ in range(2))
        torch.cuda.synchronize()
        kernels.paged_read(gpu_ctx, pool.kv, pool.table.cuda(), pool.lens.cuda(), kb, vb, seq_start=i32(start).cuda())
        done(gpu_ctx)
        for got, x in ((kb, k), (vb, v)):
            exact = held(x)
            assert torch.equal(got.cpu().isnan(), exact.isnan())
            assert torch.equal(got.cpu().nan_to_num(0), exact.to(TYPES[back]).nan_to_num(0))
            far = ~exact.isnan()
            d = quantised(x.unflatten(-1, (-1, 32)))[0].expand(-1, -1, -1, 32).flatten(-2)
            off = (exact - x.double().clamp(-16384, 16384)).abs()
            assert bool((off[far] <= d[far] / 2).all())


@pytest.mark.parametrize("rot,interleaved", [(64, False), (64, True), (32, False), (36, True), (6, False)])
def test_append_to_4_bits_with_norm_and_rotation(gpu_ctx, rot, interleaved):
    """What the call stores is what it stores in f32, quantised: the same bytes as in two calls."""
    hd, kv, heads = 64, 2, 4
    bring, before = [9, 1, 30], [0, 16, 7]
    lens = [a + b for a, b in zip(before, bring)]
    start, t = i32([0] + np.cumsum(bring).tolist()), sum(bring)
    q, k, v = (randn(50 + i, (t, n, hd), BF16) for i, n in enumerate((heads, kv, kv)))
    gain = 1 + 0.1 * torch.randn(hd, generator=gen(55))
    plan = RopePlan(gpu_ctx, rot, 1e4, interleaved)
    four, wide = Pool(gpu_ctx, 51, lens, KV4, 16, kv, hd), Pool(gpu_ctx, 51, lens, F32, 16, kv, hd)
    outs = []
    for pool in (four, wide):
        out = torch.zeros(q.shape, dtype=q.dtype, device="cuda")
        torch.cuda.synchronize()
        kernels.paged_append(gpu_ctx, pool.kv, pool.table.cuda(), pool.lens.cuda(), k.cuda(), v.cuda(), rope=plan,
                             seq_start=start.cuda(), q=q.cuda(), q_out=out, q_norm=gain.cuda(), k_norm=gain.cuda())
        done(gpu_ctx)
        outs.append(out.cpu())
    assert torch.equal(*outs)
    rows, back = ([torch.empty(t, kv, hd, device="cuda") for _ in range(2)] for _ in range(2))
    for pool, to in ((wide, rows), (four, back)):
        table, ln, st = on_gpu(pool.table, pool.lens, start)
        kernels.paged_read(gpu_ctx, pool.kv, table, ln, *to, seq_start=st)
        done(gpu_ctx)
    for x, got in zip(rows, back):
        assert torch.equal(got.cpu().double(), held(x.cpu()))


def test_append_to_4_bits_one_token_each(gpu_ctx):
    lens = [1, 0, 17, 40, 16]
    pool = Pool(gpu_ctx, 56, lens, KV4, 16, 3, 96)
    k, v = randn(57, (5, 3, 96), F16), randn(58, (5, 3, 96), F16)
    kb, vb = (torch.full((5, 3, 96), 7.0, device="cuda") for _ in range(2))
    before = pool.k.cpu().clone()
    table, ln, kd, vd = on_gpu(pool.table, pool.lens, k, v)
    kernels.paged_append(gpu_ctx, pool.kv, table, ln, kd, vd)
    kernels.paged_read(gpu_ctx, pool.kv, table, ln, kb, vb)
    done(gpu_ctx)
    for s, n in enumerate(lens):
        for got, x in ((kb, k), (vb, v)):
            assert torch.equal(got[s].cpu().double(), held(x[s]) if n else torch.zeros(3, 96, dtype=torch.float64))
    changed = (pool.k.cpu() != before).any(-1).any(-1)
    assert set(changed.nonzero().flatten().tolist()) <= {int(pool.table[s, (n - 1) // 16]) for s, n in enumerate(lens) if n}


@pytest.mark.parametrize("ct", [F32, F16, BF16, KV4])
@pytest.mark.parametrize("back", [F32, F16, BF16])
def test_read(gpu_ctx, ct, back):
    """All that the sequences hold, padding left as it is, missing pages as zeros, keys or values alone, strided rows."""
    lens = [33, 0, 100, 16]
    pool = Pool(gpu_ctx, 60, lens, ct, 24, 2, 64, "hps")
    table = pool.table.clone()
    table[2, 1] = -5
    start, t = i32([0] + np.cumsum(lens).tolist()), sum(lens)
    both = torch.full((t + 4, 5, 64), 7.0, dtype=TYPES[back], device="cuda")
    for only in ("kv", "k", "v"):
        both.fill_(7.0)
        torch.cuda.synchronize()
        kernels.paged_read(gpu_ctx, pool.kv, table.cuda(), pool.lens.cuda(), both[:, :2] if "k" in only else None,
                           both[:, 3:] if "v" in only else None, seq_start=start.cuda())
        done(gpu_ctx)
        got = both.cpu()
        assert bool((got[t:] == 7.0).all()) and bool((got[:, 2] == 7.0).all())
        for s, n in enumerate(lens):
            rows = slice(int(start[s]), int(start[s + 1]))
            for name, x, at in (("k", pool.history(s)[0], slice(0, 2)), ("v", pool.history(s)[1], slice(3, 5))):
                if name not in only:
                    assert bool((got[rows, at] == 7.0).all())
                    continue
                want = x.clone()
                if s == 2:
                    want[24:48] = 0
                assert torch.equal(got[rows, at], want.to(TYPES[back])), (only, s, name)


def test_library_pool_of_4_bits(gpu_ctx):
    """A pool of the library's: zeros at first, then what is stored."""
    kv = PagedKv.create(gpu_ctx, KV4, 6, 16, 2, 64)
    table, lens = i32([[3, 1], [0, 5]]).cuda(), i32([20, 32]).cuda()
    start = i32([0, 20, 52]).cuda()
    back = torch.full((52, 2, 64), 7.0, device="cuda")
    torch.cuda.synchronize()
    kernels.paged_read(gpu_ctx, kv, table, lens, back, seq_start=start)
    done(gpu_ctx)
    assert bool((back == 0).all())
    k = randn(61, (52, 2, 64), F32)
    kd, vd = on_gpu(k, k)
    kernels.paged_append(gpu_ctx, kv, table, lens, kd, vd, seq_start=start)
    kernels.paged_read(gpu_ctx, kv, table, lens, None, back, seq_start=start)
    done(gpu_ctx)
    assert torch.equal(back.cpu().double(), held(k))
    kv.close()


# ---- together, as a server runs them -------------------------------------------------------------------
@pytest.mark.parametrize("ct,dt", [(BF16, BF16), (KV4, F32), (F32, F32), (KV4, BF16)])
def test_conversations(gpu_ctx, ct, dt):
    """Prompts in chunks, then drafts, then single tokens, each appended and attended to: what the whole conversation's
    formulas say of the values that the cache holds."""
    print("conversations", ct, dt, flush=True)
    nh, kv, hd, page = 8, 2, 64, 16
    chunks = [[40, 7, 0], [25, 0, 64], [3, 3, 3], [1, 1, 1], [1, 1, 1]]
    total = [sum(c[s] for c in chunks) for s in range(3)]
    pool = Pool(gpu_ctx, 70, total, ct, page, kv, hd)
    plan = RopePlan(gpu_ctx, 64, 1e4)
    slopes = slopes_of(nh)
    lens = [0, 0, 0]
    for c, chunk in enumerate(chunks):
        t = sum(chunk)
        single = chunk == [1, 1, 1]
        lens = [a + b for a, b in zip(lens, chunk)]
        start = None if single else i32([0] + np.cumsum(chunk).tolist()).cuda()
        q, k, v = (randn(71 + 10 * c + i, (t, n, hd), dt) for i, n in enumerate((nh, kv, kv)))
        qr, out = torch.zeros(t, nh, hd, dtype=TYPES[dt], device="cuda"), torch.zeros(t, nh, hd, dtype=TYPES[dt], device="cuda")
        every = i32([0] + np.cumsum(lens).tolist())
        kb, vb = (torch.zeros(sum(lens), kv, hd, device="cuda") for _ in range(2))
        ln, table, kd, vd, qd, sd, ev = on_gpu(i32(lens), pool.table, k, v, q, slopes, every)
        kernels.paged_append(gpu_ctx, pool.kv, table, ln, kd, vd, rope=plan, seq_start=start, q=qd, q_out=qr)
        kernels.paged_prompt_attention(gpu_ctx, pool.kv, table, ln, qr, out, seq_start=start, cap=20.0, slopes=sd)
        kernels.paged_read(gpu_ctx, pool.kv, table, ln, kb, vb, seq_start=ev)
        done(gpu_ctx)
        at, row = 0, 0
        for s in range(3):
            hist = tuple(x[at:at + lens[s]].cpu().double() for x in (kb, vb))
            n = chunk[s]
            if n:
                want, _, tol, _ = attention64(qr[row:row + n].cpu(), hist, torch.arange(lens[s] - n, lens[s]), 1 / 8, dt, ct,
                                              cap=20.0, slopes=slopes)
                close(out[row:row + n], want, tol * (1 + half_step(dt)) + half_step(dt) * want.abs() + TINY[dt],
                      f"chunk {c} of {s}")
            at += lens[s]
            row += n
    plan.close()


def test_captured_calls(gpu_ctx):
    """A graph of append, attention and reading follows lengths, starts and pages at each replay; two graphs with workspaces of
    their own; eager work between the replays."""
    nh, kv, hd, page, n, t = 4, 1, 64, 16, 3, 24
    stream = torch.cuda.Stream()
    ctx = Context(0)
    ctx.set_stream(stream.cuda_stream)
    lens_max = 2000
    for ct in (BF16, KV4):
        pool = Pool(ctx, 80, [lens_max] * n, ct, page, kv, hd)
        table = pool.table.cuda()
        static = {"lens": i32([30, 40, 50]).cuda(), "start": i32([0, 8, 16, 24]).cuda(), "q": torch.zeros(t, nh, hd, device="cuda"),
                  "k": torch.zeros(t, kv, hd, device="cuda"), "v": torch.zeros(t, kv, hd, device="cuda")}
        outs = [torch.zeros(t, nh, hd, device="cuda") for _ in range(2)]
        lses = [torch.zeros(t, nh, device="cuda") for _ in range(2)]
        kb = torch.zeros(t, kv, hd, device="cuda")
        size = max(pool.kv.prompt_workspace(nh, n, t), 16)
        wss = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(2)]

        def step(i):
            kernels.paged_append(ctx, pool.kv, table, static["lens"], static["k"], static["v"], seq_start=static["start"])
            kernels.paged_prompt_attention(ctx, pool.kv, table, static["lens"], static["q"], outs[i], seq_start=static["start"],
                                           cap=10.0, lse=lses[i], workspace=wss[i])
            kernels.paged_read(ctx, pool.kv, table, static["lens"], kb, seq_start=static["start"])

        graphs = []
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(stream):
                step(i)
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                step(i)
            graphs.append(g)
        for turn, (lens, start) in enumerate((([30, 40, 50], [0, 8, 16, 24]), ([1990, 9, 0], [0, 20, 24, 24]),
                                              ([3, 2000, 1500], [0, 1, 2, 10]), ([100, 200, 300], [0, 8, 16, 24]))):
            static["lens"].copy_(i32(lens))
            static["start"].copy_(i32(start))
            for name in ("q", "k", "v"):
                static[name].copy_(randn(81 + turn, static[name].shape, F32))
            got = []
            for i in (0, 1, 0):
                outs[i].fill_(7.0)
                torch.cuda.synchronize()
                graphs[i].replay()
                torch.cuda.synchronize()
                got.append((outs[i].cpu().clone(), lses[i].cpu().clone(), kb.cpu().clone()))
            outs[0].fill_(7.0)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                step(0)
            torch.cuda.synchronize()
            want = (outs[0].cpu(), lses[0].cpu(), kb.cpu())
            rows = start[-1]
            for g in got:
                assert all(torch.equal(a[:rows], b[:rows]) for a, b in zip(g, want)), turn
                assert bool((g[0][rows:] == 7.0).all())
        del graphs
    ctx.close()


def test_another_stream(gpu_ctx):
    """Work in order on a stream of the caller's."""
    pool = Pool(gpu_ctx, 90, [300, 200], KV4, 16, 2, 64)
    q = randn(91, (60, 8, 64), F32)
    want = run(gpu_ctx, pool, q, [0, 40, 60])
    stream = torch.cuda.Stream()
    ctx = Context(0)
    ctx.set_stream(stream.cuda_stream)
    table, lens, start = pool.table.cuda(), pool.lens.cuda(), i32([0, 40, 60]).cuda()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        x = q.cuda(non_blocking=True)
        out, lse = torch.zeros_like(x), torch.zeros(60, 8, device="cuda")
        kernels.paged_prompt_attention(ctx, pool.kv, table, lens, x, out, seq_start=start, lse=lse)
        out2 = out.clone()
    torch.cuda.synchronize()
    assert torch.equal(out2.cpu(), want[0]) and torch.equal(lse.cpu(), want[1])
    ctx.close()


def test_strides_and_host_arrays(gpu_ctx):
    """Rows of a fused projection, rows between others, arrays in host memory: the same bits."""
    for ct in (F32, KV4):
        pool = Pool(gpu_ctx, 92, [70, 33], ct, 16, 2, 64)
        q = randn(93, (50, 4, 64), F32)
        start = [0, 40, 45]
        want, wl = run(gpu_ctx, pool, q, start, window=20, slopes=slopes_of(4), prefix=i32([2, 0]))
        fused = torch.full((50, 10, 64), 7.0, device="cuda")
        fused[:, 1:5] = q.cuda()
        torch.cuda.synchronize()
        kernels.paged_prompt_attention(gpu_ctx, pool.kv, pool.table.cuda(), pool.lens.cuda(), fused[:, 1:5], fused[:, 6:10],
                                       seq_start=i32(start).cuda(), window=20, slopes=slopes_of(4).cuda(), prefix=i32([2, 0]).cuda())
        done(gpu_ctx)
        assert torch.equal(fused[:45, 6:].cpu(), want[:45]) and bool((fused[45:, 6:] == 7.0).all())
        assert bool((fused[:, 0] == 7.0).all()) and bool((fused[:, 5] == 7.0).all())
        out, lse = np.full((50, 4, 64), 7.0, np.float32), np.full((50, 4), 7.0, np.float32)
        # (host arrays are checked: pages that are needed have to be there)
        kernels.paged_prompt_attention(gpu_ctx, pool.kv, pool.table.numpy(), pool.lens.numpy(), q.numpy(), out,
                                       seq_start=np.array(start, np.int32), window=20, slopes=slopes_of(4).numpy(),
                                       prefix=np.array([2, 0], np.int32), lse=lse)
        assert np.array_equal(out, want.numpy()) and np.array_equal(lse, wl.numpy())
        kb = np.full((45, 2, 64), 7.0, np.float32)
        kernels.paged_read(gpu_ctx, pool.kv, pool.table.numpy(), pool.lens.numpy(), kb, seq_start=np.array(start, np.int32))
        assert np.array_equal(kb[:40], pool.history(0)[0][30:].float().numpy())


def test_past_32_bits(gpu_ctx):
    """Pages whose elements lie past 2^32 bytes and elements of a pool."""
    for ct in (BF16, KV4):
        page, kv, hd, far = 256, 4, 128, 20_000 if ct == BF16 else 60_000
        shape = (far + 3, page, kv, hd) if ct == BF16 else (far + 3, kv, kv4_bytes(page, hd))
        k, v = (torch.zeros(shape, dtype=torch.bfloat16 if ct == BF16 else torch.uint8, device="cuda") for _ in range(2))
        assert k.numel() > 1 << 32 if ct == KV4 else k.numel() > 1 << 31
        handle = PagedKv(gpu_ctx, k, v) if ct == BF16 else PagedKv.four_bit(gpu_ctx, k, v, page, hd)
        table, lens, start = i32([[far + 2, 1], [0, far]]).cuda(), i32([400, 300]).cuda(), i32([0, 400, 700]).cuda()
        kk, vv = randn(95, (700, kv, hd), BF16), randn(96, (700, kv, hd), BF16)
        q = randn(97, (700, 4, hd), BF16)
        out, kb = torch.zeros(q.shape, dtype=q.dtype, device="cuda"), torch.zeros(kk.shape, device="cuda")
        one = torch.zeros(2, 4, hd, dtype=q.dtype, device="cuda")
        kd, vd, qd, last = on_gpu(kk, vv, q, q[[399, 699]])
        kernels.paged_append(gpu_ctx, handle, table, lens, kd, vd, seq_start=start)
        kernels.paged_prompt_attention(gpu_ctx, handle, table, lens, qd, out, seq_start=start)
        kernels.paged_attention(gpu_ctx, handle, table, lens, last, one)
        kernels.paged_read(gpu_ctx, handle, table, lens, kb, seq_start=start)
        done(gpu_ctx)
        hk, hv = (held(x) if ct == KV4 else x.double() for x in (kk, vv))
        assert torch.equal(kb.cpu().double(), hk)
        for a, b, s in ((0, 400, 0), (400, 700, 1)):
            want, _, tol, _ = attention64(q[a:b], (hk[a:b], hv[a:b]), torch.arange(b - a), 1 / math.sqrt(hd), BF16, ct)
            tol = tol * (1 + half_step(BF16)) + half_step(BF16) * want.abs()
            close(out[a:b], want, tol, f"sequence {s}")
            close(one[s], want[-1], tol[-1], f"last token of {s}")
        handle.close()
        del k, v, kd, vd, qd


# ---- refusals ----------------------------------------------------------------------------------------
def refused(code, f):
    with pytest.raises(BBError) as e:
        f()
    assert e.value.code == code, e.value


def test_refusals(gpu_ctx):
    c = gpu_ctx
    ARG, DT, SHAPE, RANGE = _lib.BB_ERR_ARG, _lib.BB_ERR_DTYPE, _lib.BB_ERR_SHAPE, _lib.BB_ERR_RANGE
    pool = Pool(c, 99, [40, 50], F32, 16, 2, 64)
    table, lens, start = pool.table.cuda(), pool.lens.cuda(), i32([0, 10, 20]).cuda()
    q = torch.zeros(20, 4, 64, device="cuda")
    out = torch.zeros_like(q)

    def call(**kw):
        a = dict(q=q, out=out, seq_start=start)
        a.update(kw)
        return kernels.paged_prompt_attention(c, pool.kv, table, lens, **a)

    refused(ARG, lambda: call(cap=-1.0))
    refused(ARG, lambda: call(cap=NAN))
    refused(ARG, lambda: call(scale=INF))
    refused(ARG, lambda: call(out=q))
    refused(SHAPE, lambda: call(seq_start=None))
    refused(ARG, lambda: call(q=q[:, :3].contiguous(), out=out[:, :3].contiguous()))
    refused(ARG, lambda: call(lse=out.view(-1)[:80].view(20, 4)))
    refused(ARG, lambda: call(out=pool.k.view(-1)[:20 * 256].view(20, 4, 64)))
    refused(RANGE, lambda: call(workspace=torch.zeros(16, dtype=torch.uint8, device="cuda")))
    for bad in (lambda: call(window=-1), lambda: call(scale=0), lambda: call(seq_start=start[:2]), lambda: call(slopes=torch.zeros(3, device="cuda")),
                lambda: call(prefix=i32([1]).cuda()), lambda: call(lse=torch.zeros(20, 3, device="cuda")), lambda: call(out=out.half()),
                lambda: call(seq_start=start.cpu()), lambda: call(q=q[:, :, ::2])):
        with pytest.raises(ValueError):
            bad()
    # what host arrays hold
    hq, ho = np.zeros((20, 4, 64), np.float32), np.zeros((20, 4, 64), np.float32)

    def host(table=pool.table, lens=pool.lens, start=(0, 10, 20), **kw):
        return kernels.paged_prompt_attention(c, pool.kv, table.numpy(), lens.numpy(), hq, ho,
                                              seq_start=np.array(start, np.int32), **kw)

    host()
    refused(RANGE, lambda: host(start=(1, 10, 20)))
    refused(RANGE, lambda: host(start=(0, 30, 20)))
    refused(RANGE, lambda: host(start=(0, 10, 21)))
    refused(RANGE, lambda: host(lens=i32([5, 50])))
    refused(RANGE, lambda: host(lens=i32([-1, 50])))
    refused(RANGE, lambda: host(lens=i32([4000, 50])))
    gone = pool.table.clone()
    gone[0, 0] = -1
    refused(RANGE, lambda: host(table=gone))
    host(table=gone, window=5)
    refused(RANGE, lambda: host(table=gone, window=5, prefix=np.array([1, 0], np.int32)))
    refused(RANGE, lambda: host(prefix=np.array([-1, 0], np.int32)))
    # too much for one call
    n = ctypes.c_size_t()
    lib = _lib.lib()
    assert lib.bb_paged_prompt_attention_workspace(c.handle, pool.kv.handle, 4, 2, 1 << 22, ctypes.byref(n)) == RANGE
    assert lib.bb_paged_prompt_attention_workspace(c.handle, pool.kv.handle, 65534, 2, 1 << 21, ctypes.byref(n)) == RANGE
    assert lib.bb_paged_prompt_attention_workspace(c.handle, pool.kv.handle, 3, 2, 8, ctypes.byref(n)) == ARG
    # none at all
    kernels.paged_prompt_attention(c, pool.kv, table[:0], lens[:0], q[:0], out[:0], seq_start=i32([0]).cuda())
    kernels.paged_read(c, pool.kv, table[:0], lens[:0], torch.zeros(0, 2, 64, device="cuda"))
    # 4-bit pools
    refused(SHAPE, lambda: kv4_bytes(16, 48))
    refused(SHAPE, lambda: PagedKv.create(c, KV4, 4, 16, 2, 80))
    refused(DT, lambda: PagedKv.create(c, 2, 4, 16, 2, 64))
    size = kv4_bytes(16, 64)
    k = torch.zeros(4, 2, size, dtype=torch.uint8, device="cuda")
    v = torch.zeros_like(k)
    refused(ARG, lambda: PagedKv.four_bit(c, k, k, 16, 64))
    refused(ARG, lambda: PagedKv.four_bit(c, k[:1].expand(4, 2, size), v[:1].expand(4, 2, size), 16, 64))
    wide = torch.zeros(9, size + 8, dtype=torch.uint8, device="cuda")
    refused(ARG, lambda: PagedKv.four_bit(c, wide[:4, :size].unsqueeze(1), wide[4:8, :size].unsqueeze(1), 16, 64))
    for bad in (lambda: PagedKv.four_bit(c, k, v[:3], 16, 64), lambda: PagedKv.four_bit(c, k, v, 17, 64),
                lambda: PagedKv.four_bit(c, k.cpu(), v.cpu(), 16, 64), lambda: PagedKv.four_bit(c, k.short(), v.short(), 16, 64),
                lambda: kernels.paged_read(c, pool.kv, table, lens)):
        with pytest.raises(ValueError):
            bad()
    rows = torch.zeros(20, 2, 64, device="cuda")
    refused(ARG, lambda: kernels.paged_read(c, pool.kv, table, lens, rows, rows, seq_start=start))
    refused(ARG, lambda: kernels.paged_read(c, pool.kv, table, lens, pool.k.view(-1)[:20 * 128].view(20, 2, 64), seq_start=start))
    refused(SHAPE, lambda: kernels.paged_read(c, pool.kv, table, lens, rows))


def test_capture_without_a_workspace_is_refused(gpu_ctx):
    pool = Pool(gpu_ctx, 98, [400], BF16, 16, 1, 64)
    stream = torch.cuda.Stream()
    ctx = Context(0)
    ctx.set_stream(stream.cuda_stream)
    q, table, lens, start = torch.zeros(4, 4, 64, device="cuda"), pool.table.cuda(), pool.lens.cuda(), i32([0, 4]).cuda()
    out = torch.zeros_like(q)
    assert pool.kv.prompt_workspace(4, 1, 4) > 0
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        out.zero_()
        refused(_lib.BB_ERR_ARG, lambda: kernels.paged_prompt_attention(ctx, pool.kv, table, lens, q, out, seq_start=start))
    torch.cuda.synchronize()
    del g
    ctx.close()
