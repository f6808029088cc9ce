"""The paged-cache operators (bb_rope, bb_paged_append, bb_paged_attention) against their formulas in
64 bits: types, head layouts, lengths from none to long ones, odd sizes and page sizes, strides,
windows, pages that are not there, what lies behind the last position, captured calls.

Tolerances count roundings. u = 2^-24 is half a step of f32. A sum of n terms is off by at most
n·u of the terms' absolute sum, and by independent roundings of about sqrt(n)·u of it: 8·sqrt(n)·u is
allowed. A stored value of type t is off by finfo(t).eps / 2 of itself.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

from bebelm_amd import BBError, _lib, kernels, synth
from bebelm_amd.model import BF16, F16, F32, AttnOp, Context, PagedKv, RopePlan

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -25, BF16: 2.0 ** -134}   # half a step of the smallest values


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(seed, shape, dt, spread=1.0):
    return (spread * torch.randn(shape, generator=gen(seed))).to(TYPES[dt])


def half_step(dt):
    return torch.finfo(TYPES[dt]).eps / 2


def done(ctx):
    ctx.synchronize()
    torch.cuda.synchronize()


def close(got, want, tol, what):
    got, want = got.double().cpu(), want.double().cpu()
    tol = torch.as_tensor(tol, dtype=torch.float64).expand_as(want)
    off = (got - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / tol).max()):.3g} times"


# ---- the formulas in 64 bits --------------------------------------------------------------------
RULES = {"none": {}, "linear": {"factor": 4.0}, "base": {"factor": 8.0},
         "parts": {"factor": 8.0, "original_positions": 4096.0}}


def frequencies(rot, base, scaling, factor=1.0, original_positions=0.0, low_rotations=1.0, high_rotations=32.0):
    f = []
    for i in range(rot // 2):
        b = np.longdouble(base)
        if scaling == "base":
            b = b * np.longdouble(factor) ** (np.longdouble(rot) / (rot - 2))
        v = b ** (-np.longdouble(2 * i) / rot)
        if scaling == "linear":
            v = v / factor
        if scaling == "parts":
            r = original_positions * v / (2 * np.pi)
            g = min(1, max(0, (r - low_rotations) / (high_rotations - low_rotations)))
            v = v * (g + (1 - g) / factor)
        f.append(v)
    return np.array(f, np.longdouble)


def turned(x, pos, f, interleaved, m=1.0):
    """(x [tokens, heads, hd] turned, the absolute sums of each value's two products) in float64."""
    x, half = x.double(), len(f)
    # (the angles and their remainder in extended precision)
    a = np.asarray(pos, np.longdouble)[:, None] * f[None]
    a = np.remainder(a, 2 * np.longdouble("3.14159265358979323846264338327950288"))
    c, s = (torch.from_numpy(np.asarray(w, np.float64))[:, None] * m for w in (np.cos(a), np.sin(a)))
    i, j = (torch.arange(half) * 2, torch.arange(half) * 2 + 1) if interleaved else (torch.arange(half),
                                                                                     torch.arange(half) + half)
    out, mag = x.clone(), x.abs()
    out[..., i] = x[..., i] * c - x[..., j] * s
    out[..., j] = x[..., i] * s + x[..., j] * c
    mag[..., i] = mag[..., j] = abs(m) * (x[..., i].abs() + x[..., j].abs())
    return out, mag


# cos and sin are off by at most 2^-25.3 (the reduced angle) and 2^-23 (the function), the products and
# the sum round three times more: 2.7·2^-23 of the absolute sum; the angle itself by pos·f·2^-51
def turn_tol(want, mag, pos, f, dt, more=0.0):
    far = torch.as_tensor(np.abs(np.asarray(pos, np.float64)) * float(f.max()) * 2.0 ** -51)[:, None, None]
    return (2.7 * 2.0 ** -23 + more + far) * mag * (1 + half_step(dt)) + half_step(dt) * want.abs() + TINY[dt]


def normed(x, gain, eps):
    x = x.double()
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * gain.double()


# sum of squares: at most 22 roundings in a row; half of that reaches the root; division, root, reciprocal, two
# products: 17 u
NORM_TOL = 17 * U


class Pool:
    """A pool, the page table of sequences of the given lengths, and where their positions are."""

    def __init__(self, ctx, seed, lens, dt, page, kv, hd, order="phd", fill=None, spare=2, extra=1):
        g = gen(seed)
        need = [(max(n, 0) + page - 1) // page for n in lens]
        self.n_pages = sum(need) + spare
        ids = torch.randperm(self.n_pages, generator=g).int()
        self.table = torch.full((len(lens), max(need + [1]) + extra), 1 << 30, dtype=torch.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = ids[at:at + n]
            at += n
        shape = {"p": self.n_pages, "s": page, "h": kv}
        dims = {"phd": "psh", "hnd": "phs", "hps": "hps"}[order]
        def make(i):
            x = torch.randn([shape[c] for c in dims] + [hd], generator=gen(seed + i))
            x = x.to(TYPES[dt]) if fill is None else torch.full_like(x, fill).to(TYPES[dt])
            return x.cuda().permute(*[dims.index(c) for c in "psh"], 3)
        self.k, self.v = make(1), make(2)
        self.kv = PagedKv(ctx, self.k, self.v)
        self.page, self.lens_list, self.lens = page, lens, torch.tensor(lens, dtype=torch.int32)

    def where(self, s):
        j = torch.arange(self.lens_list[s])
        return self.table[s][j // self.page].long(), j % self.page

    def history(self, s):
        p, r = self.where(s)
        return self.k.cpu()[p, r], self.v.cpu()[p, r]


def attention64(q, hist, scale, window=0):
    """(out, lse, tolerance without the output's rounding, lse's tolerance) of q [heads, hd]."""
    k, v = (t.double() for t in hist)
    n, heads, kv = k.shape[0], q.shape[0], k.shape[1]
    if window:
        k, v = k[max(0, n - window):], v[max(0, n - window):]
        n = k.shape[0]
    if n == 0:
        z = torch.zeros(q.shape, dtype=torch.float64)
        return z, torch.full((heads,), -math.inf, dtype=torch.float64), z, torch.zeros(heads, dtype=torch.float64)
    g = heads // kv
    qk = q.double().reshape(kv, g, -1)
    kt, vt = k.permute(1, 2, 0).contiguous(), v.permute(1, 0, 2).contiguous()
    s = (qk @ kt) * scale
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse[..., None])
    out = (p @ vt).reshape(heads, -1)
    # a score: its sum over hd, the scale's and the logarithm base's products; exp: 2 u and its argument's rounding
    hd = k.shape[-1]
    d = ((8 * math.sqrt(hd) + 4) * U * abs(scale) * (qk.abs() @ kt.abs()) + 4 * U * s.abs()).amax(-1) + 4 * U
    sums = (8 * math.sqrt(n) + 16) * U
    tol = ((2 * d + 2 * sums)[..., None] * (p @ vt.abs())).reshape(heads, -1)
    return out, lse.reshape(-1), tol, (d + sums + 4 * U * lse.abs()).reshape(-1)


def check_attention(pool, q, out, lse, scale, window, dt, what):
    for s in range(len(pool.lens_list)):
        want, wl, tol, tl = attention64(q[s].cpu(), pool.history(s), scale, window)
        close(out[s], want, tol * (1 + half_step(dt)) + half_step(dt) * want.abs() + TINY[dt], f"{what} out {s}")
        if lse is not None:
            empty = torch.isneginf(wl)
            assert torch.equal(torch.isneginf(lse[s].cpu()), empty), f"{what} lse {s}: empty rows"
            if not empty.any():
                close(lse[s], wl, tl + U * wl.abs(), f"{what} lse {s}")


def attend(ctx, pool, q, window=0, scale=None, workspace=None, kv=None):
    out = torch.full(q.shape, float("nan"), dtype=q.dtype, device="cuda")
    lse = torch.full(q.shape[:2], float("nan"), device="cuda")
    torch.cuda.synchronize()
    kernels.paged_attention(ctx, kv or pool.kv, pool.table.cuda(), pool.lens.cuda(), q.cuda(), out, scale=scale,
                            window=window, lse=lse, workspace=workspace)
    done(ctx)
    return out, lse


# ---- rotary positions -----------------------------------------------------------------------------
ROPE_SIZES = [(1, 1, 2, 2), (1, 40, 64, 64), (3, 5, 64, 32), (7, 2, 80, 26), (2, 3, 10, 6), (5, 1, 256, 256),
              (4500, 2, 48, 16), (33, 9, 96, 96), (2, 2, 255, 254), (3, 4, 64, 46), (5, 3, 100, 36), (2, 3, 33, 18)]


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("size", ROPE_SIZES)
def test_rope(gpu_ctx, dt, interleaved, size):
    t, h, hd, rot = size
    print("rope", dt, interleaved, size, flush=True)
    for i, (rule, more) in enumerate(RULES.items()):
        if rule == "base" and rot < 4:
            continue
        m = 1.0 if rule == "none" else 1.25
        plan = RopePlan(gpu_ctx, rot, 1e4, interleaved, rule, magnitude=m, **more)
        f = frequencies(rot, 1e4, rule, **more)
        x = randn(100 * t + i, (t, h, hd), dt)
        pos = torch.randint(-50, 200_000, (t,), generator=gen(i), dtype=torch.int32)
        xd, out = x.cuda(), torch.full(x.shape, float("nan"), dtype=TYPES[dt], device="cuda")
        torch.cuda.synchronize()
        kernels.rope(gpu_ctx, plan, xd, pos.cuda(), out)
        done(gpu_ctx)
        want, mag = turned(x, pos.numpy(), f, interleaved, m)
        close(out, want, turn_tol(want, mag, pos.numpy(), f, dt), f"{rule}")
        assert torch.equal(out[..., rot:].cpu().view(torch.uint8), x[..., rot:].contiguous().view(torch.uint8))
        assert torch.equal(xd.cpu(), x)
        kernels.rope(gpu_ctx, plan, xd, pos.cuda())   # in place: the same bits
        done(gpu_ctx)
        assert torch.equal(xd, out)
        plan.close()


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_strides(gpu_ctx, interleaved):
    """A slice of a fused projection, heads first, and rows so far apart that bytes between them show."""
    plan = RopePlan(gpu_ctx, 32, 1e6, interleaved)
    f = frequencies(32, 1e6, "none")
    pos = torch.tensor([5, 0, 1 << 20, (1 << 31) - 1, -(1 << 31)], dtype=torch.int32)
    fused = randn(1, (5, 12, 64), F32)
    for name, view in (("slice", lambda a: a[:, 2:9]), ("odd", lambda a: a[:, 4:, :50]),
                       ("heads first", lambda a: a.permute(1, 0, 2)[:5, :3])):
        x = fused.cuda()
        out = torch.full_like(x, 7.0)
        p = pos[:view(x).shape[0]].contiguous()
        torch.cuda.synchronize()
        kernels.rope(gpu_ctx, plan, view(x), p.cuda(), view(out))
        done(gpu_ctx)
        want, mag = turned(view(fused), p.numpy(), f, interleaved)
        close(view(out), want, turn_tol(want, mag, p.numpy(), f, F32), name)
        view(out).fill_(7.0)
        assert bool((out == 7.0).all()), f"{name}: written between the rows"


def test_rope_host_arrays_and_none(gpu_ctx):
    plan = RopePlan(gpu_ctx, 16, 1e4)
    x = np.random.default_rng(3).standard_normal((6, 2, 16)).astype(np.float32)
    out = np.full((6, 4, 16), 9.0, np.float32)
    pos = np.arange(6, dtype=np.int32)
    kernels.rope(gpu_ctx, plan, x, pos, out[:, 1:3])
    f = frequencies(16, 1e4, "none")
    want, mag = turned(torch.from_numpy(x), pos, f, False)
    close(torch.from_numpy(out[:, 1:3].copy()), want, turn_tol(want, mag, pos, f, F32), "host")
    assert (out[:, [0, 3]] == 9.0).all()
    kernels.rope(gpu_ctx, plan, x[:0], pos[:0])


def test_rope_keeps_what_is_not_a_number(gpu_ctx):
    plan = RopePlan(gpu_ctx, 16, 1e4)
    x = torch.zeros(1, 2, 32, device="cuda")
    x[0, 0, 3], x[0, 1, 30] = float("nan"), float("inf")
    out = torch.empty_like(x)
    torch.cuda.synchronize()
    kernels.rope(gpu_ctx, plan, x, torch.tensor([1], dtype=torch.int32, device="cuda"), out)
    done(gpu_ctx)
    nan = torch.isnan(out).nonzero().tolist()
    assert nan == [[0, 0, 3], [0, 0, 11]] and out[0, 1, 30] == float("inf") and float(out[0, 1].nan_to_num(posinf=0).sum()) == 0


# ---- append ---------------------------------------------------------------------------------------
def check_append(ctx, seed, dt, ct, heads, kv, hd, page, before, bring, rot=0, interleaved=False, norm=False, pos=None,
                 with_q=True, order="phd", padding=0, decode=False):
    lens = [a + b for a, b in zip(before, bring)]
    pool = Pool(ctx, seed, lens, ct, page, kv, hd, order=order)
    start = np.concatenate([[0], np.cumsum(bring)]).astype(np.int32)
    t = int(start[-1]) + padding
    q, k, v = (randn(seed + i, (t, n, hd), dt) for i, n in ((3, heads), (4, kv), (5, kv)))
    # a fused projection: the three side by side for each token
    fused = torch.cat((q, k, v), 1).cuda()
    qd, kd, vd = fused[:, :heads], fused[:, heads:heads + kv], fused[:, heads + kv:]
    q_out = torch.full((t, heads, hd), 7.0, dtype=TYPES[dt], device="cuda")
    gains = [1 + 0.1 * torch.randn(hd, generator=gen(seed + i)) for i in (6, 7)] if norm else [None, None]
    plan = RopePlan(ctx, rot, 1e6, interleaved) if rot else None
    kb, vb = pool.k.cpu().clone(), pool.v.cpu().clone()
    posd = torch.tensor(pos, dtype=torch.int32) if pos is not None else None
    torch.cuda.synchronize()
    kernels.paged_append(ctx, pool.kv, pool.table.cuda(), pool.lens.cuda(), kd, vd, rope=plan,
                         pos=posd.cuda() if posd is not None else None,
                         seq_start=None if decode else torch.from_numpy(start).cuda(),
                         q=qd if with_q else None, q_out=q_out if with_q else None,
                         q_norm=gains[0].cuda() if norm and with_q else None,
                         k_norm=gains[1].cuda() if norm else None, eps=1e-5)
    done(ctx)
    f = frequencies(rot, 1e6, "none") if rot else np.zeros(0, np.longdouble)
    more = NORM_TOL if norm else 0.0
    got_k, got_v = pool.k.cpu(), pool.v.cpu()
    for s, n in enumerate(bring):
        if n == 0:
            continue
        rows = slice(int(start[s]), int(start[s + 1]))
        page_ids, row = pool.where(s)
        page_ids, row = page_ids[-n:], row[-n:]
        p = np.asarray(pos[rows]) if pos is not None else np.arange(lens[s] - n, lens[s])
        kk, qq = (normed(x[rows], g, 1e-5) if norm else x[rows].double() for x, g in ((k, gains[1]), (q, gains[0])))
        if rot:
            wk, mk = turned(kk, p, f, interleaved)
            wq, mq = turned(qq, p, f, interleaved)
            tk, tq = turn_tol(wk, mk, p, f, ct, more), turn_tol(wq, mq, p, f, dt, more)
        else:
            wk, wq = kk, qq
            tk, tq = (w.abs() * (more + half_step(d)) + TINY[d] for w, d in ((wk, ct), (wq, dt)))
        close(got_k[page_ids, row], wk, tk, f"keys of {s}")
        assert torch.equal(got_v[page_ids, row], v[rows].to(TYPES[ct])), f"values of {s}"
        if with_q:
            close(q_out[rows], wq, tq, f"queries of {s}")
        got_k[page_ids, row] = kb[page_ids, row]
        got_v[page_ids, row] = vb[page_ids, row]
    # everything else is as it was
    assert torch.equal(got_k, kb) and torch.equal(got_v, vb), "written outside of the tokens' positions"
    assert bool((q_out[int(start[-1]):] == 7.0).all()) and (with_q or bool((q_out == 7.0).all()))
    assert torch.equal(fused.cpu(), torch.cat((q, k, v), 1))


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("ct", [F32, F16, BF16])
def test_append_types(gpu_ctx, dt, ct):
    for norm in (False, True):
        print("append", dt, ct, norm, flush=True)
        check_append(gpu_ctx, 11, dt, ct, 8, 2, 64, 16, [0, 15, 16, 40], [5, 1, 33, 7], rot=64, norm=norm)


APPEND_SHAPES = [
    # heads, kv, hd, rot, interleaved, page, before, bring
    (4, 4, 80, 80, False, 24, [3, 0, 100], [1, 60, 0]),
    (5, 1, 96, 48, True, 1, [0, 9], [4, 5]),
    (3, 3, 8, 4, False, 7, [6, 0, 0, 2], [0, 1, 0, 30]),
    (16, 1, 256, 256, True, 128, [200], [129]),
    (24, 2, 40, 26, False, 16, [0] * 70, [i % 3 for i in range(70)]),
    (2, 2, 64, 0, False, 16, [17, 0], [3, 3]),
    (6, 2, 64, 46, True, 16, [5, 9], [3, 20]),
    (6, 2, 72, 54, False, 16, [5, 9], [3, 20]),
]


@pytest.mark.parametrize("shape", range(len(APPEND_SHAPES)))
@pytest.mark.parametrize("order", ["phd", "hnd", "hps"])
def test_append_shapes(gpu_ctx, shape, order):
    heads, kv, hd, rot, il, page, before, bring = APPEND_SHAPES[shape]
    for norm in (False, True):
        print("append", shape, order, norm, flush=True)
        check_append(gpu_ctx, 20 + shape, BF16, F16, heads, kv, hd, page, before, bring, rot, il, norm, order=order,
                     padding=3)


def test_append_one_token_each(gpu_ctx):
    # decode batches: every sequence one token, and an empty place among them; without queries; given positions
    check_append(gpu_ctx, 31, F32, F32, 4, 2, 64, 16, [0, 15, 16, 31, 4000], [1] * 5, rot=64, norm=True, decode=True)
    check_append(gpu_ctx, 32, F32, BF16, 4, 2, 64, 16, [8], [1], rot=32, with_q=False, decode=True)
    pos = list(range(1000, 1009))
    check_append(gpu_ctx, 33, F16, F16, 4, 2, 64, 16, [0, 3], [4, 5], rot=64, interleaved=True, pos=pos)


def test_append_long_batch(gpu_ctx):
    # more tokens than blocks take one at a time, and a sequence search of more than one round
    check_append(gpu_ctx, 34, BF16, BF16, 4, 2, 64, 16, [i for i in range(130)], [37] * 130, rot=64, padding=5)


def test_append_leaves_out_what_has_no_place(gpu_ctx):
    """Empty places of a batch, pages that are not in the pool, lengths past the table."""
    pool = Pool(gpu_ctx, 41, [20, 16, 33, 5], F32, 16, 2, 64)
    pool.table[0, 1] = -1          # position 19's page
    pool.table[2, 2] = pool.n_pages  # position 32's
    lens = torch.tensor([20, 0, 33, 16 * pool.table.shape[1] + 1], dtype=torch.int32)
    k = torch.ones(4, 2, 64, device="cuda")
    q = torch.ones(4, 4, 64, device="cuda")
    q_out = torch.full_like(q, 7.0)
    kb, vb = pool.k.clone(), pool.v.clone()
    torch.cuda.synchronize()
    kernels.paged_append(gpu_ctx, pool.kv, pool.table.cuda(), lens.cuda(), k, k, q=q, q_out=q_out)
    done(gpu_ctx)
    assert torch.equal(pool.k, kb) and torch.equal(pool.v, vb)
    # a token whose page is missing has a position (its query is turned), the others have none
    assert [float(q_out[i, 0, 0]) for i in range(4)] == [1.0, 7.0, 1.0, 7.0]
    # starts that do not ascend: every token lands in some sequence's own pages or nowhere
    bad = torch.tensor([0, 9, 2, 3, 4], dtype=torch.int32, device="cuda")
    lens = torch.tensor([1, 2, 3, 4], dtype=torch.int32, device="cuda")
    kernels.paged_append(gpu_ctx, pool.kv, pool.table.cuda(), lens, k, k, seq_start=bad)
    done(gpu_ctx)


# ---- attention ------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("ct", [F32, F16, BF16])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_types(gpu_ctx, dt, ct, hd):
    print("attention", dt, ct, hd, flush=True)
    pool = Pool(gpu_ctx, 51, [1, 0, 15, 16, 17, 700, 64, 2500], ct, 16, 2, hd)
    q = randn(52, (8, 8, hd), dt, 1.5)
    out, lse = attend(gpu_ctx, pool, q)
    check_attention(pool, q, out, lse, 1 / math.sqrt(hd), 0, dt, "types")
    again, lse2 = attend(gpu_ctx, pool, q)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


HEADS = [(1, 1, 8), (32, 8, 64), (7, 7, 24), (16, 1, 128), (17, 1, 64), (40, 1, 80), (10, 2, 96), (4, 4, 256), (33, 3, 40),
         (64, 2, 256), (12, 6, 104)]


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_attention_heads(gpu_ctx, heads, dt):
    nh, kv, hd = heads
    print("attention", heads, dt, flush=True)
    pool = Pool(gpu_ctx, 61, [130, 1, 0, 63], dt, 16, kv, hd)
    q = randn(62, (4, nh, hd), dt, 2.0)
    out, lse = attend(gpu_ctx, pool, q)
    check_attention(pool, q, out, lse, 1 / math.sqrt(hd), 0, dt, "heads")


@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 33, 64, 100, 256])
@pytest.mark.parametrize("order", ["phd", "hnd", "hps"])
def test_attention_pages(gpu_ctx, page, order):
    lens = [page, page + 1, max(0, page - 1), 2 * page, 517, 0, 1, 1200]
    for dt in (F32, F16):
        print("attention", page, order, dt, flush=True)
        pool = Pool(gpu_ctx, 71, lens, dt, page, 3, 64, order=order)
        q = randn(72, (len(lens), 6, 64), dt)
        out, lse = attend(gpu_ctx, pool, q)
        check_attention(pool, q, out, lse, 0.125, 0, dt, "pages")


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 64, 100, 999, 1000, 5000, 1 << 40])
def test_attention_window(gpu_ctx, window):
    lens = [1000, 1, 0, 64, 17, 333]
    for page in (16, 24):
        pool = Pool(gpu_ctx, 81, lens, BF16, page, 2, 64)
        # positions before the window: pages that are gone
        for s, n in enumerate(lens):
            pool.table[s, :max(0, n - window) // page] = -1
        want = Pool(gpu_ctx, 81, lens, BF16, page, 2, 64)
        q = randn(82, (6, 4, 64), F32)
        out, lse = attend(gpu_ctx, pool, q, window=window, scale=0.3)
        check_attention(want, q, out, lse, 0.3, window if window < 1 << 31 else 0, F32, "window")


def test_attention_reads_nothing_behind_a_sequence(gpu_ctx):
    """A pool of NaN (and of infinities) but for the sequences' positions."""
    for fill in (float("nan"), float("inf")):
        for dt, page, hd in ((F32, 16, 64), (BF16, 16, 128), (F16, 24, 80), (BF16, 5, 64), (F16, 64, 256)):
            lens = [5, 33, 0, 1, 700]
            pool = Pool(gpu_ctx, 91, lens, dt, page, 2, hd, fill=fill)
            for s in range(len(lens)):
                p, r = pool.where(s)
                pool.k[p.cuda(), r.cuda()] = randn(92 + s, (lens[s], 2, hd), dt).cuda()
                pool.v[p.cuda(), r.cuda()] = randn(99 + s, (lens[s], 2, hd), dt).cuda()
            q = randn(93, (5, 8, hd), dt)
            out, lse = attend(gpu_ctx, pool, q)
            check_attention(pool, q, out, lse, 1 / math.sqrt(hd), 0, dt, f"fill {fill}")


def test_attention_without_pages(gpu_ctx):
    """Pages that are not in the pool: their positions are not there; with none left, zeros and -inf."""
    pool = Pool(gpu_ctx, 101, [80, 40, 16, 50], F32, 16, 2, 64)
    q = randn(102, (4, 4, 64), F32)
    table = pool.table.clone()
    pool.table[0, 1], pool.table[0, 4] = -5, pool.n_pages
    pool.table[1, :] = -1
    pool.table[2, 0] = (1 << 31) - 1
    out, lse = attend(gpu_ctx, pool, q)
    there = table.clone()
    for s in range(4):
        j = torch.arange(pool.lens_list[s])
        j = j[[0 <= int(pool.table[s, i // 16]) < pool.n_pages for i in j.tolist()]]
        p, r = there[s][j // 16].long(), j % 16
        want, wl, tol, tl = attention64(q[s], (pool.k.cpu()[p, r], pool.v.cpu()[p, r]), 0.125)
        close(out[s], want, tol + U * want.abs() + TINY[F32], f"out {s}")
        if torch.isneginf(wl).any():
            assert bool((out[s] == 0).all()) and bool(torch.isneginf(lse[s]).all())
        else:
            close(lse[s], wl, tl + U * wl.abs(), f"lse {s}")
    # lengths below 0 and past the table: none, and all of the table
    pool = Pool(gpu_ctx, 103, [32, 32], F32, 16, 2, 64, extra=0)
    q = randn(104, (2, 4, 64), F32)
    want, wl = attend(gpu_ctx, pool, q)
    pool.lens = torch.tensor([-3, 1 << 30], dtype=torch.int32)
    out, lse = attend(gpu_ctx, pool, q)
    assert bool((out[0] == 0).all()) and bool(torch.isneginf(lse[0]).all())
    assert torch.equal(out[1], want[1]) and torch.equal(lse[1], wl[1])


def test_attention_extremes(gpu_ctx):
    """Scores far apart, equal ones, infinite ones, values that are not numbers."""
    for dt in (F32, F16, BF16):
        pool = Pool(gpu_ctx, 111, [300, 300, 300, 300, 20, 300], dt, 16, 1, 64)
        p, r = pool.where(0)
        pool.k[p.cuda(), r.cuda()] = (30.0 * randn(112, (300, 1, 64), F32)).to(TYPES[dt]).cuda()  # one weight of 1
        p, r = pool.where(1)
        pool.k[p.cuda(), r.cuda()] = 0.0                                                          # equal weights
        p, r = pool.where(4)
        pool.k[p.cuda(), r.cuda()] = float("-inf")                                                # no weight at all
        q = randn(113, (6, 3, 64), dt)
        q[4] = q[4].abs() + 0.5
        q[2] = 0.0
        p, r = pool.where(5)
        pool.v[int(p[250]), int(r[250]), 0, 7] = float("nan")
        out, lse = attend(gpu_ctx, pool, q)
        for s in (0, 1, 2, 3):
            want, wl, tol, tl = attention64(q[s], pool.history(s), 0.125)
            close(out[s], want, tol * (1 + half_step(dt)) + half_step(dt) * want.abs() + TINY[dt], f"{dt} out {s}")
            close(lse[s], wl, tl + U * wl.abs(), f"{dt} lse {s}")
        assert bool((out[4] == 0).all()) and bool(torch.isneginf(lse[4]).all())
        assert torch.isnan(out[5, :, 7]).all() and int(torch.isnan(out[5]).sum()) == 3
        # an infinite key: the formula has no number either
        q[3] = q[3].abs() + 0.5
        p, r = pool.where(3)
        pool.k[int(p[100]), int(r[100])] = float("inf")
        out, lse = attend(gpu_ctx, pool, q)
        assert torch.isnan(out[3]).all()


def test_attention_wide_queries(gpu_ctx):
    """f32 queries and keys over many powers of two: nothing is rounded to the cache's type on the way."""
    for ct in (F32, F16, BF16):
        for lo, hi in ((-20, 3), (-3, 14)):
            pool = Pool(gpu_ctx, 121, [100, 1000], ct, 16, 2, 64)
            q = randn(122, (2, 4, 64), F32) * torch.exp2(torch.randint(lo, hi, (2, 4, 64), generator=gen(123)).float())
            scale = 0.02 * 2.0 ** -max(hi - 4, 0)
            out, lse = attend(gpu_ctx, pool, q, scale=scale)
            check_attention(pool, q, out, lse, scale, 0, F32, f"{ct} 2^{lo}..2^{hi}")
    # queries past f16's range and below it
    pool = Pool(gpu_ctx, 124, [50], F16, 16, 1, 64)
    for e in (-40, 40):
        q = randn(125, (1, 2, 64), F32) * 2.0 ** e
        out, lse = attend(gpu_ctx, pool, q, scale=0.125 * 2.0 ** -e)
        check_attention(pool, q, out, lse, 0.125 * 2.0 ** -e, 0, F32, f"2^{e}")


def test_attention_subnormal_keys_and_values(gpu_ctx):
    """f16 values below 2^-14 count as what they are, bf16 ones over their whole range too."""
    for ct, e in ((F16, -18), (BF16, -120), (F32, -120)):
        pool = Pool(gpu_ctx, 126, [40, 300], ct, 16, 2, 64)
        for x in (pool.k, pool.v):
            x.copy_((torch.randn(x.shape, generator=gen(127)) * 2.0 ** e).to(TYPES[ct]))
        q = randn(128, (2, 4, 64), F32) * 2.0 ** 10
        scale = 2.0 ** (-10 - e - 3)
        out, lse = attend(gpu_ctx, pool, q, scale=scale)
        check_attention(pool, q, out, lse, scale, 0, F32, f"2^{e}")


def test_attention_rows_at_odd_strides(gpu_ctx):
    """Rows of q and out that start at any element."""
    for dt in (F32, F16, BF16):
        for ct, hd in ((F32, 64), (BF16, 64), (F16, 128), (BF16, 24)):
            pool = Pool(gpu_ctx, 129, [40, 300, 5], ct, 16, 2, hd)
            row = 4 * hd + 3
            base = torch.randn(3 * row + 7, generator=gen(130)).to(TYPES[dt])
            view = lambda a: a.as_strided((3, 4, hd), (row, hd, 1))
            dev, out = base.cuda(), torch.full((3 * row + 7,), 7.0, dtype=TYPES[dt], device="cuda")
            torch.cuda.synchronize()
            kernels.paged_attention(gpu_ctx, pool.kv, pool.table.cuda(), pool.lens.cuda(), view(dev), view(out))
            done(gpu_ctx)
            check_attention(pool, view(base), view(out), None, 1 / math.sqrt(hd), 0, dt, f"{dt} {ct}")
            view(out).fill_(7.0)
            assert bool((out == 7.0).all())


def test_one_pool_of_keys_and_values(gpu_ctx):
    """Keys and values side by side in each page, and in each position."""
    for shape, pick in (((9, 2, 16, 2, 64), lambda a, i: a[:, i]), ((9, 16, 2, 2, 64), lambda a, i: a[:, :, i]),
                        ((9, 16, 2, 2, 64), lambda a, i: a[:, :, :, i])):
        both = torch.zeros(shape, dtype=torch.bfloat16, device="cuda")
        pool = PagedKv(gpu_ctx, pick(both, 0), pick(both, 1))
        k, v, q = randn(153, (70, 2, 64), BF16), randn(154, (70, 2, 64), BF16), randn(155, (2, 4, 64), BF16)
        table = torch.tensor([[8, 0, 3, 5], [1, 2, 7, 4]], dtype=torch.int32)
        start = torch.tensor([0, 50, 70], dtype=torch.int32)
        lens = torch.tensor([50, 20], dtype=torch.int32)
        out = torch.empty(2, 4, 64, dtype=torch.bfloat16, device="cuda")
        args = [x.cuda() for x in (table, lens, k, v, start, q)]
        torch.cuda.synchronize()
        kernels.paged_append(gpu_ctx, pool, args[0], args[1], args[2], args[3], seq_start=args[4])
        kernels.paged_attention(gpu_ctx, pool, args[0], args[1], args[5], out)
        done(gpu_ctx)
        for s in range(2):
            rows = slice(int(start[s]), int(start[s + 1]))
            want, _, tol, _ = attention64(q[s], (k[rows], v[rows]), 0.125)
            close(out[s], want, tol * (1 + half_step(BF16)) + half_step(BF16) * want.abs() + TINY[BF16], f"out {s}")
        pool.close()


def test_attention_ragged_batches(gpu_ctx):
    """Many sequences of all lengths: splits of every kind."""
    for seed, (n, longest, kv, g, hd, dt) in enumerate([(300, 60, 2, 4, 64, BF16), (70, 5000, 1, 2, 64, F16),
                                                        (3, 40000, 2, 3, 128, BF16), (1000, 9, 1, 1, 64, F32),
                                                        (40, 900, 8, 4, 64, F32), (270, 2500, 1, 2, 64, BF16),
                                                        (5, 3000, 1, 24, 64, F16), (4, 2000, 2, 17, 128, F32),
                                                        (600, 300, 2, 1, 256, F16)]):
        print("ragged", n, longest, flush=True)
        lens = [int(longest ** u) if u > 0.1 else 0 for u in torch.rand(n, generator=gen(seed)).tolist()]
        lens[-1] = longest
        pool = Pool(gpu_ctx, 131 + seed, lens, dt, 16, kv, hd)
        q = randn(132, (n, kv * g, hd), dt)
        out, lse = attend(gpu_ctx, pool, q)
        k, v = pool.k.cpu(), pool.v.cpu()
        for s in range(0, n, 7 if n > 100 else 1):
            p, r = pool.where(s)
            want, wl, tol, tl = attention64(q[s], (k[p, r], v[p, r]), 1 / math.sqrt(hd))
            close(out[s], want, tol * (1 + half_step(dt)) + half_step(dt) * want.abs() + TINY[dt], f"out {s}")
            if lens[s]:
                close(lse[s], wl, tl + U * wl.abs(), f"lse {s}")
        empty = torch.tensor(lens) == 0
        assert bool((out.cpu()[empty] == 0).all()) and bool(torch.isneginf(lse.cpu()[empty]).all())


def test_attention_past_32_bits(gpu_ctx):
    """A pool of more than 2^32 elements, its last pages in use; append and attention."""
    page, kv, hd = 256, 8, 128
    n_pages = (1 << 32) // (page * kv * hd) + 40
    k = torch.empty(n_pages, page, kv, hd, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    pool = PagedKv(gpu_ctx, k, v)
    ids = [n_pages - 1, 3, n_pages - 7, n_pages // 2 + 1]
    lens = 3 * page + 10
    hist = [randn(141 + i, (lens, kv, hd), BF16) for i in range(2)]
    table = torch.tensor([ids], dtype=torch.int32, device="cuda")
    start = torch.tensor([0, lens], dtype=torch.int32, device="cuda")
    n = torch.tensor([lens], dtype=torch.int32, device="cuda")
    kd, vd = (h.cuda() for h in hist)
    torch.cuda.synchronize()
    kernels.paged_append(gpu_ctx, pool, table, n, kd, vd, seq_start=start)
    done(gpu_ctx)
    for i, p in enumerate(ids):
        rows = slice(i * page, min(lens, (i + 1) * page))
        assert torch.equal(k[p, :rows.stop - rows.start].cpu(), hist[0][rows])
        assert torch.equal(v[p, :rows.stop - rows.start].cpu(), hist[1][rows])
    q = randn(143, (1, 16, hd), BF16)
    qd, out, lse = q.cuda(), torch.empty(1, 16, hd, dtype=torch.bfloat16, device="cuda"), torch.empty(1, 16, device="cuda")
    torch.cuda.synchronize()
    kernels.paged_attention(gpu_ctx, pool, table, n, qd, out, lse=lse)
    done(gpu_ctx)
    want, wl, tol, tl = attention64(q[0], hist, 1 / math.sqrt(hd))
    close(out[0], want, tol * (1 + half_step(BF16)) + half_step(BF16) * want.abs() + TINY[BF16], "out")
    pool.close()


def test_attention_strided_queries_and_host_arrays(gpu_ctx):
    pool = Pool(gpu_ctx, 151, [40, 3, 0], F32, 16, 2, 64)
    fused = randn(152, (3, 12, 64), F32)
    fd, od = fused.cuda(), torch.full((3, 9, 64), 7.0, device="cuda")
    torch.cuda.synchronize()
    wide = torch.zeros(3, 64, dtype=torch.int32)
    wide[:, :pool.table.shape[1]] = pool.table
    kernels.paged_attention(gpu_ctx, pool.kv, wide.cuda()[:, :pool.table.shape[1]], pool.lens.cuda(), fd[:, :4], od[:, 4:8])
    done(gpu_ctx)
    check_attention(pool, fused[:, :4], od[:, 4:8], None, 0.125, 0, F32, "strided")
    assert bool((od[:, [0, 1, 2, 3, 8]] == 7.0).all())
    out = np.full((3, 6, 64), 7.0, np.float32)
    lse = np.zeros((3, 4), np.float32)
    table = pool.table.numpy().copy()
    kernels.paged_attention(gpu_ctx, pool.kv, table, pool.lens.numpy(), fused[:, :4].numpy(), out[:, 1:5], lse=lse)
    check_attention(pool, fused[:, :4], torch.from_numpy(out[:, 1:5].copy()), torch.from_numpy(lse), 0.125, 0, F32, "host")
    assert (out[:, [0, 5]] == 7.0).all()
    x = np.ones((1, 2, 64), np.float32)
    kernels.paged_append(gpu_ctx, pool.kv, table[1:2], pool.lens.numpy()[1:2], x, 2 * x)
    done(gpu_ctx)
    p, r = pool.where(1)
    assert bool((pool.k[int(p[2]), int(r[2])] == 1).all()) and bool((pool.v[int(p[2]), int(r[2])] == 2).all())


def test_pool_of_the_library(gpu_ctx):
    """A pool that the library allocates gives what a view gives, and starts zeroed."""
    lens = [20, 7]
    pool = Pool(gpu_ctx, 161, lens, BF16, 16, 2, 64)
    kv = PagedKv.create(gpu_ctx, BF16, pool.n_pages, 16, 2, 64)
    kp, vp = kv.pages()
    assert kp % 256 == 0 and vp > kp
    k, v, q = randn(162, (27, 2, 64), BF16).cuda(), randn(163, (27, 2, 64), BF16).cuda(), randn(164, (2, 4, 64), BF16)
    start = torch.tensor([0, 20, 27], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    zeros, _ = attend(gpu_ctx, pool, q, kv=kv)
    assert bool((zeros == 0).all())
    for pages in (pool.kv, kv):
        kernels.paged_append(gpu_ctx, pages, pool.table.cuda(), pool.lens.cuda(), k, v, seq_start=start)
    a, b = attend(gpu_ctx, pool, q), attend(gpu_ctx, pool, q, kv=kv)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    check_attention(pool, q, *a, 0.125, 0, BF16, "view")
    kv.close()


# ---- captured calls, streams, the operators together --------------------------------------------
def test_captured_step(gpu_ctx):
    """Append and attention captured into two graphs of different batches on one context, replayed in
    turn with growing sequences and eager work between: the replays follow the lengths on the device."""
    stream = torch.cuda.Stream()
    gpu_ctx.set_stream(stream.cuda_stream)
    try:
        graphs = []
        for seed, lens in ((171, [15, 900, 0, 31]), (172, [3000])):
            top = [n + 8 for n in lens]
            pool = Pool(gpu_ctx, seed, top, BF16, 16, 2, 64)
            n = len(lens)
            plan = RopePlan(gpu_ctx, 64, 1e6)
            q, k, v = (torch.empty(n, h, 64, device="cuda") for h in (8, 2, 2))
            q_out, out, lse = torch.empty_like(q), torch.empty_like(q), torch.empty(n, 8, device="cuda")
            ln, table = torch.tensor(lens, dtype=torch.int32, device="cuda"), pool.table.cuda()
            ws = torch.empty(max(pool.kv.attention_workspace(8, n), 16), dtype=torch.uint8, device="cuda")

            def step(pool=pool, table=table, ln=ln, k=k, v=v, plan=plan, q=q, q_out=q_out, out=out, lse=lse, ws=ws):
                kernels.paged_append(gpu_ctx, pool.kv, table, ln, k, v, rope=plan, q=q, q_out=q_out)
                kernels.paged_attention(gpu_ctx, pool.kv, table, ln, q_out, out, lse=lse, workspace=ws)

            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                step()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                step()
            graphs.append((graph, pool, ln, (q, k, v, q_out, out, lse), step, lens, table, plan))
        for i in range(4):
            for graph, pool, ln, (q, k, v, q_out, out, lse), step, lens, _, _ in graphs:
                now = [n + i + 1 if n or i % 2 else 0 for n in lens]
                ln.copy_(torch.tensor(now, dtype=torch.int32))
                for j, x in enumerate((q, k, v)):
                    x.copy_(randn(180 + 10 * i + j, x.shape, F32))
                out.fill_(float("nan"))
                torch.cuda.synchronize()
                graph.replay()
                torch.cuda.synchronize()
                got = [x.clone() for x in (q_out, out, lse, pool.k, pool.v)]
                pool.lens_list = now
                check_attention(pool, q_out.cpu(), out, lse, 0.125, 0, F32, f"replay {i}")
                out.fill_(float("nan"))
                torch.cuda.synchronize()
                with torch.cuda.stream(stream):
                    step()
                torch.cuda.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(got, (q_out, out, lse, pool.k, pool.v)))
        # what may not be captured is refused, and the capture lives on
        _, pool, ln, (q, k, v, q_out, out, lse), step, lens, table, plan = graphs[0]
        host = np.zeros((1, 1, 64), np.float32)
        other = torch.cuda.CUDAGraph()
        with torch.cuda.graph(other, stream=stream):
            with pytest.raises(BBError, match="workspace"):
                kernels.paged_attention(gpu_ctx, pool.kv, table, ln, q, out)
            with pytest.raises(BBError, match="captured"):
                kernels.rope(gpu_ctx, plan, host, np.zeros(1, np.int32))
            step()
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        other.replay()
        torch.cuda.synchronize()
        check_attention(pool, q_out.cpu(), out, lse, 0.125, 0, F32, "replay of the third")
    finally:
        gpu_ctx.set_stream(0)


def test_two_contexts_at_once(gpu_ctx):
    """Two contexts on two streams, many calls of each under way together, on one pool."""
    pool = Pool(gpu_ctx, 181, [3000, 17, 900, 0, 2000], BF16, 16, 2, 64)
    other = Context(0)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    try:
        table, lens = pool.table.cuda(), pool.lens.cuda()
        qs = [[randn(182 + 10 * c + i, (5, 8, 64), F32).cuda() for i in range(6)] for c in range(2)]
        outs = [[torch.empty_like(q) for q in c] for c in qs]
        torch.cuda.synchronize()
        for ctx, st in zip((gpu_ctx, other), streams):
            ctx.set_stream(st.cuda_stream)
        for i in range(6):
            for c, ctx in enumerate((gpu_ctx, other)):
                kernels.paged_attention(ctx, pool.kv, table, lens, qs[c][i], outs[c][i])
        torch.cuda.synchronize()
        for c in range(2):
            for i in range(6):
                check_attention(pool, qs[c][i].cpu(), outs[c][i], None, 0.125, 0, F32, f"context {c} call {i}")
    finally:
        gpu_ctx.set_stream(0)
        other.close()


def test_decode_beside_the_attention_operator(gpu_ctx):
    """Conversations of one attention layer stepped together through the paged operators give what
    AttnOp gives each of them alone (its sums are in another order and its angles in f32)."""
    w = synth.attn_weights(5, hidden=512, n_heads=8, n_kv_heads=2, head_dim=64)
    op = AttnOp(gpu_ctx, w)
    prompts = [33, 5, 1, 64]
    n, hidden = len(prompts), 512
    rng = np.random.default_rng(7)
    xs = [0.5 * rng.standard_normal((p + 3, hidden)).astype(np.float32) for p in prompts]
    want, caches = [], []
    for x, p in zip(xs, prompts):
        cache = op.new_cache(128)
        out = np.empty_like(x)
        op.forward(cache, 0, x[:p], p, out[:p])
        for i in range(p, p + 3):
            op.forward(cache, i, x[i:i + 1], 1, out[i:i + 1])
        want.append(out)
        caches.append(cache)
    top = [p + 3 for p in prompts]
    pool = Pool(gpu_ctx, 191, top, F32, 16, 2, 64)
    plan = RopePlan(gpu_ctx, 64, w.freq_base)
    table = pool.table.cuda()
    gains = [torch.from_numpy(np.ascontiguousarray(g, np.float32)).cuda() for g in (w.q_norm, w.k_norm)]

    def project(t, x, rows):
        y = torch.empty(x.shape[0], rows, device="cuda")
        kernels.matmul(gpu_ctx, t.dtype, t, x.shape[1], rows, x, x.shape[0], y)
        return y

    def layer(x, lens, start):
        q, k, v = (project(t, x, r).view(x.shape[0], r // 64, 64) for t, r in ((op.q, 512), (op.k, 128), (op.v, 128)))
        ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
        st = None if start is None else torch.tensor(start, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        kernels.paged_append(gpu_ctx, pool.kv, table, ln, k, v, rope=plan, seq_start=st, q=q, q_norm=gains[0],
                             k_norm=gains[1], eps=w.eps)
        return q, ln

    # the prompts in one ragged batch, then three steps of all conversations together
    x = torch.from_numpy(np.concatenate([a[:p] for a, p in zip(xs, prompts)])).cuda()
    layer(x, prompts, np.concatenate([[0], np.cumsum(prompts)]).tolist())
    for i in range(3):
        x = torch.from_numpy(np.stack([a[p + i] for a, p in zip(xs, prompts)])).cuda()
        q, ln = layer(x, [p + i + 1 for p in prompts], None)
        out = torch.empty_like(q)
        torch.cuda.synchronize()
        kernels.paged_attention(gpu_ctx, pool.kv, table, ln, q, out)
        y = project(op.o, out.view(n, 512), hidden)
        done(gpu_ctx)
        for s, p in enumerate(prompts):
            a, b = y[s].double().cpu().numpy(), want[s][p + i].astype(np.float64)
            # the projections quantise their input to 8 bits: a value next to a step may fall to its other
            # side, which moves an output by 1/127 of a weight's share (512 inputs): 1% of the norm
            assert np.linalg.norm(a - b) <= 1e-2 * np.linalg.norm(b), (i, s)
    for s in range(n):
        k, v = caches[s].read()
        hk, hv = pool.history(s)
        assert np.array_equal(hv.numpy().reshape(-1), v)
        # angles: AttnOp's f32 sequence is off by a few roundings of positions below 67
        assert np.abs(hk.numpy().reshape(-1) - k).max() <= 2 * 67 * 64 * U * np.abs(k).max()
        caches[s].close()
    op.close()


# ---- refusals -------------------------------------------------------------------------------------
def refused(code, f):
    with pytest.raises(BBError) as e:
        f()
    assert e.value.code == code, e.value


def test_refusals(gpu_ctx):
    c = gpu_ctx
    ARG, DT, SHAPE, RANGE = _lib.BB_ERR_ARG, _lib.BB_ERR_DTYPE, _lib.BB_ERR_SHAPE, _lib.BB_ERR_RANGE
    # plans
    refused(SHAPE, lambda: RopePlan(c, 0, 1e4))
    refused(SHAPE, lambda: RopePlan(c, 7, 1e4))
    refused(SHAPE, lambda: RopePlan(c, 258, 1e4))
    refused(ARG, lambda: RopePlan(c, 8, 0.0))
    refused(ARG, lambda: RopePlan(c, 8, float("nan")))
    refused(ARG, lambda: RopePlan(c, 8, 1e4, scaling="linear", factor=0.0))
    refused(SHAPE, lambda: RopePlan(c, 2, 1e4, scaling="base", factor=2.0))
    refused(ARG, lambda: RopePlan(c, 8, 1e4, scaling="parts", factor=2.0))
    refused(ARG, lambda: RopePlan(c, 8, 1e4, scaling="parts", factor=2.0, original_positions=10, low_rotations=3,
                                  high_rotations=3))
    refused(ARG, lambda: RopePlan(c, 8, 1e4, magnitude=float("inf")))
    refused(RANGE, lambda: RopePlan(c, 64, 1e-300))
    with pytest.raises(ValueError):
        RopePlan(c, 8, 1e4, scaling="other")
    plan = RopePlan(c, 32, 1e4)
    x, pos = torch.zeros(4, 2, 64, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    refused(SHAPE, lambda: kernels.rope(c, plan, x[..., :16], pos))
    refused(ARG, lambda: kernels.rope(c, plan, x[1:3], pos[:2], x[2:4]))               # overlaps
    refused(ARG, lambda: kernels.rope(c, plan, x, pos, torch.zeros(1, 2, 64, device="cuda").expand(4, 2, 64)))
    refused(ARG, lambda: kernels.rope(c, plan, x.view(-1)[1:1 + 64].view(1, 1, 64), pos[:1]))   # misaligned
    for bad in (lambda: kernels.rope(c, plan, x.double(), pos), lambda: kernels.rope(c, plan, x, pos.long()),
                lambda: kernels.rope(c, plan, x, pos[:3]), lambda: kernels.rope(c, plan, x, pos.cpu()),
                lambda: kernels.rope(c, plan, x, pos, x.half()), lambda: kernels.rope(c, plan, x[..., ::2], pos)):
        with pytest.raises(ValueError):
            bad()
    # pools
    k = torch.zeros(4, 16, 2, 64, device="cuda")
    v = torch.zeros_like(k)
    refused(ARG, lambda: PagedKv(c, k, k))
    flat = torch.zeros(4 * 16 * 2 * 64 + 64, device="cuda")
    refused(ARG, lambda: PagedKv(c, flat[:-64].view(4, 16, 2, 64), flat[64:].view(4, 16, 2, 64)))
    refused(SHAPE, lambda: PagedKv(c, k[..., :20], v[..., :20]))
    refused(SHAPE, lambda: PagedKv.create(c, F32, 4, 16, 2, 264))
    refused(ARG, lambda: PagedKv(c, k[:1].expand(4, 16, 2, 64), v[:1].expand(4, 16, 2, 64)))
    flat = torch.zeros(8, 90, device="cuda")
    refused(ARG, lambda: PagedKv(c, flat[:4, :64].view(4, 1, 1, 64), flat[4:, :64].view(4, 1, 1, 64)))  # 90·4 % 16
    refused(DT, lambda: PagedKv.create(c, 12, 4, 16, 2, 64))
    refused(ARG, lambda: PagedKv.create(c, F32, 0, 16, 2, 64))
    refused(RANGE, lambda: PagedKv.create(c, F32, 1 << 31, 16, 2, 64))
    for bad in (lambda: PagedKv(c, k, v[:3]), lambda: PagedKv(c, k.cpu(), v.cpu()), lambda: PagedKv(c, k.double(), v.double()),
                lambda: PagedKv(c, k[..., ::2], v[..., ::2])):
        with pytest.raises(ValueError):
            bad()
    kv = PagedKv(c, k, v)
    table = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    lens = torch.ones(3, dtype=torch.int32, device="cuda")
    kk = torch.zeros(3, 2, 64, device="cuda")
    q = torch.zeros(3, 4, 64, device="cuda")
    out = torch.zeros_like(q)
    # append
    refused(SHAPE, lambda: kernels.paged_append(c, kv, table, lens, kk[:2], kk[:2]))
    big = RopePlan(c, 128, 1e4)
    refused(SHAPE, lambda: kernels.paged_append(c, kv, table, lens, kk, kk, rope=big))
    refused(ARG, lambda: kernels.paged_append(c, kv, table, lens, kk, kk, k_norm=torch.ones(64, device="cuda"), eps=-1.0))
    refused(ARG, lambda: kernels.paged_append(c, kv, table, lens, kk, kk, q=kk, k_norm=torch.ones(64, device="cuda"),
                                              eps=float("nan")))
    refused(ARG, lambda: kernels.paged_append(c, kv, table, lens, kk, kk, q=q, q_out=q[:1].expand(3, 4, 64)))
    refused(ARG, lambda: kernels.paged_append(c, kv, table, lens, kk, kk, q=q[:, :2], q_out=kk))   # onto the keys
    many = torch.zeros(4, 4, 64, device="cuda")
    refused(ARG, lambda: kernels.paged_append(c, kv, table, lens, kk, kk, q=many[:3], q_out=many[1:]))
    inside = k[0, :3]                                                              # rows of the pool itself
    refused(ARG, lambda: kernels.paged_append(c, kv, table, lens, inside, kk))
    refused(ARG, lambda: kernels.paged_append(c, kv, table, lens, kk, v[1, 2:5]))
    refused(ARG, lambda: kernels.paged_append(c, kv, table, lens, kk, kk, q=inside))
    for bad in (lambda: kernels.paged_append(c, kv, table, lens, kk.half(), kk),
                lambda: kernels.paged_append(c, kv, table, lens[:2], kk, kk),
                lambda: kernels.paged_append(c, kv, table.long(), lens, kk, kk),
                lambda: kernels.paged_append(c, kv, table, lens, kk[..., :32], kk[..., :32]),
                lambda: kernels.paged_append(c, kv, table, lens, kk, kk, seq_start=lens),
                lambda: kernels.paged_append(c, kv, table, lens, kk, kk.cpu())):
        with pytest.raises(ValueError):
            bad()
    # attention
    att = kernels.paged_attention
    refused(ARG, lambda: att(c, kv, table, lens, q, q))
    refused(ARG, lambda: att(c, kv, table, lens, q[:, :3], out[:, :3]))          # 3 heads on 2
    refused(ARG, lambda: att(c, kv, table, lens, q, out, scale=float("inf")))
    wide = torch.zeros(1, 1 << 27, dtype=torch.int32, device="cuda")              # 2^31 positions
    refused(RANGE, lambda: att(c, kv, wide, lens[:1], q[:1], out[:1]))
    need = kv.attention_workspace(4, 3)
    if need > 16:
        refused(RANGE, lambda: att(c, kv, table, lens, q, out, workspace=torch.zeros(need - 16, dtype=torch.uint8, device="cuda")))
    refused(ARG, lambda: att(c, kv, table, lens, kk, inside))
    ws = torch.zeros(need + 1024, dtype=torch.uint8, device="cuda")
    refused(ARG, lambda: att(c, kv, table, lens, q, out, lse=ws[:48].view(torch.float32).view(3, 4), workspace=ws))
    refused(ARG, lambda: att(c, kv, table, lens, q, out, workspace=ws[8:]))
    for bad in (lambda: att(c, kv, table, lens, q, out.half()), lambda: att(c, kv, table, lens, q, out[:2]),
                lambda: att(c, kv, table, lens, q, out, lse=out), lambda: att(c, kv, table, lens, q, out, scale=0.0),
                lambda: att(c, kv, table, lens, q, out, workspace=torch.zeros(1 << 20))):
        with pytest.raises(ValueError):
            bad()
    # what host arrays hold is looked at first
    h = dict(t=table.cpu().numpy(), n=lens.cpu().numpy(), k=kk.cpu().numpy(), q=q.cpu().numpy(), o=out.cpu().numpy())
    for n in (-1, 33):
        refused(RANGE, lambda: att(c, kv, h["t"], np.array([1, n, 1], np.int32), h["q"], h["o"]))
    for page in (-1, 4):
        t = h["t"].copy()
        t[2, 0] = page
        refused(RANGE, lambda: att(c, kv, t, h["n"], h["q"], h["o"]))
        refused(RANGE, lambda: kernels.paged_append(c, kv, t, h["n"], h["k"], h["k"]))
    for start in ([1, 1, 2, 3], [0, 2, 1, 3], [0, 1, 2, 4], [0, 0, 0, 2]):
        refused(RANGE, lambda: kernels.paged_append(c, kv, h["t"], h["n"], h["k"], h["k"], seq_start=np.array(start, np.int32)))
    closed = RopePlan(c, 32, 1e4)
    closed.close()
    with pytest.raises(ValueError):
        kernels.paged_append(c, kv, table, lens, kk, kk, rope=closed)
    refused(ARG, lambda: kernels.rope(c, closed, x, pos))
    done(c)
    assert bool((k == 0).all()) and bool((v == 0).all())


def test_spans_past_any_memory_are_refused(gpu_ctx):
    """Strides whose products with the counts could pass 64 bits, in the call's arrays and in a view."""
    c, lib = gpu_ctx, _lib.lib()
    plan = RopePlan(c, 32, 1e4)
    pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    x = torch.ones(64, device="cuda")
    for at in range(4):
        st = [64] * 4
        st[at] = 1 << 36
        assert lib.bb_rope(c.handle, plan.handle, F32, x.data_ptr(), st[0], st[1], 1, 1, 64, pos.data_ptr(), x.data_ptr(),
                           st[2], st[3], _lib.LOC_DEVICE) == _lib.BB_ERR_RANGE, at
    done(c)
    assert bool((x == 1).all())
    k, v = torch.zeros(1024, device="cuda"), torch.zeros(1024, device="cuda")
    for pages, size, heads, strides in ((1 << 20, 1, 1, (1 << 35, 0, 0)), (1 << 30, 1, 1, (1 << 25, 0, 0)),
                                        (3, 1, 1, (1 << 36, 0, 0)), (1, 1 << 19, 2, (0, 64, 1 << 36))):
        view = ctypes.c_void_p()
        assert lib.bb_paged_kv_view(c.handle, F32, k.data_ptr(), v.data_ptr(), pages, size, heads, 64, *strides,
                                    ctypes.byref(view)) == _lib.BB_ERR_RANGE, (pages, size, heads, strides)
        assert not view.value


# ---- rows of one buffer side by side -------------------------------------------------------------
def fused_parts(buf, heads, kv, order):
    """q, k and v as the columns of one projection's rows, in the given order ('-': a head of something else)."""
    at, got = 0, {}
    for c in order:
        n = {"q": heads, "k": kv, "v": kv, "-": 1}[c]
        got[c] = buf[:, at:at + n]
        at += n
    return got["q"], got["k"], got["v"]


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("order", ["qkv", "kvq", "k-q-v"])
@pytest.mark.parametrize("norm", [False, True])
def test_append_in_place_in_a_fused_projection(gpu_ctx, dt, order, norm):
    """q turned where it lies, between k and v of the same rows: the bits of a call with a q_out of its own."""
    heads, kv, hd = 6, 2, 64
    plan = RopePlan(gpu_ctx, hd, 1e6)
    gains = [(1 + 0.1 * torch.randn(hd, generator=gen(i))).cuda() if norm else None for i in (201, 202)]
    for bring, lens in (([1, 1], [5, 30]), ([3, 0, 9], [3, 17, 40])):
        t = sum(bring)
        start = None if bring == [1, 1] else torch.tensor([0, 3, 3, 12], dtype=torch.int32)
        base = randn(203, (t, heads + 2 * kv + order.count("-"), hd), dt)
        results = []
        for where in ("apart", "in place", "host"):
            pool = Pool(gpu_ctx, 204, lens, BF16, 16, kv, hd)
            index = [pool.table, pool.lens, start]
            g = gains
            if where == "host" and dt == F32:
                buf = base.numpy().copy()
                index = [i if i is None else i.numpy() for i in index]
                g = [i if i is None else i.cpu().numpy() for i in gains]
            else:
                buf = base.cuda()
                index = [i if i is None else i.cuda() for i in index]
            q, k, v = fused_parts(buf, heads, kv, order)
            out = torch.empty(t, heads, hd, dtype=TYPES[dt], device="cuda") if where == "apart" else None
            torch.cuda.synchronize()
            got = kernels.paged_append(gpu_ctx, pool.kv, index[0], index[1], k, v, rope=plan, seq_start=index[2], q=q,
                                       q_out=out, q_norm=g[0], k_norm=g[1])
            done(gpu_ctx)
            _, k0, v0 = fused_parts(base, heads, kv, order)
            assert torch.equal(torch.as_tensor(k).cpu(), k0) and torch.equal(torch.as_tensor(v).cpu(), v0)
            results.append((torch.as_tensor(got).cpu().clone(), pool.k.cpu(), pool.v.cpu()))
        for other in results[1:]:
            assert all(torch.equal(a, b) for a, b in zip(results[0], other))


def test_attention_and_rope_between_rows_of_their_output(gpu_ctx):
    """Queries and outputs as the halves of one buffer's rows; turned heads beside the ones they come from."""
    pool = Pool(gpu_ctx, 211, [40, 300, 0, 5], BF16, 16, 2, 64)
    both = torch.full((4, 9, 64), 7.0, device="cuda")
    both[:, 1:5] = randn(212, (4, 4, 64), F32).cuda()
    q = both[:, 1:5].clone()
    want, _ = attend(gpu_ctx, pool, q)
    kernels.paged_attention(gpu_ctx, pool.kv, pool.table.cuda(), pool.lens.cuda(), both[:, 1:5], both[:, 5:])
    done(gpu_ctx)
    assert torch.equal(both[:, 5:], want) and torch.equal(both[:, 1:5], q) and bool((both[:, 0] == 7.0).all())
    host = both.cpu().numpy()
    host[:, 5:] = 0.0
    kernels.paged_attention(gpu_ctx, pool.kv, pool.table.numpy(), pool.lens.numpy(), host[:, 1:5], host[:, 5:])
    assert np.array_equal(host, both.cpu().numpy())
    plan = RopePlan(gpu_ctx, 64, 1e4)
    pos = torch.arange(5, dtype=torch.int32, device="cuda")
    for shape, pick in (((5, 6, 64), lambda a, i: a[:, 3 * i:3 * i + 3]), ((5, 6, 64), lambda a, i: a[:, i::2]),
                        ((3, 10, 64), lambda a, i: a.permute(1, 0, 2)[5 * i:5 * i + 5]),
                        ((3, 10, 64), lambda a, i: a.permute(1, 0, 2)[i::2])):
        both = randn(213, shape, F32).cuda()
        x = pick(both, 0).contiguous()
        out = torch.empty_like(x)
        torch.cuda.synchronize()
        kernels.rope(gpu_ctx, plan, x, pos, out)
        kernels.rope(gpu_ctx, plan, pick(both, 0), pos, pick(both, 1))
        done(gpu_ctx)
        assert torch.equal(pick(both, 1), out) and torch.equal(pick(both, 0), x)


def test_rows_that_share_elements_are_refused(gpu_ctx):
    c, ARG = gpu_ctx, _lib.BB_ERR_ARG
    pool = Pool(c, 221, [20, 20, 20], F32, 16, 2, 64)
    table, lens = pool.table.cuda(), pool.lens.cuda()
    row = 8 * 64
    buf = torch.zeros(4 * row, device="cuda")

    def at(offset, heads, stride=row):
        return buf.as_strided((3, heads, 64), (stride, 64, 1), offset)

    q, k, v = at(0, 4), at(256, 2), at(384, 2)
    append = lambda q_out, **kw: kernels.paged_append(c, pool.kv, table, lens, **{**dict(k=k, v=v, q=q), **kw}, q_out=q_out)
    refused(ARG, lambda: append(at(64, 4)))                    # half on q, half on k
    refused(ARG, lambda: append(at(192, 2), q=at(0, 2)))       # its second head is k's first
    refused(ARG, lambda: append(at(row - 64, 2), q=at(128, 2)))  # v's last head
    refused(ARG, lambda: append(at(row - 64, 2), k=at(0, 2), v=at(128, 2), q=at(256, 2)))   # the next row's k
    refused(ARG, lambda: append(at(384, 2, row + 64), k=at(0, 2), v=at(128, 2), q=at(256, 2)))  # other strides
    att = lambda a, b: kernels.paged_attention(c, pool.kv, table, lens, a, b)
    refused(ARG, lambda: att(at(0, 4), at(192, 4)))
    refused(ARG, lambda: att(at(64, 4), at(384, 4)))
    refused(ARG, lambda: att(at(0, 4), at(row, 4)))            # the next sequence's rows
    plan, pos = RopePlan(c, 64, 1e4), torch.zeros(3, dtype=torch.int32, device="cuda")
    refused(ARG, lambda: kernels.rope(c, plan, at(0, 4), pos, at(192, 4)))
    refused(ARG, lambda: kernels.rope(c, plan, at(0, 4)[:, ::2], pos, at(32, 4)[:, ::2]))
    refused(ARG, lambda: kernels.rope(c, plan, at(0, 4), pos, at(row + 64, 4)))
    done(c)
    assert bool((buf == 0).all())


# ---- what a call does not look at ------------------------------------------------------------------
def test_host_append_needs_no_page_of_a_sequence_without_tokens(gpu_ctx):
    """A sequence that brings nothing may have any entries: also the one of its partly filled last page."""
    pool = Pool(gpu_ctx, 231, [20, 37, 3], F32, 16, 2, 64)
    table = pool.table.numpy().copy()
    table[1] = -1
    k = randn(232, (5, 2, 64), F32)
    start = np.array([0, 4, 4, 5], np.int32)
    before = pool.k.cpu(), pool.v.cpu()
    kernels.paged_append(gpu_ctx, pool.kv, table, pool.lens.numpy(), k.numpy(), 2 * k.numpy(), seq_start=start)
    done(gpu_ctx)
    got = pool.k.cpu(), pool.v.cpu()
    for s in (0, 2):
        p, r = (i[-(start[s + 1] - start[s]):] for i in pool.where(s))
        for x, old, want in zip(got, before, (k, 2 * k)):
            assert torch.equal(x[p, r], want[start[s]:start[s + 1]])
            x[p, r] = old[p, r]
    assert all(torch.equal(a, b) for a, b in zip(got, before))
    # the entries that it stores through are looked at, and lengths that no table holds
    table[0, 1] = -1
    refused(_lib.BB_ERR_RANGE, lambda: kernels.paged_append(gpu_ctx, pool.kv, table, pool.lens.numpy(), k.numpy(),
                                                            k.numpy(), seq_start=start))
    table = pool.table.numpy()
    for n in (-1, 16 * table.shape[1] + 1):
        refused(_lib.BB_ERR_RANGE, lambda: kernels.paged_append(gpu_ctx, pool.kv, table, np.array([20, n, 3], np.int32),
                                                                k.numpy(), k.numpy(), seq_start=start))


@pytest.mark.parametrize("where", ["cpu", "cuda"])
@pytest.mark.parametrize("pages", [0, 3])
def test_a_batch_of_no_sequences(gpu_ctx, where, pages):
    pool = Pool(gpu_ctx, 241, [20], F32, 16, 2, 64)
    before = pool.k.clone()
    new = lambda *shape, **kw: torch.zeros(*shape, device=where, **kw)
    table, lens = new(0, pages, dtype=torch.int32), new(0, dtype=torch.int32)
    q, k = new(0, 4, 64), new(0, 2, 64)
    assert kernels.paged_append(gpu_ctx, pool.kv, table, lens, k, k, q=q) is q
    assert kernels.paged_attention(gpu_ctx, pool.kv, table, lens, q, new(0, 4, 64)).numel() == 0
    # tokens that are all padding
    q = new(3, 4, 64) + 7.0
    kernels.paged_append(gpu_ctx, pool.kv, table, lens, new(3, 2, 64), new(3, 2, 64), q=q,
                         seq_start=new(1, dtype=torch.int32))
    done(gpu_ctx)
    assert torch.equal(pool.k, before) and bool((q == 7.0).all())


def test_the_decode_part_of_a_mixed_batch(gpu_ctx):
    """Index arrays, gains and sums as slices that begin at any word: three prompts' entries lie before those of the
    sequences that take one step."""
    pool = Pool(gpu_ctx, 251, [20, 37, 3, 40, 700, 18, 1], F32, 16, 1, 64, extra=2)
    other = Pool(gpu_ctx, 251, [20, 37, 3, 40, 700, 18, 1], F32, 16, 1, 64, extra=2)
    plan = RopePlan(gpu_ctx, 64, 1e6)
    table = torch.zeros(7, pool.table.shape[1] + 1, dtype=torch.int32)
    table[:, 1:] = pool.table
    table, lens = table.cuda(), pool.lens.cuda()
    pos = torch.arange(900, 907, dtype=torch.int32, device="cuda")
    words = torch.arange(-1, 5, dtype=torch.int32, device="cuda")   # [1:]: 0, 1, 2, 3, 4
    gains = (1 + 0.1 * torch.randn(129, generator=gen(252))).cuda()
    q, k, v = (randn(253 + i, (4, n, 64), F32).cuda() for i, n in enumerate((3, 1, 1)))
    lse = torch.full((7, 3), 7.0, device="cuda")
    got = []
    for p, own in ((pool, lambda x: x), (other, lambda x: x.clone())):
        q_out, out = torch.empty_like(q), torch.empty_like(q)
        sums = own(lse[3:])
        assert own(lens[3:]).data_ptr() % 16 == (0 if p is other else 12)
        torch.cuda.synchronize()
        kernels.paged_append(gpu_ctx, p.kv, own(table[3:, 1:]), own(lens[3:]), k, v, rope=plan, pos=own(pos[3:]),
                             seq_start=own(words[1:]), q=q, q_out=q_out, q_norm=own(gains[1:65]), k_norm=own(gains[65:]))
        kernels.paged_attention(gpu_ctx, p.kv, own(table[3:, 1:]), own(lens[3:]), q_out, out, lse=sums)
        x = kernels.rope(gpu_ctx, plan, q, own(pos[3:]), torch.empty_like(q))
        done(gpu_ctx)
        got.append((q_out, out, sums.clone(), x, p.k, p.v))
    assert all(torch.equal(a, b) for a, b in zip(*got))
    assert bool((lse[:3] == 7.0).all()) and not bool((lse[3:] == 7.0).any())
    # a word that begins inside another is refused
    x = got[0][3]
    assert _lib.lib().bb_rope(gpu_ctx.handle, plan.handle, F32, q.data_ptr(), 192, 64, 1, 3, 64, pos.data_ptr() + 2,
                              x.data_ptr(), 192, 64, _lib.LOC_DEVICE) == _lib.BB_ERR_ARG


# ---- windows over every form of page ---------------------------------------------------------------
@pytest.mark.parametrize("page", [1, 5, 8, 13, 16, 24, 40])
@pytest.mark.parametrize("ct,dt,hd", [(F32, F32, 64), (F16, F16, 80), (BF16, F32, 128), (BF16, BF16, 24)])
def test_attention_window_over_other_pages(gpu_ctx, page, ct, dt, hd):
    """Whole and odd pages, tiles of 16 and 32 positions: what lies before the window (and behind the last position)
    makes no difference, be its pages in the pool and full of NaN, or gone."""
    print("window", page, ct, dt, hd, flush=True)
    lens = [700, 3, 0, 64, 17, 333, 130]
    for window in (1, 31, 33, 100, 650):
        pool = Pool(gpu_ctx, 261, lens, ct, page, 2, hd, fill=float("nan"))
        hist = []
        for s, n in enumerate(lens):
            p, r = (i[max(0, n - window):] for i in pool.where(s))
            kv = [randn(262 + 2 * s + i, (len(p), 2, hd), ct) for i in range(2)]
            for x, h in zip((pool.k, pool.v), kv):
                x[p.cuda(), r.cuda()] = h.cuda()
            hist.append(kv)
            if s % 2:
                pool.table[s, :max(0, n - window) // page] = -1
        q = randn(290, (len(lens), 6, hd), dt)
        out, lse = attend(gpu_ctx, pool, q, window=window)
        for s in range(len(lens)):
            want, wl, tol, tl = attention64(q[s], hist[s], 1 / math.sqrt(hd))
            close(out[s], want, tol * (1 + half_step(dt)) + half_step(dt) * want.abs() + TINY[dt], f"{window} out {s}")
            if lens[s]:
                close(lse[s], wl, tl + U * wl.abs(), f"{window} lse {s}")
            else:
                assert bool(torch.isneginf(lse[s]).all())


# ---- what the tests above leave out ----------------------------------------------------------------
@pytest.mark.parametrize("low,high", [(1.0, 32.0), (0.25, 4.0), (0.0, 0.5), (8.0, 1000.0), (-3.0, 2.0), (1e5, 1e6)])
def test_rope_parts_between_other_rotations(gpu_ctx, low, high):
    more = {"factor": 16.0, "original_positions": 8192.0, "low_rotations": low, "high_rotations": high}
    plan = RopePlan(gpu_ctx, 128, 1e4, scaling="parts", magnitude=1.5, **more)
    f = frequencies(128, 1e4, "parts", **more)
    x, pos = randn(301, (9, 2, 128), F32), torch.randint(0, 130_000, (9,), generator=gen(302), dtype=torch.int32)
    out = torch.empty(9, 2, 128, device="cuda")
    xd, pd = x.cuda(), pos.cuda()
    torch.cuda.synchronize()
    kernels.rope(gpu_ctx, plan, xd, pd, out)
    done(gpu_ctx)
    want, mag = turned(x, pos.numpy(), f, False, 1.5)
    close(out, want, turn_tol(want, mag, pos.numpy(), f, F32), f"{low}..{high}")


def test_append_with_starts_that_do_not_ascend(gpu_ctx):
    """Device starts are not checked: a token's sequence is the number of sequences that end at or before it, its
    place counts from that one's end, and nothing but such places is written."""
    pool = Pool(gpu_ctx, 311, [20, 16, 33, 5], F32, 16, 2, 64)
    start, lens, t = [0, 9, 2, 3, 4], [12, 2, 3, 4], 12
    k, v = randn(312, (t, 2, 64), F32), randn(313, (t, 2, 64), F32)
    want = [pool.k.cpu(), pool.v.cpu()]
    for i in range(t):
        s = sum(e <= i for e in start[1:])
        at = lens[s] - start[s + 1] + i if s < 4 else -1
        page = int(pool.table[s, at // 16]) if 0 <= at < 16 * pool.table.shape[1] else -1
        if 0 <= page < pool.n_pages:
            for w, x in zip(want, (k, v)):
                w[page, at % 16] = x[i]
    args = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (lens, start)]
    kd, vd, table = k.cuda(), v.cuda(), pool.table.cuda()
    torch.cuda.synchronize()
    kernels.paged_append(gpu_ctx, pool.kv, table, args[0], kd, vd, seq_start=args[1])
    done(gpu_ctx)
    assert torch.equal(pool.k.cpu(), want[0]) and torch.equal(pool.v.cpu(), want[1])


def test_sums_past_32_bits(gpu_ctx):
    """The log sums of pages past 2^32 elements, a long sequence split over many blocks among them."""
    page, kv, hd = 64, 2, 64
    n_pages = (1 << 32) // (page * kv * hd) + 200
    pools = [torch.empty(n_pages, page, kv, hd, dtype=torch.float16, device="cuda") for _ in range(2)]
    ids = torch.cat((torch.arange(n_pages - 150, n_pages), torch.tensor([0, 7, n_pages // 2])))
    lens = [len(ids) * page - 11, 3 * page]
    table = torch.full((2, len(ids)), -1, dtype=torch.int32)
    table[0], table[1, :3] = ids, ids[-3:]
    for i, x in enumerate(pools):
        x[ids.cuda()] = randn(321 + i, (len(ids), page, kv, hd), F16).cuda()
    pool = PagedKv(gpu_ctx, *pools)
    q, out, lse = randn(323, (2, 8, hd), F16), torch.empty(2, 8, hd, dtype=torch.float16, device="cuda"), torch.empty(2, 8, device="cuda")
    args = table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), q.cuda()
    torch.cuda.synchronize()
    kernels.paged_attention(gpu_ctx, pool, *args, out, lse=lse)
    done(gpu_ctx)
    for s, n in enumerate(lens):
        pages = ids if s == 0 else ids[-3:]
        hist = [x[pages.cuda()].cpu().flatten(0, 1)[:n] for x in pools]
        want, wl, tol, tl = attention64(q[s], hist, 0.125)
        close(out[s], want, tol * (1 + half_step(F16)) + half_step(F16) * want.abs() + TINY[F16], f"out {s}")
        close(lse[s], wl, tl + U * wl.abs(), f"lse {s}")
    pool.close()


def test_a_batch_too_large_to_count_is_refused(gpu_ctx):
    """65536 sequences of 8 kv heads under a table of 2^17 positions; half of them are served."""
    pool = torch.zeros(2, 16, 8, 8, device="cuda"), torch.zeros(2, 16, 8, 8, device="cuda")
    kv = PagedKv(gpu_ctx, *pool)
    n = 65536
    table, lens = torch.zeros(n, 8192, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda")
    q, out = torch.ones(n, 8, 8, device="cuda"), torch.full((n, 8, 8), 7.0, device="cuda")
    refused(_lib.BB_ERR_RANGE, lambda: kernels.paged_attention(gpu_ctx, kv, table, lens, q, out))
    done(gpu_ctx)
    assert bool((out == 7.0).all())
    half = n // 2
    lens[half - 1] = 16
    torch.cuda.synchronize()
    kernels.paged_attention(gpu_ctx, kv, table[:half], lens[:half], q[:half], out[:half])
    done(gpu_ctx)
    assert bool((out[:half] == 0.0).all()) and bool((out[half:] == 7.0).all())
