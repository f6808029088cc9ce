"""The paged-cache operators a server of many conversations calls for each decoder layer: rotary
positions, appending a batch's keys and values to a paged cache (with the q/k norm and the rotation
on the way) and one new token per conversation attending over its pages.

`run` is the operators' plain form (elementary torch operations in float32, angles in float64), or
with `own` set the library's entry points on the same inputs. `exact` states the definitions again
in float64. Head shapes are the decoder's own (32 query and 8 kv heads of 64) and generic ones.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BASE = 1e6          # the decoder's rotary base
EPS = 1e-5


def _rope(layout="half", rot=64, scaling="none", factor=1.0, original=0, magnitude=1.0):
    return {"layout": layout, "rot": rot, "scaling": scaling, "factor": factor, "original": original,
            "magnitude": magnitude}


def listed():
    return [
        # rotation of one token's queries and keys: nothing but latency
        {"name": "rope_token_1", "kind": "rope", "tokens": 1, "heads": 40, "hd": 64, "dtype": "f32", "far": 4096,
         **_rope()},
        # a long prompt's queries, half of each head rotated in interleaved pairs, a context stretched
        # past the trained one: positions up to a million
        {"name": "rope_prompt_4097", "kind": "rope", "tokens": 4097, "heads": 32, "hd": 128, "dtype": "bf16",
         "far": 1_000_000, **_rope("interleaved", 64, "parts", 8.0, 8192, 1.2)},
        # one conversation's next token into a cache in the activations' own type
        {"name": "append_token_1", "kind": "append", "seqs": 1, "tokens": 0, "far": 4096, "heads": 32, "kv": 8,
         "hd": 64, "dtype": "f32", "cache": "f32", "page": 16, "norm": True, **_rope()},
        # a decode batch: every conversation's next token, f32 activations into a bf16 cache
        {"name": "append_batch_48", "kind": "append", "seqs": 48, "tokens": 0, "far": 8192, "heads": 32, "kv": 8,
         "hd": 64, "dtype": "f32", "cache": "bf16", "page": 16, "norm": True, **_rope()},
        # several prompts of different lengths absorbed in one ragged batch
        {"name": "append_prompts_5003", "kind": "append", "seqs": 7, "tokens": 5003, "far": 4096, "heads": 32, "kv": 8,
         "hd": 128, "dtype": "bf16", "cache": "bf16", "page": 32, "norm": False, **_rope(rot=128)},
        # the first tokens of a conversation: a cache of one page and a bit
        {"name": "attend_1_17", "kind": "attend", "seqs": 1, "longest": 17, "even": True, "heads": 32, "kv": 8,
         "hd": 64, "dtype": "f32", "cache": "f32", "page": 16, "window": 0},
        # one long conversation on a bf16 cache, f32 activations
        {"name": "attend_1_9001", "kind": "attend", "seqs": 1, "longest": 9001, "even": True, "heads": 32, "kv": 8,
         "hd": 64, "dtype": "f32", "cache": "bf16", "page": 16, "window": 0},
        # a decode batch of conversations of very different lengths, two places of it empty
        {"name": "attend_34_ragged", "kind": "attend", "seqs": 34, "longest": 16384, "even": False, "heads": 32,
         "kv": 8, "hd": 64, "dtype": "bf16", "cache": "bf16", "page": 16, "window": 0},
        # one kv head for each query head, an odd head size, pages that are no power of two
        {"name": "attend_7_own_heads", "kind": "attend", "seqs": 7, "longest": 3001, "even": False, "heads": 16,
         "kv": 16, "hd": 80, "dtype": "f16", "cache": "f16", "page": 24, "window": 0},
        # all query heads on one kv head, a very long document, the last tokens only in reach
        {"name": "attend_2_one_kv_head", "kind": "attend", "seqs": 2, "longest": 131072, "even": True, "heads": 16,
         "kv": 1, "hd": 128, "dtype": "bf16", "cache": "bf16", "page": 64, "window": 100_000},
        # the largest: a full server batch of long conversations
        {"name": "attend_64_8192", "kind": "attend", "seqs": 64, "longest": 8192, "even": True, "heads": 32, "kv": 8,
         "hd": 128, "dtype": "f16", "cache": "f16", "page": 16, "window": 0},
        # the step of one layer as a server runs it: append, then attend, f32 cache
        {"name": "step_24", "kind": "step", "seqs": 24, "longest": 4096, "even": False, "heads": 32, "kv": 8,
         "hd": 64, "dtype": "f32", "cache": "f32", "page": 16, "window": 0, "norm": True, **_rope()},
    ]


LARGEST = 64 * 8192 * 8 * 128   # cached key values of the largest listed case


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def _draw_rope(rng, hd):
    rot = rng.choice([hd, hd, hd // 2, 2 * rng.randint(2, hd // 2)])
    scaling = rng.choice(["none", "none", "linear", "base", "parts"])
    if scaling == "none":
        return _rope(rng.choice(["half", "interleaved"]), rot)
    return _rope(rng.choice(["half", "interleaved"]), rot, scaling, rng.choice([2.0, 4.0, 8.0, 32.0]),
                 rng.choice([4096, 8192, 32768]), rng.choice([1.0, 1.0, 1.1, 1.35]))


def draw(rng):
    kind = rng.choice(["rope", "append", "append", "attend", "attend", "attend", "attend", "step"])
    hd = rng.choice([64, 64, 128, 128, 32, 80, 96, 256])
    if kind == "rope":
        return {"kind": kind, "tokens": _log(rng, 1, 4096), "heads": _log(rng, 1, 40), "hd": hd,
                "dtype": rng.choice(list(TYPES)), "far": _log(rng, 256, 1_000_000), **_draw_rope(rng, hd)}
    kv, group = rng.choice([(8, 4), (8, 4), (4, 8), (2, 5), (16, 1), (1, 16), (1, 24)])
    dtype = rng.choice(list(TYPES))
    case = {"kind": kind, "heads": kv * group, "kv": kv, "hd": hd, "dtype": dtype,
            "cache": dtype if rng.random() < 0.6 else rng.choice(list(TYPES)),
            "page": rng.choice([1, 8, 16, 16, 16, 24, 32, 64, 128, 256])}
    if kind == "append":
        seqs = _log(rng, 1, 256)
        tokens = rng.choice([0, seqs + _log(rng, 1, 4096)])
        far = _log(rng, 64, min(32768, max(64, (1 << 28) // (seqs * kv * hd))))
        return {**case, "seqs": seqs, "tokens": tokens, "far": far,
                "norm": rng.random() < 0.5, **_draw_rope(rng, hd)}
    most = LARGEST // (2 * kv * hd)   # an f32 cache costs twice as much
    seqs = _log(rng, 1, min(256, most))
    longest = _log(rng, 1, min(131072, most // seqs))
    case.update(seqs=seqs, longest=longest, even=rng.random() < 0.4,
                window=rng.choice([0, 0, 0, _log(rng, 1, 8192)]))
    if kind == "step":
        case.update(norm=rng.random() < 0.5, **_draw_rope(rng, hd))
    return case


# ---- inputs ------------------------------------------------------------------------------------
def _gen(seed, stream, device="cuda"):
    g = torch.Generator(device=device)
    g.manual_seed((1_000_003 * int(seed) + 7919 * stream + 17) % (1 << 62))
    return g


def _normal(seed, stream, shape, dtype, spread=1.0):
    x = torch.randn(shape, generator=_gen(seed, stream), device="cuda", dtype=torch.float32)
    return (spread * x).to(TYPES[dtype])


def _pool(case, seed, stream, n_pages):
    """Pages of one pool, standard normal values (keys and values after their norms)."""
    return torch.empty(n_pages, case["page"], case["kv"], case["hd"], device="cuda",
                       dtype=TYPES[case["cache"]]).normal_(generator=_gen(seed, stream))


def _pages(seed, lens, page, spare=3):
    """(page table with -1 past each sequence's pages, pages of the pool): a sequence's pages lie
    anywhere in the pool, as they do after many conversations came and went."""
    need = [(n + page - 1) // page for n in lens]
    order = torch.randperm(sum(need) + spare, generator=_gen(seed, 11, "cpu"))
    table = torch.full((len(lens), max(1, max(need))), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table.cuda(), sum(need) + spare


def _lengths(case):
    """Positions in reach of the sequences: all the longest, or spread over their logarithm with the
    first the longest and two places of a larger batch empty. The same for every seed (a pool keeps
    its size); the seed says which sequence has which."""
    n, longest = case["seqs"], case["longest"]
    if case["even"]:
        return [longest] * n
    u = torch.rand(n, generator=_gen(0, 12, "cpu")).tolist()
    lens = [max(1, round(math.exp(x * math.log(longest)))) for x in u]
    lens[0] = longest
    if n >= 8:
        lens[n // 2] = lens[n - 1] = 0
    return lens


def _arrivals(case):
    """(positions cached before, tokens that the batch brings) of the sequences of an append."""
    n, t = case["seqs"], case["tokens"] or case["seqs"]
    cuts = torch.sort(torch.randperm(t - 1, generator=_gen(0, 13, "cpu"))[:n - 1])[0] + 1 if n > 1 else []
    edges = [0] + [int(c) for c in cuts] + [t]
    before = torch.randint(0, case["far"], (n,), generator=_gen(0, 15, "cpu")).tolist()
    return [(a, hi - lo) for a, lo, hi in zip(before, edges, edges[1:])]


def _shuffled(seed, items):
    return [items[i] for i in torch.randperm(len(items), generator=_gen(seed, 16, "cpu")).tolist()]


class _Program:
    """What a process keeps: one context, and one torch stream that is the current one from its making on, so that
    what fills the inputs, the calls and what reads their results are in order."""
    ctx = None
    stream = None

    @classmethod
    def context(cls):
        if cls.ctx is None:
            from bebelm_amd.model import Context
            cls.stream = torch.cuda.Stream()
            cls.ctx = Context(torch.cuda.current_device())
            cls.ctx.set_stream(cls.stream.cuda_stream)
            cls.stream.wait_stream(torch.cuda.current_stream())
            torch.cuda.set_stream(cls.stream)
        return cls.ctx


def _plan(case):
    from bebelm_amd.model import RopePlan
    return RopePlan(_Program.context(), case["rot"], BASE, interleaved=case["layout"] == "interleaved",
                    scaling=case["scaling"], factor=case["factor"], original_positions=case["original"],
                    magnitude=case["magnitude"])


def prepare(case, seed):
    kind, dtype, hd = case["kind"], case["dtype"], case["hd"]
    s = {"case": case}
    if own:
        _Program.context()   # (the inputs are made on its stream)
    if kind == "rope":
        t = case["tokens"]
        first = int(torch.randint(0, max(1, case["far"] - t), (1,), generator=_gen(seed, 14, "cpu")))
        s["x"] = _normal(seed, 1, (t, case["heads"], hd), dtype)
        s["pos"] = torch.arange(first, first + t, dtype=torch.int32, device="cuda")
        s["out"] = torch.empty_like(s["x"])
        if own:
            s["plan"] = _plan(case)
        return s
    if kind == "append":
        come = _shuffled(seed, _arrivals(case))
        lens = [a + b for a, b in come]
        tokens = case["tokens"] or case["seqs"]
        if case["tokens"]:
            edges = [0]
            for _, n in come:
                edges.append(edges[-1] + n)
            s["start"] = torch.tensor(edges, dtype=torch.int32, device="cuda")
    else:
        lens, tokens = _shuffled(seed, _lengths(case)), case["seqs"]
    s["table"], n_pages = _pages(seed, lens, case["page"])
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["k_pages"], s["v_pages"] = _pool(case, seed, 2, n_pages), _pool(case, seed, 3, n_pages)
    # queries a little wider than keys: some positions stand out, most count
    s["q"] = _normal(seed, 4, (tokens, case["heads"], hd), dtype, 1.5)
    if kind != "attend":
        s["k"], s["v"] = (_normal(seed, i, (tokens, case["kv"], hd), dtype) for i in (5, 6))
        s["q_rot"] = torch.zeros_like(s["q"])
        if case["norm"]:
            s["q_norm"] = 1.0 + 0.05 * _normal(seed, 7, (hd,), "f32")
            s["k_norm"] = 1.0 + 0.05 * _normal(seed, 8, (hd,), "f32")
        if own:
            s["plan"] = _plan(case)
    if kind != "append":
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(case["seqs"], case["heads"], device="cuda")
    if own:
        from bebelm_amd.model import PagedKv
        s["kv"] = PagedKv(_Program.context(), s["k_pages"], s["v_pages"])
    return s


# ---- plain forms -------------------------------------------------------------------------------
def _angles(case, pos):
    """float64 angles [tokens, rot / 2]."""
    rot, factor = case["rot"], case["factor"]
    base = BASE
    if case["scaling"] == "base":
        base = BASE * factor ** (rot / (rot - 2))
    i = torch.arange(0, rot, 2, dtype=torch.float64, device=pos.device)
    freq = torch.exp(i * (-math.log(base) / rot))
    if case["scaling"] == "linear":
        freq = freq / factor
    if case["scaling"] == "parts":
        keep = ((case["original"] * freq / (2 * math.pi) - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        freq = freq * (keep + (1.0 - keep) / factor)
    return pos.to(torch.float64)[:, None] * freq


def _rotate(case, x, pos):
    """float32 rotation of x [tokens, heads, hd]."""
    rot, m = case["rot"], case["magnitude"]
    a = _angles(case, pos)
    c, s = (m * torch.cos(a)).float()[:, None], (m * torch.sin(a)).float()[:, None]
    out = x.float().clone()
    first, second = ((slice(0, rot // 2), slice(rot // 2, rot)) if case["layout"] == "half" else
                     (slice(0, rot, 2), slice(1, rot, 2)))
    u, v = x[..., first].float(), x[..., second].float()
    out[..., first] = u * c - v * s
    out[..., second] = u * s + v * c
    return out


def _normed(x, gain):
    x = x.float()
    return x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)) * gain


def _places(s, tokens):
    """(whether each token has a place, its index in its sequence, its page, its row in the page)."""
    case, lens = s["case"], s["lens"].long()
    t = torch.arange(tokens, device="cuda")
    if "start" in s:
        start = s["start"].long()
        seq = torch.searchsorted(start, t, right=True) - 1
        index = lens[seq] - start[seq + 1] + t
    else:
        seq, index = t, lens - 1
    at = index.clamp(min=0)
    return index >= 0, index, s["table"][seq, at // case["page"]].long(), at % case["page"]


def _append(s):
    case, q, k = s["case"], s["q"], s["k"]
    there, index, page, row = _places(s, k.shape[0])
    if case["norm"]:
        q, k = _normed(q, s["q_norm"]), _normed(k, s["k_norm"])
    k, q = _rotate(case, k, index), _rotate(case, q, index)
    if case["kind"] == "step":  # empty places of the batch: nothing is written
        q = torch.where(there[:, None, None], q, s["q_rot"].float())
        old = (s["k_pages"][page, row].float(), s["v_pages"][page, row].float())
        k = torch.where(there[:, None, None], k, old[0])
        v = torch.where(there[:, None, None], s["v"].float(), old[1])
    else:
        v = s["v"].float()
    s["k_pages"][page, row] = k.to(s["k_pages"].dtype)
    s["v_pages"][page, row] = v.to(s["v_pages"].dtype)
    s["q_rot"].copy_(q)
    return s["k_pages"], s["v_pages"], s["q_rot"]


def _attend(s, q):
    case, lens, table = s["case"], s["lens"].long(), s["table"].long().clamp(min=0)
    kv, group, hd = case["kv"], case["heads"] // case["kv"], case["hd"]
    out, lse = s["out"], s["lse"]
    n = table.shape[1] * case["page"]
    some = max(1, (1 << 28) // (n * kv * hd))   # sequences at a time: about a gigabyte of keys
    for a in range(0, case["seqs"], some):
        ln, tb = lens[a:a + some], table[a:a + some]
        k = s["k_pages"][tb].reshape(len(tb), n, kv, hd).permute(0, 2, 3, 1).float().contiguous()
        qs = q[a:a + some].float().reshape(len(tb), kv, group, hd)
        scores = torch.matmul(qs, k) * (1.0 / math.sqrt(hd))
        j = torch.arange(n, device="cuda")
        seen = j[None] < ln[:, None]
        if case["window"]:
            seen = seen & (j[None] >= ln[:, None] - case["window"])
        scores = scores.masked_fill(~seen[:, None, None], -math.inf)
        top = scores.amax(-1, keepdim=True)
        top = torch.where(top == -math.inf, torch.zeros_like(top), top)
        p = torch.exp(scores - top)
        total = p.sum(-1, keepdim=True)
        v = s["v_pages"][tb].reshape(len(tb), n, kv, hd).permute(0, 2, 1, 3).float().contiguous()
        o = torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)
        out[a:a + some] = o.reshape(len(tb), -1, hd).to(out.dtype)
        lse[a:a + some] = (torch.log(total) + top).reshape(len(tb), -1)
    return out, lse   # an empty sequence: zeros, and the logarithm of nothing, -inf


def _own_append(s):
    from bebelm_amd import kernels
    kernels.paged_append(_Program.ctx, s["kv"], s["table"], s["lens"], s["k"], s["v"], rope=s["plan"],
                         seq_start=s.get("start"), q=s["q"], q_out=s["q_rot"], q_norm=s.get("q_norm"),
                         k_norm=s.get("k_norm"), eps=EPS)
    return s["k_pages"], s["v_pages"], s["q_rot"]


def _own_attend(s, q):
    from bebelm_amd import kernels
    kernels.paged_attention(_Program.ctx, s["kv"], s["table"], s["lens"], q, s["out"], window=s["case"]["window"],
                            lse=s["lse"])
    return s["out"], s["lse"]


def run(state):
    case = state["case"]
    if own:
        if case["kind"] == "rope":
            from bebelm_amd import kernels
            return kernels.rope(_Program.ctx, state["plan"], state["x"], state["pos"], state["out"])
        done = _own_append(state) if case["kind"] != "attend" else ()
        if case["kind"] == "append":
            return done
        return (*done, *_own_attend(state, state["q_rot"] if done else state["q"]))
    if case["kind"] == "rope":
        state["out"].copy_(_rotate(case, state["x"], state["pos"]))
        return state["out"]
    done = _append(state) if case["kind"] != "attend" else ()
    if case["kind"] == "append":
        return done
    return (*done, *_attend(state, state["q_rot"] if done else state["q"]))


# ---- what a pass cannot do without ---------------------------------------------------------------
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def work(case):
    kind, hd, e = case["kind"], case["hd"], _SIZE[case["dtype"]]
    if kind == "rope":
        n = case["tokens"] * case["heads"]
        return {"bytes": 2 * n * hd * e + 4 * case["tokens"], "flops": 3 * n * case["rot"]}
    c, row, nh = _SIZE[case["cache"]], case["kv"] * hd, case["heads"]
    nbytes = flops = 0
    if kind != "attend":
        t = (case["tokens"] or case["seqs"]) if kind == "append" else sum(n > 0 for n in _lengths(case))
        nbytes += t * (2 * row * (e + c) + 2 * nh * hd * e) + 8 * t
        flops += t * (nh + case["kv"]) * (3 * case["rot"] + (4 * hd if case["norm"] else 0))
    if kind != "append":
        seen = sum(min(n, case["window"] or n) for n in _lengths(case))
        nbytes += 2 * seen * row * c + 2 * case["seqs"] * nh * hd * e + 4 * seen / case["page"] + 4 * case["seqs"] * nh
        flops += 4 * nh * hd * seen
    return {"bytes": nbytes, "flops": flops}


# ---- the definitions in 64 bits -------------------------------------------------------------------
def _exact_turn(case, x, pos):
    """x [tokens, heads, hd] float64 as complex pairs times magnitude * e^(i angle)."""
    rot = case["rot"]
    f = []
    for i in range(rot // 2):
        if case["scaling"] == "base":
            v = (BASE * case["factor"] ** (rot / (rot - 2.0))) ** (-2.0 * i / rot)
        else:
            v = BASE ** (-2.0 * i / rot)
        if case["scaling"] == "linear":
            v /= case["factor"]
        elif case["scaling"] == "parts":
            turns = case["original"] * v / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - 1.0) / 31.0))
            v = keep * v + (1.0 - keep) * v / case["factor"]
        f.append(v)
    angle = torch.outer(pos.double(), torch.tensor(f, dtype=torch.float64, device=x.device))
    turn = torch.polar(torch.full_like(angle, case["magnitude"]), angle)[:, None]
    head = x[..., :rot]
    if case["layout"] == "half":
        z = turn * torch.complex(head[..., :rot // 2], head[..., rot // 2:])
        head = torch.cat((z.real, z.imag), -1)
    else:
        z = turn * torch.view_as_complex(head.reshape(*head.shape[:-1], rot // 2, 2).contiguous())
        head = torch.view_as_real(z).flatten(-2)
    return torch.cat((head, x[..., rot:]), -1)


def _exact_append(s):
    case, lens, table = s["case"], s["lens"].tolist(), s["table"].cpu()
    edges = s["start"].tolist() if "start" in s else list(range(len(lens) + 1))
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    if case["norm"]:
        q, k = (x / (x.square().sum(-1, keepdim=True) / case["hd"] + EPS).sqrt() * s[g].double()
                for x, g in ((q, "q_norm"), (k, "k_norm")))
    kp, vp, qr = s["k_pages"].double(), s["v_pages"].double(), s["q_rot"].double()
    for b, n in enumerate(lens):
        a, z = edges[b], edges[b + 1]
        if n == 0:
            continue
        at = torch.arange(n - (z - a), n)
        page, row = table[b][at // case["page"]].long().cuda(), (at % case["page"]).cuda()
        pos = at.cuda()
        kp[page, row] = _exact_turn(case, k[a:z], pos)
        vp[page, row] = v[a:z]
        qr[a:z] = _exact_turn(case, q[a:z], pos)
    return kp, vp, qr


def _exact_attend(s, q, k_pages, v_pages):
    case, lens, table = s["case"], s["lens"].tolist(), s["table"].long()
    group, page = case["heads"] // case["kv"], case["page"]
    out = torch.zeros(case["seqs"], case["heads"], case["hd"], dtype=torch.float64, device="cuda")
    lse = torch.full((case["seqs"], case["heads"]), -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        if n == 0:
            continue
        first = max(0, n - case["window"]) if case["window"] else 0
        pages = table[b, first // page:(n + page - 1) // page]
        skip = first - first // page * page
        k, v = (x[pages].flatten(0, 1)[skip:skip + n - first].double() for x in (k_pages, v_pages))
        for g in range(case["kv"]):
            h = slice(g * group, (g + 1) * group)
            z = q[b, h].double() @ k[:, g].T / math.sqrt(case["hd"])
            lse[b, h] = torch.logsumexp(z, -1)
            out[b, h] = torch.exp(z - lse[b, h, None]) @ v[:, g]
    return out, lse


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rope":
        return _exact_turn(case, s["x"].double(), s["pos"])
    if case["kind"] == "attend":
        return _exact_attend(s, s["q"], s["k_pages"], s["v_pages"])
    done = _exact_append(s)
    if case["kind"] == "append":
        return done
    # the attention reads what the cache and the rotated queries hold: values in their own types
    k, v, q = (x.to(t.dtype) for x, t in zip(done, (s["k_pages"], s["v_pages"], s["q_rot"])))
    return (*done, *_exact_attend(s, q, k, v))
