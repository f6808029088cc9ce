"""More operators of the paged cache: several new tokens per conversation attending over its pages
(prompts, chunks of prompts, drafts to verify) with capped scores, a bias by distance, a window and a
prefix that every token sees; one new token with the same scores; and a cache held in 4 bits, appended
to, read back and attended over.

`run` is the operators' plain form (elementary torch operations in float32, block steps and divisions
in float64), or with `own` set the library's entry points on the same inputs. `exact` states the definitions
again in float64. Head shapes are the decoder's own (32 query and 8 kv heads of 64) and generic ones.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _attend(name, seqs, tokens, before, heads, kv, hd, dtype, cache, page=16, cap=0.0, slopes=False, window=0,
            prefix=0, even=True):
    return {"name": name, "kind": "attend", "seqs": seqs, "tokens": tokens, "before": before, "even": even,
            "heads": heads, "kv": kv, "hd": hd, "dtype": dtype, "cache": cache, "page": page, "cap": cap,
            "slopes": slopes, "window": window, "prefix": prefix}


def listed():
    return [
        # the first words of a conversation: nothing but latency
        _attend("prompt_17", 1, 17, 0, 32, 8, 64, "f32", "f32"),
        # a chunk of 512 tokens, as the decoder takes a prompt, in the middle of it, all in f32
        _attend("prompt_512_after_1536", 1, 512, 1536, 32, 8, 64, "f32", "f32"),
        # several prompts of different lengths in one ragged batch, some behind a cached beginning; the first 200
        # positions of each are seen by every token (a description that is read in both directions)
        _attend("prompts_5003_prefix", 7, 5003, 2000, 32, 8, 128, "bf16", "bf16", 32, prefix=200, even=False),
        # the largest: a long document from its beginning
        _attend("prompt_16384", 1, 16384, 0, 32, 8, 128, "bf16", "bf16"),
        # layers with capped scores and a sliding window, wide heads
        _attend("prompts_capped_window", 2, 6001, 0, 16, 8, 256, "f16", "f16", 64, cap=50.0, window=1024, even=False),
        # five drafted tokens of each conversation verified at once over its long cache
        _attend("verify_16x5", 16, 80, 8192, 32, 8, 128, "bf16", "bf16"),
        # the next token of conversations of very different lengths, two places of the batch empty, capped scores
        _attend("next_34_capped", 34, 0, 16384, 32, 8, 64, "bf16", "bf16", cap=30.0, even=False),
        # the next token of one long conversation with a bias by distance, f32 activations on a bf16 cache
        _attend("next_1_slopes", 1, 0, 9001, 32, 8, 64, "f32", "bf16", slopes=True),
        # a decode batch's next keys and values into a 4-bit cache, and back as the values that it holds
        {"name": "append4_batch_48", "kind": "append", "seqs": 48, "tokens": 0, "before": 8192, "kv": 8, "hd": 64,
         "dtype": "f32", "page": 16},
        # several prompts absorbed into a 4-bit cache
        {"name": "append4_prompts_5003", "kind": "append", "seqs": 7, "tokens": 5003, "before": 4096, "kv": 8,
         "hd": 128, "dtype": "bf16", "page": 32},
        # a full server batch of long conversations on a 4-bit cache
        _attend("next4_64_8192", 64, 0, 8192, 32, 8, 128, "f16", "4"),
        # chunks of four prompts behind long beginnings, on a 4-bit cache
        _attend("prompts4_2048", 4, 2048, 8192, 32, 8, 128, "bf16", "4"),
    ]


LARGEST = 32 * 128 * 16384 * 16384 // 2   # products of queries and keys in the largest listed case
MOST_CACHE = 64 * 8192 * 8 * 128          # cached key values of the longest caches


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    kind = rng.choice(["append", "append", "next", "next", "prompt", "prompt", "prompt"])
    dtype = rng.choice(list(TYPES))
    page = rng.choice([1, 8, 16, 16, 16, 24, 32, 64, 128, 256])
    kv, group = rng.choice([(8, 4), (8, 4), (4, 8), (2, 5), (16, 1), (1, 16), (1, 24)])
    cache = rng.choice([dtype, dtype, "4", "4", rng.choice(list(TYPES))])
    hd = rng.choice([64, 64, 128, 128, 32, 96, 256] if kind == "append" or cache == "4"
                    else [64, 64, 128, 128, 32, 80, 96, 256])
    if kind == "append":
        seqs = _log(rng, 1, 256)
        return {"kind": "append", "seqs": seqs, "tokens": rng.choice([0, seqs + _log(rng, 1, 4096)]),
                "before": _log(rng, 64, min(32768, max(64, (1 << 28) // (seqs * kv * hd)))), "kv": kv, "hd": hd,
                "dtype": dtype, "page": page}
    most = MOST_CACHE // (4 * kv * hd)
    scores = {"cap": rng.choice([0.0, 0.0, 20.0, 30.0, 50.0]), "slopes": rng.random() < 0.3,
              "window": rng.choice([0, 0, 0, _log(rng, 1, 4096)]), "even": rng.random() < 0.4}
    if kind == "next":
        seqs = _log(rng, 1, min(256, most))
        return {**_attend("", seqs, 0, _log(rng, 1, min(65536, most // seqs)), kv * group, kv, hd, dtype, cache, page,
                          prefix=rng.choice([0, 0, 4]) if scores["window"] else 0), **scores}
    seqs = _log(rng, 1, 64)
    tokens = seqs * _log(rng, 1, 12) if rng.random() < 0.3 else seqs + _log(rng, 1, 8192)
    before = _log(rng, 1, min(16384, max(1, most // seqs)))
    # (no dearer than the largest listed case, the padded batch of the plain form included)
    cost = kv * group * hd * 4 * tokens
    before = max(0, min(before, LARGEST // cost - 4 * tokens))
    return {**_attend("", seqs, tokens, before, kv * group, kv, hd, dtype, cache, page,
                      prefix=rng.choice([0, 0, _log(rng, 1, 1000)])), **scores}


# ---- inputs ------------------------------------------------------------------------------------
def _gen(seed, stream, device="cuda"):
    g = torch.Generator(device=device)
    g.manual_seed((1_000_003 * int(seed) + 7919 * stream + 29) % (1 << 62))
    return g


def _normal(seed, stream, shape, dtype, spread=1.0):
    x = torch.randn(shape, generator=_gen(seed, stream), device="cuda", dtype=torch.float32)
    return (spread * x).to(TYPES[dtype])


def _pages(seed, lens, page, spare=3):
    """(page table with -1 past each sequence's pages, pages of the pool): a sequence's pages lie
    anywhere in the pool, as they do after many conversations came and went."""
    need = torch.tensor([(n + page - 1) // page for n in lens])
    total, wide = int(need.sum()), max(1, int(need.max()))
    order = torch.randperm(total + spare, generator=_gen(seed, 11, "cpu")).to(torch.int32)
    table = torch.full((len(lens), wide), -1, dtype=torch.int32)
    table[torch.arange(wide)[None] < need[:, None]] = order[:total]
    return table.cuda(), total + spare


def _batch(case):
    """(positions cached before, new tokens) of each sequence: the same for every seed (a pool keeps its size),
    which says only which sequence has which. Tokens 0: each sequence's next one, two places of a larger ragged
    batch empty."""
    n, t, far = case["seqs"], case["tokens"], case["before"]
    u = torch.rand(n, generator=_gen(0, 12, "cpu")).tolist()
    spread = [max(1, round(math.exp(x * math.log(far)))) if far > 0 else 0 for x in u]
    if t == 0:
        lens = [far] * n if case.get("even", False) else [far] + spread[1:]
        if n >= 8 and not case.get("even", True):
            lens[n // 2] = lens[n - 1] = 0
        return [(m - 1, 1) if m else (0, 0) for m in lens]
    if case.get("even", False):
        return [(far, t // n + (1 if i < t % n else 0)) for i in range(n)]
    cuts = torch.sort(torch.randperm(t - 1, generator=_gen(0, 13, "cpu"))[:n - 1])[0] + 1 if n > 1 else []
    edges = [0] + [int(c) for c in cuts] + [t]
    return [(0 if i % 2 else m, hi - lo) for i, (m, lo, hi) in enumerate(zip(spread, edges, edges[1:]))]


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


def prepare(case, seed):
    if own:
        _Program.context()   # (the inputs are made on its stream)
    hd, kv, page, dtype = case["hd"], case["kv"], case["page"], case["dtype"]
    come = _batch(case)
    come = [come[i] for i in torch.randperm(len(come), generator=_gen(seed, 16, "cpu")).tolist()]
    lens, new = [a + b for a, b in come], [b for _, b in come]
    # (an empty place of a decode batch has a row all the same)
    rows = new if case["tokens"] else [1] * len(new)
    tokens = sum(rows)
    s = {"case": case, "tokens": tokens, "most": max(rows)}
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["table"], n_pages = _pages(seed, lens, page)
    edges = torch.cumsum(torch.tensor([0] + rows), 0).to(torch.int32)
    s["start"] = edges.cuda()
    if case["kind"] == "append":
        s["k"], s["v"] = (_normal(seed, i, (tokens, kv, hd), dtype) for i in (5, 6))
        shape = (n_pages, kv, _chunk(page, hd))
        s["k_pages"], s["v_pages"] = (torch.zeros(shape, dtype=torch.uint8, device="cuda") for _ in range(2))
        s["k_back"], s["v_back"] = (torch.empty(tokens, kv, hd, device="cuda") for _ in range(2))
    else:
        # standard normal keys and values, as after their norms
        for name, i in (("k_pages", 2), ("v_pages", 3)):
            if case["cache"] == "4":
                s[name] = torch.empty(n_pages, kv, _chunk(page, hd), dtype=torch.uint8, device="cuda")
                g, some = _gen(seed, i), max(1, (1 << 26) // (kv * page * hd))
                for a in range(0, n_pages, some):
                    part = s[name][a:a + some]
                    _fill(part, torch.randn(len(part), kv, page, hd, generator=g, device="cuda"))
            else:
                s[name] = torch.empty(n_pages, page, kv, hd, device="cuda",
                                      dtype=TYPES[case["cache"]]).normal_(generator=_gen(seed, i))
        # queries a little wider than keys: some positions stand out, most count
        s["q"] = _normal(seed, 4, (tokens, case["heads"], hd), dtype, 1.5)
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(tokens, case["heads"], device="cuda")
        if case["slopes"]:
            # steep for the first head, flat for the last
            h = torch.arange(1, case["heads"] + 1, device="cuda", dtype=torch.float32)
            s["slopes"] = torch.exp2(-8.0 * h / case["heads"])
        if case["prefix"]:
            s["prefix"] = torch.full((len(lens),), case["prefix"], dtype=torch.int32, device="cuda")
    if own:
        from bebelm_amd.model import PagedKv
        four = case["kind"] == "append" or case["cache"] == "4"
        s["handle"] = (PagedKv.four_bit(_Program.context(), s["k_pages"], s["v_pages"], page, hd) if four
                       else PagedKv(_Program.context(), s["k_pages"], s["v_pages"]))
    return s


# ---- a cache in 4 bits ----------------------------------------------------------------------------
# Blocks of 32 elements of a head: 16 bytes of codes (element 2i in the low half of byte i) and a 16-bit head: its
# step d, an f16 number of 5 significant bits (bits 6 to 14), and its offset z in 7 bits (bits 0 to 5, and bit 15 for
# -64). An element stands for d·(code + z). d is the smallest step with 15d >= max - min, 63d >= max and 47d >= -min
# (values past ±16384 are taken as that, a block with one that is not finite is NaN), z = round(min / d), codes
# round(x / d) - z in 0..15. A page's head is its positions' codes, then their heads of blocks (an even number of
# them), in a multiple of 16 bytes.
def _heads_of(hd):
    return (hd // 32 + 1) // 2 * 2


def _chunk(page, hd):
    return (page * (hd // 2 + 2 * _heads_of(hd)) + 15) // 16 * 16


def _quantised(x):
    """(codes uint8 [..., hd / 2], heads int16 [..., blocks]) of x [..., hd]."""
    x = x.float()
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    odd = ~torch.isfinite(b).all(-1, keepdim=True)
    b = torch.where(odd, torch.zeros_like(b), b.clamp(-16384.0, 16384.0)).double()
    lo, hi = b.amin(-1, keepdim=True), b.amax(-1, keepdim=True)
    need = torch.maximum((hi - lo) / 15.0, torch.maximum(hi / 63.0, -lo / 47.0))
    unit = torch.exp2(torch.clamp(torch.frexp(need)[1].double() - 5.0, min=-18.0))
    d = torch.ceil(need / unit) * unit
    by = torch.where(d > 0, d, torch.ones_like(d))
    z = torch.round(lo / by)
    code = (torch.round(b / by) - z).clamp(0.0, 15.0).to(torch.uint8)
    z = z.to(torch.int32)
    head = d.to(torch.float16).view(torch.int16).to(torch.int32) | (z & 63) | ((z < 0).to(torch.int32) << 15)
    head = torch.where(odd, torch.full_like(head, 0x7fc0), head)
    code = torch.where(odd, torch.zeros_like(code), code)
    return (code[..., 0::2] | (code[..., 1::2] << 4)).flatten(-2), head.squeeze(-1).to(torch.int16)


def _values(codes, heads):
    """float32 values [..., hd] of codes [..., hd / 2] and heads [..., blocks]."""
    h = heads.to(torch.int32)
    d = (h & 0x7fc0).to(torch.int16).view(torch.float16).float()
    z = ((h & 63) - ((h >> 15) & 1) * 64).float()
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    c = c.reshape(*c.shape[:-1], heads.shape[-1], 32).float()
    return ((c + z[..., None]) * d[..., None]).flatten(-2)


def _parts(pages, page, hd):
    """Views of a pool of 4-bit pages: codes [pages, kv, page, hd / 2] and heads int16 [pages, kv, page, blocks]."""
    n, kv, _ = pages.shape
    codes = pages[:, :, :page * hd // 2].unflatten(-1, (page, hd // 2))
    at = page * hd // 2
    heads = pages[:, :, at:at + page * 2 * _heads_of(hd)].view(torch.int16).unflatten(-1, (page, _heads_of(hd)))
    return codes, heads[..., :hd // 32]


def _fill(pages, x):
    """x [pages, kv, page, hd] as the whole contents of `pages`."""
    pages.zero_()
    codes, heads = _parts(pages, x.shape[2], x.shape[3])
    c, h = _quantised(x)
    codes.copy_(c)
    heads.copy_(h)


def _cached(s, name, table):
    """float32 [sequences, kv, positions, hd] of the pages of a table's rows."""
    case = s["case"]
    pages, at = s[name], table.clamp(min=0).long()
    if case["kind"] == "append" or case["cache"] == "4":
        codes, heads = _parts(pages, case["page"], case["hd"])
        x = _values(codes[at], heads[at])            # [sequences, pages, kv, page, hd]
        return x.transpose(1, 2).flatten(2, 3)
    return pages[at].flatten(1, 2).transpose(1, 2).float()


# ---- plain forms -------------------------------------------------------------------------------
def _append(s):
    case, page, lens, start = s["case"], s["case"]["page"], s["lens"].long(), s["start"].long()
    t = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(start, t, right=True) - 1
    index = lens[seq] - start[seq + 1] + t
    there = index >= 0   # (an empty place of a batch: nothing is written, zeros are read)
    at = index.clamp(min=0)
    where, row = s["table"][seq, at // page].long().clamp(min=0), at % page
    for pages, x, back in ((s["k_pages"], s["k"], s["k_back"]), (s["v_pages"], s["v"], s["v_back"])):
        codes, heads = _parts(pages, page, case["hd"])
        c, h = _quantised(x)
        codes[where, :, row] = torch.where(there[:, None, None], c, codes[where, :, row])
        heads[where, :, row] = torch.where(there[:, None, None], h, heads[where, :, row])
        back.copy_(torch.where(there[:, None, None], _values(codes[where, :, row], heads[where, :, row]), 0.0))
    return s["k_back"], s["v_back"]


def _attended(s):
    case, lens, start = s["case"], s["lens"].long(), s["start"].long()
    kv, group, hd, page = case["kv"], case["heads"] // case["kv"], case["hd"], case["page"]
    out, lse, most, table = s["out"], s["lse"], s["most"], s["table"]
    n = table.shape[1] * page
    some = max(1, (1 << 28) // (n * kv * hd))                       # sequences at a time: about a gigabyte of keys
    some = min(some, case["seqs"])
    rows = max(1, min(most, (1 << 28) // (some * n * case["heads"])))   # new tokens of each at a time
    j = torch.arange(n, device="cuda")
    for a in range(0, case["seqs"], some):
        ln, first, last = lens[a:a + some], start[:-1][a:a + some], start[1:][a:a + some]
        k = _cached(s, "k_pages", table[a:a + some]).transpose(2, 3).contiguous()
        v = _cached(s, "v_pages", table[a:a + some]).contiguous()
        for b in range(0, most, rows):
            m = torch.arange(b, min(b + rows, most), device="cuda")
            token = first[:, None] + m                              # [sequences, rows]
            real = token < last[:, None]
            q = s["q"][torch.where(real, token, 0)].float()         # [sequences, rows, heads, hd]
            q = q.unflatten(2, (kv, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)
            x = (torch.matmul(q, k) * (1.0 / math.sqrt(hd))).unflatten(2, (len(m), group))
            if case["cap"]:
                x = case["cap"] * torch.tanh(x / case["cap"])
            index = ln[:, None] - last[:, None] + token             # the tokens' own positions
            away = index[:, :, None] - j                            # [sequences, rows, positions]
            if case["slopes"]:
                x = x - s["slopes"].view(1, kv, 1, group, 1) * away.abs()[:, None, :, None].float()
            seen = away >= 0
            if case["window"]:
                seen = seen & (away < case["window"])
            if case["prefix"]:
                seen = seen | (j < s["prefix"].long()[a:a + some, None, None])
            seen = seen & (j < ln[:, None, None])
            x = x.masked_fill(~seen[:, None, :, None], -math.inf).flatten(2, 3)
            top = x.amax(-1, keepdim=True)
            top = torch.where(top == -math.inf, torch.zeros_like(top), top)
            p = torch.exp(x - top)
            total = p.sum(-1, keepdim=True)
            o = torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)
            o = o.unflatten(2, (len(m), group)).permute(0, 2, 1, 3, 4).flatten(2, 3)
            z = (torch.log(total) + top).unflatten(2, (len(m), group)).permute(0, 2, 1, 3, 4).flatten(2)
            out[token[real]] = o[real].to(out.dtype)
            lse[token[real]] = z[real]
    return out, lse   # a row that sees nothing: zeros, and the logarithm of nothing, -inf


def _own_append(s):
    from bebelm_amd import kernels
    start = s["start"] if s["case"]["tokens"] else None
    kernels.paged_append(_Program.ctx, s["handle"], s["table"], s["lens"], s["k"], s["v"], seq_start=start)
    kernels.paged_read(_Program.ctx, s["handle"], s["table"], s["lens"], s["k_back"], s["v_back"], seq_start=start)
    return s["k_back"], s["v_back"]


def _own_attended(s):
    from bebelm_amd import kernels
    case = s["case"]
    start = s["start"] if case["tokens"] else None
    kernels.paged_prompt_attention(_Program.ctx, s["handle"], s["table"], s["lens"], s["q"], s["out"], seq_start=start,
                                   window=case["window"], cap=case["cap"], slopes=s.get("slopes"),
                                   prefix=s.get("prefix"), lse=s["lse"])
    return s["out"], s["lse"]


def run(state):
    if state["case"]["kind"] == "append":
        return _own_append(state) if own else _append(state)
    return _own_attended(state) if own else _attended(state)


# ---- what a pass cannot do without ---------------------------------------------------------------
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _row_bytes(case):
    """Bytes of a position's keys (or values) of all heads."""
    if case["kind"] == "append" or case["cache"] == "4":
        return case["kv"] * (case["hd"] // 2 + 2 * (case["hd"] // 32))
    return case["kv"] * case["hd"] * _SIZE[case["cache"]]


def work(case):
    e, hd, kv = _SIZE[case["dtype"]], case["hd"], case["kv"]
    come = _batch(case)
    if case["kind"] == "append":
        t = sum(n for _, n in come)
        # written, read back, and its values as f32
        return {"bytes": t * 2 * (kv * hd * (e + 4) + 2 * _row_bytes(case)) + 8 * t, "flops": 8 * t * kv * hd}
    heads, window = case["heads"], case["window"]
    nbytes = flops = 0
    for before, n in come:
        length = before + n
        prefix = min(case["prefix"], length)
        first = max(0, before - window + 1) if window else 0      # what the first new token sees begins here
        nbytes += 2 * _row_bytes(case) * (length - first + min(prefix, first)) + 4 * length / case["page"]
        index = torch.arange(before, length, dtype=torch.int64)
        low = (index - window + 1).clamp(min=0) if window else torch.zeros_like(index)
        seen = index + 1 - low + torch.minimum(low, torch.full_like(low, prefix))
        seen = seen + (prefix - 1 - index).clamp(min=0)
        flops += 4 * heads * hd * int(seen.sum())
    t = case["tokens"] or case["seqs"]
    return {"bytes": nbytes + t * heads * (2 * hd * e + 4), "flops": flops}


# ---- the definitions in 64 bits -------------------------------------------------------------------
def _exact_blocks(x):
    """float64 values that a 4-bit cache holds for x [tokens, kv, hd]."""
    b = x.double().unflatten(-1, (-1, 32))
    fine = b.abs() < math.inf
    b = torch.clip(torch.where(fine, b, 0.0), -(2.0 ** 14), 2.0 ** 14)
    lo, hi = b.min(-1, keepdim=True).values, b.max(-1, keepdim=True).values
    # the steps there are, in order: multiples of 2^-18 up to 2^-13, then 16 to a power of two
    steps = [i * 2.0 ** -18 for i in range(32)]
    steps += [(16 + i) * 2.0 ** (e - 4) for e in range(-13, 16) for i in range(16)]
    steps = torch.tensor(steps, dtype=torch.float64, device=x.device)
    at = torch.maximum(torch.searchsorted(15.0 * steps, (hi - lo).contiguous()),
                       torch.searchsorted(63.0 * steps, hi.contiguous()))
    d = steps[torch.maximum(at, torch.searchsorted(47.0 * steps, (-lo).contiguous()))]

    def nearest(y):   # ties to even
        q = y / torch.where(d == 0, 1.0, d)
        low = torch.floor(q)
        part = q - low
        up = (part > 0.5) | ((part == 0.5) & (torch.remainder(low, 2.0) == 1.0))
        return low + up

    z = nearest(lo)
    value = d * torch.clip(nearest(b), z, z + 15.0)
    return torch.where(fine.all(-1, keepdim=True), value, math.nan).flatten(-2)


def _exact_rows(s, name, b, a, z):
    """float64 [positions a..z, kv, hd] of sequence b."""
    case, page = s["case"], s["case"]["page"]
    at = torch.arange(a, z, device="cuda")
    where, row = s["table"][b].long()[at // page], at % page
    if case["cache"] != "4":
        return s[name][where, row].double()
    raw = s[name][where]                                         # [positions, kv, bytes]
    hd, kv = case["hd"], case["kv"]
    i = torch.arange(hd, device="cuda")
    byte = raw.gather(2, (row[:, None] * (hd // 2) + i // 2)[:, None].expand(-1, kv, -1)).long()
    code = torch.where(i % 2 == 1, byte // 16, byte % 16)
    place = page * (hd // 2) + 2 * (row[:, None] * _heads_of(hd) + i // 32)
    low = raw.gather(2, place[:, None].expand(-1, kv, -1)).long()
    high = raw.gather(2, (place + 1)[:, None].expand(-1, kv, -1)).long()
    exponent, mantissa = (high // 4) % 32, (high % 4) * 4 + low // 64
    d = torch.where(exponent == 0, mantissa * 2.0 ** -18, (16.0 + mantissa) * torch.exp2(exponent.double() - 19.0))
    offset = low % 64 - torch.where(high >= 128, 64, 0)
    return d * (code + offset).double()


def _exact_attended(s):
    case, lens, start = s["case"], s["lens"].tolist(), s["start"].tolist()
    group, hd = case["heads"] // case["kv"], case["hd"]
    out = torch.zeros(s["tokens"], case["heads"], hd, dtype=torch.float64, device="cuda")
    lse = torch.full((s["tokens"], case["heads"]), -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        t0, t1 = start[b], start[b + 1]
        if n == 0 or t0 == t1:
            continue
        base = n - (t1 - t0)
        for a in range(t0, t1, 2048):
            z = min(a + 2048, t1)
            i = torch.arange(a - t0 + base, z - t0 + base, device="cuda", dtype=torch.float64)[:, None]
            # (no key past the last of these tokens and the prefix, none before what the window and the prefix leave)
            end = min(n, max(base + z - t0, case["prefix"]))
            begin = max(0, base + a - t0 + 1 - case["window"]) if case["window"] and not case["prefix"] else 0
            j = torch.arange(begin, end, device="cuda", dtype=torch.float64)[None]
            far = torch.abs(i - j)
            hidden = j > i
            if case["window"]:
                hidden = hidden | (i - j >= case["window"])
            if case["prefix"]:
                hidden = hidden & (j >= case["prefix"])
            k, v = (_exact_rows(s, x, b, begin, end) for x in ("k_pages", "v_pages"))
            for h in range(case["heads"]):
                x = s["q"][a:z, h].double() @ k[:, h // group].T.contiguous() / math.sqrt(hd)
                if case["cap"]:
                    x = case["cap"] * torch.tanh(x / case["cap"])
                if case["slopes"]:
                    x = x - s["slopes"][h].double() * far
                x = torch.where(hidden, -math.inf, x)
                sums = torch.logsumexp(x, -1)
                lse[a:z, h] = sums
                w = torch.exp(x - torch.where(sums == -math.inf, 0.0, sums)[:, None])
                out[a:z, h] = w @ v[:, h // group].contiguous()
    return out, lse


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] != "append":
        return _exact_attended(s)
    lens, start = s["lens"].tolist(), s["start"].tolist()
    there = torch.tensor([lens[b] > 0 for b in range(case["seqs"]) for _ in range(start[b], start[b + 1])],
                         device="cuda")
    return tuple(torch.where(there[:, None, None], _exact_blocks(s[x]), 0.0) for x in ("k", "v"))
