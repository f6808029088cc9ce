"""Kernel-level mirror of the reference's src/kernels API over the C ABI.

  quantize_q8(x) -> Q8Vec                  kernels/matmul.rs:141
  matvec(dtype, w, n_in, n_out, x, y)      kernels/matmul.rs:850
  matmul(dtype, w, n_in, n_out, x, t, y)   kernels/matmul.rs:908
  FusedJob / matvec_fused_batch            kernels/matmul.rs:995-1053
  swiglu / sigmoid_slice                   kernels/activation.rs:16, :25
  add_scaled / add_assign                  kernels/elementwise.rs:12, :4
  rmsnorm                                  kernels/rmsnorm.rs:10
  logits_from_hidden                       model.rs:380-388
  conv_step / conv_prefill                 kernels/conv.rs:18, :48
  softmax                                  kernels/softmax.rs:9
  attention_decode                         kernels/attention.rs:17
  rope_neox                                kernels/rope.rs:17
The paged-cache operators have no counterpart there:
  rope                                     rotary positions of any layout and frequency rule
  paged_append / paged_attention           a batch of conversations on one pool of cache pages
  paged_prompt_attention / paged_read      several tokens of each attending over it, what it holds
Each function takes the Context first; `w` is an uploaded Tensor (plus a byte offset where the
reference passes a sub-slice of the weight bytes).
"""
import ctypes
from dataclasses import dataclass

import numpy as np

from . import _lib
from ._lib import check, lib
from .model import F32, INT32, _codes, _dtype, _ptr, _same_loc


@dataclass
class Q8Vec:
    q: object       # int8 [n]
    scales: object  # f32 [n/256]
    sums: object    # i32 [n/32]


def quantize_q8(ctx, x, out=None):
    n = x.shape[-1] if hasattr(x, "shape") else len(x)
    if out is None:
        out = Q8Vec(np.empty(n, np.int8), np.empty(n // 256, np.float32), np.empty(n // 32, np.int32))
    loc = _same_loc(x, out.q, out.scales, out.sums)
    check(lib().bb_quantize_q8(ctx.handle, _ptr(x)[0], n, _ptr(out.q)[0], _ptr(out.scales)[0], _ptr(out.sums)[0], loc))
    return out


def matvec(ctx, dtype, w, n_in, n_out, x, y, byte_off=0):
    loc = _same_loc(x, y)
    check(lib().bb_matvec(ctx.handle, dtype, w.handle, byte_off, n_in, n_out, _ptr(x)[0], _ptr(y)[0], loc))
    return y


def matmul(ctx, dtype, w, n_in, n_out, x, n_tokens, y, byte_off=0):
    loc = _same_loc(x, y)
    check(lib().bb_matmul(ctx.handle, dtype, w.handle, byte_off, n_in, n_out, _ptr(x)[0], n_tokens, _ptr(y)[0], loc))
    return y


@dataclass
class FusedJob:
    """FusedJob (matmul.rs:995-1005): qx (Q8Vec) for the integer dot, or qx None and x (f32) for
    the f32 fused dot."""
    dtype: int
    w: object
    n_in: int
    n_out: int
    qx: object = None
    byte_off: int = 0
    x: object = None


def matvec_fused_batch(ctx, jobs, out):
    arr = (_lib.FusedJob * len(jobs))()
    arrays = [out]
    for i, j in enumerate(jobs):
        if j.qx is not None:
            arr[i] = _lib.FusedJob(j.dtype, j.w.handle, j.byte_off, j.n_in, j.n_out, _ptr(j.qx.q)[0],
                                   _ptr(j.qx.scales)[0], _ptr(j.qx.sums)[0], None)
            arrays += [j.qx.q, j.qx.scales, j.qx.sums]
        else:
            arr[i] = _lib.FusedJob(j.dtype, j.w.handle, j.byte_off, j.n_in, j.n_out, None, None, None, _ptr(j.x)[0])
            arrays += [j.x]
    loc = _same_loc(*arrays)
    check(lib().bb_matvec_fused_batch(ctx.handle, arr, len(jobs), _ptr(out)[0], loc))
    return out


def swiglu(ctx, gate, up, out):
    check(lib().bb_swiglu(ctx.handle, _ptr(gate)[0], _ptr(up)[0], _ptr(out)[0], _n(out), _same_loc(gate, up, out)))
    return out


def sigmoid_slice(ctx, x):
    check(lib().bb_sigmoid_slice(ctx.handle, _ptr(x)[0], _n(x), _same_loc(x)))
    return x


def add_scaled(ctx, out, b, s):
    check(lib().bb_add_scaled(ctx.handle, _ptr(out)[0], _ptr(b)[0], ctypes.c_float(s), _n(out), _same_loc(out, b)))
    return out


def add_assign(ctx, a, b):
    check(lib().bb_add_assign(ctx.handle, _ptr(a)[0], _ptr(b)[0], _n(a), _same_loc(a, b)))
    return a


def rmsnorm(ctx, x, gain, eps, out, n_vec=1):
    n = _n(gain)
    check(lib().bb_rmsnorm(ctx.handle, _ptr(x)[0], _ptr(gain)[0], ctypes.c_float(eps), n, n_vec, _ptr(out)[0],
                           _same_loc(x, gain, out)))
    return out


def logits_from_hidden(ctx, tok_embd, gain, eps, h, logits):
    """Model::logits_from_hidden (model.rs:380-388): rmsnorm, then the token_embd matvec."""
    loc = _same_loc(h, gain, logits)
    check(lib().bb_logits_from_hidden(ctx.handle, tok_embd.handle, _ptr(gain)[0], eps, _ptr(h)[0], _ptr(logits)[0], loc))
    return logits


def conv_step(ctx, state, bx, weight, channels, l_cache, out):
    """conv.rs:18-39: out[c] = w[c, L-1]·bx[c] + Σ_k w[c, k]·state[k, c]."""
    loc = _same_loc(state, bx, weight, out)
    check(lib().bb_conv_step(ctx.handle, _ptr(state)[0], _ptr(bx)[0], _ptr(weight)[0], channels, l_cache, _ptr(out)[0],
                             loc))
    return out


def conv_prefill(ctx, state, bx, weight, channels, l_cache, n_tokens, out):
    """conv.rs:48-68 over n_tokens positions; state is updated in place."""
    loc = _same_loc(state, bx, weight, out)
    check(lib().bb_conv_prefill(ctx.handle, _ptr(state)[0], _ptr(bx)[0], _ptr(weight)[0], channels, l_cache, n_tokens,
                                _ptr(out)[0], loc))
    return out


def softmax(ctx, x, n_vec=1):
    """softmax.rs:9-22 on each of n_vec rows, in place."""
    n = _n(x) // n_vec
    check(lib().bb_softmax(ctx.handle, _ptr(x)[0], n, n_vec, _same_loc(x)))
    return x


def attention_decode(ctx, q, k, v, n_ctx, n_heads, n_kv_heads, head_dim, out):
    """attention.rs:17-55."""
    loc = _same_loc(q, k, v, out)
    check(lib().bb_attention_decode(ctx.handle, _ptr(q)[0], _ptr(k)[0], _ptr(v)[0], n_ctx, n_heads, n_kv_heads,
                                    head_dim, _ptr(out)[0], loc))
    return out


def rope_neox(ctx, x, head_dim, pos, freq_base):
    """rope.rs:17-30 on each head vector of x, in place."""
    check(lib().bb_rope_neox(ctx.handle, _ptr(x)[0], head_dim, _n(x) // head_dim, pos, ctypes.c_float(freq_base),
                             _same_loc(x)))
    return x


# ---- arrays of the paged-cache operators (checked with few calls each: a step makes these for every
# layer, and a decode step's kernels take a few microseconds)
def _place(ctx, *arrays):
    """Where the arrays are: all in host memory, or all on the context's GPU."""
    where = None
    for a in arrays:
        if a is not None:
            d = -1 if isinstance(a, np.ndarray) else a.get_device()
            if d != where:
                if where is not None:
                    raise ValueError("all arrays of one call must be host or all device")
                where = d
    if where < 0:
        return _lib.LOC_HOST
    if where != ctx.device:
        raise ValueError(f"tensors on GPU {where}, context on GPU {ctx.device}")
    return _lib.LOC_DEVICE


def _data(a):
    return a.ctypes.data if isinstance(a, np.ndarray) else a.data_ptr()


def _whole(a):
    return a.flags["C_CONTIGUOUS"] if isinstance(a, np.ndarray) else a.is_contiguous()


def _strides(a):
    """In elements."""
    return [i // a.itemsize for i in a.strides] if isinstance(a, np.ndarray) else a.stride()


def _heads(a, what, code, n, heads, hd, packed=True):
    """(address, token stride, head stride) of a [n, heads, head_dim] of the given type, checked."""
    if a.shape != (n, heads, hd):
        raise ValueError(f"{what} must be {[n, heads, hd]}, is {list(a.shape)}")
    if _codes.get(a.dtype) != code and _dtype(a) != code:
        raise ValueError(f"{what}: {a.dtype} is not the type of the other arrays")
    if _whole(a):
        return _data(a), heads * hd, hd
    st = _strides(a)
    if hd > 1 and st[2] != 1:
        raise ValueError(f"{what}: the elements of a head must be adjacent")
    if packed and heads > 1 and st[1] != hd:
        raise ValueError(f"{what}: the heads of a token must be adjacent")
    if min(st) < 0:
        raise ValueError(f"{what}: negative strides")
    return _data(a), (st[0] if n > 1 else heads * hd), (st[1] if heads > 1 else hd)


def _flat(a, what, code, *shape):
    """Address of a contiguous array of the given type and shape (None: 0)."""
    if a is None:
        return 0
    if a.shape != shape or _dtype(a) != code:
        raise ValueError(f"{what} must be {'int32' if code == INT32 else 'float32'} {list(shape)}, is {a.dtype} {list(a.shape)}")
    if not _whole(a):
        raise ValueError(f"{what} must be contiguous")
    return _data(a)


def _floating(a, what):
    code = _dtype(a)
    if code == INT32:
        raise ValueError(f"{what} must be float32, float16 or bfloat16")
    return code


def _seqs(page_table, lens):
    """(sequences, bb_paged_seqs)"""
    if len(page_table.shape) != 2 or _dtype(page_table) != INT32:
        raise ValueError("page_table must be int32 [sequences, pages]")
    n, pages = page_table.shape
    row = pages
    if not _whole(page_table):
        st = _strides(page_table)
        if (pages > 1 and st[1] != 1) or st[0] < 0:
            raise ValueError("page_table: the entries of a sequence must be adjacent")
        row = st[0] if n > 1 else pages
    return n, _lib.PAGED_SEQS.pack(n, pages, row, _data(page_table), _flat(lens, "lens", INT32, n))


def rope(ctx, plan, x, pos, out=None):
    """x [tokens, heads, head_dim] (any token and head strides) turned by pos int32 [tokens] as the
    RopePlan says, into out (x itself by default)."""
    out = x if out is None else out
    t, h, hd = x.shape
    code = _floating(x, "x")
    xa, xt, xh = _heads(x, "x", code, t, h, hd, False)
    oa, ot, oh = _heads(out, "out", code, t, h, hd, False)
    check(lib().bb_rope(ctx.handle, plan.handle, code, xa, xt, xh, t, h, hd, _flat(pos, "pos", INT32, t), oa, ot, oh,
                        _place(ctx, x, pos, out)))
    return out


def paged_append(ctx, kv, page_table, lens, k, v, rope=None, pos=None, seq_start=None, q=None, q_out=None, q_norm=None,
                 k_norm=None, eps=1e-5):
    """Stores k and v [tokens, n_kv_heads, head_dim] at the end of their sequences in the PagedKv's
    pages; on the way k (and q [tokens, n_heads, head_dim], into q_out, q itself by default) is normed
    with k_norm (q_norm) and turned as the RopePlan `rope` says, by pos int32 [tokens] or each token's
    index in its sequence. q, k and v may be slices of one projection's rows. page_table int32 [sequences, pages] and lens int32 [sequences] count the
    call's tokens; seq_start int32 [sequences + 1] says which tokens each sequence brings (None: one
    each). Returns q_out."""
    t, hd, nkv, code = k.shape[0], kv.head_dim, kv.n_kv_heads, _floating(k, "k")
    n, seqs = _seqs(page_table, lens)
    ka, ks, _ = _heads(k, "k", code, t, nkv, hd)
    va, vs, _ = _heads(v, "v", code, t, nkv, hd)
    qa = qs = oa = os = heads = 0
    if q is not None:
        q_out = q if q_out is None else q_out
        heads = q.shape[1]
        qa, qs, _ = _heads(q, "q", code, t, heads, hd)
        oa, os, _ = _heads(q_out, "q_out", code, t, heads, hd)
    elif q_out is not None:
        raise ValueError("q_out without q")
    plan = None
    if rope is not None:
        plan = rope.handle
        if not plan:
            raise ValueError("the RopePlan is closed")
    tokens = _lib.PAGED_TOKENS.pack(t, code, ka, va, ks, vs, qa, oa, heads, qs, os, _flat(q_norm, "q_norm", F32, hd),
                                    _flat(k_norm, "k_norm", F32, hd), eps, _flat(pos, "pos", INT32, t),
                                    _flat(seq_start, "seq_start", INT32, n + 1))
    check(lib().bb_paged_append(ctx.handle, kv.handle, plan, seqs, tokens,
                                _place(ctx, k, v, page_table, lens, pos, seq_start, q, q_out, q_norm, k_norm)))
    return q_out


def paged_attention(ctx, kv, page_table, lens, q, out, scale=None, window=0, lse=None, workspace=None):
    """One query token per sequence, q [sequences, n_heads, head_dim], over the sequence's positions
    in the PagedKv's pages (the last `window` of them; 0: all), into out; lse float32 [sequences,
    n_heads] gets the softmax's log sums. scale None: 1/sqrt(head_dim). workspace: a device tensor of
    kv.attention_workspace(n_heads, sequences) bytes for this call alone (None: the context's; a call
    captured into a graph needs one)."""
    n, seqs = _seqs(page_table, lens)
    heads, hd, code = q.shape[1], kv.head_dim, _floating(q, "q")
    qa, qs, _ = _heads(q, "q", code, n, heads, hd)
    oa, os, _ = _heads(out, "out", code, n, heads, hd)
    if scale is None:
        scale = 0.0
    elif scale == 0:
        raise ValueError("scale must not be 0")
    if window < 0:
        raise ValueError("window must not be negative")
    ws, ws_bytes = _workspace(ctx, workspace)
    query = _lib.PAGED_QUERY.pack(code, qa, oa, heads, qs, os, scale, window, _flat(lse, "lse", F32, n, heads), ws,
                                  ws_bytes)
    check(lib().bb_paged_attention(ctx.handle, kv.handle, seqs, query, _place(ctx, q, out, page_table, lens, lse)))
    return out


def _workspace(ctx, workspace):
    """(address, bytes)"""
    if workspace is None:
        return 0, 0
    if isinstance(workspace, np.ndarray) or workspace.get_device() != ctx.device or not workspace.is_contiguous():
        raise ValueError("the workspace must be a contiguous tensor on the context's GPU")
    return workspace.data_ptr(), workspace.numel() * workspace.element_size()


def paged_prompt_attention(ctx, kv, page_table, lens, q, out, seq_start=None, scale=None, window=0, cap=0.0, slopes=None,
                           prefix=None, lse=None, workspace=None):
    """Several query tokens per sequence, q [tokens, n_heads, head_dim], each over its sequence's positions in the
    PagedKv's pages up to its own (the last `window` of them; 0: all) and those below prefix int32 [sequences], into
    out. seq_start int32 [sequences + 1] says which tokens each sequence has, its last ones (None: one each). Scores
    are capped (cap > 0: cap·tanh(score / cap)) and get -slopes[head]·distance (slopes float32 [n_heads]); lse
    float32 [tokens, n_heads] gets the softmax's log sums. scale None: 1/sqrt(head_dim). workspace: a device
    tensor of kv.prompt_workspace(n_heads, sequences, tokens) bytes for this call alone (None: the context's; a call
    captured into a graph needs one unless that is 0)."""
    n, seqs = _seqs(page_table, lens)
    t, heads, hd, code = q.shape[0], q.shape[1], kv.head_dim, _floating(q, "q")
    qa, qs, _ = _heads(q, "q", code, t, heads, hd)
    oa, os, _ = _heads(out, "out", code, t, heads, hd)
    if scale is None:
        scale = 0.0
    elif scale == 0:
        raise ValueError("scale must not be 0")
    if window < 0:
        raise ValueError("window must not be negative")
    ws, ws_bytes = _workspace(ctx, workspace)
    queries = _lib.PAGED_QUERIES.pack(t, code, qa, oa, heads, qs, os, scale, cap, window,
                                      _flat(slopes, "slopes", F32, heads), _flat(prefix, "prefix", INT32, n),
                                      _flat(seq_start, "seq_start", INT32, n + 1), _flat(lse, "lse", F32, t, heads), ws,
                                      ws_bytes)
    check(lib().bb_paged_prompt_attention(ctx.handle, kv.handle, seqs, queries,
                                          _place(ctx, q, out, page_table, lens, seq_start, slopes, prefix, lse)))
    return out


def paged_read(ctx, kv, page_table, lens, k=None, v=None, seq_start=None):
    """The keys and values that the PagedKv's pages hold at the tokens' positions (those that paged_append with the
    same page_table, lens and seq_start stores to), into k and v [tokens, n_kv_heads, head_dim] (either may be None)."""
    some = k if k is not None else v
    if some is None:
        raise ValueError("neither k nor v to read")
    n, seqs = _seqs(page_table, lens)
    t, hd, nkv, code = some.shape[0], kv.head_dim, kv.n_kv_heads, _floating(some, "k" if k is not None else "v")
    ka, ks, _ = _heads(k, "k", code, t, nkv, hd) if k is not None else (0, 0, 0)
    va, vs, _ = _heads(v, "v", code, t, nkv, hd) if v is not None else (0, 0, 0)
    rows = _lib.PAGED_ROWS.pack(t, code, ka, va, ks, vs, _flat(seq_start, "seq_start", INT32, n + 1))
    check(lib().bb_paged_read(ctx.handle, kv.handle, seqs, rows, _place(ctx, k, v, page_table, lens, seq_start)))
    return k, v


def _n(a):
    return a.numel() if hasattr(a, "numel") else a.size
