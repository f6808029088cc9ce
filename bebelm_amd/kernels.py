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
Each function takes the Context first; `w` is an uploaded Tensor (plus a byte offset where the
reference passes a sub-slice of the weight bytes).
"""
import ctypes
from dataclasses import dataclass

import numpy as np

from . import _lib
from ._lib import check, lib
from .model import _dtype, _on, _ptr, _same_loc


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


def _strides(a):
    """Strides in elements."""
    return tuple(a.stride()) if hasattr(a, "data_ptr") else tuple(n // a.itemsize for n in a.strides)


def _data(a):
    return a.data_ptr() if hasattr(a, "data_ptr") else a.ctypes.data


def _loc_of(ctx, *arrays):
    """Where the arrays are (those of any strides among them), all in one place."""
    _on(ctx, *arrays)
    locs = {bool(getattr(a, "is_cuda", False)) for a in arrays if a is not None}
    if len(locs) != 1:
        raise ValueError("all arrays of one call must be host or all device")
    return _lib.LOC_DEVICE if locs.pop() else _lib.LOC_HOST


def _heads(a, what, n=None, heads=None, hd=None, packed=True):
    """Strides (token, head) of [tokens, heads, head_dim], checked."""
    if len(a.shape) != 3 or any(w is not None and w != g for w, g in zip((n, heads, hd), a.shape)):
        raise ValueError(f"{what} must be [tokens, heads, head_dim], is {tuple(a.shape)}")
    st, (t, h, d) = _strides(a), a.shape
    if d > 1 and st[2] != 1:
        raise ValueError(f"{what}: the elements of a head must be adjacent")
    if packed and h > 1 and st[1] != d:
        raise ValueError(f"{what}: the heads of a token must be adjacent")
    if any(s < 0 for s in st):
        raise ValueError(f"{what}: negative strides")
    return (st[0] if t > 1 else h * d), (st[1] if h > 1 else d)


def _ints(a, what, shape):
    if a is None:
        return None
    if str(a.dtype).replace("torch.", "") != "int32" or tuple(a.shape) != shape:
        raise ValueError(f"{what} must be int32 {list(shape)}, is {a.dtype} {list(a.shape)}")
    return _ptr(a)[0]


def _floats(a, what, shape):
    if a is None:
        return None
    if str(a.dtype).replace("torch.", "") != "float32" or tuple(a.shape) != shape:
        raise ValueError(f"{what} must be float32 {list(shape)}, is {a.dtype} {list(a.shape)}")
    return _ptr(a)[0]


def _seqs(kv, page_table, lens):
    if len(page_table.shape) != 2 or str(page_table.dtype).replace("torch.", "") != "int32":
        raise ValueError("page_table must be int32 [sequences, pages]")
    n, pages = page_table.shape
    st = _strides(page_table)
    if (pages > 1 and st[1] != 1) or st[0] < 0:
        raise ValueError("page_table: the entries of a sequence must be adjacent")
    return _lib.PagedSeqs(n, pages, st[0] if n > 1 else pages, _data(page_table), _ints(lens, "lens", (n,)))


def rope(ctx, plan, x, pos, out=None):
    """x [tokens, heads, head_dim] (any token and head strides) turned by pos int32 [tokens] as the
    RopePlan says, into out (x itself by default)."""
    out = x if out is None else out
    t, h, hd = x.shape
    xs, os = _heads(x, "x", packed=False), _heads(out, "out", t, h, hd, packed=False)
    if _dtype(x) != _dtype(out):
        raise ValueError("x and out must be of one type")
    loc = _loc_of(ctx, x, pos, out)
    check(lib().bb_rope(ctx.handle, plan.handle, _dtype(x), _data(x), *xs, t, h, hd, _ints(pos, "pos", (t,)),
                        _data(out), *os, loc))
    return out


def paged_append(ctx, kv, page_table, lens, k, v, rope=None, pos=None, seq_start=None, q=None, q_out=None, q_norm=None,
                 k_norm=None, eps=1e-5):
    """Stores k and v [tokens, n_kv_heads, head_dim] at the end of their sequences in the PagedKv's
    pages; on the way k (and q [tokens, n_heads, head_dim], into q_out, q itself by default) is normed
    with k_norm (q_norm) and turned as the RopePlan `rope` says, by pos int32 [tokens] or each token's
    index in its sequence. page_table int32 [sequences, pages] and lens int32 [sequences] count the
    call's tokens; seq_start int32 [sequences + 1] says which tokens each sequence brings (None: one
    each). Returns q_out."""
    t = k.shape[0]
    seqs = _seqs(kv, page_table, lens)
    ks = _heads(k, "k", t, kv.n_kv_heads, kv.head_dim)
    vs = _heads(v, "v", t, kv.n_kv_heads, kv.head_dim)
    if q is not None and q_out is None:
        q_out = q
    if len({_dtype(a) for a in (k, v, q, q_out) if a is not None}) != 1:
        raise ValueError("k, v, q and q_out must be of one type")
    if rope is not None and not rope.handle:
        raise ValueError("the RopePlan is closed")
    heads, qs, qos = 0, (0, 0), (0, 0)
    if q is not None:
        heads = q.shape[1]
        qs, qos = _heads(q, "q", t, None, kv.head_dim), _heads(q_out, "q_out", t, heads, kv.head_dim)
    loc = _loc_of(ctx, page_table, lens, k, v, pos, seq_start, q, q_out, q_norm, k_norm)
    tok = _lib.PagedTokens(t, _dtype(k), _data(k), _data(v), ks[0], vs[0], _data(q) if q is not None else None,
                           _data(q_out) if q_out is not None else None, heads, qs[0], qos[0],
                           _floats(q_norm, "q_norm", (kv.head_dim,)), _floats(k_norm, "k_norm", (kv.head_dim,)), eps,
                           _ints(pos, "pos", (t,)), _ints(seq_start, "seq_start", (seqs.n_seqs + 1,)))
    check(lib().bb_paged_append(ctx.handle, kv.handle, rope.handle if rope is not None else None, ctypes.byref(seqs),
                                ctypes.byref(tok), loc))
    return q_out


def paged_attention(ctx, kv, page_table, lens, q, out, scale=None, window=0, lse=None, workspace=None):
    """One query token per sequence, q [sequences, n_heads, head_dim], over the sequence's positions
    in the PagedKv's pages (the last `window` of them; 0: all), into out; lse float32 [sequences,
    n_heads] gets the softmax's log sums. scale None: 1/sqrt(head_dim). workspace: a device tensor of
    kv.attention_workspace(n_heads, sequences) bytes for this call alone (None: the context's; a call
    captured into a graph needs one)."""
    seqs = _seqs(kv, page_table, lens)
    n, heads = seqs.n_seqs, q.shape[1]
    qs = _heads(q, "q", n, None, kv.head_dim)
    os = _heads(out, "out", n, heads, kv.head_dim)
    if _dtype(q) != _dtype(out):
        raise ValueError("q and out must be of one type")
    loc = _loc_of(ctx, page_table, lens, q, out, lse)
    if workspace is not None:
        if not (getattr(workspace, "is_cuda", False) and workspace.is_contiguous()):
            raise ValueError("the workspace must be a contiguous device tensor")
        _on(ctx, workspace)
    if scale is not None and scale == 0:
        raise ValueError("scale must not be 0")
    pq = _lib.PagedQuery(_dtype(q), _data(q), _data(out), heads, qs[0], os[0], 0.0 if scale is None else scale,
                         int(window), _floats(lse, "lse", (n, heads)),
                         workspace.data_ptr() if workspace is not None else None,
                         workspace.numel() * workspace.element_size() if workspace is not None else 0)
    check(lib().bb_paged_attention(ctx.handle, kv.handle, ctypes.byref(seqs), ctypes.byref(pq), loc))
    return out


def _n(a):
    return a.numel() if hasattr(a, "numel") else a.size
