"""Device-resident entry points (include/fgm_cuda.h, "device pointers").

Every buffer is a CUDA tensor on the current device; work is enqueued on the
current torch stream (or ``stream=``) and nothing waits.  torch is used only
for allocation and stream handles; the arithmetic is the library's.
"""
from __future__ import annotations

import ctypes as C

import torch

from ._lib import FgmCudaError, call, lib


def _s(stream):
    if stream is not None:
        return stream.cuda_stream
    # torch.cuda.current_stream() without its Stream object: this runs on every call
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


def _p(t):
    return None if t is None else t.data_ptr()


def gemm_q4g(M, N, K, A, a_scale, Bq, b_scale, group, C, ldc=None, n0=0, n1=None, stream=None):
    n1 = N // 16 if n1 is None else n1
    call("fgm_cuda_gemm_q4g", M, N, K, _p(A), _p(a_scale), _p(Bq), _p(b_scale), group, _p(C),
         N if ldc is None else ldc, n0, n1, _s(stream))


def gemm_q8c(M, N, K, A, a_scale, B, b_scale, C, ldc=None, n0=0, n1=None, stream=None):
    n1 = N // 16 if n1 is None else n1
    call("fgm_cuda_gemm_q8c", M, N, K, _p(A), _p(a_scale), _p(B), _p(b_scale), _p(C),
         N if ldc is None else ldc, n0, n1, _s(stream))


def _warm_args(warm):
    """(weights, scales) tensors of the next launch -> the four warm arguments."""
    w, s = (tuple(warm) + (None, None))[:2] if warm is not None else (None, None)
    nbytes = lambda t: 0 if t is None else t.numel() * t.element_size()
    return _p(w), nbytes(w), _p(s), nbytes(s)


def gemm_q4g_warm(M, N, K, A, a_scale, Bq, b_scale, group, C, warm, ldc=None, n0=0, n1=None,
                  stream=None):
    """gemm_q4g that also prefetches warm = (next weights, next scales) into L2."""
    n1 = N // 16 if n1 is None else n1
    call("fgm_cuda_gemm_q4g_warm", M, N, K, _p(A), _p(a_scale), _p(Bq), _p(b_scale), group,
         _p(C), N if ldc is None else ldc, n0, n1, *_warm_args(warm), _s(stream))


def gemm_q8c_warm(M, N, K, A, a_scale, B, b_scale, C, warm, ldc=None, n0=0, n1=None,
                  stream=None):
    """gemm_q8c that also prefetches warm = (next weights, next scales) into L2."""
    n1 = N // 16 if n1 is None else n1
    call("fgm_cuda_gemm_q8c_warm", M, N, K, _p(A), _p(a_scale), _p(B), _p(b_scale), _p(C),
         N if ldc is None else ldc, n0, n1, *_warm_args(warm), _s(stream))


def gemm_q4g_acc(M, N, K, A, Bq, group, acc, n0=0, n1=None, stream=None):
    n1 = N // 16 if n1 is None else n1
    call("fgm_cuda_gemm_q4g_acc", M, N, K, _p(A), _p(Bq), group, _p(acc), n0, n1, _s(stream))


def gemm_q8c_acc(M, N, K, A, B, acc, n0=0, n1=None, stream=None):
    n1 = N // 16 if n1 is None else n1
    call("fgm_cuda_gemm_q8c_acc", M, N, K, _p(A), _p(B), _p(acc), n0, n1, _s(stream))


def prep_rows(src, lda, qs, pa, m, k, hsz, rot=None, qa=None, r0=0, r1=None, stream=None):
    r1 = m if r1 is None else r1
    call("fgm_cuda_prep_rows", _p(src), lda, _p(rot), _p(qa), _p(qs), _p(pa), m, k, hsz, r0, r1,
         _s(stream))


def linear_q4g(src, lda, hsz, M, N, K, Bq, b_scale, group, C, ldc=None, n0=0, n1=None,
               stream=None):
    """Gemm::run for one int4 projection: f32 rows in, C out (prep fused for M <= 16)."""
    n1 = N // 16 if n1 is None else n1
    call("fgm_cuda_linear_q4g", _p(src), lda, hsz, M, N, K, _p(Bq), _p(b_scale), group, _p(C),
         N if ldc is None else ldc, n0, n1, _s(stream))


def linear_q8c(src, lda, hsz, M, N, K, B, b_scale, C, ldc=None, n0=0, n1=None, stream=None):
    """Gemm::run for one int8 projection (tensor cores for prepared weights, M >= 64)."""
    n1 = N // 16 if n1 is None else n1
    call("fgm_cuda_linear_q8c", _p(src), lda, hsz, M, N, K, _p(B), _p(b_scale), _p(C),
         N if ldc is None else ldc, n0, n1, _s(stream))


def packed_a(m: int, k: int, device=None) -> torch.Tensor:
    """An uninitialised packed-activation buffer of ``packed_a_len(m, k)`` bytes."""
    return torch.empty((m + 15) // 16 * 16 * k, dtype=torch.int8, device=device or "cuda")


def gemm_q8c_rows(M, N, K, A, a_scale, B, b_scale, C, lda=None, ldc=None, n0=0, n1=None,
                  stream=None):
    """Prefill int8 GEMM from row-major int8 activations (prepared weight)."""
    n1 = N // 16 if n1 is None else n1
    call("fgm_cuda_gemm_q8c_rows", M, N, K, _p(A), K if lda is None else lda, _p(a_scale), _p(B),
         _p(b_scale), _p(C), N if ldc is None else ldc, n0, n1, _s(stream))


def gemm_q8c_noalloc(M, N, K, A, a_scale, B, b_scale, C, ldc=None, n0=0, n1=None, stream=None):
    """gemm_q8c on the tensor-core kernel with no device allocation (prepared
    weight, M*K <= 4 MiB; concurrent calls on one device race)."""
    n1 = N // 16 if n1 is None else n1
    call("fgm_cuda_gemm_q8c_noalloc", M, N, K, _p(A), _p(a_scale), _p(B), _p(b_scale), _p(C),
         N if ldc is None else ldc, n0, n1, _s(stream))


def q8c_prepare(B, N, K, stream=None):
    """Make the tensor-core operand copy of a device int8 weight (large-M path)."""
    call("fgm_cuda_q8c_prepare", _p(B), N, K, _s(stream))


def q8c_release(B):
    call("fgm_cuda_q8c_release", _p(B))


# ------------------------------------------- decode-chain glue, attention
def rmsnorm(out, x, w, rows, n, eps, stream=None):
    """ops.c:59-92 over rows of n (w None: the no-scale form)."""
    call("fgm_cuda_rmsnorm", _p(out), _p(x), _p(w), rows, n, eps, _s(stream))


def gelu_mul(out, gate, up, rows, n, stream=None):
    """ops.c:119-131: out = gelu_tanh(gate) * up."""
    call("fgm_cuda_gelu_mul", _p(out), _p(gate), _p(up), rows, n, _s(stream))


def add(a, b, stream=None):
    call("fgm_cuda_add", _p(a), _p(b), a.numel(), _s(stream))


def mul(a, b, stream=None):
    call("fgm_cuda_mul", _p(a), _p(b), a.numel(), _s(stream))


def scale(a, s, stream=None):
    call("fgm_cuda_scale", _p(a), s, a.numel(), _s(stream))


def softcap(x, rows, n, cap, stream=None):
    call("fgm_cuda_softcap", _p(x), rows, n, cap, _s(stream))


def rope(x, x_ld, rows, n_heads, head_dim, inv_freq, pos, cs=None, stream=None):
    """ops.c:135-147 in place; pos: int32 device tensor [rows]; cs: a device
    copy of rope_table(...) (the reference's libm cos / sin), else the device
    evaluates them."""
    if cs is None:
        call("fgm_cuda_rope", _p(x), x_ld, rows, n_heads, head_dim, _p(inv_freq), _p(pos),
             _s(stream))
    else:
        call("fgm_cuda_rope_cs", _p(x), x_ld, rows, n_heads, head_dim, _p(inv_freq), _p(cs),
             cs.shape[0], _p(pos), _s(stream))


def rope_table(positions, head_dim, inv_freq):
    """Host [positions][head_dim] f32: cosf | sinf of (float)p * inv_freq[j]
    (ops.c:137-139) from this host's libm; inv_freq: numpy f32 [head_dim/2]."""
    import numpy as np
    inv = np.ascontiguousarray(inv_freq, dtype=np.float32)
    out = np.empty((positions, head_dim), np.float32)
    call("fgm_cuda_rope_table", out.ctypes.data, positions, head_dim, inv.ctypes.data)
    return out


def quant_act(x, rows, k, q, scale, stream=None):
    """ops.c:181-204 (quant_kv: one row)."""
    call("fgm_cuda_quant_act", _p(x), rows, k, _p(q), _p(scale), _s(stream))


def store_v_t(vt, vt_stride, src, src_ld, rows, n, slot, stream=None):
    """ops.c:653-660 for `rows` caches."""
    call("fgm_cuda_store_v_t", _p(vt), vt_stride, _p(src), src_ld, rows, n, slot, _s(stream))


def attend_q8(out, out_ld, q, q_ld, kc, kc_stride, ks, ks_stride, vt, vt_stride, vs, vs_stride,
              rows, n_heads, kv_heads, head_dim, start, end, ring=0, stream=None):
    """ops.c:378-640 for `rows` query rows, each against its own int8 KV cache."""
    call("fgm_cuda_attend_q8", _p(out), out_ld, _p(q), q_ld, _p(kc), kc_stride, _p(ks), ks_stride,
         _p(vt), vt_stride, _p(vs), vs_stride, rows, n_heads, kv_heads, head_dim, start, end, ring,
         _s(stream))


def norm_prep(h, proj, w_post, w_pre, rows, n, eps, qs, pa, stream=None):
    """forward.rs:476-480, :625-654: h += rmsnorm(proj, w_post) (when proj is
    given), then the packed rows of rmsnorm(h, w_pre)."""
    call("fgm_cuda_norm_prep", _p(h), _p(proj), _p(w_post), _p(w_pre), rows, n, eps, _p(qs), _p(pa),
         _s(stream))


def gelu_mul_prep(gate, up, rows, n, qs, pa, act=None, ld=None, stream=None):
    """forward.rs:641-643: packed rows of gelu(gate) * up (rows ld apart)."""
    call("fgm_cuda_gelu_mul_prep", _p(gate), _p(up), n if ld is None else ld, rows, n, _p(act),
         _p(qs), _p(pa), _s(stream))


def qkv_post(q, k, v, rows, n_heads, kv_heads, head_dim, q_norm, k_norm, eps, inv_freq, pos, ring,
             cap, kc, kc_stride, ks, ks_stride, vt, vt_stride, vs, vs_stride, q_ld=None, kv_ld=None,
             cs=None, stream=None):
    """forward.rs:482-545: head norms, rope, int8 K / V rows into the caches
    (cs: a device copy of rope_table(...), as for rope)."""
    q_ld = n_heads * head_dim if q_ld is None else q_ld
    kv_ld = kv_heads * head_dim if kv_ld is None else kv_ld
    call("fgm_cuda_qkv_post_cs", _p(q), q_ld, _p(k), _p(v), kv_ld, rows, n_heads, kv_heads,
         head_dim, _p(q_norm), _p(k_norm), eps, _p(inv_freq), _p(cs),
         0 if cs is None else cs.shape[0], _p(pos), ring, cap, _p(kc), kc_stride, _p(ks),
         ks_stride, _p(vt), vt_stride, _p(vs), vs_stride, _s(stream))


# ----------------------------- several tokens per sequence over one KV cache
class KvCache(C.Structure):
    """One layer's int8 KV caches of several sequences (fgm_cuda_kv): a view of
    tensors the caller owns, kept alive by it.

    kc [rows][cap][kv_heads * head_dim] int8, ks / vs [rows][cap] f32, vt
    [rows][ceil(cap / 4) * 4 * kv_heads * head_dim] int8 in any shape after
    the first dimension, acc [rows][cap] f32 and tpos [rows][cap] int32 where
    used; rows may be strided, what lies behind a row is contiguous."""
    _fields_ = [("kc", C.c_void_p), ("ks", C.c_void_p), ("vt", C.c_void_p), ("vs", C.c_void_p),
                ("acc", C.c_void_p), ("tpos", C.c_void_p),
                ("kc_stride", C.c_size_t), ("ks_stride", C.c_size_t), ("vt_stride", C.c_size_t),
                ("vs_stride", C.c_size_t), ("acc_stride", C.c_size_t), ("tpos_stride", C.c_size_t),
                ("rows", C.c_int), ("kv_heads", C.c_int), ("head_dim", C.c_int),
                ("cap", C.c_int), ("ring", C.c_int)]

    def __init__(self, kc, ks, vt, vs, kv_heads, head_dim, ring=0, acc=None, tpos=None):
        super().__init__()
        rows, cap = kc.shape[0], kc.shape[1]
        kvd = kv_heads * head_dim
        if tuple(kc.shape) != (rows, cap, kvd):
            raise ValueError(f"kc has shape {tuple(kc.shape)}, not [rows][cap][{kvd}]")
        for name, t, dtype, n in (("kc", kc, torch.int8, cap * kvd), ("ks", ks, torch.float32, cap),
                                  ("vt", vt, torch.int8, (cap + 3) // 4 * 4 * kvd),
                                  ("vs", vs, torch.float32, cap), ("acc", acc, torch.float32, cap),
                                  ("tpos", tpos, torch.int32, cap)):
            if t is None:
                continue
            if t.dtype != dtype or t.shape[0] != rows or (rows and t[0].numel() < n):
                raise ValueError(f"{name}: {t.dtype} {tuple(t.shape)}, need {dtype} with {n} "
                                 f"elements in each of {rows} rows")
            if rows and not t[0].is_contiguous():
                raise ValueError(f"{name}: a row has to be contiguous")
            setattr(self, name, t.data_ptr())
            setattr(self, name + "_stride", t.stride(0))
        self.rows, self.kv_heads, self.head_dim, self.cap, self.ring = (rows, kv_heads, head_dim,
                                                                        cap, ring)
        self._keep = (kc, ks, vt, vs, acc, tpos)


def kv_layers(views):
    """Several layers' KvCache views as one array for kv_accept."""
    arr = (KvCache * len(views))(*views)
    arr._keep_views = list(views)
    return arr


_NOT_INT32 = {"mask": torch.int64, "take": torch.uint8}


def _flat(**tensors):
    """The entries take whole tensors by address: one of another type, or a
    strided one, would be misread."""
    for name, t in tensors.items():
        if t is not None and (t.dtype != _NOT_INT32.get(name, torch.int32) or
                              not t.is_contiguous()):
            raise ValueError(f"{name} has to be contiguous "
                             f"{_NOT_INT32.get(name, torch.int32)}, not {t.dtype} with strides "
                             f"{t.stride()}")


def _rows(**tensors):
    """The same for rows of f32 at a distance the caller gives."""
    for name, t in tensors.items():
        if t is not None and (t.dtype != torch.float32 or
                              (t.shape[-1] > 1 and t.stride(-1) != 1)):
            raise ValueError(f"{name} has to be torch.float32 with its last dimension contiguous, "
                             f"not {t.dtype} with strides {t.stride()}")


def _lse(lse, rows, n_heads):
    if lse is None:
        return None, 0, 0
    if (lse.dtype != torch.float32 or lse.dim() != 2 or lse.shape[0] < rows or
            lse.shape[1] < n_heads):
        raise ValueError(f"lse: {lse.dtype} {tuple(lse.shape)}, need torch.float32 of "
                         f"[{rows}][{n_heads}]")
    return lse.data_ptr(), lse.stride(0), lse.stride(1)


def _on(stream):
    return torch.cuda.stream(stream or torch.cuda.current_stream())


def attend_workspace(kv, n_heads, T):
    """A workspace for the attention entries on this cache, zeroed as its first
    use needs it; to be kept from call to call, by one stream at a time."""
    n = call("fgm_cuda_attend_workspace", C.byref(kv), n_heads, T)
    if n == 0 and kv.rows:
        raise FgmCudaError(-1, lib().fgm_cuda_last_error().decode())
    return torch.zeros(max(int(n), 1), dtype=torch.uint8, device="cuda")


def _ws(ws, kv, n_heads, T, stream):
    if ws is None:  # from torch's allocator, on the stream that uses it
        with _on(stream):
            ws = attend_workspace(kv, n_heads, T)
    return ws


def tree_mask(mask, pos, parent, lens, stream=None):
    """Ancestor words mask [rows][T][ceil(T / 64)] (int64) and positions pos
    [rows * T] of the trees parent [rows][T] (int32)."""
    rows, T = parent.shape
    _flat(mask=mask, pos=pos, parent=parent, lens=lens)
    call("fgm_cuda_tree_mask", _p(mask), _p(pos), _p(parent), _p(lens), rows, T, _s(stream))


def attend_tree_q8(out, q, kv, n_heads, T, lens, mask=None, pos=None, window=0, lse=None, ws=None,
                   q_ld=None, out_ld=None, stream=None):
    """T nodes of each sequence attend to its cache and to one another (mask
    None: to the nodes before them); lse [rows * T][n_heads], of any strides, if
    wanted.  A window goes by the slots' indexes, so not with a cache that
    kv_evict_q8 has moved rows in."""
    _flat(lens=lens, mask=mask, pos=pos)
    _rows(q=q, out=out)
    lse = _lse(lse, kv.rows * T, n_heads)
    ws = _ws(ws, kv, n_heads, T, stream)
    ld = n_heads * kv.head_dim
    call("fgm_cuda_attend_tree_q8", C.byref(kv), _p(q), ld if q_ld is None else q_ld, n_heads, T,
         _p(lens), _p(mask), _p(pos), window, _p(out), ld if out_ld is None else out_ld,
         *lse, _p(ws), ws.numel(), _s(stream))


def attend_accum_q8(q, kv, n_heads, T, lens, lse, mask=None, pos=None, window=0, take=None,
                    decay=1.0, ws=None, q_ld=None, stream=None):
    """kv's acc = decay * acc + the weights of the taken nodes (take: uint8
    [rows * T]) of such an attention, from its lse."""
    _flat(lens=lens, mask=mask, pos=pos, take=take)
    _rows(q=q)
    lse = _lse(lse, kv.rows * T, n_heads)
    ws = _ws(ws, kv, n_heads, T, stream)
    call("fgm_cuda_attend_accum_q8", C.byref(kv), _p(q),
         n_heads * kv.head_dim if q_ld is None else q_ld, n_heads, T, _p(lens), _p(mask), _p(pos),
         window, *lse, _p(take), decay, _p(ws), ws.numel(), _s(stream))


def attend_acc_q8(out, q, kv, n_heads, lens, decay=1.0, ws=None, q_ld=None, out_ld=None,
                  stream=None):
    """One token per sequence: attention over slots [0, lens[b]] and its weights added to kv's acc."""
    _flat(lens=lens)
    _rows(q=q, out=out)
    ws = _ws(ws, kv, n_heads, 1, stream)
    ld = n_heads * kv.head_dim
    call("fgm_cuda_attend_acc_q8", C.byref(kv), _p(q), ld if q_ld is None else q_ld, n_heads,
         _p(lens), decay, _p(out), ld if out_ld is None else out_ld, _p(ws), ws.numel(),
         _s(stream))


def tree_verify(path, n_acc, next_token, parent, token, target, stream=None):
    """The accepted path of each drafted tree: path [rows][T] (then -1), its
    length n_acc and the token after it."""
    rows, T = parent.shape
    _flat(path=path, n_acc=n_acc, next_token=next_token, parent=parent, token=token, target=target)
    call("fgm_cuda_tree_verify", _p(path), _p(n_acc), _p(next_token), _p(parent), _p(token),
         _p(target), rows, T, _s(stream))


def kv_accept(layers, T, lens, path, n_acc, lens_new=None, stream=None):
    """Move the accepted path's rows behind the committed ones in every layer
    (layers: kv_layers(...) or one KvCache)."""
    _flat(lens=lens, path=path, n_acc=n_acc, lens_new=lens_new)
    one = isinstance(layers, KvCache)
    call("fgm_cuda_kv_accept", C.byref(layers) if one else layers, 1 if one else len(layers), T,
         _p(lens), _p(path), _p(n_acc), _p(lens_new), _s(stream))


def kv_evict_q8(kv, lens, budget, sink, recent, slot_map, lens_out, acc_out=None, tpos_out=None,
                stream=None):
    """Keep `budget` slots of each cache (protected, then by accumulated
    weight); slot_map [rows][budget] says where each slot's row came from."""
    _flat(lens=lens, slot_map=slot_map, lens_out=lens_out)
    for name, t, dtype in (("acc_out", acc_out, torch.float32), ("tpos_out", tpos_out, torch.int32)):
        if t is not None and (t.dtype != dtype or t.dim() != 2 or t.shape[0] < kv.rows or
                              t.shape[1] < budget or (t.shape[1] > 1 and t.stride(1) != 1)):
            raise ValueError(f"{name}: {t.dtype} {tuple(t.shape)} with strides {t.stride()}, need "
                             f"{dtype} of [{kv.rows}][{budget}] with contiguous rows")
    stride = (acc_out if acc_out is not None else tpos_out).stride(0) \
        if acc_out is not None or tpos_out is not None else 0
    if acc_out is not None and tpos_out is not None and tpos_out.stride(0) != stride:
        raise ValueError("acc_out and tpos_out need the same row stride")
    call("fgm_cuda_kv_evict_q8", C.byref(kv), _p(lens), budget, sink, recent, _p(slot_map),
         _p(lens_out), _p(acc_out), _p(tpos_out), stride, _s(stream))


def qkv_post_tree(kv, q, k, v, n_heads, T, q_norm, k_norm, eps, inv_freq, pos, lens, q_ld=None,
                  kv_ld=None, cs=None, stream=None):
    """qkv_post for the nodes of a tree: rope at pos (None: at lens[b] + i), K / V rows into
    slots lens[b] + i."""
    _flat(pos=pos, lens=lens)
    _rows(q=q, k=k, v=v)
    kvd = kv.kv_heads * kv.head_dim
    call("fgm_cuda_qkv_post_tree", C.byref(kv), _p(q),
         n_heads * kv.head_dim if q_ld is None else q_ld, _p(k), _p(v),
         kvd if kv_ld is None else kv_ld, n_heads, T, _p(q_norm), _p(k_norm), eps, _p(inv_freq),
         _p(cs), 0 if cs is None else cs.shape[0], _p(pos), _p(lens), _s(stream))


# ------------------------------------------------------- decode work list
class _Work(C.Structure):
    """fgm_cuda_work (include/fgm_cuda.h)."""
    _fields_ = [("kind", C.c_int), ("N", C.c_int), ("K", C.c_int), ("group", C.c_int),
                ("n0", C.c_int), ("n1", C.c_int), ("ldc", C.c_int), ("lda", C.c_int),
                ("hsz", C.c_int), ("deps", C.c_int * 2),
                ("A", C.c_void_p), ("a_scale", C.c_void_p), ("B", C.c_void_p),
                ("b_scale", C.c_void_p), ("C", C.c_void_p), ("src", C.c_void_p),
                ("pa", C.c_void_p), ("qs", C.c_void_p)]


WORK_Q4G, WORK_Q8C, WORK_PREP = 0, 1, 2


class WorkList:
    """A decode step's projections as one persistent launch
    (fgm_cuda_worklist_*).  Add entries in an order where every entry's
    dependencies come first, then ``build(M)`` once and ``run()`` per step.
    The tensors passed in must stay alive (and in place) as long as the list."""

    def __init__(self):
        self._items, self._keep, self.handle = [], [], None

    def _add(self, w, deps, keep):
        d = list(deps) + [-1, -1]
        w.deps[0], w.deps[1] = d[0], d[1]
        self._items.append(w)
        self._keep.extend(keep)
        return len(self._items) - 1

    def prep(self, src, lda, K, pa, qs, hsz=0, deps=()):
        """Rows [0, M) of src (f32) -> packed pa and scales qs (fgm_prep_rows)."""
        w = _Work(kind=WORK_PREP, K=K, lda=lda, hsz=hsz, src=_p(src), pa=_p(pa), qs=_p(qs))
        return self._add(w, deps, (src, pa, qs))

    def gemm_q4g(self, N, K, A, a_scale, Bq, b_scale, group, C, ldc=None, n0=0, n1=None,
                 deps=()):
        n1 = N // 16 if n1 is None else n1
        w = _Work(kind=WORK_Q4G, N=N, K=K, group=group, n0=n0, n1=n1,
                  ldc=N if ldc is None else ldc, A=_p(A), a_scale=_p(a_scale), B=_p(Bq),
                  b_scale=_p(b_scale), C=_p(C))
        return self._add(w, deps, (A, a_scale, Bq, b_scale, C))

    def gemm_q8c(self, N, K, A, a_scale, B, b_scale, C, ldc=None, n0=0, n1=None, deps=()):
        n1 = N // 16 if n1 is None else n1
        w = _Work(kind=WORK_Q8C, N=N, K=K, n0=n0, n1=n1, ldc=N if ldc is None else ldc,
                  A=_p(A), a_scale=_p(a_scale), B=_p(B), b_scale=_p(b_scale), C=_p(C))
        return self._add(w, deps, (A, a_scale, B, b_scale, C))

    def build(self, M):
        arr = (_Work * len(self._items))(*self._items)
        h = C.c_void_p()
        call("fgm_cuda_worklist_create", M, arr, len(self._items), C.byref(h))
        self.handle = h
        return self

    def run(self, stream=None):
        call("fgm_cuda_worklist_run", self.handle, _s(stream))

    def close(self):
        if self.handle is not None:
            call("fgm_cuda_worklist_destroy", self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
