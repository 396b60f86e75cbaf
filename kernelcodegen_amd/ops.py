"""Device operators: torch tensors in, the gfx950 kernels underneath.

Names and argument meaning follow the reference's Frontend operators
(include/Frontend/Operators.h:73-102): Matmul, Relu, BatchedMatmul, Softmax,
and the fused attention the FMHAOptimizer recognises
(src/Optimizer/Optimizer.cc:586-672).  Everything goes through the C-ABI; a
failing status raises lib.KcgError.

Attention layers that serve have operators of their own (the reference has none):
qk_norm_rope and its gradient make the queries and keys, KvCache with kv_cache_write and
kv_cache_read holds them, fmha_cache attends over it.
"""
import ctypes

import torch

from . import lib

EPILOGUE_NONE = 0
EPILOGUE_RELU = 1
F32 = 0
BF16 = 1
E4M3 = 2
_DTYPES = {torch.float32: F32, torch.bfloat16: BF16}


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr())


def _dev_f32(t, name):
    if not (t.is_cuda and t.dtype == torch.float32 and t.is_contiguous()):
        raise ValueError("%s must be a contiguous fp32 device tensor" % name)


def _check(t, name, dtype, shape, device):
    """The kernels take raw pointers: a tensor of another dtype, shape, device or layout
    would make them read or write out of bounds, so it is refused here."""
    if not isinstance(t, torch.Tensor):
        raise ValueError("%s must be a tensor" % name)
    if not t.is_cuda or t.device != device:
        raise ValueError("%s must be on device %s" % (name, device))
    if t.dtype != dtype:
        raise ValueError("%s must have dtype %s, not %s" % (name, dtype, t.dtype))
    if tuple(t.shape) != tuple(shape):
        raise ValueError("%s must have shape %s, not %s" % (name, tuple(shape), tuple(t.shape)))
    if not t.is_contiguous():
        raise ValueError("%s must be contiguous" % name)


def _sched(sched, cls):
    if sched is None:
        return None
    if isinstance(sched, cls):
        return ctypes.byref(sched)
    return ctypes.byref(cls(**sched))


def matmul_workspace_bytes(M, N, K, sched=None):
    """Bytes of workspace with which matmul() can run its K-split plan (0: there is none)."""
    return int(lib.load().kcg_gemm_f32_ws_bytes(M, N, K, _sched(sched, lib.GemmSched)))


def matmul(A, B, relu=False, out=None, sched=None, workspace=None):
    """C = A.B (row-major fp32), optionally with the ReLU epilogue fused.

    workspace: a contiguous device tensor the call may use for partial sums
    (kcg_gemm_f32_ws; see matmul_workspace_bytes).  Nothing else may use it until the
    call has completed on the current stream.
    """
    _dev_f32(A, "A")
    _dev_f32(B, "B")
    M, K = A.shape
    K2, N = B.shape
    if K != K2:
        raise ValueError("Can't apply Matmul Operation due to imcompatible K-dim.")
    if B.device != A.device:
        raise ValueError("A and B must be on the same device")
    if out is None:
        out = torch.empty((M, N), dtype=torch.float32, device=A.device)
    _check(out, "out", torch.float32, (M, N), A.device)
    epilogue = EPILOGUE_RELU if relu else EPILOGUE_NONE
    if workspace is not None:
        if not (isinstance(workspace, torch.Tensor) and workspace.is_cuda and workspace.device == A.device
                and workspace.is_contiguous()):
            raise ValueError("workspace must be a contiguous tensor on %s" % A.device)
        st = lib.load().kcg_gemm_f32_ws(_ptr(A), _ptr(B), _ptr(out), M, N, K, epilogue,
                                        _sched(sched, lib.GemmSched), _ptr(workspace),
                                        workspace.numel() * workspace.element_size(), lib.current_stream())
    else:
        st = lib.load().kcg_gemm_f32(_ptr(A), _ptr(B), _ptr(out), M, N, K, epilogue,
                                     _sched(sched, lib.GemmSched), lib.current_stream())
    lib.check(st)
    return out


def relu(x, inplace=False, out=None):
    _dev_f32(x, "x")
    if out is not None:
        _dev_f32(out, "out")
        if out.numel() != x.numel() or out.device != x.device:
            raise ValueError("relu: out must have as many elements as x, on the same device")
    y = x if inplace else (out if out is not None else torch.empty_like(x))
    lib.check(lib.load().kcg_relu_f32(_ptr(x), _ptr(y), x.numel(), lib.current_stream()))
    return y


def batched_matmul(A, B, trans_a=False, trans_b=False, out=None):
    """C[b] = op(A[b]).op(B[b]); leading dims are the batch (Layout::colMajor = trans)."""
    _dev_f32(A, "A")
    _dev_f32(B, "B")
    batch_shape = tuple(A.shape[:-2])
    if tuple(B.shape[:-2]) != batch_shape:
        raise ValueError("BatchedMatmul: A, B dim not matched.")
    K, M = (A.shape[-2], A.shape[-1]) if trans_a else (A.shape[-1], A.shape[-2])
    K2, N = (B.shape[-1], B.shape[-2]) if trans_b else (B.shape[-2], B.shape[-1])
    if K != K2:
        raise ValueError("Can't apply BatchedMatmul Operation due to imcompatible K-dim.")
    batch = 1
    for d in batch_shape:
        batch *= d
    if B.device != A.device:
        raise ValueError("A and B must be on the same device")
    if out is None:
        out = torch.empty(batch_shape + (M, N), dtype=torch.float32, device=A.device)
    _check(out, "out", torch.float32, batch_shape + (M, N), A.device)
    st = lib.load().kcg_batched_matmul_f32(_ptr(A), int(trans_a), _ptr(B), int(trans_b), _ptr(out),
                                           batch, M, N, K, lib.current_stream())
    lib.check(st)
    return out


def softmax_(x):
    """In-place softmax over the last axis (the reference operator is in place)."""
    _dev_f32(x, "x")
    n = x.shape[-1]
    lib.check(lib.load().kcg_softmax_f32(_ptr(x), x.numel() // n, n, lib.current_stream()))
    return x


def fmha(Q, K, V, scale=1.0, causal=False, out=None, out_dtype=None, sched=None):
    """O = softmax(scale * Q.K^T [+causal]) . V for [B,H,S,D] tensors.

    fp32 tensors run the fp32 kernel; bf16 tensors the bf16 kernel (fp32
    accumulation and softmax), writing `out_dtype` (bf16 by default).
    """
    if not isinstance(Q, torch.Tensor) or Q.dim() != 4:
        raise ValueError("Q, K, V must share one [B,H,S,D] shape")
    if Q.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("fmha supports float32 and bfloat16")
    if not Q.is_cuda:
        raise ValueError("Q, K, V must be contiguous device tensors")
    for t, name in ((Q, "Q"), (K, "K"), (V, "V")):
        _check(t, name, Q.dtype, Q.shape, Q.device)
    B_, H, S, D = Q.shape
    if Q.dtype == torch.float32:
        if out_dtype not in (None, torch.float32):
            raise ValueError("fp32 attention writes fp32: out_dtype must be float32")
        want = torch.float32
    else:
        if out_dtype not in (None, torch.bfloat16, torch.float32):
            raise ValueError("bf16 attention writes bfloat16 or float32, not %s" % out_dtype)
        want = out_dtype or (out.dtype if out is not None else torch.bfloat16)
        if want not in (torch.bfloat16, torch.float32):
            raise ValueError("out must be bfloat16 or float32, not %s" % want)
    if out is not None:
        _check(out, "out", want, Q.shape, Q.device)
    L = lib.load()
    if Q.dtype == torch.float32:
        if out is None:
            out = torch.empty_like(Q)
        st = L.kcg_fmha_f32(_ptr(Q), _ptr(K), _ptr(V), _ptr(out), B_, H, S, D, float(scale),
                            int(causal), _sched(sched, lib.FmhaSched), lib.current_stream())
    else:
        if out is None:
            out = torch.empty(Q.shape, dtype=want, device=Q.device)
        o_dtype = BF16 if out.dtype == torch.bfloat16 else F32
        st = L.kcg_fmha_bf16(_ptr(Q), _ptr(K), _ptr(V), _ptr(out), o_dtype, B_, H, S, D,
                             float(scale), int(causal), _sched(sched, lib.FmhaSched),
                             lib.current_stream())
    lib.check(st)
    return out


# ---- attention layers that serve --------------------------------------------------------


# A small call takes as long as its checks: each helper below first asks everything in one
# expression and looks for what is wrong only where that fails.
_Tensor, _contiguous, _pack_rows = torch.Tensor, torch.contiguous_format, lib.pack_rows
_TOO_MANY = 1 << 31  # (extents are 32-bit numbers in the C interface)


def _rows(t, name, dtype, index, shape=None):
    """kcg_rows of a [B,S,H,D] (or [tokens,H,D]) tensor on device `index`: any strides but a
    contiguous last axis."""
    if isinstance(t, _Tensor) and t.dtype == dtype and t.get_device() == index and (
            shape is None or t.shape == shape) and t.numel() < _TOO_MANY:
        stride = t.stride()
        if len(stride) == 4 and stride[3] == 1:
            return _pack_rows(t.data_ptr(), stride[0], stride[1], stride[2])
        if len(stride) == 3 and stride[2] == 1:
            return _pack_rows(t.data_ptr(), 0, stride[0], stride[1])
    if not isinstance(t, _Tensor) or t.dim() not in (3, 4):
        raise ValueError("%s must be a [B,S,H,D] or [tokens,H,D] tensor" % name)
    if t.get_device() != index:
        raise ValueError("%s must be on device cuda:%d" % (name, index))
    if t.dtype != dtype:
        raise ValueError("%s must have dtype %s, not %s" % (name, dtype, t.dtype))
    if shape is not None and t.shape != shape:
        raise ValueError("%s must have shape %s, not %s" % (name, tuple(shape), tuple(t.shape)))
    if t.numel() >= _TOO_MANY:
        raise ValueError("%s must have fewer than 2^31 elements" % name)
    raise ValueError("the last axis of %s must be contiguous" % name)


def _new_rows(t):
    """kcg_rows of a contiguous tensor that was made here."""
    shape = t.shape
    H, D = shape[-2], shape[-1]
    return _pack_rows(t.data_ptr(), shape[-3] * H * D, H * D, D)


def _plain(t, name, dtype, shape, index):
    """Address of a contiguous tensor of this type and shape on device `index`."""
    if not (isinstance(t, _Tensor) and t.dtype == dtype and t.get_device() == index and t.shape == shape
            and t.is_contiguous()):
        _check(t, name, dtype, shape, torch.device("cuda", index))
    return t.data_ptr()


def _call(fn, index, *args):
    """Calls a C entry point on the current stream of device `index`, whichever device is current."""
    if index == torch.cuda.current_device():
        st = fn(*args, lib.raw_stream(index))
    else:
        with torch.cuda.device(index):
            st = fn(*args, lib.raw_stream(index))
    if st:
        lib.check(st)


def _workspace(workspace, need, index, device):
    """(address, bytes) of a workspace, and the tensor that holds it."""
    if workspace is None:
        if not need:
            return None, 0, None
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
        return workspace.data_ptr(), need, workspace
    if not (isinstance(workspace, torch.Tensor) and workspace.get_device() == index and workspace.is_contiguous()):
        raise ValueError("workspace must be a contiguous tensor on cuda:%d" % index)
    return workspace.data_ptr(), workspace.numel() * workspace.element_size(), workspace


def _norm_rope_args(q, k, q_weight, k_weight, positions, inv_freq, eps, interleaved):
    if not isinstance(q, _Tensor) or not q.is_cuda:
        raise ValueError("q must be a device tensor")
    index, dtype = q.get_device(), q.dtype
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError("q must be float32 or bfloat16, not %s" % dtype)
    rq, rk = _rows(q, "q", dtype, index), _rows(k, "k", dtype, index)
    shape, k_shape = tuple(q.shape), tuple(k.shape)
    tokens, D = shape[:-2], shape[-1]
    if k_shape[:-2] != tokens or k_shape[-1] != D:
        raise ValueError("k must have q's tokens and head dimension")
    if not isinstance(inv_freq, _Tensor) or inv_freq.dim() != 1:
        raise ValueError("inv_freq must be a tensor of one frequency for each rotated pair")
    pairs = inv_freq.shape[0]
    args = (_plain(q_weight, "q_weight", dtype, (D,), index), _plain(k_weight, "k_weight", dtype, (D,), index),
            _plain(positions, "positions", torch.int32, tokens, index),
            _plain(inv_freq, "inv_freq", torch.float32, (pairs,), index), code,
            tokens[0] if len(tokens) == 2 else 1, tokens[-1], shape[-2], k_shape[-2], D, 2 * pairs,
            1 if interleaved else 0, eps)
    return index, rq, rk, args


def qk_norm_rope(q, k, q_weight, k_weight, positions, inv_freq, eps=1e-6, interleaved=False, out=None):
    """Per-head RMS norm with a learned weight, then the position rotation, of q and k in one pass.

    q [B,S,Hq,D] and k [B,S,Hk,D] (or [tokens,H,D]) may have any strides but a contiguous
    last axis, so parts of a fused projection's output are taken as they are.  positions: int32
    [B,S]; inv_freq: fp32, one frequency per rotated pair (2 * len(inv_freq) elements of a head
    are rotated: elements i and i + len, or 2i and 2i + 1 if `interleaved`).  Returns the new
    (q, k), written to the pair `out` if given; out=(q, k) works in place.  Like every operator here it
    records nothing for autograd, also where an input requires a gradient: qk_norm_rope_backward is called
    by hand.  kcg_qk_norm_rope.
    """
    index, rq, rk, args = _norm_rope_args(q, k, q_weight, k_weight, positions, inv_freq, eps, interleaved)
    if out is None:
        q_out = torch.empty_like(q, memory_format=_contiguous)
        k_out = torch.empty_like(k, memory_format=_contiguous)
        ro, rp = _new_rows(q_out), _new_rows(k_out)
    else:
        q_out, k_out = out
        ro = _rows(q_out, "out[0]", q.dtype, index, q.shape)
        rp = _rows(k_out, "out[1]", q.dtype, index, k.shape)
    _call(lib.load().kcg_qk_norm_rope, index, rq, rk, ro, rp, *args)
    return q_out, k_out


def qk_norm_rope_backward(dq, dk, q, k, q_weight, k_weight, positions, inv_freq, eps=1e-6, interleaved=False,
                          workspace=None):
    """Gradients (q, k, q_weight, k_weight) of qk_norm_rope from those of its outputs.

    The other arguments are the forward call's inputs.  workspace: a contiguous device tensor
    of at least kcg_qk_norm_rope_backward_ws_bytes bytes (allocated if not given).
    """
    index, rq, rk, args = _norm_rope_args(q, k, q_weight, k_weight, positions, inv_freq, eps, interleaved)
    dtype, shape, k_shape = q.dtype, q.shape, k.shape
    rdq, rdk = _rows(dq, "dq", dtype, index, shape), _rows(dk, "dk", dtype, index, k_shape)
    L = lib.load()
    gq, gk = torch.empty_like(q, memory_format=_contiguous), torch.empty_like(k, memory_format=_contiguous)
    gwq, gwk = torch.empty_like(q_weight), torch.empty_like(k_weight)
    # (a shape that has no workspace is one that the call refuses)
    address, size, held = _workspace(workspace, L.kcg_qk_norm_rope_backward_ws_bytes(*args[5:10]) or 16, index, q.device)
    _call(L.kcg_qk_norm_rope_backward, index, rdq, rdk, rq, rk, _new_rows(gq), _new_rows(gk), args[0], args[1],
          gwq.data_ptr(), gwk.data_ptr(), *args[2:], address, size)
    return gq, gk, gwq, gwk


class KvCache:
    """A paged key/value cache over tensors of the caller.

    k, v: [pages, heads, page_size, dim], bfloat16 or float8_e4m3fn, contiguous; for
    float8_e4m3fn also k_exp, v_exp: uint8 [pages, heads, page_size], a row standing for its
    values times 2^(exponent - 127).  page_size is 16, 32, 64, 128 or 256, dim 64 or 128.  The
    handle keeps the tensors alive and their addresses at hand: they must not be resized.
    """

    def __init__(self, k, v, k_exp=None, v_exp=None):
        if not isinstance(k, _Tensor) or k.dim() != 4 or not k.is_cuda:
            raise ValueError("k must be a [pages, heads, page_size, dim] device tensor")
        if k.dtype not in (torch.bfloat16, torch.float8_e4m3fn):
            raise ValueError("a cache holds bfloat16 or float8_e4m3fn, not %s" % k.dtype)
        _check(k, "k", k.dtype, k.shape, k.device)
        _check(v, "v", k.dtype, k.shape, k.device)
        if k.dtype == torch.float8_e4m3fn:
            _check(k_exp, "k_exp", torch.uint8, k.shape[:3], k.device)
            _check(v_exp, "v_exp", torch.uint8, k.shape[:3], k.device)
        elif k_exp is not None or v_exp is not None:
            raise ValueError("a bfloat16 cache has no exponents")
        self.k, self.v, self.k_exp, self.v_exp = k, v, k_exp, v_exp
        self.index, self.device = k.get_device(), k.device
        pages, self.heads, self.page_size, self.dim = k.shape
        eight = k.dtype == torch.float8_e4m3fn
        if max(k.shape) > 0x7fffffff:
            raise ValueError("the cache's extents must be 32-bit numbers")
        self._c = lib.KvCache(k.data_ptr(), v.data_ptr(), k_exp.data_ptr() if eight else None,
                              v_exp.data_ptr() if eight else None, E4M3 if eight else BF16, pages, self.page_size,
                              self.heads, self.dim)

    @classmethod
    def empty(cls, pages, heads, page_size, dim, dtype=torch.float8_e4m3fn, device="cuda"):
        """A cache with memory of its own.  What it holds before the first write is undefined."""
        k, v = (torch.empty((pages, heads, page_size, dim), dtype=dtype, device=device) for _ in range(2))
        if dtype != torch.float8_e4m3fn:
            return cls(k, v)
        return cls(k, v, *(torch.empty((pages, heads, page_size), dtype=torch.uint8, device=device) for _ in range(2)))


def _cache_device(cache):
    if not isinstance(cache, KvCache):
        raise ValueError("cache must be a KvCache")
    return cache.index


def kv_cache_write(cache, k, v, slots):
    """Writes keys and values [B,S,heads,dim] (or [tokens,heads,dim]) to the int32 slots [B,S].

    A slot is page * page_size + place; -1 (padding) and any other slot outside the cache is
    not written, and of tokens with the same slot the last one is.  fp32 or bf16 rows are
    rounded to the cache's type; kcg_kv_cache_write says how.
    """
    index = _cache_device(cache)
    if not isinstance(k, _Tensor) or k.dtype not in _DTYPES:
        raise ValueError("k must be a float32 or bfloat16 tensor")
    dtype, shape = k.dtype, k.shape
    rk, rv = _rows(k, "k", dtype, index), _rows(v, "v", dtype, index, shape)
    if shape[-2:] != (cache.heads, cache.dim):
        raise ValueError("k must have the cache's heads and dim %s" % ((cache.heads, cache.dim),))
    _call(lib.load().kcg_kv_cache_write, index, cache._c, rk, rv, _DTYPES[dtype],
          _plain(slots, "slots", torch.int32, shape[:-2], index), shape[0] if len(shape) == 4 else 1, shape[-3])


def kv_cache_read(cache, slots, out_dtype=torch.bfloat16, out=None):
    """Keys and values of the int32 slots [B,S] (or [tokens]) as rows [..., heads, dim].

    A slot outside the cache gives rows of zeros.  out: the pair of tensors to write, with any
    strides but a contiguous last axis.
    """
    index = _cache_device(cache)
    if not isinstance(slots, _Tensor) or slots.dim() not in (1, 2):
        raise ValueError("slots must be an int32 tensor [B,S] or [tokens]")
    shape = tuple(slots.shape)
    at = _plain(slots, "slots", torch.int32, shape, index)
    B, S = shape if len(shape) == 2 else (1, shape[0])
    shape += (cache.heads, cache.dim)
    if out is None:
        if out_dtype not in _DTYPES:
            raise ValueError("a cache is read as float32 or bfloat16")
        k = torch.empty(shape, dtype=out_dtype, device=cache.device)
        v = torch.empty_like(k)
        rk, rv = _new_rows(k), _new_rows(v)
    else:
        k, v = out
        out_dtype = k.dtype if isinstance(k, _Tensor) else None
        if out_dtype not in _DTYPES:
            raise ValueError("a cache is read as float32 or bfloat16")
        rk, rv = _rows(k, "out[0]", out_dtype, index, shape), _rows(v, "out[1]", out_dtype, index, shape)
    _call(lib.load().kcg_kv_cache_read, index, cache._c, at, rk, rv, _DTYPES[out_dtype], B, S)
    return k, v


def fmha_cache_workspace_bytes(cache, table_width, batch, drafts, heads):
    """Bytes of workspace with which fmha_cache can split long sequences as it prefers to."""
    _cache_device(cache)
    return int(lib.load().kcg_fmha_cache_ws_bytes(cache._c, table_width, batch, drafts, heads))


def fmha_cache(q, cache, block_table, context_lens, draft_lens=None, tree_mask=None, scale=1.0, out=None,
               out_dtype=None, workspace=None):
    """Attention of each sequence's newest tokens (one, a chain or a tree of drafts) over a cache.

    q: bf16 [B,N,Hq,dim], N up to 64.  Sequence b has context_lens[b] keys that every query sees
    and behind them those of its draft_lens[b] (default: N) drafted tokens, all already written;
    block_table[b, j // page_size] is key j's page.  tree_mask: int64 [B,N], bit j of [b,n] says
    that drafted token n sees drafted token j (default: a chain, j <= n).  Lengths and table are
    int32.  Rows of `out` from draft_lens[b] on stay as they were.  kcg_fmha_cache says the rest.
    """
    index = _cache_device(cache)
    if not isinstance(q, _Tensor) or q.dim() != 4:
        raise ValueError("q must be a [B,N,H,dim] tensor")
    rq = _rows(q, "q", torch.bfloat16, index)
    shape = q.shape
    B, N, Hq, D = shape
    if D != cache.dim or Hq % cache.heads:
        raise ValueError("q must have the cache's dim and a multiple of its heads")
    if not isinstance(block_table, _Tensor) or block_table.dim() != 2:
        raise ValueError("block_table must be an int32 tensor [B, pages]")
    width = block_table.shape[1]
    if width >= _TOO_MANY:
        raise ValueError("block_table must have fewer than 2^31 pages to a sequence")
    table = _plain(block_table, "block_table", torch.int32, (B, width), index)
    context = _plain(context_lens, "context_lens", torch.int32, (B,), index)
    drafts = None if draft_lens is None else _plain(draft_lens, "draft_lens", torch.int32, (B,), index)
    tree = None if tree_mask is None else _plain(tree_mask, "tree_mask", torch.int64, (B, N), index)
    if out is None:
        out_dtype = out_dtype or torch.bfloat16
        out = (torch.empty if draft_lens is None else torch.zeros)(shape, dtype=out_dtype, device=cache.device)
    elif not isinstance(out, _Tensor) or out_dtype not in (None, out.dtype):
        raise ValueError("out must be a tensor of dtype out_dtype")
    out_dtype = out.dtype
    if out_dtype not in _DTYPES:
        raise ValueError("attention over a cache writes bfloat16 or float32, not %s" % out_dtype)
    L = lib.load()
    need = 0 if workspace is not None else L.kcg_fmha_cache_ws_bytes(cache._c, width, B, N, Hq)
    address, size, held = _workspace(workspace, need, index, cache.device)
    _call(L.kcg_fmha_cache, index, rq, cache._c, table, width, context, drafts, tree,
          _rows(out, "out", out_dtype, index, shape), _DTYPES[out_dtype], B, N, Hq, scale, address, size)
    return out
