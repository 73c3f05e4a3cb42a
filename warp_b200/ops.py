"""Torch-tensor front end of the C ABI (include/warp_cuda.h).

Names follow the reference functions whose arithmetic each call computes:

    mvq_matvec      waste_mvq_rows_f32      (src/model.c:423-519)
    vq_build_lut    vq_build_lut / lutb_range_avx512 (model.c:3864, simd_avx512.c:90)
    vq_apply        vq_apply / vq_rows      (model.c:4152, 3909-3977)
    vq_dequant      tools/kimi_ref.py:240-273 (expert dequant)
    vq4p_lut        vq_build_lut (4 x 64) + vq_quant_lut (model.c:3815, 4063)
    vq4p_apply      waste_vq_rows_p6        (model.c:4076-4113)
    vq_encode       waste_vq_encode         (src/vq.c:99)
    qwen_moe_route  waste_qwen_moe_route    (src/qwen_moe.c:10-44)
    MoELayer        qwen_moe_layer / moe_layer (model.c:8180, 5488)

The attention half of a decoder block, which the reference computes per model
family on the CPU, is served by operators of its own shape:

    rope_inv_freq   rotary frequencies, plain or stretched for long contexts
    qk_norm_rope    norms of queries and keys for each head, and the rotation
    kv_slots        where a step's tokens go in the pages, once for all layers
    kv_append       qk_norm_rope with keys and values written to the pages
    paged_attention attention over the pages, with or without a shared prefix

and a step that checks drafted tokens, several continuations of a request at once:

    page_pool       the pages that are free, for step_plan
    step_plan       pages, slots, positions and tree masks of a step, on the device
    tree_attention  paged_attention where a request's queries are the nodes of a tree
    pick_tokens     penalties, biases and masks on logits, and the largest of each row
    tree_accept     the path of drafted tokens that were picked, its keys put in order

Every tensor argument must already be on the CUDA device; calls are
asynchronous on torch's current stream.  A failure raises ffi.WarpError.
"""
import ctypes
import math
import struct

import torch

from . import ffi
from .container import ENTRIES, STAGES, VEC, parse_header


def _p(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream():
    # torch.cuda.current_stream().cuda_stream without the Stream object around it
    return ctypes.c_void_p(torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice()))


def _cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("warp_b200 ops take CUDA tensors")


def mvq_matvec(W, ws, X, out, in_, group, bits, rowbytes=None):
    """Y[b][o] = sum_k f16(ws[o,k]) * sum_i q(o,k*g+i) * X[b][k*g+i]."""
    _cuda(W, ws, X)
    if rowbytes is None:
        rowbytes = (in_ + group - 1) // group * group * bits // 8
    X2 = X.reshape(-1, in_).contiguous()
    if X2.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("activations must be fp32 or bf16")
    Y = torch.empty(X2.shape[0], out, dtype=torch.float32, device=X.device)
    ffi.check(ffi.load().warp_mvq_matvec(
        _p(W), _p(ws), _p(X2), int(X2.dtype == torch.bfloat16), _p(Y), X2.shape[0], out,
        in_, group, bits, rowbytes, _stream()))
    return Y


def vq_build_lut(booksT, x, cb_base):
    """lut[v][s][c] = FMA chain over d of x[8v+d] * booksT[cb_base+s][d][c]."""
    _cuda(booksT, x)
    nv = x.numel() // VEC
    lut = torch.empty(nv, STAGES, ENTRIES, dtype=torch.float32, device=x.device)
    ffi.check(ffi.load().warp_vq_lut_build(_p(lut), _p(booksT), _p(x.contiguous()), nv,
                                           cb_base, _stream()))
    return lut


def vq_apply(idx, scale, lut, M, ordered=False):
    """y[r] = f16(scale[r]) * sum_v T_v[i0] + T_v[i1] + T_v[i2]."""
    _cuda(idx, scale, lut)
    y = torch.empty(M, dtype=torch.float32, device=lut.device)
    ffi.check(ffi.load().warp_vq_apply(_p(y), _p(idx), _p(scale), _p(lut), M, lut.shape[0],
                                       int(ordered), _stream()))
    return y


def vq4p_lut(booksT, x, cb_base=0):
    """VQ4P int8 table of x: (q [nv][4][64] int8, lscale [ceil(nv/32)])."""
    _cuda(booksT, x)
    nv = x.numel() // VEC
    q = torch.empty(nv, 4, 64, dtype=torch.int8, device=x.device)
    ls = torch.empty((nv + 31) // 32, dtype=torch.float32, device=x.device)
    ffi.check(ffi.load().warp_vq4p_lut(_p(q), _p(ls), _p(booksT.contiguous()), booksT.shape[0],
                                       _p(x.contiguous()), nv, cb_base, _stream()))
    return q, ls


def vq4p_apply(idx, scale, q, lscale, M):
    """waste_vq_rows_p6: y[r] = f16(scale[r]) * sum_blk lscale[blk] * sum(lookups)."""
    _cuda(idx, scale, q, lscale)
    y = torch.empty(M, dtype=torch.float32, device=q.device)
    ffi.check(ffi.load().warp_vq4p_apply(_p(y), _p(idx), _p(scale), _p(q), _p(lscale), M,
                                         q.shape[0], _stream()))
    return y


def vq_matmul(X, idx, scale, books, M, cb_base=0):
    """Y[t][r] = f16(scale[r]) * sum_k W~[r][k] X[t][k] on the tensor cores
    (fp16 operands, fp32 accumulation); X [T][N] fp32 -> Y [T][M] fp32."""
    _cuda(X, idx, scale, books)
    X2 = X.reshape(-1, X.shape[-1]).contiguous().float()
    T, N = X2.shape
    Y = torch.empty(T, M, dtype=torch.float32, device=X.device)
    ffi.check(ffi.load().warp_vq_matmul(_p(Y), _p(X2), T, _p(idx), _p(scale), _p(books), M, N,
                                        cb_base, _stream()))
    return Y


def umma_status(clear=True):
    ffi.check(ffi.load().warp_umma_status(int(clear)))


def vq_dequant(idx, scale, books, M, N, cb_base):
    """Dequantized VQ3R matrix, fp32 [M][N], bit-exact."""
    _cuda(idx, scale, books)
    W = torch.empty(M, N, dtype=torch.float32, device=books.device)
    ffi.check(ffi.load().warp_vq_dequant(_p(W), _p(idx), _p(scale), _p(books), M, N,
                                         cb_base, _stream()))
    return W


def vq_encode(X, books):
    """Residual nearest-centroid codes, X [n][8] fp32, books [stages][256][8]."""
    _cuda(X, books)
    X = X.reshape(-1, VEC).contiguous()
    codes = torch.empty(X.shape[0], books.shape[0], dtype=torch.uint8, device=X.device)
    ffi.check(ffi.load().warp_vq_encode(_p(X), X.shape[0], _p(books.contiguous()),
                                        books.shape[0], _p(codes), _stream()))
    return codes


def qwen_moe_route(logits, K, renorm=True):
    """Softmax top-k in selection order; logits [T][E]."""
    _cuda(logits)
    L = logits.reshape(-1, logits.shape[-1]).contiguous().float()
    T, E = L.shape
    idx = torch.empty(T, K, dtype=torch.int32, device=L.device)
    w = torch.empty(T, K, dtype=torch.float32, device=L.device)
    ffi.check(ffi.load().warp_qwen_route(_p(L), T, E, K, int(renorm), _p(idx), _p(w),
                                         _stream()))
    return idx, w


def moe_route(logits, K, score_func, bias=None, renorm=True, routed_scale=1.0):
    """moe_layer's routing (router_scores + biased selection + renorm +
    routed_scale); logits [T][E]."""
    _cuda(logits, bias)
    L = logits.reshape(-1, logits.shape[-1]).contiguous().float()
    T, E = L.shape
    idx = torch.empty(T, K, dtype=torch.int32, device=L.device)
    w = torch.empty(T, K, dtype=torch.float32, device=L.device)
    ffi.check(ffi.load().warp_moe_route(_p(L), T, E, K, int(score_func), _p(bias), int(renorm),
                                        float(routed_scale), _p(idx), _p(w), _stream()))
    return idx, w


def rmsnorm(x, w=None, eps=1e-6, out=None):
    """waste_rmsnorm over the last dimension."""
    _cuda(x, w)
    x2 = x.reshape(-1, x.shape[-1]).contiguous()
    if out is None:
        out = torch.empty_like(x2)
    ffi.check(ffi.load().warp_rmsnorm(_p(x2), _p(w), _p(out), x2.shape[0], x2.shape[1],
                                      eps, _stream()))
    return out


_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def rope_inv_freq(rot_dim, base=10000.0, scaling="none", factor=1.0, trained=None,
                  beta_fast=32.0, beta_slow=1.0, device=None):
    """(inv_freq, rot_scale): fp64 radians a position for each of rot_dim/2
    pairs, base^(-2i/rot_dim), and the factor on cos and sin.  scaling:

        "none"    as it is
        "linear"  positions divided by `factor`
        "ntk"     base * factor^(rot_dim/(rot_dim-2))
        "yarn"    pairs that turn more than beta_fast times over `trained`
                  positions as they are, fewer than beta_slow divided by
                  `factor`, a ramp between; rot_scale 0.1 ln(factor) + 1
    """
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError("rot_dim must be even and at least 2")
    if scaling not in ("none", "linear", "ntk", "yarn"):
        raise ValueError(f"unknown scaling {scaling!r}")
    if scaling != "none" and not factor >= 1.0:
        raise ValueError("factor must be at least 1")
    if scaling == "ntk":
        if rot_dim == 2:
            raise ValueError("ntk scaling needs rot_dim above 2")
        base = base * factor ** (rot_dim / (rot_dim - 2))
    f = float(base) ** -(torch.arange(0, rot_dim, 2, dtype=torch.float64) / rot_dim)
    scale = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        if not trained:
            raise ValueError("yarn scaling needs the trained context length")

        def pair(turns):
            return rot_dim * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo = max(0, math.floor(pair(beta_fast)))
        hi = min(rot_dim - 1, math.ceil(pair(beta_slow)))
        i = torch.arange(rot_dim // 2, dtype=torch.float64)
        ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        f = f * (1 - ramp) + f / factor * ramp
        scale = 0.1 * math.log(factor) + 1.0
    return f.to(device), scale


def _device(x):
    """The number of torch's current device, on whose current stream calls run, for
    a call with tensor x."""
    if not x.is_cuda:           # without a device there is no current one to ask for
        _cuda(x)
    return torch._C._cuda_getDevice()


def _elsewhere(x):
    """Refuses a tensor whose device is not the current one."""
    _cuda(x)
    raise ValueError(f"a tensor is on {x.device}, which is not the current device")


def _vec_ok(x, n, dtype, dev):
    if x.get_device() != dev:
        _elsewhere(x)
    return x.dtype is dtype and x.numel() == n and x.is_contiguous()


def _rows(x, name, T, D, dtype, dev):
    """(heads, token stride, head stride, address) of [T][heads][D] on the
    device with contiguous heads; the stride of an axis of one entry is 0, as
    it has no meaning."""
    if x.get_device() != dev:
        _elsewhere(x)
    shape, strides = x.shape, x.stride()
    if len(shape) != 3 or shape[0] != T or shape[2] != D or x.dtype is not dtype or \
            (strides[2] != 1 and D > 1):
        raise ValueError(f"{name} must be [tokens][heads][head_dim] with contiguous heads, all "
                         "of one dtype, token count and head_dim")
    heads = shape[1]
    return heads, strides[0] if T > 1 else 0, strides[1] if heads > 1 else 0, x.data_ptr()


def _rope_pack(q, k, v, positions, inv_freq, q_norm, k_norm, eps, interleaved, rot_scale, q_out,
               k_out, out_dtype):
    x = k if q is None else q
    if x is None:
        raise ValueError("neither queries nor keys")
    dt = x.dtype
    if x.dim() != 3 or dt not in _TYPES:
        raise ValueError("queries and keys must be [tokens][heads][head_dim], fp32, fp16 or bf16")
    dev = _device(x)
    T, nk, D = x.shape
    nq = qt = qh = qp = kt = kh = kp = vt = vh = vp = qn = kn = f = p = rot = 0
    if q is not None:
        nq, qt, qh, qp = _rows(q, "q", T, D, dt, dev)
        nk = 0
    if k is not None:
        nk, kt, kh, kp = _rows(k, "k", T, D, dt, dev)
    if v is not None:
        nv, vt, vh, vp = _rows(v, "v", T, D, dt, dev)
        if nv != nk:
            raise ValueError("v must have k's heads")
    if inv_freq is not None:
        rot = 2 * inv_freq.numel()
        if not _vec_ok(inv_freq, rot // 2, torch.float64, dev):
            raise ValueError("inv_freq must be contiguous float64")
        if positions is None or not _vec_ok(positions, T, torch.int32, dev):
            raise ValueError("positions must be contiguous int32 [tokens]")
        f, p = inv_freq.data_ptr(), positions.data_ptr()
    if q_norm is not None:
        if not _vec_ok(q_norm, D, torch.float32, dev):
            raise ValueError("q_norm must be contiguous float32 [head_dim]")
        qn = q_norm.data_ptr()
    if k_norm is not None:
        if not _vec_ok(k_norm, D, torch.float32, dev):
            raise ValueError("k_norm must be contiguous float32 [head_dim]")
        kn = k_norm.data_ptr()
    return ffi.ROPE_DESC.pack(
        T, nq, nk, D, _TYPES[dt], _TYPES.get(out_dtype, -1), qp, kp, vp, qt, qh, kt, kh, vt, vh,
        0 if q_out is None else q_out.data_ptr(), 0 if k_out is None else k_out.data_ptr(),
        qn, kn, eps, f, rot, interleaved, rot_scale, p)


def _dense(x, dtype):
    """A new contiguous tensor of x's shape."""
    return torch.empty_like(x, dtype=dtype, memory_format=torch.contiguous_format)


def qk_norm_rope(q, k, positions, inv_freq, q_norm=None, k_norm=None, eps=1e-6,
                 interleaved=False, rot_scale=1.0, out_dtype=None):
    """Per-head RMSNorm (with q_norm / k_norm, fp32 [head_dim]) and rotary
    positions of queries and keys in one launch (warp_qk_norm_rope).

    q [T][Hq][D] and k [T][Hk][D], any strides with contiguous heads (parts of
    one projection's rows, say); either may be None.  positions int32 [T];
    inv_freq fp64 [R/2] rotates the first R dimensions (rope_inv_freq; None:
    no rotation).  Returns contiguous (q_out, k_out) in out_dtype: the inputs'
    own, or any for fp32 inputs."""
    if out_dtype is None and (q is not None or k is not None):
        out_dtype = (q if q is not None else k).dtype
    q_out = None if q is None else _dense(q, out_dtype)
    k_out = None if k is None else _dense(k, out_dtype)
    d = _rope_pack(q, k, None, positions, inv_freq, q_norm, k_norm, eps, interleaved, rot_scale,
                   q_out, k_out, out_dtype)
    ffi.check(ffi.load().warp_qk_norm_rope(d, _stream()))
    return q_out, k_out


def _pages_pack(k_pages, v_pages, dev, skip=0):
    """The description of pages; `skip`: axes before theirs."""
    if k_pages.get_device() != dev or v_pages.get_device() != dev:
        _elsewhere(k_pages if k_pages.get_device() != dev else v_pages)
    shape, ks, vs = k_pages.shape, k_pages.stride(), v_pages.stride()
    same = shape == v_pages.shape
    if skip:
        shape, ks, vs = shape[skip:], ks[skip:], vs[skip:]
    if len(shape) != 4 or not same or k_pages.dtype is not v_pages.dtype or \
            (shape[3] > 1 and (ks[3] != 1 or vs[3] != 1)):
        raise ValueError("k_pages and v_pages must be [pages][page_size][kv_heads][head_dim] "
                         "of one shape and dtype with contiguous heads")
    n, size, heads, dim = shape
    if n == 1 or size == 1 or heads == 1:   # the stride of an axis of one entry has no meaning
        ks, vs = ([s if e > 1 else 0 for s, e in zip(x, shape)] for x in (ks, vs))
    return ffi.KV_PAGES.pack(k_pages.data_ptr(), v_pages.data_ptr(),
                             _TYPES.get(k_pages.dtype, -1), size, heads, dim, n, ks[0], ks[1],
                             ks[2], vs[0], vs[1], vs[2])


def kv_append(q, k, v, k_pages, v_pages, slots, positions, inv_freq, q_norm=None, k_norm=None,
              eps=1e-6, interleaved=False, rot_scale=1.0):
    """qk_norm_rope with the keys' results and the values written to the pages
    in the same launch (warp_kv_append); returns q's result, in the pages'
    dtype (None for q None).

    k_pages / v_pages [pages][page_size][Hk][D], fp16 or bf16, any strides with
    contiguous heads (a transposed [pages][Hk][page_size][D], say); slots int64
    [T]: token t's slot (page * page_size + offset; negative: not stored), as
    kv_slots makes them."""
    if k is None or v is None:
        raise ValueError("kv_append needs keys and values")
    dev = _device(k)
    c = _pages_pack(k_pages, v_pages, dev)
    q_out = None if q is None else _dense(q, k_pages.dtype)
    d = _rope_pack(q, k, v, positions, inv_freq, q_norm, k_norm, eps, interleaved, rot_scale,
                   q_out, None, k_pages.dtype)
    if not _vec_ok(slots, k.shape[0], torch.int64, dev):
        raise ValueError("slots must be contiguous int64 [tokens]")
    ffi.check(ffi.load().warp_kv_append(d, c, slots.data_ptr(), _stream()))
    return q_out


def kv_slots(q_start, kv_len, pages, page_size, tokens, base=0):
    """(positions int32 [T], slots int64 [T]) of a step's tokens for kv_append
    (warp_kv_slots): q_start int32 [B+1], kv_len int32 [B] own keys with the
    new ones counted, pages int32 [B][n]; base: the shared prefix's length.
    Keys past a row's pages or in a page of negative number have no slot, and
    attn_status raises."""
    B, row, wide = _batch(q_start, kv_len, pages, _device(kv_len))
    positions = torch.empty(tokens, dtype=torch.int32, device=q_start.device)
    slots = torch.empty(tokens, dtype=torch.int64, device=q_start.device)
    ffi.check(ffi.load().warp_kv_slots(
        q_start.data_ptr(), kv_len.data_ptr(), B, tokens, pages.data_ptr(), row, wide,
        page_size, base, positions.data_ptr(), slots.data_ptr(), _stream()))
    return positions, slots


def _batch(q_start, kv_len, pages, dev):
    """(requests, row stride and width of the page table)."""
    B = kv_len.numel()
    if not _vec_ok(kv_len, B, torch.int32, dev):
        raise ValueError("kv_len must be contiguous int32 [batch]")
    if not _vec_ok(q_start, B + 1, torch.int32, dev):
        raise ValueError("q_start must be contiguous int32 [batch + 1]")
    if pages.get_device() != dev:
        _elsewhere(pages)
    shape, strides = pages.shape, pages.stride()
    if len(shape) != 2 or shape[0] != B or pages.dtype is not torch.int32 or \
            (strides[1] != 1 and shape[1] > 1):
        raise ValueError("pages must be int32 [batch][pages a request], rows contiguous")
    return B, strides[0] if B > 1 else 0, shape[1]


def paged_attention(q, k_pages, v_pages, pages, kv_len, q_start, max_q, max_kv, scale=None,
                    causal=True, prefix_pages=None, prefix_len=0, out=None):
    """Attention of ragged queries over paged keys and values
    (warp_paged_attention).

    q [T][Hq][D] fp16 or bf16, D 64 or 128; k_pages / v_pages as for
    kv_append, Hq a multiple of Hk.  Request b owns tokens q_start[b] ..
    q_start[b+1]-1 and kv_len[b] keys in the pages of pages[b] (all int32 on
    the device); max_q and max_kv bound both on the host.  causal: the queries
    are the request's last positions; False: every query sees every key.  With
    prefix_len, all queries also see the first prefix_len keys of prefix_pages
    (int32 [n]), before their own.  A query that sees nothing gets zeros; a
    token of no request is not written.  scale: 1/sqrt(D) by default.  Returns
    [T][Hq][D] in q's dtype."""
    return _attention(q, k_pages, v_pages, pages, kv_len, q_start, max_q, max_kv, scale, causal,
                      prefix_pages, prefix_len, out)


def _attention(q, k_pages, v_pages, pages, kv_len, q_start, max_q, max_kv, scale, causal,
               prefix_pages, prefix_len, out, seen=None):
    dev = _device(q)
    c = _pages_pack(k_pages, v_pages, dev)
    B, row, wide = _batch(q_start, kv_len, pages, dev)
    dt = q.dtype
    if q.dim() != 3 or dt not in _TYPES:
        raise ValueError("q must be [tokens][heads][head_dim], fp16 or bf16")
    T, _, D = q.shape
    Hq, qt, qh, qp = _rows(q, "q", T, D, dt, dev)
    if out is None:
        out = _dense(q, dt)
    else:
        if out.get_device() != dev:
            _elsewhere(out)
        if out.shape != q.shape or out.dtype is not dt or not out.is_contiguous():
            raise ValueError("out must be contiguous, of q's shape and dtype")
    pp = 0
    if prefix_len:
        if prefix_pages is None or prefix_len > prefix_pages.numel() * k_pages.shape[1]:
            raise ValueError("prefix_pages hold fewer than prefix_len keys")
        if not _vec_ok(prefix_pages, prefix_pages.numel(), torch.int32, dev):
            raise ValueError("prefix_pages must be contiguous int32 [n]")
        pp = prefix_pages.data_ptr()
    if seen is not None:
        words = _seen_ok(seen, T, max_q, dev)
    d = ffi.ATTN_DESC.pack(
        B, T, Hq, k_pages.shape[2], D, _TYPES[dt], qp, qt, qh,
        out.data_ptr(), q_start.data_ptr(), kv_len.data_ptr(), pages.data_ptr(), row, wide, max_q,
        max_kv, causal, (D or 1) ** -0.5 if scale is None else scale, pp, prefix_len)
    lib = ffi.load()
    need = (lib.warp_attn_scratch if seen is None else lib.warp_tree_scratch)(d, c)
    if need < 0:
        ffi.check(need)
    # from torch's allocator: ordered by the stream, and private to a graph
    # where one is being captured
    scratch = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    at = scratch.data_ptr() if need else None
    if seen is None:
        ffi.check(lib.warp_paged_attention(d, c, at, _stream()))
    else:
        ffi.check(lib.warp_tree_attention(d, c, seen.data_ptr(), words, at, _stream()))
    return out


def page_pool(pages, device="cuda"):
    """A pool with all of `pages` pages free, for step_plan: int32 [1 + pages], how
    many are free and their numbers, of which page 0 comes off first."""
    return torch.arange(pages, -1, -1, dtype=torch.int32, device=device)


def step_plan(q_start, kv_len, pages, page_size, tokens, base=0, held=None, pool=None,
              parents=None, max_q=0):
    """A step's plan from its requests' lengths, on the device (warp_step_plan):
    (positions int32 [T], slots int64 [T]) of its tokens, as kv_slots makes them.

    q_start int32 [B+1], kv_len int32 [B] own keys with the new ones counted,
    pages int32 [B][n].  With held (int32 [B], pages that each row has) and pool
    (page_pool) the rows first give back the pages that kv_len does not need and
    take those that it does, in place; a length of 0 gives all back.  A pool that
    runs empty leaves held short and the keys without a slot, and attn_status raises.

    With parents (int32 [T]: a node's parent among its request's tokens, -1 for
    the first) each request's tokens are the nodes of a tree, max_q at most: their
    positions go by depth, and a third result, seen int64 [T][ceil(max_q / 64)], has
    bit m of a node's words set for each node m that it sees: its ancestors
    and itself."""
    dev = _device(kv_len)
    B, row, wide = _batch(q_start, kv_len, pages, dev)
    hp = pp = np = up = sp = 0
    if held is not None or pool is not None:
        if held is None or pool is None:
            raise ValueError("held and pool go together")
        if not _vec_ok(held, B, torch.int32, dev):
            raise ValueError("held must be contiguous int32 [batch]")
        np = pool.numel() - 1
        if not _vec_ok(pool, np + 1, torch.int32, dev) or np < 0:
            raise ValueError("pool must be contiguous int32 [1 + pages]")
        hp, pp = held.data_ptr(), pool.data_ptr()
    seen = None
    if parents is not None:
        if not _vec_ok(parents, tokens, torch.int32, dev):
            raise ValueError("parents must be contiguous int32 [tokens]")
        if max_q < 1:
            raise ValueError("a tree's nodes need their bound max_q")
        seen = torch.empty(tokens, (max_q + 63) // 64, dtype=torch.int64, device=kv_len.device)
        up, sp = parents.data_ptr(), seen.data_ptr()
    positions = torch.empty(tokens, dtype=torch.int32, device=kv_len.device)
    slots = torch.empty(tokens, dtype=torch.int64, device=kv_len.device)
    d = ffi.PLAN_DESC.pack(B, tokens, q_start.data_ptr(), kv_len.data_ptr(), pages.data_ptr(), row,
                           wide, page_size, base, hp, pp, np, up, sp, max_q, positions.data_ptr(),
                           slots.data_ptr())
    ffi.check(ffi.load().warp_step_plan(d, _stream()))
    return (positions, slots) if parents is None else (positions, slots, seen)


def _seen_ok(seen, T, max_q, dev):
    """Words of a row of masks [T][words]."""
    if seen.get_device() != dev:
        _elsewhere(seen)
    if seen.dim() != 2 or seen.shape[0] != T or seen.dtype is not torch.int64 or \
            not seen.is_contiguous() or seen.shape[1] * 64 < min(max_q, T):
        raise ValueError("seen must be contiguous int64 [tokens][words] with a bit for each of "
                         "max_q nodes")
    return seen.shape[1]


def tree_attention(q, k_pages, v_pages, pages, kv_len, q_start, seen, max_q, max_kv, scale=None,
                   prefix_pages=None, prefix_len=0, out=None):
    """paged_attention where a request's queries are the nodes of a tree
    (warp_tree_attention): its own keys before its last n, one a query, are
    seen by all its queries, and of the last n query i sees those whose bits
    are set in its row of seen (step_plan's).  A query that sees nothing gets
    zeros."""
    if seen is None:
        raise ValueError("a tree needs its masks")
    return _attention(q, k_pages, v_pages, pages, kv_len, q_start, max_q, max_kv, scale, False,
                      prefix_pages, prefix_len, out, seen)


def _table(x, name, rows, wide, dtype, dev):
    """Row stride of [rows][wide], or of [wide] for all rows: 0."""
    if x.get_device() != dev:
        _elsewhere(x)
    shape, strides = x.shape, x.stride()
    if len(shape) not in (1, 2) or x.dtype is not dtype or shape[-1] < wide or \
            (len(shape) == 2 and shape[0] != rows) or (strides[-1] != 1 and shape[-1] > 1):
        raise ValueError(f"{name} must be {dtype} [rows][{wide}] or [{wide}], rows contiguous")
    return strides[0] if len(shape) == 2 and rows > 1 else 0


def pick_tokens(logits, q_start=None, max_q=None, history=None, history_len=None, repetition=None,
                frequency=None, presence=None, bias=None, allowed=None, drafted=None, seen=None,
                out=None):
    """The token of the largest adjusted logit of each row, int32 [T]; -1 where
    none is above -inf (warp_pick_tokens).

    logits [T][V] fp32, fp16 or bf16, rows contiguous; row t belongs to request t,
    or to the one with q_start[b] <= t < q_start[b+1] (int32 [B+1]).  max_q bounds
    the rows of a request; by default all of them are taken, with seen as many as its
    words have bits.  A row past the bound gets -1, and attn_status raises.  With c the
    number of times that a token is in the row's context,

        x > 0 ? x / repetition : x * repetition, then less frequency * c and
        presence, where c > 0 (float32 [B] each); plus bias (float32 [V] or
        [B][V]); -inf where allowed (int32 [T][ceil(V / 32)] or [ceil(V / 32)],
        a bit a token, the lowest first) has no bit.

    The bias is added behind the penalties, which do not see it (a sampler that
    penalises biased logits has it in front), and one context serves all three.
    The context: the first history_len[b] (int32 [B]) tokens of history[b] (int32
    [B][H]), and with drafted (int32 [T]) and seen (step_plan's) the drafted
    tokens of the nodes that the row's node sees.  out, of logits' shape and
    dtype, takes the adjusted logits; it may be logits itself.  A row of no
    request is not written."""
    dev = _device(logits)
    if logits.get_device() != dev:
        _elsewhere(logits)
    dt = logits.dtype
    if logits.dim() != 2 or dt not in _TYPES or logits.shape[1] < 1 or \
            (logits.stride(1) != 1 and logits.shape[1] > 1):
        raise ValueError("logits must be [rows][vocabulary], fp32, fp16 or bf16, rows contiguous")
    T, V = logits.shape
    row = logits.stride(0) if T > 1 else 0
    B = T
    if max_q is None:
        max_q = max(1, T if seen is None or seen.dim() != 2 else min(T, 64 * seen.shape[1]))
    qp = op = orow = hp = lp = hrow = wide = bp = brow = ap = arow = dp = sp = words = 0
    if q_start is not None:
        B = q_start.numel() - 1
        if B < 0 or not _vec_ok(q_start, B + 1, torch.int32, dev):
            raise ValueError("q_start must be contiguous int32 [batch + 1]")
        qp = q_start.data_ptr()
    if out is not None:
        if out.get_device() != dev:
            _elsewhere(out)
        if out.shape != logits.shape or out.dtype is not dt or (out.stride(1) != 1 and V > 1):
            raise ValueError("out must be of logits' shape and dtype, rows contiguous")
        op, orow = out.data_ptr(), out.stride(0) if T > 1 else 0
        if T > 1 and orow < V:
            raise ValueError("rows of out overlap")
    if history is not None or history_len is not None:
        if history is None or history_len is None:
            raise ValueError("history and history_len go together")
        if not _vec_ok(history_len, B, torch.int32, dev):
            raise ValueError("history_len must be contiguous int32 [batch]")
        if history.dim() != 2:
            raise ValueError("history must be int32 [batch][places]")
        hrow = _table(history, "history", B, 0, torch.int32, dev)
        hp, lp, wide = history.data_ptr(), history_len.data_ptr(), history.shape[1]
    if drafted is not None or seen is not None:
        if drafted is None or seen is None or q_start is None:
            raise ValueError("drafted, seen and q_start go together")
        if not _vec_ok(drafted, T, torch.int32, dev):
            raise ValueError("drafted must be contiguous int32 [rows]")
        words = _seen_ok(seen, T, max_q, dev)
        dp, sp = drafted.data_ptr(), seen.data_ptr()
    scalars = []
    for x in (repetition, frequency, presence):
        if x is not None and not _vec_ok(x, B, torch.float32, dev):
            raise ValueError("repetition, frequency and presence must be contiguous float32 [batch]")
        scalars.append(0 if x is None else x.data_ptr())
    if bias is not None:
        brow = _table(bias, "bias", B, V, torch.float32, dev)
        bp = bias.data_ptr()
    if allowed is not None:
        arow = _table(allowed, "allowed", T, (V + 31) // 32, torch.int32, dev)
        ap = allowed.data_ptr()
    if qp and not max_q:                    # which the kernels take for no work
        return torch.full((T,), -1, dtype=torch.int32, device=logits.device)
    picked = torch.empty(T, dtype=torch.int32, device=logits.device)
    d = ffi.PICK_DESC.pack(T, B, V, _TYPES[dt], max_q, logits.data_ptr(), row, op, orow,
                           picked.data_ptr(), qp, hp, lp, hrow, wide, *scalars, bp, brow, ap, arow,
                           dp, sp, words)
    lib = ffi.load()
    need = lib.warp_pick_scratch(d)
    if need < 0:
        ffi.check(need)
    scratch = torch.empty(need, dtype=torch.uint8, device=logits.device) if need else None
    ffi.check(lib.warp_pick_tokens(d, scratch.data_ptr() if need else None, _stream()))
    return picked


def tree_accept(drafted, picked, seen, q_start, kv_len, max_q, caches=(), pages=None):
    """The drafted tokens checked against what was picked, and the caches put in
    order (warp_tree_accept): (count int32 [B], path int32 [B][max_q], chosen int32
    [B][max_q], kv_after int32 [B]).

    drafted and picked int32 [T] of the nodes (a negative drafted token is never
    accepted); seen and max_q as for step_plan; kv_len int32 [B] with the nodes
    counted.  path holds the `count` nodes of the longest path from node 0 on which
    each drafted token is what was picked behind its parent, chosen what was picked behind
    them (the step's new tokens), both -1 from there on; kv_after = kv_len - nodes
    + count.

    caches: (k_pages, v_pages) of all layers, [layers][pages][page_size][Hk][D], or
    a list of each layer's pair, all of one layout and apart from one another; their keys
    and values of the path move behind the keys before the tree, pages int32 [B][n] being
    the page table."""
    dev = _device(kv_len)
    T, B = drafted.numel(), kv_len.numel()
    words = _seen_ok(seen, T, max_q, dev)
    if not _vec_ok(drafted, T, torch.int32, dev) or not _vec_ok(picked, T, torch.int32, dev):
        raise ValueError("drafted and picked must be contiguous int32 [tokens]")
    n = row = wide = tp = 0
    c = ks = vs = None
    if len(caches):
        if pages is None:
            raise ValueError("caches need the page table")
        _, row, wide = _batch(q_start, kv_len, pages, dev)
        tp = pages.data_ptr()
        n, c, ks, vs = _caches_pack(caches, dev)
    elif not _vec_ok(kv_len, B, torch.int32, dev):
        raise ValueError("kv_len must be contiguous int32 [batch]")
    elif not _vec_ok(q_start, B + 1, torch.int32, dev):
        raise ValueError("q_start must be contiguous int32 [batch + 1]")
    count, after = torch.empty_like(kv_len), torch.empty_like(kv_len)
    path = kv_len.new_empty((B, max_q))
    chosen = torch.empty_like(path)
    d = ffi.ACCEPT_DESC.pack(B, T, max_q, drafted.data_ptr(), picked.data_ptr(), seen.data_ptr(),
                             words, q_start.data_ptr(), kv_len.data_ptr(), tp, row, wide,
                             count.data_ptr(), path.data_ptr(), chosen.data_ptr(),
                             after.data_ptr())
    ffi.check(ffi.load().warp_tree_accept(d, c, n, ks, vs, _stream()))
    return count, path, chosen, after


def _caches_pack(caches, dev):
    """(layers, their layout, addresses of their keys and of their values)."""
    if isinstance(caches[0], torch.Tensor):
        k, v = caches
        if k.dim() != 5 or v.dim() != 5:
            raise ValueError("caches must be a pair [layers][pages][page_size][kv_heads][head_dim]")
        n = k.shape[0]
        if not n:
            return 0, None, None, None
        c = _pages_pack(k, v, dev, 1)
        at = []
        for x in (k, v):
            first, step = x.data_ptr(), x.stride(0) * x.element_size()
            at.append(struct.pack(f"@{n}P", *(range(first, first + n * step, step) if step
                                              else [first] * n)))
        return n, c, *at
    packed = [_pages_pack(k, v, dev) for k, v in caches]
    if any(x[16:] != packed[0][16:] for x in packed):
        raise ValueError("caches must have one shape, dtype and layout")
    at = [struct.pack(f"@{len(caches)}P", *(x.data_ptr() for x in side)) for side in zip(*caches)]
    return len(caches), packed[0], *at


def attn_status(clear=True):
    """Raises if an attention kernel left something out (a page or slot out of
    range, a length over its bound, a wait that gave up) since the last clear."""
    ffi.check(ffi.load().warp_attn_status(int(clear)))


class MoELayer:
    """One resident MoE layer on the device (warp_moe_layer_*).

    bank: uint8 CUDA tensor of E expert records (rec_bytes each, sorted by id);
    books/booksT: the layer's decoded codebooks; router: fp32 [E][hidden];
    shared: optional dict(gate_w, gate_s, up_w, up_s, down_w, down_s, inter,
    group, bits) of CUDA tensors; shared_gate: optional fp32 [hidden].
    tile_bank (default) re-tiles the bank in place on creation (see
    warp_moe_desc.tile_bank): read the records you need in container layout
    before creating the layer.
    """

    def __init__(self, bank, rec_bytes, books, booksT, router, hidden, inter, n_experts,
                 top_k, renorm=True, shared=None, shared_gate=None, max_tokens=1,
                 tile_bank=True, ep_rank=0, ep_size=1, prefill_tokens=0, router_kind=0,
                 score_func=0, score_bias=None, routed_scale=1.0, ep_mode=0):
        _cuda(bank, books, booksT, router, score_bias)
        self.keep = [bank, books, booksT, router, shared_gate, score_bias] + \
            (list(shared.values()) if shared else [])
        self.hidden, self.inter, self.E, self.K = hidden, inter, n_experts, top_k
        self.max_tokens = max_tokens
        d = ffi.MoEDesc()
        d.hidden, d.inter, d.n_experts, d.top_k, d.renorm = hidden, inter, n_experts, top_k, int(renorm)
        d.bank, d.rec_bytes = bank.data_ptr(), rec_bytes
        d.booksT, d.books, d.n_books = booksT.data_ptr(), books.data_ptr(), books.shape[0]
        d.router = router.data_ptr()
        if shared:
            d.shared_gate_w = shared["gate_w"].data_ptr()
            d.shared_up_w = shared["up_w"].data_ptr()
            d.shared_down_w = shared["down_w"].data_ptr()
            d.shared_gate_s = shared["gate_s"].data_ptr()
            d.shared_up_s = shared["up_s"].data_ptr()
            d.shared_down_s = shared["down_s"].data_ptr()
            d.shared_inter, d.shared_group = shared["inter"], shared["group"]
            d.shared_bits = shared["bits"]
        if shared_gate is not None:
            d.shared_gate = shared_gate.data_ptr()
        d.tile_bank = int(tile_bank)
        d.ep_rank, d.ep_size = int(ep_rank), int(ep_size)
        d.prefill_tokens = int(prefill_tokens)
        d.router_kind, d.score_func = int(router_kind), int(score_func)
        if score_bias is not None:
            d.score_bias = score_bias.data_ptr()
        d.routed_scale = float(routed_scale)
        d.ep_mode = int(ep_mode)
        self.ep_rank, self.ep_size = int(ep_rank), int(ep_size)
        self.desc = d
        h = ctypes.c_void_p()
        ffi.check(ffi.load().warp_moe_layer_create(ctypes.byref(d), max_tokens,
                                                   ctypes.byref(h)))
        self.handle = h

    def forward(self, x, residual=None, out=None, want_route=False):
        _cuda(x)
        x2 = x.reshape(-1, self.hidden)
        T = x2.shape[0]
        if out is None:
            out = torch.empty(T, self.hidden, dtype=torch.float32, device=x.device)
        idx = w = None
        if want_route:
            idx = torch.empty(T, self.K, dtype=torch.int32, device=x.device)
            w = torch.empty(T, self.K, dtype=torch.float32, device=x.device)
        ffi.check(ffi.load().warp_moe_layer_forward(
            self.handle, _p(x2), T, _p(residual), _p(out), _p(idx), _p(w), _stream()))
        return (out, idx, w) if want_route else out

    def forward_block(self, h, out, norm_w=None, eps=1e-6, want_route=False):
        """out = h + MoE(RMSNorm(h) * norm_w): the norm kernel into the
        layer's buffer, then the layer with residual h (warp_moe_block_forward);
        out must not alias h."""
        _cuda(h, out, norm_w)
        h2 = h.reshape(-1, self.hidden)
        T = h2.shape[0]
        idx = w = None
        if want_route:
            idx = torch.empty(T, self.K, dtype=torch.int32, device=h.device)
            w = torch.empty(T, self.K, dtype=torch.float32, device=h.device)
        ffi.check(ffi.load().warp_moe_block_forward(
            self.handle, _p(h2), T, _p(norm_w), float(eps), _p(out), _p(idx), _p(w), _stream()))
        return (out, idx, w) if want_route else out

    def prefill(self, x, residual=None, out=None, want_route=False):
        """The layer for T tokens on the tensor cores (warp_moe_layer_prefill)."""
        _cuda(x)
        x2 = x.reshape(-1, self.hidden).contiguous()
        T = x2.shape[0]
        if out is None:
            out = torch.empty(T, self.hidden, dtype=torch.float32, device=x.device)
        idx = w = None
        if want_route:
            idx = torch.empty(T, self.K, dtype=torch.int32, device=x.device)
            w = torch.empty(T, self.K, dtype=torch.float32, device=x.device)
        ffi.check(ffi.load().warp_moe_layer_prefill(
            self.handle, _p(x2), T, _p(residual), _p(out), _p(idx), _p(w), _stream()))
        return (out, idx, w) if want_route else out

    def slots_per_token(self):
        """S: top_k route slots plus the shared expert's column blocks."""
        return ffi.load().warp_moe_layer_slots_per_token(self.handle)

    def slots(self, T=1, device=None):
        """A zeroed slot buffer for forward_ep: [T][S][hidden] fp32."""
        return torch.zeros(T, self.slots_per_token(), self.hidden, dtype=torch.float32,
                           device=device)

    def forward_ep(self, x, slots, want_route=False):
        """Expert-parallel first half: this rank's routed outputs and its
        share of the shared expert into slots (warp_moe_layer_forward_ep)."""
        _cuda(x, slots)
        x2 = x.reshape(-1, self.hidden)
        T = x2.shape[0]
        if slots.shape != (T, self.slots_per_token(), self.hidden) or not slots.is_contiguous():
            raise ValueError("slots must be a contiguous [T][S][hidden] tensor (S: "
                             "slots_per_token)")
        idx = w = None
        if want_route:
            idx = torch.empty(T, self.K, dtype=torch.int32, device=x.device)
            w = torch.empty(T, self.K, dtype=torch.float32, device=x.device)
        ffi.check(ffi.load().warp_moe_layer_forward_ep(
            self.handle, _p(x2), T, _p(slots), _p(idx), _p(w), _stream()))
        return (idx, w) if want_route else None

    def combine(self, slots, residual=None, out=None):
        """Second half, after the slots were all-reduced over the ranks."""
        _cuda(slots)
        T = slots.shape[0]
        if out is None:
            out = torch.empty(T, self.hidden, dtype=torch.float32, device=slots.device)
        ffi.check(ffi.load().warp_moe_layer_combine(self.handle, _p(slots), T, _p(residual),
                                                    _p(out), _stream()))
        return out

    PHASES = ("router", "gate_up_gather", "swiglu", "down_gather", "shared", "combine")

    def set_timing(self, on):
        ffi.check(ffi.load().warp_moe_layer_set_timing(self.handle, int(on)))

    def collect(self):
        """Add the phase times of the last graph replay (timing on at capture)."""
        ffi.check(ffi.load().warp_moe_layer_collect(self.handle))

    def timings(self):
        """(forwards, {phase: total ms}) since set_timing(True)."""
        ms = (ctypes.c_double * 6)()
        n = ffi.load().warp_moe_layer_timings(self.handle, ms)
        return n, dict(zip(self.PHASES, list(ms)))

    def status(self):
        ffi.check(ffi.load().warp_moe_layer_status(self.handle, _stream()))

    def close(self):
        if getattr(self, "handle", None):
            ffi.load().warp_moe_layer_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def record_offsets(bank_bytes_first_record):
    return parse_header(bank_bytes_first_record)
