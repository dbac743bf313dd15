"""Paged KV cache operators: append (QK norm, rotation, rows into pages) and attention, for ragged batches of sequences.

The pages are plain tensors ``[n_pages, kv heads, page, 128]``: bf16, or ``float8_e4m3fn`` with ``k_scale`` / ``v_scale``
``[n_pages, kv heads]`` (fp32 powers of two, one per block of ``page`` tokens and head). Row ``r`` of sequence ``b`` is row
``r % page`` of page ``block_table[b, r // page]``. ``kv_len[b]`` counts the rows of a sequence including the tokens of the
call; ``cu_q[b]`` is the first token of sequence ``b`` in the call (``None``: one token per sequence). Token ``i`` of the ``n``
of sequence ``b`` stands at row ``kv_len[b] - n + i``; ``kv_len[b] <= 0`` marks a padding entry.

Lengths and tables live on the device: nothing here synchronises, and a captured graph replays with other lengths in the same
tensors. Kernels run on the current stream of the device that holds the tensors; scratch comes from PyTorch's allocator for each
call, so calls on different streams and graphs share nothing. A page id or position that does not fit sets ``err``
(:data:`..lib.ERR_NAMES` 6) and its rows are left out; nothing out of range is read or written. A kernel whose internal wait ran out (a
device fault) leaves NaN in the call's rows, whether there is an ``err`` or not.

The contiguous, one-sequence siblings are :func:`..lib.qk_norm_rope_kv`, :func:`..lib.qk_norm_rope_rows`,
:func:`..lib.flash_decode` and :func:`..lib.window_attention`; :class:`..runtime.paged_kv.PagedKVCache` owns pages and tables.
"""
from __future__ import annotations

import struct
from typing import Optional

import torch

from . import lib as K

HEAD_DIM = 128
PAGE_SIZES = (16, 32, 64, 128)
_F32, _BF16, _I32, _E4M3 = torch.float32, torch.bfloat16, torch.int32, torch.float8_e4m3fn
# The argument blocks as bytes (:class:`..lib.IhbPaged`, :class:`..lib.IhbPagedAppend`, :class:`..lib.IhbPagedAttn`; native layout, 0 is
# NULL): packed in 1 us where filling the structures takes 4.
_CACHE = "PPPPiiiiiiqPPPP"
_APPEND = struct.Struct("@" + _CACHE + "PiiqPiqPPfPPiP")
_ATTN = struct.Struct("@" + _CACHE + "PiiqqPiqqPPqiifP")
_PTR = struct.Struct("@P")


# The checks below run on every call, beside kernels that take a few microseconds: plain conditions, messages formed only when they are
# needed, every attribute of a tensor read once.
def _bad(what: str) -> None:
    raise ValueError(what)


def _cache(T: int, k_pages, v_pages, block_table, kv_len, cu_q, k_scale, v_scale, err, dev: int) -> tuple:
    """The cache part of an argument block, checked. ``dev``: index of the device that all tensors must be on."""
    shape = k_pages.shape
    if len(shape) != 4 or v_pages.shape != shape or shape[3] != HEAD_DIM:
        _bad(f"pages must be [n_pages, kv heads, page, {HEAD_DIM}], k and v alike")
    n_pages, nkv, page, _ = shape
    if page not in PAGE_SIZES:
        _bad(f"page size must be one of {PAGE_SIZES}, got {page}")
    if n_pages < 1 or nkv < 1:
        _bad("there must be pages and KV heads")
    if not (k_pages.is_contiguous() and v_pages.is_contiguous()):
        _bad("pages must be contiguous")
    kp, vp = k_pages.data_ptr(), v_pages.data_ptr()
    if (kp | vp) & 15:
        _bad("pages must start on a 16-byte boundary")
    dtype = k_pages.dtype
    if v_pages.dtype != dtype:
        _bad("pages must be bfloat16 or float8_e4m3fn, k and v alike")
    ksp = vsp = 0
    if dtype == _E4M3:
        if k_scale is None or v_scale is None:
            _bad("e4m3 pages need k_scale and v_scale")
        per_page = (n_pages, nkv)
        for s in (k_scale, v_scale):
            if s.dtype != _F32 or s.shape != per_page or not s.is_contiguous() or s.get_device() != dev:
                _bad("page scales must be contiguous fp32 [n_pages, kv heads] on the pages' device")
        ksp, vsp = k_scale.data_ptr(), v_scale.data_ptr()
    elif dtype != _BF16:
        _bad("pages must be bfloat16 or float8_e4m3fn")
    elif k_scale is not None or v_scale is not None:
        _bad("bf16 pages have no scales")
    lens = kv_len.shape
    if kv_len.dtype != _I32 or len(lens) != 1 or lens[0] < 1 or not kv_len.is_contiguous():
        _bad("kv_len must be contiguous int32 [B]")
    B = lens[0]
    tshape = block_table.shape
    if len(tshape) != 2 or tshape[0] != B or tshape[1] < 1 or block_table.dtype != _I32:
        _bad("block_table must be int32 [B, blocks] with contiguous rows")
    if tshape[1] * page > 1 << 30 or nkv > 4096:
        _bad("a sequence can have at most 2^30 rows, a cache 4096 KV heads")
    tstride = block_table.stride()
    if tstride[1] != 1 and tshape[1] != 1:
        _bad("block_table must be int32 [B, blocks] with contiguous rows")
    cup = ep = 0
    if cu_q is None:
        if T != B:
            _bad(f"without cu_q there is one token per sequence: {T} tokens, {B} sequences")
    else:
        if cu_q.dtype != _I32 or cu_q.shape != (B + 1,) or not cu_q.is_contiguous() or cu_q.get_device() != dev:
            _bad("cu_q must be contiguous int32 [B + 1] on the pages' device")
        cup = cu_q.data_ptr()
    if err is not None:
        if err.dtype != _I32 or err.numel() < 1 or err.get_device() != dev:
            _bad("err must be an int32 word on the pages' device")
        ep = err.data_ptr()
    if k_pages.get_device() != dev or v_pages.get_device() != dev or kv_len.get_device() != dev or block_table.get_device() != dev:
        _bad("all tensors must be on one device")
    return kp, vp, ksp, vsp, n_pages, nkv, page, B, T, tshape[1], tstride[0], block_table.data_ptr(), kv_len.data_ptr(), cup, ep


# the stream pointer without a Stream object around it where this build of torch has that (2 us less per call)
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda dev: torch.cuda.current_stream(dev).cuda_stream)


def _launch(fn, args: bytes, dev: int, what: str) -> None:
    if dev == torch.cuda.current_device():
        code = fn(args, _stream(dev))
    else:                                   # the caller's current device is another one: launch on the tensors' own
        with torch.cuda.device(dev):
            code = fn(args, _stream(dev))
    if code:
        K.check(code, what)


def paged_append(qkv: torch.Tensor, nq: int, nkv: int, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                 kv_len: torch.Tensor, cos_t: torch.Tensor, sin_t: torch.Tensor, *, cu_q: Optional[torch.Tensor] = None,
                 positions: Optional[torch.Tensor] = None, q_gamma: Optional[torch.Tensor] = None,
                 k_gamma: Optional[torch.Tensor] = None, eps: float = 1e-6, k_scale: Optional[torch.Tensor] = None,
                 v_scale: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None,
                 err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Normalises (gammas given), rotates and appends: ``qkv [T, (nq + 2 nkv) * 128]`` fp32 or bf16 (rows may be strided).

    Q heads go, normed and rotated, to ``q_out [T, nq, 128]`` (fp32 or bf16; ``None``: in place, the returned tensor is a view
    of ``qkv``); K (normed, rotated) and V rows go to the pages. ``cos_t`` / ``sin_t`` ``[n_pos, 64]`` fp32 are indexed by the
    token's row, or by ``positions[t]`` (int32) where a token's angle is not its row (token trees).

    e4m3 pages: a page's scale is the least power of two with ``amax / 448 <= scale`` over the rows it holds (exponent -60 to
    60; infinities saturate, NaN stays NaN, neither counts). Scales and bytes are what exact arithmetic gives (bf16 pages and queries:
    fp32, rounded once). Writing row 0 starts a page anew; otherwise the scale only grows, and rows already there are brought to it in
    place, so a page that is written to must belong to one sequence. Rows behind the last token and pages of other sequences are left
    as they are."""
    if nq < 1 or nkv < 1:
        _bad("nq and nkv must be positive")
    shape = qkv.shape
    if len(shape) != 2 or shape[1] != (nq + 2 * nkv) * HEAD_DIM:
        _bad("qkv must be [T, (nq + 2 nkv) * 128]")
    T, dev, dtype = shape[0], qkv.get_device(), qkv.dtype
    if T < 1:
        _bad("there must be a token")
    stride = qkv.stride()
    if stride[1] != 1:
        _bad("qkv must be [T, (nq + 2 nkv) * 128] with contiguous rows")
    if dtype != _F32 and dtype != _BF16:
        _bad("qkv must be float32 or bfloat16")
    qp = qkv.data_ptr()
    if stride[0] & 7 or qp & 15:
        _bad("qkv rows must start on 16-byte boundaries (strides multiples of 8)")
    c = _cache(T, k_pages, v_pages, block_table, kv_len, cu_q, k_scale, v_scale, err, dev)
    if c[5] != nkv:
        _bad(f"pages have {c[5]} KV heads, the call names {nkv}")
    cs = cos_t.shape
    if (len(cs) != 2 or cs[1] != HEAD_DIM // 2 or cs[0] < 1 or sin_t.shape != cs or cos_t.dtype != _F32 or sin_t.dtype != _F32
            or not cos_t.is_contiguous() or not sin_t.is_contiguous()):
        _bad("cos_t and sin_t must be contiguous fp32 [n_pos, 64]")
    cp, sp = cos_t.data_ptr(), sin_t.data_ptr()
    gq = gk = pp = op = 0
    if q_gamma is not None or k_gamma is not None:
        if q_gamma is None or k_gamma is None:
            _bad("q_gamma and k_gamma come together")
        for t in (q_gamma, k_gamma):
            if t.dtype != _F32 or t.shape != (HEAD_DIM,) or not t.is_contiguous() or t.get_device() != dev:
                _bad("gammas must be contiguous fp32 [128] on the pages' device")
        gq, gk = q_gamma.data_ptr(), k_gamma.data_ptr()
    if (cp | sp | gq | gk) & 15:
        _bad("rope tables and gammas must start on 16-byte boundaries")
    if positions is not None:
        if positions.dtype != _I32 or positions.shape != (T,) or not positions.is_contiguous() or positions.get_device() != dev:
            _bad("positions must be contiguous int32 [T] on the pages' device")
        pp = positions.data_ptr()
    q_bf16, q_stride = 0, 0
    if q_out is None:
        if T > 1 and stride[0] < shape[1]:
            _bad("qkv rows overlap: they cannot be rewritten in place")
    else:
        os = q_out.stride() if q_out.dim() == 3 else None
        op, od = q_out.data_ptr(), q_out.dtype
        if (os is None or q_out.shape != (T, nq, HEAD_DIM) or (od != _F32 and od != _BF16) or os[2] != 1 or (nq > 1 and os[1] != HEAD_DIM)
                or os[0] & 7 or (T > 1 and os[0] < nq * HEAD_DIM) or op & 15 or q_out.get_device() != dev):
            _bad("q_out must be fp32 or bf16 [T, nq, 128] with whole rows on 16-byte boundaries, on the pages' device")
        q_bf16, q_stride = od == _BF16, os[0]
    if cos_t.get_device() != dev or sin_t.get_device() != dev:
        _bad("all tensors must be on one device")
    if dev < 0:
        _bad("the paged cache kernels need CUDA tensors")
    a = _APPEND.pack(*c, qp, dtype == _BF16, nq, stride[0], op, q_bf16, q_stride, gq, gk, eps, cp, sp, cs[0], pp)
    _launch(K.load().ihb_paged_append, a, dev, "ihb_paged_append")
    return q_out if q_out is not None else qkv[:, :nq * HEAD_DIM].unflatten(1, (nq, HEAD_DIM))


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, kv_len: torch.Tensor, *,
                    cu_q: Optional[torch.Tensor] = None, max_q: Optional[int] = None, mask: Optional[torch.Tensor] = None,
                    k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                    err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of ``q [T, nq, 128]`` (fp32 or bf16, any token / head strides that are multiples of 8) over the pages.

    A token sees its own row and those before it; with ``mask [T, >= max_q]`` (bool or uint8; a view of any row stride, rows may
    overlap or be one) it sees all rows ahead of the call's and row ``j`` of its sequence's tokens where ``mask[t, j]`` is set (token
    trees). A token that sees nothing gets zeros (and ``lse`` -inf); values in rows that a token does not see never reach it, NaN and
    infinities included. ``max_q``, required with ``cu_q``: an upper bound of the tokens per sequence (a sequence with more sets ``err``
    and may leave rows of ``out`` unwritten). ``scale`` defaults to 128 ** -0.5. ``out [T, nq, 128]`` fp32 or bf16 (default: new, of
    ``q``'s type; tokens behind ``cu_q[B]`` are left as they are, so a new tensor holds nothing there). ``lse [T, nq]`` fp32 receives
    the natural log of each softmax denominator, for merging with attention over other rows.

    Sums, maxima and denominators are fp32. What else is rounded, relative to the result: fp32 queries 2^-20 over both kinds of pages;
    bf16 queries over e4m3 pages 2^-11 (probabilities in fp16; in windows of more than 32 rows, tokens x query heads of a KV head, what
    lies below 2^-17 of a query's largest element is lost too); over bf16 pages 2^-16, and 2^-8 where ``out`` is bf16 and a window has
    more than 128 rows. Infinities in a value row that every token sees come out as infinity or NaN. Scales of e4m3 pages are taken
    between 2^-60 and 2^60, scores (to base 2) up to 2^24 in magnitude."""
    shape = q.shape
    if len(shape) != 3 or shape[2] != HEAD_DIM or shape[0] < 1:
        _bad(f"q must be [T, nq, {HEAD_DIM}]")
    T, nq, _ = shape
    dev, dtype, qs, qp = q.get_device(), q.dtype, q.stride(), q.data_ptr()
    if dtype != _F32 and dtype != _BF16:
        _bad("q must be float32 or bfloat16")
    if qs[2] != 1 or (qs[0] | qs[1]) & 7 or qp & 15:
        _bad("q strides must be multiples of 8 (the last 1), its start of 16 bytes")
    c = _cache(T, k_pages, v_pages, block_table, kv_len, cu_q, k_scale, v_scale, err, dev)
    nkv = c[5]
    if nq % nkv or nq < 1:
        _bad(f"{nq} query heads do not share {nkv} KV heads evenly")
    if nq > 256 * nkv:
        _bad("a KV head can have at most 256 query heads")
    if max_q is None:
        if cu_q is not None:
            _bad("cu_q needs max_q, an upper bound of the tokens per sequence")
        max_q = 1
    elif max_q < 1 or (cu_q is None and max_q != 1):
        _bad("max_q must be positive, and 1 without cu_q")
    elif max_q > T:
        max_q = T
    if scale is None:
        scale = HEAD_DIM ** -0.5
    elif not 0.0 < scale < 1e30:
        _bad("scale must be positive and finite")
    lp = mp = 0
    mask_stride = mask_cols = 0
    if lse is not None:
        if lse.dtype != _F32 or lse.shape != (T, nq) or not lse.is_contiguous() or lse.get_device() != dev:
            _bad("lse must be contiguous fp32 [T, nq] on the pages' device")
        lp = lse.data_ptr()
    if mask is not None:
        if mask.dtype not in (torch.bool, torch.uint8) or mask.dim() != 2 or mask.shape[0] != T or mask.shape[1] < max_q or mask.get_device() != dev:
            _bad("mask must be bool or uint8 [T, >= max_q] on the pages' device")
        mask_stride, last = mask.stride()
        mask_cols = mask.shape[1]
        if last != 1 and mask_cols > 1:
            _bad("mask must have contiguous rows")
        mp = mask.data_ptr()
    if out is None:
        if dev < 0:
            _bad("the paged cache kernels need CUDA tensors")
        out = torch.empty(shape, dtype=dtype, device=q.device)
        op, od, os = out.data_ptr(), dtype, (nq * HEAD_DIM, HEAD_DIM)
    else:
        op, od, os = out.data_ptr(), out.dtype, out.stride()
        if (out.shape != shape or (od != _F32 and od != _BF16) or os[2] != 1 or (os[0] | os[1]) & 3 or op & 15 or out.get_device() != dev):
            _bad("out must be fp32 or bf16 [T, nq, 128], strides multiples of 4, its start of 16 bytes, on the pages' device")
        # tokens around heads, or heads around tokens, nothing in between
        if not ((nq == 1 or os[1] >= HEAD_DIM) and (T == 1 or os[0] >= (nq - 1) * os[1] + HEAD_DIM)
                or (T == 1 or os[0] >= HEAD_DIM) and (nq == 1 or os[1] >= (T - 1) * os[0] + HEAD_DIM)):
            _bad("rows of out overlap")
        if dev < 0:
            _bad("the paged cache kernels need CUDA tensors")
    a = _ATTN.pack(*c, qp, dtype == _BF16, nq, qs[0], qs[1], op, od == _BF16, os[0], os[1], lp, mp, mask_stride, mask_cols, max_q, scale, 0)
    lib = K.load()
    scratch = torch.empty(lib.ihb_paged_attention_scratch(a), dtype=torch.uint8, device=q.device)
    _launch(lib.ihb_paged_attention, a[:-_PTR.size] + _PTR.pack(scratch.data_ptr()), dev, "ihb_paged_attention")
    return out
