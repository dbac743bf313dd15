"""Paged KV cache operators: append (QK norm, rotation, rows into pages) and attention, for ragged batches of sequences.

The pages are plain tensors ``[n_pages, kv heads, page, 128]``: bf16, or ``float8_e4m3fn`` with ``k_scale`` / ``v_scale``
``[n_pages, kv heads]`` (fp32 powers of two, one per block of ``page`` tokens and head). Row ``r`` of sequence ``b`` is row
``r % page`` of page ``block_table[b, r // page]``. ``kv_len[b]`` counts the rows of a sequence including the tokens of the
call; ``cu_q[b]`` is the first token of sequence ``b`` in the call (``None``: one token per sequence). Token ``i`` of the ``n``
of sequence ``b`` stands at row ``kv_len[b] - n + i``; ``kv_len[b] <= 0`` marks a padding entry.

Lengths and tables live on the device: nothing here synchronises, and a captured graph replays with other lengths in the same
tensors. Kernels run on the current stream of the device that holds the tensors; scratch comes from PyTorch's allocator for each
call, so calls on different streams and graphs share nothing. A page id or position that does not fit sets ``err``
(:data:`..lib.ERR_NAMES` 6) and its rows are left out; nothing out of range is read or written.

The contiguous, one-sequence siblings are :func:`..lib.qk_norm_rope_kv`, :func:`..lib.qk_norm_rope_rows`,
:func:`..lib.flash_decode` and :func:`..lib.window_attention`; :class:`..runtime.paged_kv.PagedKVCache` owns pages and tables.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import lib as K

HEAD_DIM = 128
PAGE_SIZES = (16, 32, 64, 128)
_IO = (torch.float32, torch.bfloat16)


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _cache(T: int, k_pages, v_pages, block_table, kv_len, cu_q, k_scale, v_scale, err, dev) -> K.IhbPaged:
    """The cache part of an argument block, checked."""
    _need(k_pages.dim() == 4 and k_pages.shape == v_pages.shape and k_pages.shape[3] == HEAD_DIM,
          f"pages must be [n_pages, kv heads, page, {HEAD_DIM}], k and v alike")
    n_pages, nkv, page, _ = k_pages.shape
    _need(page in PAGE_SIZES, f"page size must be one of {PAGE_SIZES}, got {page}")
    _need(n_pages > 0 and nkv > 0, "there must be pages and KV heads")
    _need(k_pages.is_contiguous() and v_pages.is_contiguous(), "pages must be contiguous")
    _need(k_pages.data_ptr() % 16 == 0 and v_pages.data_ptr() % 16 == 0, "pages must start on a 16-byte boundary")
    if k_pages.dtype == torch.float8_e4m3fn and v_pages.dtype == torch.float8_e4m3fn:
        _need(k_scale is not None and v_scale is not None, "e4m3 pages need k_scale and v_scale")
        for s in (k_scale, v_scale):
            _need(s.dtype == torch.float32 and s.shape == (n_pages, nkv) and s.is_contiguous() and s.device == dev,
                  "page scales must be contiguous fp32 [n_pages, kv heads] on the pages' device")
    else:
        _need(k_pages.dtype == torch.bfloat16 and v_pages.dtype == torch.bfloat16, "pages must be bfloat16 or float8_e4m3fn")
        _need(k_scale is None and v_scale is None, "bf16 pages have no scales")
    B = kv_len.shape[0] if kv_len.dim() == 1 else 0
    _need(B > 0 and kv_len.dtype == torch.int32 and kv_len.is_contiguous(), "kv_len must be contiguous int32 [B]")
    _need(block_table.dim() == 2 and block_table.shape[0] == B and block_table.shape[1] > 0 and block_table.dtype == torch.int32
          and block_table.stride(1) == 1, "block_table must be int32 [B, blocks] with contiguous rows")
    if cu_q is not None:
        _need(cu_q.dtype == torch.int32 and cu_q.shape == (B + 1,) and cu_q.is_contiguous(), "cu_q must be contiguous int32 [B + 1]")
    else:
        _need(T == B, f"without cu_q there is one token per sequence: {T} tokens, {B} sequences")
    if err is not None:
        _need(err.dtype == torch.int32 and err.numel() >= 1, "err must be an int32 word")
    for t in (k_pages, v_pages, block_table, kv_len, cu_q, err):
        _need(t is None or t.device == dev, "all tensors must be on one device")
    return K.IhbPaged(k_pages.data_ptr(), v_pages.data_ptr(), K.ptr(k_scale), K.ptr(v_scale), n_pages, nkv, page, B, T,
                      block_table.shape[1], block_table.stride(0), block_table.data_ptr(), kv_len.data_ptr(), K.ptr(cu_q), K.ptr(err))


def _launch(fn, args, dev: torch.device, what: str) -> None:
    if dev.type != "cuda":
        raise ValueError("the paged cache kernels need CUDA tensors")
    if dev.index == torch.cuda.current_device():
        K.check(fn(C.byref(args), K.stream_ptr()), what)
    else:                                   # the caller's current device is another one: launch on the tensors' own
        with torch.cuda.device(dev):
            K.check(fn(C.byref(args), K.stream_ptr()), what)


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
    60; infinities saturate, NaN stays NaN, neither counts). Writing row 0 starts a page anew; otherwise the scale only grows, and
    rows already there are brought to it in place, so a page that is written to must belong to one sequence. Rows behind the last
    token and pages of other sequences are left as they are."""
    _need(nq > 0 and nkv > 0, "nq and nkv must be positive")
    _need(qkv.dim() == 2 and qkv.shape[1] == (nq + 2 * nkv) * HEAD_DIM and qkv.stride(1) == 1, "qkv must be [T, (nq + 2 nkv) * 128]")
    T, dev = qkv.shape[0], qkv.device
    _need(T > 0, "there must be a token")
    _need(qkv.dtype in _IO, "qkv must be float32 or bfloat16")
    vec = 8                                                     # bytes or two fp32: what one access takes
    _need(qkv.stride(0) % 2 == 0 and qkv.data_ptr() % vec == 0, "qkv rows must start on 8-byte (fp32) or 4-byte (bf16) boundaries")
    _need(q_out is not None or T == 1 or qkv.stride(0) >= qkv.shape[1], "qkv rows overlap: they cannot be rewritten in place")
    c = _cache(T, k_pages, v_pages, block_table, kv_len, cu_q, k_scale, v_scale, err, dev)
    _need(c.nkv == nkv, f"pages have {c.nkv} KV heads, the call names {nkv}")
    _need(cos_t.shape == sin_t.shape and cos_t.dim() == 2 and cos_t.shape[1] == HEAD_DIM // 2 and cos_t.shape[0] > 0
          and cos_t.dtype == torch.float32 and sin_t.dtype == torch.float32 and cos_t.is_contiguous() and sin_t.is_contiguous(),
          "cos_t and sin_t must be contiguous fp32 [n_pos, 64]")
    _need((q_gamma is None) == (k_gamma is None), "q_gamma and k_gamma come together")
    for t in (q_gamma, k_gamma):
        _need(t is None or (t.dtype == torch.float32 and t.shape == (HEAD_DIM,) and t.is_contiguous() and t.data_ptr() % vec == 0),
              "gammas must be contiguous fp32 [128]")
    if positions is not None:
        _need(positions.dtype == torch.int32 and positions.shape == (T,) and positions.is_contiguous(), "positions must be contiguous int32 [T]")
    if q_out is not None:
        _need(q_out.shape == (T, nq, HEAD_DIM) and q_out.dtype in _IO and q_out.stride(2) == 1 and (nq == 1 or q_out.stride(1) == HEAD_DIM)
              and q_out.stride(0) % 2 == 0 and (T == 1 or q_out.stride(0) >= nq * HEAD_DIM) and q_out.data_ptr() % vec == 0, "q_out must be fp32 or bf16 [T, nq, 128] with whole rows")
    for t in (cos_t, sin_t, q_gamma, k_gamma, positions, q_out):
        _need(t is None or t.device == dev, "all tensors must be on one device")
    a = K.IhbPagedAppend(c, qkv.data_ptr(), qkv.dtype == torch.bfloat16, nq, qkv.stride(0), K.ptr(q_out),
                         q_out is not None and q_out.dtype == torch.bfloat16, q_out.stride(0) if q_out is not None else 0,
                         K.ptr(q_gamma), K.ptr(k_gamma), eps, cos_t.data_ptr(), sin_t.data_ptr(), cos_t.shape[0], K.ptr(positions))
    _launch(K.load().ihb_paged_append, a, dev, "ihb_paged_append")
    return q_out if q_out is not None else qkv[:, :nq * HEAD_DIM].unflatten(1, (nq, HEAD_DIM))


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, kv_len: torch.Tensor, *,
                    cu_q: Optional[torch.Tensor] = None, max_q: int = 1, mask: Optional[torch.Tensor] = None,
                    k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                    err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of ``q [T, nq, 128]`` (fp32 or bf16, any token / head strides that are multiples of 8) over the pages.

    A token sees its own row and those before it; with ``mask [T, >= max_q]`` (bool or uint8) it sees all rows ahead of the
    call's and row ``j`` of its sequence's tokens where ``mask[t, j]`` is set (token trees). A token that sees nothing gets zeros
    (and ``lse`` -inf); values in rows that a token does not see never reach it, NaN and infinities included. ``max_q``: an
    upper bound of the tokens per sequence. ``scale`` defaults to 128 ** -0.5. ``out [T, nq, 128]`` fp32 or bf16 (default: new, of
    ``q``'s type; tokens behind ``cu_q[B]`` are left as they are, so a new tensor holds nothing there). ``lse [T, nq]`` fp32
    receives the natural log of each softmax denominator, for merging with attention over other rows."""
    _need(q.dim() == 3 and q.shape[2] == HEAD_DIM and q.stride(2) == 1 and q.shape[0] > 0, f"q must be [T, nq, {HEAD_DIM}]")
    T, nq, _ = q.shape
    dev = q.device
    _need(q.dtype in _IO, "q must be float32 or bfloat16")
    _need(q.stride(0) % 8 == 0 and q.stride(1) % 8 == 0 and q.data_ptr() % 16 == 0, "q strides must be multiples of 8, its start of 16 bytes")
    c = _cache(T, k_pages, v_pages, block_table, kv_len, cu_q, k_scale, v_scale, err, dev)
    _need(nq % c.nkv == 0, f"{nq} query heads do not share {c.nkv} KV heads evenly")
    _need(max_q > 0 and (cu_q is not None or max_q == 1), "max_q must be positive, and 1 without cu_q")
    if scale is None:
        scale = HEAD_DIM ** -0.5
    _need(0.0 < scale < 1e30, "scale must be positive and finite")
    if out is None:
        out = torch.empty(T, nq, HEAD_DIM, dtype=q.dtype, device=dev)
    else:
        _need(out.shape == q.shape and out.dtype in _IO and out.stride(2) == 1 and out.device == dev
              and out.stride(0) % 4 == 0 and out.stride(1) % 4 == 0 and out.data_ptr() % 16 == 0,
              "out must be fp32 or bf16 [T, nq, 128], strides multiples of 4, its start of 16 bytes")
        _need((T == 1 or out.stride(0) >= HEAD_DIM) and (nq == 1 or out.stride(1) >= HEAD_DIM), "rows of out overlap")
    if lse is not None:
        _need(lse.dtype == torch.float32 and lse.shape == (T, nq) and lse.is_contiguous() and lse.device == dev, "lse must be contiguous fp32 [T, nq]")
    if mask is not None:
        _need(mask.dtype in (torch.bool, torch.uint8) and mask.dim() == 2 and mask.shape[0] == T and mask.shape[1] >= max_q
              and mask.stride(1) == 1 and mask.device == dev, "mask must be bool or uint8 [T, >= max_q] with contiguous rows")
    a = K.IhbPagedAttn(c, q.data_ptr(), q.dtype == torch.bfloat16, nq, q.stride(0), q.stride(1), out.data_ptr(),
                       out.dtype == torch.bfloat16, out.stride(0), out.stride(1), K.ptr(lse), K.ptr(mask),
                       mask.stride(0) if mask is not None else 0, max_q, scale, None)
    if dev.type != "cuda":
        raise ValueError("the paged cache kernels need CUDA tensors")
    lib = K.load()
    scratch = torch.empty(lib.ihb_paged_attention_scratch(C.byref(a)), dtype=torch.uint8, device=dev)
    a.scratch = scratch.data_ptr()
    _launch(lib.ihb_paged_attention, a, dev, "ihb_paged_attention")
    return out
