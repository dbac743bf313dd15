"""Paged cache kernels against plain 64-bit implementations (needs a B200).

Tolerances. q' (append): three roundings of fp32 products and the RMS (rsqrt within 2 ulp): 2^-20 of the row's largest
magnitude, plus half a step of the output type. K / V rows: e4m3 bytes within one step where a value lies next to a rounding
border in fp32 and is on it in 64 bits, else equal; scales equal. Attention: see _tol."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import paged_oracle as O
from inferencehackathon_b200.ops import paged

DEV = "cuda:0"


def _io(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _dev(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


# ---- append ---------------------------------------------------------------------------------------------------------------
APPENDS = [
    # befores, news, nq, nkv, page
    ([0], [1], 8, 1, 64),
    ([15, 16, 0, 63, 17], [1, 1, 1, 1, 1], 4, 2, 16),
    ([100, 0, 31, 5], [1, 70, 33, 0], 6, 3, 32),
    ([127, 1, 128], [129, 3, 256], 4, 4, 128),
    ([7], [200], 20, 4, 64),
    ([0, 0, 0], [16, 17, 15], 1, 1, 16),
]


@pytest.mark.parametrize("befores,news,nq,nkv,page", APPENDS)
@pytest.mark.parametrize("cache", ["fp8", "bf16"])
@pytest.mark.parametrize("io,norm", [("fp32", True), ("bf16", False), ("bf16", True)])
def test_append(befores, news, nq, nkv, page, cache, io, norm):
    gen = torch.Generator().manual_seed(sum(befores) + nq)
    lens = [b + n for b, n in zip(befores, news)]
    T = sum(news)
    table, n_pages = O.tables(lens, page, gen)
    k, v, ks, vs = O.random_pages(n_pages, nkv, page, cache, gen)
    qkv = (torch.randn(T + 2, (nq + 2 * nkv) * 128, generator=gen) * 2).to(_io(io))       # two tokens behind the last sequence
    cos, sin = O.rope_tables(max(lens) + 1)
    qg, kg = ((1 + 0.2 * torch.randn(128, generator=gen)) for _ in range(2)) if norm else (None, None)
    cu = O.cu_of(news)
    ref = O.Pages(k, v, ks, vs)
    q_ref = O.append(ref, qkv, nq, nkv, table, lens, cu, cos, sin, qg, kg)
    kd, vd, ksd, vsd, td, cud, cosd, sind, qgd, kgd, x = _dev(k, v, ks, vs, table, cu, cos, sin, qg, kg, qkv)
    ld = torch.tensor(lens, dtype=torch.int32, device=DEV)
    q_out = torch.full((T + 2, nq, 128), 7.0, dtype=_io(io), device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = paged.paged_append(x, nq, nkv, kd, vd, td, ld, cosd, sind, cu_q=cud, q_gamma=qgd, k_gamma=kgd, k_scale=ksd, v_scale=vsd,
                             q_out=q_out, err=err)
    torch.cuda.synchronize()
    assert got is q_out and int(err) == 0 and torch.equal(x.cpu(), qkv)
    assert bool((q_out[T:] == 7.0).all())                                                 # left as they were
    ref_q = q_ref[:T]
    half = torch.finfo(_io(io)).eps / 2
    tol = ref_q.abs() * half + ref_q.abs().amax(-1, keepdim=True) * 2.0 ** -20
    assert bool(((got[:T].double().cpu() - ref_q).abs() <= tol).all())
    for dst, sc, want, want_s in ((kd, ksd, ref.k, ref.ks), (vd, vsd, ref.v, ref.vs)):
        g = dst.to(torch.float32).double().cpu()
        if cache == "bf16":
            assert bool(((g - want).abs() <= want.abs() * 2.0 ** -8 + want.abs().amax(-1, keepdim=True) * 2.0 ** -20).all())
            continue
        assert torch.equal(sc.double().cpu(), want_s)
        far = (g - want).abs()
        assert bool((far <= want.abs() * 2.0 ** -3 + 2.0 ** -9).all())                    # at most the neighbour
        assert float((far > 0).double().mean()) < 1e-3                                    # and hardly ever
    # in place: the Q part of qkv is rewritten, the K / V parts stay
    kd2, vd2, ksd2, vsd2 = _dev(k, v, ks, vs)
    view = paged.paged_append(x, nq, nkv, kd2, vd2, td, ld, cosd, sind, cu_q=cud, q_gamma=qgd, k_gamma=kgd, k_scale=ksd2, v_scale=vsd2)
    assert view.data_ptr() == x.data_ptr() and torch.equal(view[:T], q_out[:T])
    assert torch.equal(x[:, nq * 128:].cpu(), qkv[:, nq * 128:]) and torch.equal(x[T:].cpu(), qkv[T:])
    assert torch.equal(kd2.view(torch.uint8), kd.view(torch.uint8)) and torch.equal(vd2.view(torch.uint8), vd.view(torch.uint8))


def test_append_token_by_token_equals_prompt():
    """Decode appends fill pages to the same scales as one prompt append, and to the same bytes but for subnormals."""
    gen = torch.Generator().manual_seed(5)
    nq, nkv, P, T = 2, 2, 32, 75
    qkv = torch.randn(T, (nq + 2 * nkv) * 128, generator=gen) * torch.exp2(torch.linspace(-5, 5, T))[:, None]
    cos, sin = _dev(*O.rope_tables(T))
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=DEV)

    def blank():
        return ([torch.zeros(3, nkv, P, 128, device=DEV).to(torch.float8_e4m3fn) for _ in range(2)]
                + [torch.full((3, nkv), float("nan"), device=DEV) for _ in range(2)])

    x = qkv.to(DEV)
    k1, v1, ks1, vs1 = blank()
    paged.paged_append(x.clone(), nq, nkv, k1, v1, table, torch.tensor([T], dtype=torch.int32, device=DEV), cos, sin,
                       cu_q=torch.tensor([0, T], dtype=torch.int32, device=DEV), k_scale=ks1, v_scale=vs1)
    k2, v2, ks2, vs2 = blank()
    for t in range(T):
        paged.paged_append(x[t:t + 1].clone(), nq, nkv, k2, v2, table, torch.tensor([t + 1], dtype=torch.int32, device=DEV), cos, sin,
                           k_scale=ks2, v_scale=vs2)
    assert torch.equal(ks1, ks2) and torch.equal(vs1, vs2)
    for a, b in ((k1, k2), (v1, v2)):
        a, b = a.float(), b.float()
        normal = a.abs() >= 2.0 ** -6
        assert torch.equal(a[normal], b[normal]) and float((a - b).abs().max()) <= 2.0 ** -9


def test_append_non_finite_positions_and_padding():
    """NaN stays NaN and infinities saturate without moving the scale; explicit rotation positions; padding entries."""
    gen = torch.Generator().manual_seed(8)
    nq, nkv, P = 2, 1, 16
    qkv = torch.randn(4, (nq + 2 * nkv) * 128, generator=gen)
    qkv[1, -128 + 3] = float("inf")
    qkv[2, -128 + 5] = float("nan")
    cos, sin = O.rope_tables(64)
    lens = [5, 0, 17]
    news = [2, 1, 1]
    pos = torch.tensor([40, 63, 9, 0], dtype=torch.int32)
    table = torch.tensor([[3, -1], [-1, -1], [0, 1]], dtype=torch.int32)
    k, v, ks, vs = O.random_pages(4, nkv, P, "fp8", gen)
    ref = O.Pages(k, v, ks, vs)
    q_ref = O.append(ref, qkv, nq, nkv, table, lens, O.cu_of(news), cos, sin, positions=pos)
    kd, vd, ksd, vsd, td, cosd, sind, x, pd, cu = _dev(k, v, ks, vs, table, cos, sin, qkv, pos, O.cu_of(news))
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    q = torch.full((4, nq, 128), float("nan"), device=DEV)
    paged.paged_append(x, nq, nkv, kd, vd, td, torch.tensor(lens, dtype=torch.int32, device=DEV), cosd, sind, cu_q=cu, positions=pd,
                       k_scale=ksd, v_scale=vsd, q_out=q, err=err)
    assert int(err) == 0
    got = q.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(q_ref))
    ok = ~torch.isnan(q_ref)
    assert float((got - q_ref)[ok].abs().max()) <= 2.0 ** -20 * float(q_ref[ok].abs().max())
    assert torch.equal(ksd.double().cpu(), ref.ks) and torch.equal(vsd.double().cpu(), ref.vs)
    gv = vd.float().double().cpu()
    assert torch.equal(torch.isnan(gv), torch.isnan(ref.v)) and abs(float(gv[3, 0, 4, 3])) == 448.0
    assert float((torch.nan_to_num(gv) - torch.nan_to_num(ref.v)).abs().max()) == 0.0     # V is not rotated: the same rounding


def test_append_reports_bad_pages_and_positions():
    """A page id outside the pool, a sequence longer than its table, a rotation angle outside the tables: an error word, no write."""
    nq, nkv, P = 2, 1, 16
    cos, sin = _dev(*O.rope_tables(20))
    x = torch.ones(1, (nq + 2 * nkv) * 128, device=DEV)
    for table, n, bad in (([[9]], 1, True), ([[-2]], 1, True), ([[0]], 17, True), ([[0, 1]], 21, True), ([[0, 1]], 20, False)):
        k = torch.zeros(4, nkv, P, 128, dtype=torch.bfloat16, device=DEV)
        v, err = torch.zeros_like(k), torch.zeros(1, dtype=torch.int32, device=DEV)
        paged.paged_append(x.clone(), nq, nkv, k, v, torch.tensor(table, dtype=torch.int32, device=DEV),
                           torch.tensor([n], dtype=torch.int32, device=DEV), cos, sin, err=err)
        assert int(err) == (6 if bad else 0)
        assert bool((v == 0).all()) == bad


# ---- attention ------------------------------------------------------------------------------------------------------------
def _score_error(cache, io, tiles):
    if io == "bf16":
        return 2.0 ** -17 * 128 ** 0.5 if tiles and cache == "fp8" else 0.0
    return 2.0 ** -22 if cache == "fp8" else 2.0 ** -16


def _tol(ref, q, ref_pages, scale, cache, io, out_io, tiles=False):
    """What the roundings allow, relative to the largest |v| that is seen (a probability that is off by a relative d moves the
    output by at most d of that on both sides of the quotient, hence the 2):
      scores      q in two terms: fp16 pairs for e4m3 pages (22 bits), bf16 pairs for bf16 pages (16 bits; bf16 q is exact in
                  both); over e4m3 pages the kernel of 128-row tiles takes bf16 q as two e4m3 terms, the row's largest magnitude scaled
                  to [128, 256): what is lost is below a step of e4m3's subnormals, 2^-10, or 2^-17 of that magnitude per channel,
                  sqrt(128) of it on the norm; times |q| |k| scale; fp32 sums of 128 terms and the exponent's fp32 rounding at |s| <= 64: 2^-18
      P           fp16 (2^-11, bf16 q over e4m3 pages), fp16 pairs (2^-22) or bf16 pairs (2^-16); bf16 q in the kernel of 128-row
                  tiles over bf16 pages: one bf16 (2^-8)
      sums        fp32 over up to 2^12 terms: 2^-18 with room; ex2 2^-22
    and half a step of the output type."""
    vmax = float(torch.nan_to_num((ref_pages.v * (1.0 if ref_pages.vs is None else ref_pages.vs[:, :, None, None]))).abs().max())
    smax = float(q.double().norm(dim=-1).max()) * scale * float(
        torch.nan_to_num((ref_pages.k * (1.0 if ref_pages.ks is None else ref_pages.ks[:, :, None, None]))).norm(dim=-1).max())
    e_s = _score_error(cache, io, tiles)
    e_p = (2.0 ** -8 if tiles and io == "bf16" else 2.0 ** -16) if cache == "bf16" else (2.0 ** -11 if io == "bf16" else 2.0 ** -22)
    return vmax * 2 * (e_s * smax + e_p + 2.0 ** -18 + 2.0 ** -18) + ref.abs() * torch.finfo(_io(out_io)).eps / 2


ATTNS = [
    # lens (rows after the call), news, nq, nkv, page
    ([1], [1], 8, 1, 16),
    ([0, 1, 15, 16, 17, 64, 65], [1, 1, 1, 1, 1, 1, 1], 16, 1, 16),
    ([130, 3, 0, 257], [1, 1, 1, 1], 12, 3, 64),
    ([300, 33], [1, 1], 4, 4, 128),
    ([200, 31, 64], [3, 1, 5], 32, 2, 32),
    ([9, 100], [9, 17], 5, 1, 16),
    ([70, 0, 12], [40, 0, 12], 8, 2, 64),
    ([260], [260], 3, 1, 128),
    ([1100], [2], 20, 4, 32),
]


def _attn_case(lens, news, nq, nkv, page, cache, io, seed, masked=False, poison=True):
    gen = torch.Generator().manual_seed(seed)
    T = sum(news)
    table, n_pages = O.tables(lens, page, gen, pad=1 << 30)
    k, v, ks, vs = O.random_pages(n_pages, nkv, page, cache, gen)
    q = torch.randn(T + 1, nq, 128, generator=gen).to(_io(io))
    if poison:                                                                            # rows behind each sequence, pages of nobody
        used = set()
        for b, n in enumerate(lens):
            for i in range(max(0, -(-n // page))):
                g, live = int(table[b, i]), min(page, n - i * page)
                used.add(g)
                for t in (k, v):
                    t[g, :, live:] = torch.tensor(float("nan")).to(t.dtype)
        for g in range(n_pages):
            if g not in used:
                for t in (k, v):
                    t[g] = torch.tensor(float("nan")).to(t.dtype)
    mask = O.tree_mask(news, max(news) + 2, seed) if masked else None
    if mask is not None:
        mask = torch.cat([mask, torch.ones(1, mask.shape[1], dtype=torch.bool)])
    return k, v, ks, vs, table, q, O.cu_of(news), mask


def _run_attn(k, v, ks, vs, table, q, cu, mask, lens, news, out_io=None, lse=True, **kw):
    kd, vd, ksd, vsd, td, qd, cud, md = _dev(k, v, ks, vs, table, q, cu, mask)
    out = torch.full(q.shape, 7.0, dtype=q.dtype if out_io is None else _io(out_io), device=DEV)
    l = torch.full(q.shape[:2], 7.0, device=DEV) if lse else None
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = paged.paged_attention(qd, kd, vd, td, torch.tensor(lens, dtype=torch.int32, device=DEV), cu_q=cud, max_q=max(news), mask=md,
                                k_scale=ksd, v_scale=vsd, out=out, lse=l, err=err, **kw)
    torch.cuda.synchronize()
    assert got is out and int(err) == 0
    return out, l


@pytest.mark.parametrize("lens,news,nq,nkv,page", ATTNS)
@pytest.mark.parametrize("cache", ["fp8", "bf16"])
@pytest.mark.parametrize("io", ["fp32", "bf16"])
@pytest.mark.parametrize("masked", [False, True])
def test_attention(lens, news, nq, nkv, page, cache, io, masked):
    k, v, ks, vs, table, q, cu, mask = _attn_case(lens, news, nq, nkv, page, cache, io, 11 * sum(lens) + nq, masked)
    T = sum(news)
    ref_pages = O.Pages(k, v, ks, vs)
    ref, ref_lse = O.attention(ref_pages, q[:T], table, lens, cu, nkv, mask)
    out, lse = _run_attn(k, v, ks, vs, table, q, cu, mask, lens, news)
    assert bool((out[T:] == 7.0).all()) and bool((lse[T:] == 7.0).all())
    tol = _tol(ref, q[:T], ref_pages, 128 ** -0.5, cache, io, io, tiles=max(news) * (nq // nkv) > 32)
    far = (out[:T].double().cpu() - ref).abs()
    assert bool((far <= tol).all()), (float(far.max()), float(tol.max()))
    got = lse[:T].double().cpu()
    empty = torch.isinf(ref_lse)
    assert torch.equal(torch.isinf(got), empty) and bool((out[:T].cpu()[empty] == 0).all())
    # the denominator is summed from unrounded fp32 probabilities: only the scores' error and the fp32 sums count
    smax = float(q.double().norm(dim=-1).max()) * 128 ** -0.5 * float(torch.nan_to_num(
        (ref_pages.k * (1.0 if ref_pages.ks is None else ref_pages.ks[:, :, None, None]))).norm(dim=-1).max())
    e_s = _score_error(cache, io, max(news) * (nq // nkv) > 32)
    assert float((got - ref_lse)[~empty].abs().max()) <= e_s * smax + 2.0 ** -17


CHUNKS = [
    ([1500, 300, 129], [600, 129, 100], 8, 1, 64),
    ([513, 0, 1], [513, 0, 1], 6, 2, 16),                        # odd group, from the first token
    ([2000], [17], 64, 4, 128),                                  # two tiles of a verify window
    ([5000, 128, 640], [8, 8, 8], 16, 1, 32),                    # one full tile: both groups share its key blocks
    ([384, 384], [128, 256], 2, 1, 128),
    ([1500, 700, 2100, 129, 1900, 64, 1300, 900], [15, 1, 7, 9, 12, 3, 8, 14], 32, 2, 64),     # one and two tiles in turn
    ([130, 140, 5, 129, 128, 300], [9, 8, 5, 1, 15, 2], 64, 4, 16),
]


@pytest.mark.parametrize("lens,news,nq,nkv,page", CHUNKS)
@pytest.mark.parametrize("cache", ["fp8", "bf16"])
@pytest.mark.parametrize("io", ["bf16", "fp32"])
def test_attention_chunks(lens, news, nq, nkv, page, cache, io):
    """Windows of several tiles and key blocks, cut over the GPU."""
    k, v, ks, vs, table, q, cu, _ = _attn_case(lens, news, nq, nkv, page, cache, io, sum(lens))
    T = sum(news)
    ref_pages = O.Pages(k, v, ks, vs)
    ref, ref_lse = O.attention(ref_pages, q[:T], table, lens, cu, nkv)
    out, lse = _run_attn(k, v, ks, vs, table, q, cu, None, lens, news)
    assert bool((out[T:] == 7.0).all())
    tol = _tol(ref, q[:T], ref_pages, 128 ** -0.5, cache, io, io, tiles=True)
    far = (out[:T].double().cpu() - ref).abs()
    assert bool((far <= tol).all()), (float(far.max()), float(tol.max()))
    smax = float(q.double().norm(dim=-1).max()) * 128 ** -0.5 * float(torch.nan_to_num(
        (ref_pages.k * (1.0 if ref_pages.ks is None else ref_pages.ks[:, :, None, None]))).norm(dim=-1).max())
    assert float((lse[:T].double().cpu() - ref_lse).abs().max()) <= _score_error(cache, io, True) * smax + 2.0 ** -17
    again, _ = _run_attn(k, v, ks, vs, table, q, cu, None, lens, news)
    assert torch.equal(out, again)


WINDOWS = [
    # 33 to 128 rows: the table's width chooses the kernel
    ([5000, 128, 640], [8, 8, 8], 16, 1, 32),
    ([9, 100], [9, 17], 5, 1, 16),
    ([200, 31, 64], [3, 1, 5], 32, 2, 32),
    ([700, 0, 1300], [16, 4, 0], 8, 1, 128),
    ([130], [5], 28, 4, 64),
]


@pytest.mark.parametrize("lens,news,nq,nkv,page", WINDOWS)
@pytest.mark.parametrize("cache", ["fp8", "bf16"])
@pytest.mark.parametrize("masked", [False, True])
def test_attention_windows_with_narrow_and_wide_tables(lens, news, nq, nkv, page, cache, masked):
    """A table much wider than its sequences changes the kernel, not the result."""
    k, v, ks, vs, table, q, cu, mask = _attn_case(lens, news, nq, nkv, page, cache, "bf16", 17, masked)
    T = sum(news)
    ref_pages = O.Pages(k, v, ks, vs)
    ref, ref_lse = O.attention(ref_pages, q[:T], table, lens, cu, nkv, mask[:T] if masked else None)
    wide = torch.full((len(lens), 300000 // page), 1 << 30, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    smax = float(q.double().norm(dim=-1).max()) * 128 ** -0.5 * float(torch.nan_to_num(
        (ref_pages.k * (1.0 if ref_pages.ks is None else ref_pages.ks[:, :, None, None]))).norm(dim=-1).max())
    for t, tiles in ((table, False), (wide, True)):
        out, lse = _run_attn(k, v, ks, vs, t, q, cu, mask, lens, news)
        assert bool((out[T:] == 7.0).all())
        far = (out[:T].double().cpu() - ref).abs()
        assert bool((far <= _tol(ref, q[:T], ref_pages, 128 ** -0.5, cache, "bf16", "bf16", tiles=tiles)).all()), (tiles, float(far.max()))
        seen = torch.isfinite(ref_lse)
        got = lse[:T].double().cpu()
        assert torch.equal(seen, torch.isfinite(got))
        assert float((got - ref_lse)[seen].abs().max()) <= _score_error(cache, "bf16", tiles) * smax + 2.0 ** -17


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
def test_attention_long_contexts_are_cut_over_the_gpu(cache):
    """Contexts long enough that every range cuts items; one sequence far longer than the others."""
    lens, news, nq, nkv, page = [9000, 70, 1, 2500], [1, 1, 1, 1], 16, 2, 64
    k, v, ks, vs, table, q, cu, _ = _attn_case(lens, news, nq, nkv, page, cache, "fp32", 3)
    ref_pages = O.Pages(k, v, ks, vs)
    ref, ref_lse = O.attention(ref_pages, q[:4], table, lens, cu, nkv)
    out, lse = _run_attn(k, v, ks, vs, table, q, cu, None, lens, news)
    assert bool(((out[:4].double().cpu() - ref).abs() <= _tol(ref, q[:4], ref_pages, 128 ** -0.5, cache, "fp32", "fp32")).all())
    assert float((lse[:4].double().cpu() - ref_lse).abs().max()) <= 2e-4
    again, _ = _run_attn(k, v, ks, vs, table, q, cu, None, lens, news)
    assert torch.equal(out, again)                                                         # the fold's order is fixed


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
@pytest.mark.parametrize("news", [[6], [40], [150]])
@pytest.mark.parametrize("io", ["fp32", "bf16"])
def test_what_a_token_does_not_see_never_reaches_it(cache, news, io):
    """NaN (and infinities, in bf16 pages) in rows of the call that only later tokens see, and a token that sees nothing."""
    lens, nq, nkv, page = [news[0] + 30], 8, 2, 16
    k, v, ks, vs, table, q, cu, _ = _attn_case(lens, news, nq, nkv, page, cache, io, 4)
    n = news[0]
    clean = O.attention(O.Pages(k, v, ks, vs), q[:n], table, lens, cu, nkv)[0]
    row = lens[0] - 2                                                                     # the last but one token's row
    g, r = int(table[0, row // page]), row % page
    k[g, 0, r, 9] = torch.tensor(float("nan")).to(k.dtype)
    v[g, 1, r, 5] = torch.tensor(float("nan")).to(v.dtype)
    if cache == "bf16":
        v[g, 1, r, 6] = float("inf")
    out, _ = _run_attn(k, v, ks, vs, table, q, cu, None, lens, news)
    got = out[:n].double().cpu()
    tol = _tol(clean, q[:n], O.Pages(k, v, ks, vs), 128 ** -0.5, cache, io, io, tiles=n * 4 > 32)
    assert bool(((got - clean).abs() <= tol)[: n - 2].all())                              # earlier tokens: untouched
    assert bool(torch.isnan(got[n - 2:, :4]).all())                                       # who sees the key: NaN everywhere
    assert bool(torch.isnan(got[n - 2:, 4:, 5]).all())                                    # who sees the value: in its channel
    if cache == "bf16":
        assert bool(torch.isinf(got[n - 2:, 4:, 6]).all())
    other = [c for c in range(128) if c not in (5, 6)]
    assert bool(((got - clean).abs() <= tol)[n - 2:, 4:][..., other].all())
    # with a mask that shows a token nothing and no rows ahead of the call: zeros
    k, v, ks, vs, table, q, cu, _ = _attn_case(news, news, nq, nkv, page, cache, io, 6)
    mask = torch.eye(n + 1, dtype=torch.bool)
    mask[2] = False
    out, lse = _run_attn(k, v, ks, vs, table, q, cu, mask, news, news)
    assert bool((out[2] == 0).all()) and bool(torch.isneginf(lse[2]).all()) and bool(torch.isfinite(lse[:2]).all())


@pytest.mark.parametrize("n", [1, 24])
def test_attention_strides_types_streams_and_graph(n):
    lens, nq, nkv, page = [50 + n, n, 129 + n], 16, 2, 32
    news = [n] * 3
    k, v, ks, vs, table, q, cu, _ = _attn_case(lens, news, nq, nkv, page, "fp8", "bf16", 9)
    T = sum(news)
    q = q[:T]
    kd, vd, ksd, vsd, td, cud = _dev(k, v, ks, vs, table, cu)
    ld = torch.tensor(lens, dtype=torch.int32, device=DEV)
    kw = dict(cu_q=cud, max_q=n, k_scale=ksd, v_scale=vsd)
    want = paged.paged_attention(q.to(DEV), kd, vd, td, ld, **kw)
    # q as a view of wider rows, heads outermost, out strided, table with spare columns
    wide = torch.zeros(T, (nq + 4) * 128, dtype=torch.bfloat16, device=DEV)
    wide[:, :nq * 128] = q.to(DEV).flatten(1)
    assert torch.equal(paged.paged_attention(wide[:, :nq * 128].unflatten(1, (nq, 128)), kd, vd, td, ld, **kw), want)
    outer = q.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)
    buf = torch.full((nq, T, 136), 3.0, dtype=torch.bfloat16, device=DEV)
    got = paged.paged_attention(outer, kd, vd, td, ld, out=buf.transpose(0, 1)[..., :128], **kw)
    assert torch.equal(got, want) and bool((buf[..., 128:] == 3.0).all())
    f32 = paged.paged_attention(q.to(DEV), kd, vd, td, ld, out=torch.empty(T, nq, 128, device=DEV), **kw)
    assert torch.equal(f32.to(torch.bfloat16), want)
    table2 = torch.full((3, td.shape[1] + 5), -1, dtype=torch.int32, device=DEV)
    table2[:, :td.shape[1]] = td
    assert torch.equal(paged.paged_attention(q.to(DEV), kd, vd, table2, ld, **kw), want)
    # two streams at once, then a graph replayed with other lengths in the same tensors
    qd = q.to(DEV)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for s in (s1, s2) * 4:
        with torch.cuda.stream(s):
            outs.append(paged.paged_attention(qd, kd, vd, td, ld, **kw))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graph = torch.cuda.CUDAGraph()
    out = torch.zeros_like(want)
    with torch.cuda.graph(graph):
        paged.paged_attention(qd, kd, vd, td, ld, out=out, **kw)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    ld.copy_(torch.tensor([n + 1, n, 64 + n], dtype=torch.int32))
    short = paged.paged_attention(qd, kd, vd, td, ld, **kw)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, short) and not torch.equal(short, want)


def test_attention_reports_bad_pages():
    """A page id outside the pool: an error word, its rows are not seen; a table too short for kv_len: the rows it holds are."""
    lens, news, nq, nkv, page = [40], [1], 8, 1, 16
    k, v, ks, vs, table, q, cu, _ = _attn_case(lens, news, nq, nkv, page, "fp8", "fp32", 2)
    kd, vd, ksd, vsd, qd = _dev(k, v, ks, vs, q[:1])

    def run(t, n):
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        o = paged.paged_attention(qd, kd, vd, t.to(DEV), torch.tensor([n], dtype=torch.int32, device=DEV), k_scale=ksd, v_scale=vsd, err=err)
        return o.double().cpu(), int(err)

    pages = O.Pages(k, v, ks, vs)
    for bad in (-1, 1 << 20):
        t = table.clone()
        t[0, 0] = bad                                                                     # rows 0 .. 15 are not seen
        moved = table[:, 1:]
        want = O.attention(pages, q[:1], moved, [24], [0, 1], nkv)[0]
        got, err = run(t, 40)
        assert err == 6 and bool(((got - want).abs() <= _tol(want, q[:1], pages, 128 ** -0.5, "fp8", "fp32", "fp32")).all())
    want = O.attention(pages, q[:1], table[:, :2], [32], [0, 1], nkv)[0]
    got, err = run(table[:, :2].contiguous(), 40)
    assert err == 6 and bool(((got - want).abs() <= _tol(want, q[:1], pages, 128 ** -0.5, "fp8", "fp32", "fp32")).all())


def test_scales_of_very_different_size():
    """Pages whose scales are 2^40 apart: the small ones still count where the large ones are not attended to."""
    gen = torch.Generator().manual_seed(1)
    P, L = 16, 64
    k = torch.randn(4, 1, P, 128, generator=gen).to(torch.float8_e4m3fn)
    v = torch.randn(4, 1, P, 128, generator=gen).to(torch.float8_e4m3fn)
    ks = torch.ones(4, 1)
    vs = torch.tensor([[2.0 ** 20], [2.0 ** -20], [1.0], [2.0 ** -60]])
    q = torch.randn(1, 4, 128, generator=gen)
    table = torch.arange(4, dtype=torch.int32)[None]
    for ids in ([0, 1, 2, 3], [1, 3], [3, 2], [3]):
        t = torch.tensor([ids], dtype=torch.int32)
        n = P * len(ids)
        pages = O.Pages(k, v, ks, vs)
        want, want_lse = O.attention(pages, q, t, [n], [0, 1], 1)
        l = torch.zeros(1, 4, device=DEV)
        got = paged.paged_attention(q.to(DEV), k.to(DEV), v.to(DEV), t.to(DEV), torch.tensor([n], dtype=torch.int32, device=DEV),
                                    k_scale=ks.to(DEV), v_scale=vs.to(DEV), lse=l).double().cpu()
        seen = float((pages.v * vs[:, :, None, None].double())[ids].abs().max())
        assert float((got - want).abs().max()) <= seen * 2.0 ** -17
        assert float((l.double().cpu() - want_lse).abs().max()) <= 2.0 ** -17


@pytest.mark.parametrize("kv,io", [("fp8", "bf16"), ("fp8", "fp32"), ("bf16", "bf16")])
def test_serving_several_sequences_from_prompt_to_tokens(kv, io):
    """The two operators as a server uses them, two layers: ragged prompt chunks, decode steps of a batch, a fork of a common prefix, a token
    tree whose tail is dropped, a freed sequence. Every attention output against 64-bit attention over what the pages hold, and what
    they hold against the rows that went in."""
    from inferencehackathon_b200.runtime.paged_kv import PagedKVCache
    gen = torch.Generator().manual_seed(12)
    nq, nkv, P, layers = 8, 2, 16, 2
    cache = PagedKVCache(layers, 64, nkv, P, kv, DEV)
    cos, sin = _dev(*O.rope_tables(400))
    rows = {}                                                 # (sequence, layer) -> list of V rows [nkv, 128] that went in

    def step(new, tree=False):
        batch = cache.extend(new)
        T = batch.n_tokens
        mask = O.tree_mask(list(new.values()), batch.max_q, T) if tree else None
        for layer in range(layers):
            qkv = torch.randn(T, (nq + 2 * nkv) * 128, generator=gen).to(_io(io))
            q = cache.append(layer, qkv.to(DEV), batch, cos, sin, nq=nq)
            t = 0
            for s, n in new.items():
                have = rows.setdefault((s, layer), [])
                del have[cache.length(s) - n:]
                have += [x for x in qkv[t:t + n, (nq + nkv) * 128:].double().view(n, nkv, 128)]
                t += n
            out = cache.attend(layer, q, batch, mask=None if mask is None else mask.to(DEV))
            cache.check_error()
            ks, vs = (None, None) if cache.k_scale is None else (cache.k_scale[layer].cpu(), cache.v_scale[layer].cpu())
            pages = O.Pages(cache.k[layer].float().cpu(), cache.v[layer].float().cpu(), ks, vs)
            for t in (pages.k, pages.v):
                t.nan_to_num_(0.0)                            # pages that nothing was written to hold anything
            cu = O.cu_of(list(new.values()))
            ref, _ = O.attention(pages, q.cpu(), batch.block_table, batch.kv_len, cu, nkv, mask)
            tol = _tol(ref, q.cpu(), _live(pages, cache, rows), 128 ** -0.5, kv, io, io, tiles=batch.max_q * (nq // nkv) > 32)
            assert bool(((out.double().cpu() - ref).abs() <= tol).all())
            for s in new:
                got = pages.rows("v", torch.tensor(cache.pages(s)), 0, cache.length(s))
                want = torch.stack([r[0] for r in rows[(s, layer)]])
                big = max(float(want.abs().max()), 1.0)
                assert float((got - want).abs().max()) <= big * (2.0 ** -4 if kv == "fp8" else 2.0 ** -8)

    def _live(pages, cache, rows):
        ids = sorted({p for s in {k[0] for k in rows} for p in cache.pages(s)})
        return O.Pages(pages.k[ids], pages.v[ids], None if pages.ks is None else pages.ks[ids], None if pages.vs is None else pages.vs[ids])

    for s in "abc":
        cache.add(s)
    step({"a": 37, "b": 1, "c": 64})
    step({"a": 1, "b": 1, "c": 1})
    step({"b": 90, "a": 3})
    cache.fork("a", "d")
    for layer in range(layers):
        rows[("d", layer)] = list(rows[("a", layer)])
    step({"d": 1, "a": 1, "b": 1, "c": 1})
    step({"c": 9, "d": 4}, tree=True)
    cache.truncate("c", cache.length("c") - 6)
    step({"c": 2, "d": 1})
    cache.free("b")
    for layer in range(layers):
        del rows[("b", layer)]
    step({"a": 1, "c": 1, "d": 1})
