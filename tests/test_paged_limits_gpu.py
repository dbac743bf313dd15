"""Paged cache kernels at the edges of what their entry points allow, against plain 64-bit implementations (needs a B200).

Tolerance of an attention output: probabilities that are each off by a relative d move it by at most 2 d sum_j p_j |v_j| (numerator and
denominator); d is the rounding of P (fp16 2^-11 for bf16 queries over e4m3 pages, fp16 pairs 2^-22 for fp32 ones, bf16 pairs 2^-16, one bf16 2^-8), the
error of the scores (see test_paged_gpu.py) and 2^-17 for fp32 sums and exponents; then half a step of the output type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import paged_oracle as O
from inferencehackathon_b200.ops import paged

DEV = "cuda:0"
F64 = torch.float64


def _io(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _reference(k, v, ks, vs, q, table, lens, news, nkv, mask=None, scale=128 ** -0.5):
    """out, lse, sum_j p_j |v_j| [T, nq, 128 / - / 128] in 64 bits. NaN and infinities of V reach the rows that see them, in their channel."""
    T, nq = q.shape[:2]
    G = nq // nkv
    out = torch.full((T, nq, 128), float("nan"), dtype=F64)
    mag, lse = out.clone(), torch.full((T, nq), float("nan"), dtype=F64)
    P, t = k.shape[2], 0
    for b, (L, n) in enumerate(zip(lens, news)):
        if n == 0:
            continue
        base, ids = L - n, table[b, :-(-L // P)].long()
        j = torch.arange(L)[None, :]
        i = torch.arange(n)[:, None]
        if mask is None:
            see = j <= base + i
        else:
            see = (j < base) | torch.nn.functional.pad(mask[t:t + n, :n].bool(), (base, 0))
        for h in range(nkv):
            kk, vv = k[ids, h].to(F64), v[ids, h].to(F64)
            if ks is not None:
                kk, vv = kk * ks[ids, h].to(F64)[:, None, None], vv * vs[ids, h].to(F64)[:, None, None]
            kk, vv = kk.reshape(-1, 128)[:L].to(DEV), vv.reshape(-1, 128)[:L].to(DEV)
            odd = ~torch.isfinite(vv)
            clean = vv.masked_fill(odd, 0.0)
            s = see.to(DEV)
            for g in range(h * G, (h + 1) * G):
                w = (q[t:t + n, g].to(F64).to(DEV) @ kk.T * scale).masked_fill(~s, -math.inf)
                m = torch.logsumexp(w, 1, keepdim=True)
                p = torch.where(torch.isinf(m), torch.zeros_like(w), torch.exp(w - m))
                o = p @ clean
                if bool(odd.any()):
                    hit = s.to(F64) @ torch.isnan(vv).to(F64) > 0
                    for c in torch.isinf(vv).any(0).nonzero().flatten().tolist():
                        for r in torch.isinf(vv[:, c]).nonzero().flatten().tolist():
                            o[s[:, r], c] += vv[r, c]
                    o[hit] = float("nan")
                out[t:t + n, g], lse[t:t + n, g], mag[t:t + n, g] = o.cpu(), m[:, 0].cpu(), (p @ clean.abs()).cpu()
        t += n
    return out, lse, mag


def _check(out, ref, mag, d, out_io):
    got = out.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(torch.isinf(got), torch.isinf(ref))
    fin = torch.isfinite(ref)
    tol = 2 * d * mag + ref.abs() * (torch.finfo(_io(out_io)).eps / 2)
    far = ((got - ref).abs() - tol)[fin]
    assert float(far.max()) <= 0, (float((got - ref)[fin].abs().max()), int((far > 0).sum()))


def _score_bound(q, k, ks, cache, io, tiles, scale=128 ** -0.5):
    """Largest error of a score: what the queries' split loses (test_paged_gpu.py) times |q| |k| scale, and fp32 sums."""
    kk = torch.nan_to_num(k.to(F64) * (1.0 if ks is None else ks[:, :, None, None].to(F64)))
    smax = float(q.to(F64).norm(dim=-1).max()) * float(kk.norm(dim=-1).max()) * scale
    e = (2.0 ** -17 * 128 ** 0.5 if tiles and cache == "fp8" else 0.0) if io == "bf16" else (2.0 ** -22 if cache == "fp8" else 2.0 ** -16)
    return e * smax + 2.0 ** -17


def _p_step(cache, io, tiles):
    if cache == "fp8":
        return 2.0 ** -11 if io == "bf16" else 2.0 ** -22
    return 2.0 ** -8 if tiles and io == "bf16" else 2.0 ** -16


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
def test_many_tile_pairs_per_block_with_values_that_are_not_finite(cache):
    """Several items of two tiles for every SM, ragged last tiles, and NaN in V rows of some windows: their rows take much longer in the epilogue than
    the others' of the same tile, whose warps must not touch what is staged for them meanwhile."""
    gen = torch.Generator().manual_seed(41)
    nq, nkv, page, B = 16, 4, 32, 44
    news = [100 + 7 * (b * 5 % 19) for b in range(B)]
    lens = [n + (0 if b % 3 == 0 else 13 * (b % 7)) for b, n in enumerate(news)]
    table, n_pages = O.tables(lens, page, gen)
    k, v, ks, vs = O.random_pages(n_pages, nkv, page, cache, gen, spread=False)
    for b in range(0, B, 3):
        row = lens[b] - news[b] + news[b] // 2 + b % 5
        v[int(table[b, row // page]), b % nkv, row % page, 3 * b % 128] = torch.tensor(float("nan")).to(v.dtype)
    q = torch.randn(sum(news), nq, 128, generator=gen).to(torch.bfloat16)
    ref, ref_lse, mag = _reference(k, v, ks, vs, q, table, lens, news, nkv)
    d = _p_step(cache, "bf16", True) + _score_bound(q, k, ks, cache, "bf16", True)
    dev = [None if t is None else t.to(DEV) for t in (q, k, v, table, ks, vs, O.cu_of(news))]
    ld = torch.tensor(lens, dtype=torch.int32, device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    lse = torch.empty(q.shape[:2], device=DEV)
    first = None
    for _ in range(4):
        out = paged.paged_attention(*dev[:4], ld, cu_q=dev[6], max_q=max(news), k_scale=dev[4], v_scale=dev[5], lse=lse, err=err)
        _check(out, ref, mag, d, "bf16")
        assert int(err) == 0 and float((lse.double().cpu() - ref_lse).abs().max()) <= _score_bound(q, k, ks, cache, "bf16", True)
        first = out if first is None else first
        assert torch.equal(out.view(torch.int16), first.view(torch.int16))


class _DirtyEmpty:
    """torch for the module under test, with every new tensor full of 0xff bytes."""

    def __getattr__(self, name):
        return getattr(torch, name)

    def empty(self, *a, **kw):
        t = torch.empty(*a, **kw)
        t.view(torch.uint8).fill_(255)
        return t


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
@pytest.mark.parametrize("lens,news,nq,nkv", [([900, 1, 3000], [1, 1, 1], 16, 2), ([700, 90, 2500], [300, 90, 40], 16, 2), ([40, 0], [40, 0], 8, 1)])
def test_scratch_may_hold_anything(cache, lens, news, nq, nkv, monkeypatch):
    """The pieces that a second kernel folds are read only where the first one wrote them."""
    gen = torch.Generator().manual_seed(7)
    table, n_pages = O.tables(lens, 64, gen)
    k, v, ks, vs = O.random_pages(n_pages, nkv, 64, cache, gen)
    q = torch.randn(sum(news), nq, 128, generator=gen).to(torch.bfloat16)
    q, k, v, table, ks, vs, cu = [None if t is None else t.to(DEV) for t in (q, k, v, table, ks, vs, O.cu_of(news))]
    ld = torch.tensor(lens, dtype=torch.int32, device=DEV)
    outs = []
    for dirty in (False, True):
        if dirty:
            monkeypatch.setattr(paged, "torch", _DirtyEmpty())
        out = torch.zeros_like(q)
        paged.paged_attention(q, k, v, table, ld, cu_q=cu, max_q=max(news), k_scale=ks, v_scale=vs, out=out)
        outs.append(out)
    assert torch.equal(*outs) and bool(torch.isfinite(outs[0]).all())


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
@pytest.mark.parametrize("n", [2, 40])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("long", [200, 2 ** 31 - 1, 2 ** 31 - 300])
def test_a_length_that_its_table_does_not_hold_costs_only_its_own_rows(cache, n, masked, long):
    """Short windows and tiles: the other sequences' results are those of a call without it; its own tokens see the rows that the table holds."""
    gen = torch.Generator().manual_seed(n)
    nq, nkv, page = 8, 1, 16
    lens, news = [300, 128, 90, n], [n, n, n, n]
    table, n_pages = O.tables(lens, page, gen)
    table = table[:, :19].contiguous()
    k, v, ks, vs = O.random_pages(n_pages, nkv, page, cache, gen, spread=False)
    table[1, 8:] = -1
    table = table[:, :8].contiguous() if long == 200 else table
    lens[0] = min(lens[0], table.shape[1] * page)
    q = torch.randn(4 * n, nq, 128, generator=gen).to(torch.bfloat16)
    mask = torch.ones(4 * n, n, dtype=torch.bool).tril() if masked else None
    qd, kd, vd, td, ksd, vsd, cu, md = [None if t is None else t.to(DEV) for t in (q, k, v, table, ks, vs, O.cu_of(news), mask)]

    def run(ls):
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        o = paged.paged_attention(qd, kd, vd, td, torch.tensor(ls, dtype=torch.int32, device=DEV), cu_q=cu, max_q=n, mask=md, k_scale=ksd,
                                  v_scale=vsd, err=err)
        return o, int(err)

    good, code = run(lens)
    assert code == 0
    table[1, 8:] = table[0, 0]                                       # (rows of another page: whatever the table names is seen)
    td = table.to(DEV)
    held = table.shape[1] * page
    bad, code = run([lens[0], long, lens[2], lens[3]])
    assert code == 6
    keep = [t for t in range(4 * n) if not n <= t < 2 * n]
    d = _p_step(cache, "bf16", n * nq > 32) + _score_bound(q, k, ks, cache, "bf16", True)
    ref, _, mag = _reference(k, v, ks, vs, q[n:2 * n], table[1:2].expand(n, -1), [held] * n, [1] * n, nkv)
    assert long - n >= held                                          # (none of its tokens' own rows is held: they see all that is)
    _check(bad[n:2 * n], ref, mag, d, "bf16")
    want, _, mag = _reference(k, v, ks, vs, q, table, [lens[0], n, lens[2], lens[3]], news, nkv, mask)
    for o in (good, bad):
        _check(o[keep], want[keep], mag[keep], d, "bf16")


def _mask_views(n, width, T, gen):
    """name -> (a view [T, >= n] that is not plain contiguous bool, the same bits as a contiguous bool tensor)."""
    flat = (torch.rand(T + n - 1, generator=gen) < 0.6).to(DEV)
    row = (torch.rand(1, n, generator=gen) < 0.6).to(DEV)
    full = (torch.rand(T, n, generator=gen) < 0.6).to(DEV)
    wide = torch.ones(T, width, dtype=torch.bool, device=DEV)
    wide[:, 3:3 + n] = full
    bytes_ = torch.where(full, torch.randint(1, 256, (T, n), generator=gen).to(DEV), torch.zeros((), dtype=torch.long, device=DEV)).to(torch.uint8)
    band = flat.unfold(0, n, 1)
    return {"band of one vector": (band, band.contiguous()), "one row for all": (row.expand(T, -1), row.repeat(T, 1)),
            "columns of a wider one": (wide[:, 3:3 + n], full), "bytes": (bytes_, full), "one row, odd stride": (full.as_strided((1, n), (1, 1)), full[:1])}


@pytest.mark.parametrize("cache,io", [("fp8", "bf16"), ("bf16", "bf16"), ("bf16", "fp32")])
@pytest.mark.parametrize("n", [3, 30, 45])
def test_mask_views_are_their_contiguous_copies(cache, io, n):
    """Rows that overlap, one row for all tokens, columns of a wider mask, bytes: short windows and tiles (45 tokens of 8 heads)."""
    gen = torch.Generator().manual_seed(n)
    nq, nkv, page, news = 8, 1, 16, [n, n - 1, n]
    lens = [100 + n, n - 1, 7 + n]
    T = sum(news)
    table, n_pages = O.tables(lens, page, gen)
    k, v, ks, vs = O.random_pages(n_pages, nkv, page, cache, gen, spread=False)
    q = torch.randn(T, nq, 128, generator=gen).to(_io(io))
    qd, kd, vd, td, ksd, vsd, cu = [None if t is None else t.to(DEV) for t in (q, k, v, table, ks, vs, O.cu_of(news))]
    ld = torch.tensor(lens, dtype=torch.int32, device=DEV)
    d = _p_step(cache, io, n * nq > 32) + _score_bound(q, k, ks, cache, io, n * nq > 32)
    for name, (view, plain) in _mask_views(n, n + 24, T, gen).items():
        a = (qd, kd, vd, td, ld)
        kw = dict(cu_q=cu, max_q=n, k_scale=ksd, v_scale=vsd)
        want_lens, want_news, q_of, table_of = lens, news, q, table
        if view.shape[0] == 1:                                       # (a call of one token)
            a = (qd[:1], kd, vd, td[:1], ld[:1])
            kw = dict(max_q=1, k_scale=ksd, v_scale=vsd)
            want_lens, want_news, q_of, table_of = lens[:1], [1], q[:1], table[:1]
        ref, _, mag = _reference(k, v, ks, vs, q_of, table_of, want_lens, want_news, nkv, plain.cpu())
        got = paged.paged_attention(*a, mask=view, **kw)
        _check(got, ref, mag, d, io)
        assert torch.equal(got, paged.paged_attention(*a, mask=plain, **kw)), name


def test_tokens_beyond_the_mask_are_not_read_from_it():
    """More tokens than max_q and than a mask's columns: an error word, and no byte outside of the view counts."""
    gen = torch.Generator().manual_seed(2)
    nq, nkv, page, n = 8, 1, 16, 6
    table, n_pages = O.tables([40], page, gen)
    k, v, _, _ = O.random_pages(n_pages, nkv, page, "bf16", gen, spread=False)
    q = torch.randn(n, nq, 128, generator=gen)
    qd, kd, vd, td = (t.to(DEV) for t in (q, k, v, table))
    outs = []
    for outside in (False, True):
        wide = torch.full((n, 64), outside, dtype=torch.bool, device=DEV)
        wide[:, 5:9] = torch.ones(n, 4, dtype=torch.bool, device=DEV).tril()
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        out = torch.zeros(n, nq, 128, device=DEV)
        paged.paged_attention(qd, kd, vd, td, torch.tensor([40], dtype=torch.int32, device=DEV), cu_q=torch.tensor([0, n], dtype=torch.int32, device=DEV),
                              max_q=4, mask=wide[:, 5:9], out=out, err=err)
        assert int(err) == 6
        outs.append(out)
    assert torch.equal(*outs)


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
@pytest.mark.parametrize("io", ["fp32", "bf16"])
@pytest.mark.parametrize("n", [4, 40])
def test_a_token_that_sees_nothing_gets_zeros_whatever_its_query_holds(cache, io, n):
    """NaN and infinities in the queries of padded tokens, whose mask is empty; the other tokens of their tile are not touched."""
    gen = torch.Generator().manual_seed(n)
    nq, nkv, page = 8, 1, 32
    lens, news = [n], [n]
    table, n_pages = O.tables(lens, page, gen)
    k, v, ks, vs = O.random_pages(n_pages, nkv, page, cache, gen, spread=False)
    q = torch.randn(n, nq, 128, generator=gen)
    mask = torch.ones(n, n, dtype=torch.bool).tril()
    for t, x in ((1, float("nan")), (2, float("inf")), (n - 1, float("-inf"))):
        q[t, :, 7 * t % 128] = x
        mask[t] = False
    q = q.to(_io(io))
    qd, kd, vd, td, ksd, vsd, cu, md = [None if t is None else t.to(DEV) for t in (q, k, v, table, ks, vs, O.cu_of(news), mask)]
    lse = torch.empty(n, nq, device=DEV)
    out = paged.paged_attention(qd, kd, vd, td, torch.tensor(lens, dtype=torch.int32, device=DEV), cu_q=cu, max_q=n, mask=md, k_scale=ksd, v_scale=vsd, lse=lse)
    fine = [t for t in range(n) if t not in (1, 2, n - 1)]
    ref, _, mag = _reference(k, v, ks, vs, torch.nan_to_num(q, posinf=0.0, neginf=0.0), table, lens, news, nkv, mask)
    _check(out[fine], ref[fine], mag[fine], _p_step(cache, io, n * nq > 32) + _score_bound(torch.nan_to_num(q, posinf=0.0, neginf=0.0), k, ks, cache, io, n * nq > 32), io)
    for t in (1, 2, n - 1):
        assert bool((out[t] == 0).all()) and bool(torch.isneginf(lse[t]).all())
    md[1, 0] = True                                                  # seen: NaN
    out = paged.paged_attention(qd, kd, vd, td, torch.tensor(lens, dtype=torch.int32, device=DEV), cu_q=cu, max_q=n, mask=md, k_scale=ksd, v_scale=vsd)
    assert bool(torch.isnan(out[1]).all()) and bool((out[2] == 0).all())


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
@pytest.mark.parametrize("io", ["fp32", "bf16"])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_rows_of_zeros(cache, io, n):
    """Queries of zeros and keys of zeros, as a warm-up call or padded tokens bring them (e4m3 pages of zeros have the least scale, 2^-60): uniform
    probabilities over the keys that a token sees, for single tokens, short windows and tiles."""
    gen = torch.Generator().manual_seed(n)
    nq, nkv, page = 8, 1, 16
    lens, news = [n + 30, n, 200 + n], [n] * 3
    T = 3 * n
    table, n_pages = O.tables(lens, page, gen)
    qkv = torch.zeros(T, (nq + 2 * nkv) * 128)
    qkv[:, -128:] = torch.randn(T, 128, generator=gen)
    k, v, ks, vs = O.random_pages(n_pages, nkv, page, cache, gen, spread=False)
    k.zero_()
    if ks is not None:
        ks.fill_(2.0 ** -60)
    kd, vd, td, ksd, vsd, cu, x = [None if t is None else t.to(DEV) for t in (k, v, table, ks, vs, O.cu_of(news), qkv.to(_io(io)))]
    cos, sin = (t.to(DEV) for t in O.rope_tables(300))
    ld = torch.tensor(lens, dtype=torch.int32, device=DEV)
    q = paged.paged_append(x, nq, nkv, kd, vd, td, ld, cos, sin, cu_q=cu, q_gamma=torch.ones(128, device=DEV), k_gamma=torch.ones(128, device=DEV),
                           k_scale=ksd, v_scale=vsd)
    assert bool((q == 0).all()) and bool((kd.float() == 0).all())
    lse = torch.empty(T, nq, device=DEV)
    out = paged.paged_attention(q, kd, vd, td, ld, cu_q=cu, max_q=n, k_scale=ksd, v_scale=vsd, lse=lse)
    ref, ref_lse, mag = _reference(kd.cpu(), vd.cpu(), None if ks is None else ksd.cpu(), None if ks is None else vsd.cpu(), q.cpu(), table, lens, news, nkv)
    _check(out, ref, mag, _p_step(cache, io, n * nq > 32) + 2.0 ** -17, io)
    assert float((lse.double().cpu() - ref_lse).abs().max()) <= 2.0 ** -17


@pytest.mark.parametrize("io", ["fp32", "bf16"])
def test_scores_of_any_finite_size(io):
    """A token that sees one key has that key's value for its result, however large or small the score; of two keys 2^40 apart the larger one's."""
    gen = torch.Generator().manual_seed(3)
    nq, P = 8, 16
    k = torch.ones(1, 1, P, 128, dtype=torch.bfloat16) * 2.0 ** 60
    v = torch.randn(1, 1, P, 128, generator=gen).to(torch.bfloat16)
    q = (torch.tensor([-(2.0 ** 50), 2.0 ** 50, -(2.0 ** 20), 2.0 ** 20, -(2.0 ** -80), 0.0, -(2.0 ** 41), 1.0]) / 128)[None, :, None].expand(1, -1, 128).contiguous()
    table = torch.zeros(1, 1, dtype=torch.int32)
    for n in (1, 2):
        if n == 2:
            k[0, 0, 1] = 2.0 ** 20                                   # the scores' sign decides
        out = paged.paged_attention(q.to(_io(io)).to(DEV), k.to(DEV), v.to(DEV), table.to(DEV), torch.tensor([n], dtype=torch.int32, device=DEV))
        want = v[0, 0, 0].expand(nq, -1).clone()
        if n == 2:
            want[torch.tensor([0, 2, 6])] = v[0, 0, 1]
            rows = [0, 1, 2, 3, 6, 7]
        else:
            rows = list(range(nq))
        got = out[0].to(torch.bfloat16).cpu()
        assert torch.equal(got[rows], want[rows])


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
@pytest.mark.parametrize("io", ["fp32", "bf16"])
@pytest.mark.parametrize("nq,nkv", [(256, 1), (100, 1), (34, 2), (250, 2)])
@pytest.mark.parametrize("masked", [False, True])
def test_many_query_heads_per_kv_head(cache, io, nq, nkv, masked):
    """A token over several row tiles, decode and windows, odd groups."""
    gen = torch.Generator().manual_seed(nq)
    page = 32
    for lens, news in (([70, 0, 1, 300], [1, 1, 1, 1]), ([150, 9, 2], [5, 9, 2])):
        table, n_pages = O.tables(lens, page, gen)
        k, v, ks, vs = O.random_pages(n_pages, nkv, page, cache, gen, spread=False)
        q = torch.randn(sum(news), nq, 128, generator=gen).to(_io(io))
        mask = O.tree_mask(news, max(news), 5) if masked else None
        qd, kd, vd, td, ksd, vsd, cu, md = [None if t is None else t.to(DEV) for t in (q, k, v, table, ks, vs, O.cu_of(news), mask)]
        lse = torch.empty(sum(news), nq, device=DEV)
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        out = paged.paged_attention(qd, kd, vd, td, torch.tensor(lens, dtype=torch.int32, device=DEV), cu_q=cu, max_q=max(news), mask=md, k_scale=ksd,
                                    v_scale=vsd, lse=lse, err=err)
        tiles = max(news) * (nq // nkv) > 32
        eff = [max(n, 0) for n in lens]
        live = [m if L else 0 for L, m in zip(eff, news)]
        keep = torch.cat([torch.full((m,), bool(L), dtype=torch.bool) for L, m in zip(eff, news)])
        ref, ref_lse, mag = _reference(k, v, ks, vs, q[keep], table, eff, live, nkv, None if mask is None else mask[keep])
        bound = _score_bound(q, k, ks, cache, io, tiles)
        _check(out[keep.to(DEV)], ref, mag, _p_step(cache, io, tiles) + bound, io)
        assert float((lse[keep.to(DEV)].double().cpu() - ref_lse).abs().max()) <= bound
        gone = ~keep.to(DEV)
        assert int(err) == 0 and bool((out[gone] == 0).all()) and bool(torch.isneginf(lse[gone]).all())


def _near_ties(T, nkv, norm, io, gen, gamma, cos, sin, pos, edge, every):
    """K rows [T, nkv, 128] with normed, rotated values that lie within a few units of fp32 rounding of a tie between two e4m3 numbers, the sums that
    form them cancelling up to a hundredfold: in ``every`` pair, or in one of a row. ``edge``: the largest value of each row next to 448 instead, where
    the page scale changes."""
    y = torch.rand(T, nkv, 128, generator=gen, dtype=F64) * 300 + 100
    y = y * torch.where(torch.rand(y.shape, generator=gen) < 0.5, 1.0, -1.0)
    c, s = cos[pos].double()[:, None], sin[pos].double()[:, None]
    off = torch.rand(T, nkv, 64, generator=gen, dtype=F64) * 0.3 + 0.1
    if every:
        off.zero_()
    else:
        off.scatter_(2, torch.randint(0, 64, (T, nkv, 1), generator=gen), 0.0)
    t = (torch.randint(8, 16, (T, nkv, 64), generator=gen) + 0.5 + off) * torch.exp2(torch.randint(-1, 3, (T, nkv, 64), generator=gen).double())
    t = t * torch.where(torch.rand(t.shape, generator=gen) < 0.5, 1.0, -1.0)
    if edge:
        y = y / 4
        t = t / 4
        t[:, :, 5] = 448.0
        y[:, :, 5] = 300.0
    y[..., 64:] = (y[..., :64] * c - t) / s                          # a c - b s = t
    if norm:                                                         # y = x / rms(x) gamma: mean((y / gamma)^2) = 1
        f = torch.sqrt(((y / gamma.double()) ** 2).mean(-1, keepdim=True))
        f = torch.exp2(torch.ceil(torch.log2(f)))                    # a power of two keeps the ties
        y = y / f
        rest = 1 - ((y / gamma.double()) ** 2).mean(-1)              # the missing part in a pair that is no tie: its a c - b s is as it comes
        a = y[..., 20] / gamma[20].double()
        y[..., 20] = torch.sqrt(a * a + 128 * rest) * gamma[20].double()
        y = y * 3 / gamma.double()                                   # x: any multiple of y / gamma
    return y.to(_io(io))


@pytest.mark.parametrize("norm,edge", [(False, False), (False, True), (True, False)])       # (with a norm the largest value is the free one)
@pytest.mark.parametrize("every", [False, True])
@pytest.mark.parametrize("page,lens,news", [(16, [5, 40, 3], [5, 17, 3]), (128, [200, 7, 300], [200, 7, 131]), (64, [1, 64, 65, 130, 20], [1, 1, 1, 1, 1]),
                                            (32, [700], [700])])
def test_bytes_next_to_ties_are_those_of_64_bits(norm, edge, every, page, lens, news):
    """Every byte and scale of e4m3 pages equals the 64-bit ones, with and without gammas, odd row counts, rotation angles of their own."""
    gen = torch.Generator().manual_seed(page + norm)
    nq, nkv, T = 2, 2, sum(news)
    ang = torch.rand(2000, 64, generator=gen, dtype=F64) * 0.9 + 0.35          # no angle near a multiple of a quarter turn
    cos, sin = ang.cos().float(), ang.sin().float()
    pos = torch.randint(0, 2000, (T,), generator=gen).to(torch.int32)
    qg, kg = ((1 + 0.2 * torch.randn(128, generator=gen)) for _ in range(2)) if norm else (None, None)
    qkv = torch.randn(T, nq + 2 * nkv, 128, generator=gen)
    qkv[:, nq:nq + nkv] = _near_ties(T, nkv, norm, "fp32", gen, kg, cos, sin, pos.long(), edge, every)
    qkv = qkv.flatten(1)
    table, n_pages = O.tables(lens, page, gen)
    k, v, ks, vs = O.random_pages(n_pages, nkv, page, "fp8", gen)
    ref = O.Pages(k, v, ks, vs)
    O.append(ref, qkv, nq, nkv, table, lens, O.cu_of(news), cos, sin, qg, kg, positions=pos)
    x, kd, vd, ksd, vsd, td, cu, cosd, sind, qgd, kgd, pd = [None if t is None else t.to(DEV) for t in
                                                             (qkv, k, v, ks, vs, table, O.cu_of(news), cos, sin, qg, kg, pos)]
    paged.paged_append(x, nq, nkv, kd, vd, td, torch.tensor(lens, dtype=torch.int32, device=DEV), cosd, sind, cu_q=cu, positions=pd, q_gamma=qgd,
                       k_gamma=kgd, k_scale=ksd, v_scale=vsd)
    assert torch.equal(ksd.double().cpu(), ref.ks) and torch.equal(vsd.double().cpu(), ref.vs)
    for got, want in ((kd, ref.k), (vd, ref.v)):
        assert torch.equal(got.float().double().cpu(), want), int((got.float().double().cpu() != want).sum())


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
@pytest.mark.parametrize("lens,news,nq,nkv,page", [([700, 128, 90], [5, 8, 8], 16, 1, 32), ([300, 0, 61], [16, 0, 16], 8, 1, 128), ([130], [5], 28, 4, 64),
                                                   ([1000], [2], 128, 2, 16)])
def test_a_wider_table_does_not_cost_bits(cache, lens, news, nq, nkv, page):
    """33 to 128 rows: the table's width chooses the kernel. An fp32 result shows what is left of the probabilities in each."""
    gen = torch.Generator().manual_seed(23)
    table, n_pages = O.tables(lens, page, gen)
    k, v, ks, vs = O.random_pages(n_pages, nkv, page, cache, gen, spread=False)
    q = torch.randn(sum(news), nq, 128, generator=gen).to(torch.bfloat16)
    ref, _, mag = _reference(k, v, ks, vs, q, table, lens, news, nkv)
    wide = torch.full((len(lens), 300000 // page), 1 << 30, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    qd, kd, vd, ksd, vsd, cu = [None if t is None else t.to(DEV) for t in (q, k, v, ks, vs, O.cu_of(news))]
    for t in (table, wide):
        out = torch.empty(q.shape, device=DEV)
        paged.paged_attention(qd, kd, vd, t.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), cu_q=cu, max_q=max(news), k_scale=ksd,
                              v_scale=vsd, out=out)
        _check(out, ref, mag, _p_step(cache, "bf16", False) + _score_bound(q, k, ks, cache, "bf16", t is wide), "fp32")


@pytest.mark.parametrize("io", ["bf16", "fp32"])
@pytest.mark.parametrize("cache", ["fp8", "bf16"])
def test_an_fp32_result_of_a_prompt_has_the_bits_of_its_probabilities(cache, io):
    gen = torch.Generator().manual_seed(29)
    nq, nkv, page, lens, news = 16, 2, 64, [700, 250], [200, 250]
    table, n_pages = O.tables(lens, page, gen)
    k, v, ks, vs = O.random_pages(n_pages, nkv, page, cache, gen, spread=False)
    q = torch.randn(sum(news), nq, 128, generator=gen).to(_io(io))
    ref, _, mag = _reference(k, v, ks, vs, q, table, lens, news, nkv)
    qd, kd, vd, td, ksd, vsd, cu = [None if t is None else t.to(DEV) for t in (q, k, v, table, ks, vs, O.cu_of(news))]
    out = torch.empty(q.shape, device=DEV)
    paged.paged_attention(qd, kd, vd, td, torch.tensor(lens, dtype=torch.int32, device=DEV), cu_q=cu, max_q=max(news), k_scale=ksd, v_scale=vsd, out=out)
    _check(out, ref, mag, _p_step(cache, io, False) + _score_bound(q, k, ks, cache, io, True), "fp32")


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
@pytest.mark.parametrize("io", ["bf16", "fp32"])
@pytest.mark.parametrize("n,lens", [(1, [2000]), (12, [2000, 1999]), (100, [2000])])
def test_norm_of_the_error_over_many_keys(cache, io, n, lens):
    """Roundings of P have no sign in common: over all outputs the error's norm is that of independent ones, each at most d of its p_j v_j. A single V row
    out of place among 2000, which an elementwise bound would let pass, is far above that."""
    gen = torch.Generator().manual_seed(n)
    nq, nkv, page = 16, 2, 16
    news = [n] * len(lens)
    T, G = n * len(lens), nq // nkv
    table, n_pages = O.tables(lens, page, gen)
    k, v, ks, vs = O.random_pages(n_pages, nkv, page, cache, gen, spread=False)
    q = torch.randn(T, nq, 128, generator=gen).to(_io(io))
    qd, kd, vd, td, ksd, vsd, cu = [None if t is None else t.to(DEV) for t in (q, k, v, table, ks, vs, O.cu_of(news))]
    out = paged.paged_attention(qd, kd, vd, td, torch.tensor(lens, dtype=torch.int32, device=DEV), cu_q=cu, max_q=n, k_scale=ksd, v_scale=vsd).double()
    off = worst = split = 0.0
    for b, L in enumerate(lens):
        ids = table[b, :-(-L // page)].long()
        for h in range(nkv):
            f = 1.0 if ks is None else ks[ids, h].to(F64)[:, None, None]
            g = 1.0 if vs is None else vs[ids, h].to(F64)[:, None, None]
            kk = (k[ids, h].to(F64) * f).reshape(-1, 128)[:L].to(DEV)
            vv = (v[ids, h].to(F64) * g).reshape(-1, 128)[:L].to(DEV)
            x = qd[b * n:(b + 1) * n, h * G:(h + 1) * G].to(F64)
            w = x.flatten(0, 1) @ kk.T * 128 ** -0.5
            seen = torch.arange(L, device=DEV)[None, :] <= L - n + torch.arange(n, device=DEV).repeat_interleave(G)[:, None]
            p = torch.softmax(w.masked_fill(~seen, -math.inf), 1)
            want = p @ vv
            got = out[b * n:(b + 1) * n, h * G:(h + 1) * G].flatten(0, 1)
            off += float((got - want).pow(2).sum())
            # scores: what each channel of a query loses is independent of the others, so it counts with the norm of the key (e), and a score's error
            # moves the output by e p_j (v_j - out), at most 2 e p_j |v_j| in the mean square
            lost = (2.0 ** -17 if n * G > 32 and cache == "fp8" else 0.0) if io == "bf16" else (2.0 ** -22 if cache == "fp8" else 2.0 ** -16)
            e = lost * float(x.abs().max()) * float(kk.norm(dim=1).max()) * 128 ** -0.5 + 2.0 ** -17
            worst += float((p.pow(2) @ vv.pow(2)).sum()) * (_p_step(cache, io, n * G > 128) ** 2 + 4 * e * e) + float(want.pow(2).sum()) * (torch.finfo(_io(io)).eps / 2) ** 2
            moved = vv.clone()
            moved[1000] = vv[1001]
            split += float((p @ moved - want).pow(2).sum())
    assert off <= worst < split / 4, (off, worst, split)


@pytest.mark.parametrize("io", ["bf16", "fp32"])
@pytest.mark.parametrize("bound", [40, 1000, 2 ** 31 - 1, 10 ** 12])
def test_max_q_may_be_any_upper_bound(io, bound):
    gen = torch.Generator().manual_seed(31)
    nq, nkv, page, news = 8, 2, 32, [40] + [1] * 60 + [17]
    lens = [n + 90 for n in news]
    table, n_pages = O.tables(lens, page, gen)
    k, v, ks, vs = O.random_pages(n_pages, nkv, page, "fp8", gen, spread=False)
    q = torch.randn(sum(news), nq, 128, generator=gen).to(_io(io))
    ref, _, mag = _reference(k, v, ks, vs, q, table, lens, news, nkv)
    qd, kd, vd, td, ksd, vsd, cu = [t.to(DEV) for t in (q, k, v, table, ks, vs, O.cu_of(news))]
    out = paged.paged_attention(qd, kd, vd, td, torch.tensor(lens, dtype=torch.int32, device=DEV), cu_q=cu, max_q=bound, k_scale=ksd, v_scale=vsd)
    _check(out, ref, mag, _p_step("fp8", io, True) + _score_bound(q, k, ks, "fp8", io, True), io)


@pytest.mark.parametrize("n", [1, 3, 64])
def test_pages_beyond_32_bits(n):
    """Page ids whose rows lie more than 2^32 elements into the pool, through append and attention (short windows and tiles)."""
    gen = torch.Generator().manual_seed(n)
    nq, nkv, page, n_pages = 16, 4, 128, 70000
    k = torch.empty(n_pages, nkv, page, 128, dtype=torch.bfloat16, device=DEV)                       # 9.2 GB each
    v = torch.empty_like(k)
    lens, news = [300, n], [n, n]
    table = torch.tensor([[69999, 3, 69000], [66000, -1, -1]], dtype=torch.int32)
    small = torch.randn(2, 4, nkv, page, 128, generator=gen).to(torch.bfloat16)
    ids = [69999, 3, 69000, 66000]
    for i, g in enumerate(ids):
        k[g], v[g] = small[0, i].to(DEV), small[1, i].to(DEV)
    qkv = torch.randn(2 * n, (nq + 2 * nkv) * 128, generator=gen)
    cos, sin = O.rope_tables(301)
    td, cu, ld = table.to(DEV), O.cu_of(news).to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    q = paged.paged_append(qkv.to(DEV), nq, nkv, k, v, td, ld, cos.to(DEV), sin.to(DEV), cu_q=cu, q_out=torch.empty(2 * n, nq, 128, dtype=torch.bfloat16, device=DEV))
    here = torch.tensor([[0, 1, 2], [3, 0, 0]], dtype=torch.int32)
    ref = O.Pages(small[0], small[1])
    O.append(ref, qkv, nq, nkv, here, lens, O.cu_of(news), cos, sin)
    got_k, got_v = (torch.stack([t[g] for g in ids]).cpu() for t in (k, v))
    for got, want in ((got_k, ref.k), (got_v, ref.v)):
        assert bool(((got.double() - want).abs() <= want.abs() * 2.0 ** -8 + want.abs().amax(-1, keepdim=True) * 2.0 ** -20).all())
    out = paged.paged_attention(q, k, v, td, ld, cu_q=cu, max_q=n)
    want, _, mag = _reference(got_k, got_v, None, None, q.cpu(), here, lens, news, nkv)
    _check(out, want, mag, _p_step("bf16", "bf16", n * 4 > 128) + 2.0 ** -17, "bf16")


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
@pytest.mark.parametrize("n", [1, 40])
def test_two_captured_steps_replayed_at_once(cache, n):
    """Append and attention of two batches, captured apart, replayed on two streams at the same time, then with other lengths in the same
    tensors: what eager calls of each give."""
    cos, sin = (t.to(DEV) for t in O.rope_tables(3000))
    steps = []
    for seed in (1, 2):
        gen = torch.Generator().manual_seed(seed)
        nq, nkv, page, B = 16, 2, 32, 5
        lens, news = [n + r for r in (2000 * seed, 0, 31, 700, 90)], [n] * B
        table, n_pages = O.tables(lens, page, gen)
        k, v, ks, vs = O.random_pages(n_pages, nkv, page, cache, gen, spread=False)
        qkv = torch.randn(B * n, (nq + 2 * nkv) * 128, generator=gen).to(torch.bfloat16)
        k, v, ks, vs, table, qkv, cu = [None if t is None else t.to(DEV) for t in (k, v, ks, vs, table, qkv, O.cu_of(news))]
        lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        q = torch.empty(B * n, nq, 128, dtype=torch.bfloat16, device=DEV)
        out = torch.empty_like(q)

        def step(k=k, v=v, ks=ks, vs=vs, table=table, qkv=qkv, cu=cu, lens=lens, q=q, out=out):
            paged.paged_append(qkv, 16, 2, k, v, table, lens, cos, sin, cu_q=cu, k_scale=ks, v_scale=vs, q_out=q)
            paged.paged_attention(q, k, v, table, lens, cu_q=cu, max_q=n, k_scale=ks, v_scale=vs, out=out)

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        steps.append((step, graph, out, lens))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for change in (False, True):
        want = []
        for step, _, out, lens in steps:
            if change:
                lens.copy_(torch.tensor([n + 5, n, n + 64, n + 1, n + 33], dtype=torch.int32))
            step()
            want.append(out.clone())
        torch.cuda.synchronize()
        for _ in range(10):
            for s, (_, graph, out, _) in zip(streams, steps):
                with torch.cuda.stream(s):
                    out.zero_()
                    graph.replay()
            torch.cuda.synchronize()
            for w, (_, _, out, _) in zip(want, steps):
                assert torch.equal(out, w)


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
@pytest.mark.parametrize("B,n,nq,L", [(200, 1, 4, 16000), (100, 1, 16, 16000), (12, 40, 8, 9000)])
def test_fp32_results_keep_their_bits_over_many_keys(cache, B, n, nq, L):
    """fp32 queries, every warp adding hundreds of steps up (the sequences share their pages): the norm of the error stays below 2^-20 of the result's.
    (Independent roundings: exponents of up to 16 give 2^-21 per probability, P and q in pairs 2^-22, sums with rounded additions 2^-24 sqrt(hundreds);
    additions that cut off would give 2^-25 times hundreds.)"""
    gen = torch.Generator().manual_seed(L)
    page = 128
    table, n_pages = O.tables([L], page, gen)
    k, v, ks, vs = O.random_pages(n_pages, 1, page, cache, gen, spread=False)
    q = torch.randn(B * n, nq, 128, generator=gen)
    qd, kd, vd, td, ksd, vsd = [None if t is None else t.to(DEV) for t in (q, k, v, table, ks, vs)]
    out = paged.paged_attention(qd, kd, vd, td.expand(B, -1), torch.full((B,), L, dtype=torch.int32, device=DEV), cu_q=O.cu_of([n] * B).to(DEV), max_q=n,
                                k_scale=ksd, v_scale=vsd)
    ids = td[0].long()
    kk = (kd[ids, 0].to(F64) * (1.0 if ksd is None else ksd[ids, 0].to(F64)[:, None, None])).reshape(-1, 128)[:L]
    vv = (vd[ids, 0].to(F64) * (1.0 if vsd is None else vsd[ids, 0].to(F64)[:, None, None])).reshape(-1, 128)[:L]
    w = qd.to(F64).flatten(0, 1) @ kk.T * 128 ** -0.5
    see = torch.arange(L, device=DEV)[None, :] <= L - n + torch.arange(n, device=DEV).repeat(B).repeat_interleave(nq)[:, None]
    ref = (torch.softmax(w.masked_fill(~see, -math.inf), 1) @ vv).view(B * n, nq, 128)
    assert float((out.to(F64) - ref).norm() / ref.norm()) <= 2.0 ** -20
