"""Plain 64-bit implementations of the paged cache operators and helpers that build ragged batches (used by the tests)."""
import math

import torch

HD = 128
F64 = torch.float64


def e4m3_round(x):
    """float64 -> the nearest e4m3 number (half to even, largest 448, least step 2^-9), still float64; NaN stays."""
    nan = torch.isnan(x)
    y = torch.where(nan, torch.zeros_like(x), x).clamp(-448.0, 448.0)
    _, e = torch.frexp(y.abs().clamp(min=2.0 ** -40))
    step = torch.ldexp(torch.ones_like(y), (e - 1).clamp(min=-6) - 3)
    y = torch.round(y / step) * step
    return torch.where(nan, x, y)


def page_exponent(amax):
    """Least e in [-60, 60] with amax <= 448 * 2^e."""
    e = -60
    while e < 60 and amax > 448.0 * 2.0 ** e:
        e += 1
    return e


def norm_rope(x, gamma, eps, cos, sin):
    """x [heads, 128] float64, cos / sin [64]."""
    if gamma is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * gamma.to(F64)
    a, b = x[:, :64], x[:, 64:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=1)


class Pages:
    """Pages in float64 values (the bytes' values for e4m3) with scales."""

    def __init__(self, k, v, ks=None, vs=None):
        self.k, self.v = k.to(F64).cpu(), v.to(F64).cpu()
        self.ks = None if ks is None else ks.to(F64).cpu()
        self.vs = None if vs is None else vs.to(F64).cpu()

    def rows(self, which, ids, h, n):
        x, s = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        y = x[ids, h]
        if s is not None:
            y = y * s[ids, h][:, None, None]
        return y.reshape(-1, HD)[:n]


def append(pages, qkv, nq, nkv, table, kv_len, cu, cos, sin, q_gamma=None, k_gamma=None, eps=1e-6, positions=None):
    """Returns q' [T, nq, 128] float64 (NaN where the call leaves it alone) and updates ``pages``. bf16 pages: unrounded values."""
    P = pages.k.shape[2]
    x = qkv.to(F64).cpu().view(qkv.shape[0], nq + 2 * nkv, HD)
    table, cos, sin = table.cpu(), cos.to(F64).cpu(), sin.to(F64).cpu()
    q_gamma, k_gamma = (None if g is None else g.cpu() for g in (q_gamma, k_gamma))
    q = torch.full((qkv.shape[0], nq, HD), float("nan"), dtype=F64)
    for b, L in enumerate(int(v) for v in kv_len):
        t0, t1 = int(cu[b]), int(cu[b + 1])
        if L <= 0 or t1 == t0:
            continue
        p = L - (t1 - t0)
        t = t0
        while t < t1:
            r0 = p % P
            n = min(P - r0, t1 - t)
            g = int(table[b, p // P])
            ks, vs = [], []
            for i in range(n):
                pos = int(positions[t + i]) if positions is not None else p + i
                q[t + i] = norm_rope(x[t + i, :nq], q_gamma, eps, cos[pos], sin[pos])
                ks.append(norm_rope(x[t + i, nq:nq + nkv], k_gamma, eps, cos[pos], sin[pos]))
                vs.append(x[t + i, nq + nkv:])
            for dst, sc, new in ((pages.k, pages.ks, torch.stack(ks, 1)), (pages.v, pages.vs, torch.stack(vs, 1))):
                if sc is None:
                    dst[g, :, r0:r0 + n] = new
                    continue
                for h in range(nkv):
                    y = new[h]
                    fin = y[torch.isfinite(y)].abs()
                    want = 2.0 ** page_exponent(float(fin.max()) if fin.numel() else 0.0)
                    old = float(sc[g, h]) if r0 else 0.0
                    now = max(old, want)
                    if r0 and now > old:
                        dst[g, h, :r0] = e4m3_round(dst[g, h, :r0] * (old / now))
                    dst[g, h, r0:r0 + n] = e4m3_round(y / now)
                    sc[g, h] = now
            p += n
            t += n
    return q


def attention(pages, q, table, kv_len, cu, nkv, mask=None, scale=HD ** -0.5):
    """(out [T, nq, 128], lse [T, nq]) float64; NaN where the call leaves the rows alone."""
    T, nq, _ = q.shape
    P = pages.k.shape[2]
    x, table = q.to(F64).cpu(), table.cpu()
    mask = None if mask is None else mask.cpu().bool()
    out = torch.full((T, nq, HD), float("nan"), dtype=F64)
    lse = torch.full((T, nq), float("nan"), dtype=F64)
    for b, L in enumerate(int(v) for v in kv_len):
        t0, t1 = int(cu[b]), int(cu[b + 1])
        L = max(L, 0)
        base = L - (t1 - t0)
        ids = table[b, :-(-L // P)].long()
        for h in range(nq):
            if t1 == t0:
                break
            k = pages.rows("k", ids, h // (nq // nkv), L)
            v = pages.rows("v", ids, h // (nq // nkv), L)
            for t in range(t0, t1):
                i = t - t0
                if mask is None:
                    see = torch.arange(L) <= base + i
                else:
                    see = torch.tensor([j < base or bool(mask[t, j - base]) for j in range(L)], dtype=torch.bool)
                if not bool(see.any()):
                    out[t, h], lse[t, h] = 0.0, -math.inf
                    continue
                w = (k[see] @ x[t, h]) * scale
                lse[t, h] = torch.logsumexp(w, 0)
                out[t, h] = torch.exp(w - lse[t, h]) @ v[see]
    return out, lse


def tables(lens, P, gen, spare=3, pad=-1):
    """Shuffled page ids for rows ``lens``; unused table entries hold ``pad``."""
    blocks = [max(0, -(-n // P)) for n in lens]
    n_pages = sum(blocks) + spare
    ids = torch.randperm(n_pages, generator=gen).to(torch.int32)
    table = torch.full((len(lens), max(max(blocks), 1)), pad, dtype=torch.int32)
    at = 0
    for b, n in enumerate(blocks):
        table[b, :n] = ids[at:at + n]
        at += n
    return table, n_pages


def random_pages(n_pages, nkv, P, cache, gen, spread=True):
    """(k, v, k_scale, v_scale) on the CPU, as appends leave them; scales differ between pages."""
    out = []
    for _ in range(2):
        x = torch.randn(n_pages, nkv, P, HD, generator=gen)
        if spread:
            x = x * torch.exp2(torch.randint(-4, 3, (n_pages, nkv, 1, 1), generator=gen).float())
        if cache == "bf16":
            out.append((x.to(torch.bfloat16), None))
            continue
        s = torch.tensor([[2.0 ** page_exponent(float(x[p, h].abs().max())) for h in range(nkv)] for p in range(n_pages)])
        out.append(((x / s[:, :, None, None]).to(torch.float8_e4m3fn), s))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def rope_tables(n, theta=1e6):
    ang = torch.arange(n, dtype=F64)[:, None] * theta ** (-torch.arange(64, dtype=F64) / 64)
    return ang.cos().float(), ang.sin().float()


def tree_mask(news, width, seed=0):
    """Ancestor masks of random trees, [T, width]."""
    import random
    r = random.Random(seed)
    m = torch.zeros(sum(news), width, dtype=torch.bool)
    t0 = 0
    for n in news:
        for i in range(n):
            if i:
                m[t0 + i] = m[t0 + r.randrange(i)]
            m[t0 + i, i] = True
        t0 += n
    return m


def cu_of(news):
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32)
