"""Paged KV cache operators: what is measured.

Two operators over a cache of pages ``[n_pages, kv heads, page, 128]`` (bf16, or e4m3 with one power-of-two scale per page
and head): ``append`` (QK norm, rotation, append) and ``attend`` (attention of ragged windows over the pages). Heads are
those of this package's models: 64 query / 4 KV heads, 32 / 4, and one rank of eight of the former (8 / 1).
"""
import math
import random

import torch

own = False

HD = 128
E_MIN, E_MAX = -60, 60                 # exponents a page scale may have
EPS = 1e-6
THETA = 1e6


# ---- cases -----------------------------------------------------------------------------------------------------------
def _case(name, op, batch, ctx, ctx_min, new, new_min, nq, nkv, page, cache, io, layout=1, tree=False, lse=False):
    """``ctx``: cached rows before the call (``ctx_min`` .. ``ctx`` over the batch); ``new``: tokens of the call per sequence."""
    return {"name": name, "op": op, "batch": batch, "ctx": ctx, "ctx_min": ctx_min, "new": new, "new_min": new_min, "nq": nq,
            "nkv": nkv, "page": page, "cache": cache, "io": io, "layout": layout, "tree": tree, "lse": lse}


def listed():
    return [
        # one token of one sequence on one rank of eight: launch latency
        _case("append_token", "append", 1, 1024, 1024, 1, 1, 8, 1, 64, "fp8", "fp32"),
        # a decode step of a batch
        _case("append_batch", "append", 64, 2047, 33, 1, 1, 64, 4, 64, "fp8", "bf16"),
        # ragged prompt chunks into small bf16 pages
        _case("append_ragged_bf16", "append", 7, 701, 0, 333, 1, 32, 4, 16, "bf16", "fp32"),
        # two long prompts
        _case("append_prompt", "append", 2, 0, 0, 4097, 4001, 64, 4, 128, "fp8", "bf16"),
        # one token of one sequence on one rank of eight
        _case("decode_one", "attend", 1, 1024, 1024, 1, 1, 8, 1, 64, "fp8", "fp32"),
        # a decode step of a ragged batch, 8-bit pages
        _case("decode_batch_fp8", "attend", 64, 8191, 129, 1, 1, 64, 4, 64, "fp8", "bf16"),
        # the same over small bf16 pages, fp32 activations as the GEMMs of this package write them
        _case("decode_batch_bf16", "attend", 24, 4095, 0, 1, 1, 32, 4, 16, "bf16", "fp32"),
        # one stream deep into a long context
        _case("decode_long", "attend", 1, 131070, 131070, 1, 1, 64, 4, 128, "fp8", "bf16"),
        # speculative verification: token trees of up to 15 nodes behind each context
        _case("verify_tree", "attend", 8, 4097, 500, 15, 1, 64, 4, 64, "fp8", "bf16", tree=True, lse=True),
        # prompt chunks of several sequences behind ragged contexts
        _case("chunk_batch", "attend", 4, 8000, 77, 511, 129, 64, 4, 64, "fp8", "bf16", lse=True),
        # a prompt from its first token, bf16 pages
        _case("prompt_bf16", "attend", 1, 0, 0, 4096, 4096, 32, 4, 64, "bf16", "bf16"),
        # the last chunk of a long prompt
        _case("prompt_long", "attend", 1, 14336, 14336, 2048, 2048, 64, 4, 128, "fp8", "bf16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    nq, nkv = rng.choice([(64, 4), (32, 4), (8, 1), (8, 2), (16, 1), (32, 1), (4, 4), (20, 4)])
    page = rng.choice([16, 32, 64, 128])
    cache, io, layout = rng.choice(["fp8", "fp8", "bf16"]), rng.choice(["bf16", "fp32"]), rng.randrange(1 << 30)
    kind = rng.choice(["append", "append_prompt", "decode", "decode", "verify", "chunk"])
    if kind == "append":
        batch = _log_int(rng, 1, 128)
        ctx = _log_int(rng, 1, 2048)
        return _drawn("append", batch, ctx, rng.randrange(ctx + 1), 1, 1, nq, nkv, page, cache, io, layout)
    if kind == "append_prompt":
        batch = _log_int(rng, 1, 12)
        new = _log_int(rng, 2, 8192 // batch)
        ctx = _log_int(rng, 1, 2048) - 1
        return _drawn("append", batch, ctx, rng.randrange(ctx + 1), new, rng.randint(1, new), nq, nkv, page, cache, io, layout)
    if kind == "decode":
        batch = _log_int(rng, 1, 96)
        ctx = _log_int(rng, 1, min(131070, 262144 // batch))
        return _drawn("attend", batch, ctx, rng.randrange(ctx + 1), 1, 1, nq, nkv, page, cache, io, layout, lse=rng.random() < 0.5)
    if kind == "verify":
        batch = _log_int(rng, 1, 16)
        ctx = _log_int(rng, 1, 65536 // batch)
        new = rng.randint(2, 33)
        return _drawn("attend", batch, ctx, rng.randrange(ctx + 1), new, rng.randint(1, new), nq, nkv, page, cache, io, layout,
                      tree=rng.random() < 0.7, lse=rng.random() < 0.5)
    batch = _log_int(rng, 1, 6)
    new = _log_int(rng, 34, 2048 // batch)
    ctx = _log_int(rng, 1, 8192) - 1
    return _drawn("attend", batch, ctx, rng.randrange(ctx + 1), new, rng.randint(1, new), nq, nkv, page, cache, io, layout,
                  lse=rng.random() < 0.5)


def _drawn(*a, **k):
    c = _case("", *a, **k)
    del c["name"]
    return c


def _lens(case):
    """(rows cached before the call, tokens of the call) of each sequence; the first one has the largest of both."""
    r = random.Random(case["layout"])
    before = [r.randint(case["ctx_min"], case["ctx"]) for _ in range(case["batch"])]
    new = [r.randint(case["new_min"], case["new"]) for _ in range(case["batch"])]
    before[0], new[0] = case["ctx"], case["new"]
    return before, new


def work(case):
    before, new = _lens(case)
    tokens, rows = sum(new), sum(before) + sum(new)
    nq, nkv, es = case["nq"], case["nkv"], 2 if case["io"] == "bf16" else 4
    ec = 1 if case["cache"] == "fp8" else 2
    if case["op"] == "append":
        moved = tokens * HD * ((nq + 2 * nkv) * es + nq * es + 2 * nkv * ec) + tokens * HD * 4
        return {"bytes": moved, "flops": tokens * HD * (nq + nkv) * 7}
    scales = sum(-(-(b + n) // case["page"]) for b, n in zip(before, new)) * nkv * 8 if case["cache"] == "fp8" else 0
    pairs = sum(b * n + n * (n + 1) // 2 for b, n in zip(before, new))
    moved = 2 * tokens * nq * HD * es + rows * nkv * HD * 2 * ec + scales + (tokens * nq * 4 if case["lse"] else 0)
    return {"bytes": moved, "flops": 4 * HD * nq * pairs}


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _pow2_exponent(amax):
    """Least e with amax / 448 <= 2^e, within [E_MIN, E_MAX] (448 = 0.875 * 2^9, amax = m * 2^x with m in [0.5, 1))."""
    m, x = torch.frexp(amax)
    e = x - 9 + (m > 0.875).to(x.dtype)
    return torch.where(amax > 0, e, torch.full_like(e, E_MIN)).clamp(E_MIN, E_MAX)


def _pages(shape, cache, gen, dev):
    """Random pages as earlier appends leave them: rows of one page share a magnitude."""
    x = torch.randn(shape, generator=gen, device=dev)
    x *= torch.exp2(torch.rand(shape[0], shape[1], 1, 1, generator=gen, device=dev) * -4.0)
    if cache == "bf16":
        return x.to(torch.bfloat16), None
    scale = torch.ldexp(torch.ones((), device=dev), _pow2_exponent(x.abs().amax(dim=(2, 3))))
    return (x / scale[:, :, None, None]).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    before, new = _lens(case)
    B, P, nq, nkv = case["batch"], case["page"], case["nq"], case["nkv"]
    T = sum(new)
    blocks = [-(-(b + n) // P) for b, n in zip(before, new)]
    n_pages = sum(blocks) + 2
    ids = torch.randperm(n_pages, generator=gen, device=dev).to(torch.int32).cpu()
    table = torch.full((B, max(blocks)), int(ids[-1]), dtype=torch.int32)
    at = 0
    for b, n in enumerate(blocks):
        table[b, :n] = ids[at:at + n]
        at += n
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    io = torch.bfloat16 if case["io"] == "bf16" else torch.float32
    s = {"case": case, "T": T, "max_q": max(new), "table": table.to(dev),
         "kv_len": torch.tensor([b + n for b, n in zip(before, new)], dtype=torch.int32, device=dev),
         "cu_q": torch.tensor(cu, dtype=torch.int32, device=dev)}
    s["k"], s["k_scale"] = _pages((n_pages, nkv, P, HD), case["cache"], gen, dev)
    s["v"], s["v_scale"] = _pages((n_pages, nkv, P, HD), case["cache"], gen, dev)
    if case["op"] == "append":
        x = torch.randn(T, (nq + 2 * nkv) * HD, generator=gen, device=dev)
        x *= torch.exp(0.5 * torch.randn(1, x.shape[1], generator=gen, device=dev))
        s["qkv"] = x.to(io)
        s["q_gamma"] = 1 + 0.2 * torch.randn(HD, generator=gen, device=dev)
        s["k_gamma"] = 1 + 0.2 * torch.randn(HD, generator=gen, device=dev)
        n_pos = max(b + n for b, n in zip(before, new))
        ang = torch.arange(n_pos, dtype=torch.float64, device=dev)[:, None] * THETA ** (
            -torch.arange(HD // 2, dtype=torch.float64, device=dev) / (HD // 2))
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
        return s
    s["q"] = torch.randn(T, nq, HD, generator=gen, device=dev).to(io)
    s["mask"] = None
    if case["tree"]:
        # a node sees itself and its ancestors; its parent is any earlier node of its sequence
        N = max(new)
        mask = torch.zeros(T, N, dtype=torch.bool)
        r = random.Random(seed)
        for b, n in enumerate(new):
            for i in range(n):
                if i:
                    mask[cu[b] + i] = mask[cu[b] + r.randrange(i)]
                mask[cu[b] + i, i] = True
        s["mask"] = mask.to(dev)
    return s


# ---- the operators ---------------------------------------------------------------------------------------------------
def run(s):
    if own:
        from inferencehackathon_b200.ops import paged
        c = s["case"]
        cu = None if c["new"] == 1 else s["cu_q"]
        if c["op"] == "append":
            q = paged.paged_append(s["qkv"], c["nq"], c["nkv"], s["k"], s["v"], s["table"], s["kv_len"], s["cos"], s["sin"],
                                   cu_q=cu, q_gamma=s["q_gamma"], k_gamma=s["k_gamma"], eps=EPS, k_scale=s["k_scale"],
                                   v_scale=s["v_scale"], q_out=torch.empty(s["T"], c["nq"], HD, dtype=s["qkv"].dtype, device="cuda"))
            return _cache_out(q, s["k"], s["v"], s["k_scale"], s["v_scale"])
        lse = torch.empty(s["T"], c["nq"], dtype=torch.float32, device="cuda") if c["lse"] else None
        out = paged.paged_attention(s["q"], s["k"], s["v"], s["table"], s["kv_len"], cu_q=cu, max_q=s["max_q"], mask=s["mask"],
                                    k_scale=s["k_scale"], v_scale=s["v_scale"], lse=lse)
        return {"out": out, "lse": lse} if c["lse"] else {"out": out}
    return _plain_append(s) if s["case"]["op"] == "append" else _plain_attention(s)


def _cache_out(q, k, v, ks, vs):
    # 8-bit rows are returned as e4m3 numbers, their scales beside them
    out = {"q": q, "k": k, "v": v}
    if ks is not None:
        out["k_scale"], out["v_scale"] = ks, vs
    return out


def _tokens(s):
    """(sequence, position) of every token of the call."""
    t = torch.arange(s["T"], dtype=torch.int32, device="cuda")
    b = torch.searchsorted(s["cu_q"][1:], t, right=True)
    return b, s["kv_len"][b].long() - (s["cu_q"][b + 1] - t)


def _norm_rope(x, gamma, cos, sin):
    x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * gamma
    a, b = x[..., :HD // 2], x[..., HD // 2:]
    c, n = cos[:, None, :], sin[:, None, :]
    return torch.cat([a * c - b * n, b * c + a * n], dim=-1)


def _plain_write(pages, scale, x, page, row):
    """Rows ``x [T, nkv, 128]`` into row ``row[t]`` of page ``page[t]``; a page starts anew where its row 0 is written."""
    if scale is None:
        pages = pages.clone()
        pages[page, :, row] = x.to(pages.dtype)
        return pages, None
    n_pages, P = pages.shape[0], pages.shape[2]
    amax = torch.zeros_like(scale).index_reduce_(0, page, x.abs().amax(dim=-1), "amax")
    first = torch.full((n_pages,), P, dtype=torch.long, device=x.device).index_reduce_(0, page, row, "amin")
    touched, fresh = first < P, first == 0
    want = torch.ldexp(torch.ones_like(scale), _pow2_exponent(amax))
    old = torch.where(fresh[:, None], torch.zeros_like(scale), scale)
    now = torch.where(touched[:, None], torch.maximum(old, want), scale)
    again = (now / scale != 1) & (touched & ~fresh)[:, None]
    live = torch.arange(P, device=x.device)[None, :] < first[:, None]
    moved = (pages.float() * (scale / now)[:, :, None, None]).to(pages.dtype).view(torch.uint8)
    sel = again[:, :, None] & live[:, None, :]
    out = torch.where(sel[..., None], moved, pages.view(torch.uint8))
    rows = (x / now[page][..., None]).clamp(-448, 448).to(pages.dtype).view(torch.uint8)
    out[page, :, row] = rows
    return out.view(pages.dtype), now


def _plain_append(s):
    c = s["case"]
    nq, nkv, P = c["nq"], c["nkv"], c["page"]
    b, pos = _tokens(s)
    x = s["qkv"].float().view(s["T"], nq + 2 * nkv, HD)
    cos, sin = s["cos"][pos], s["sin"][pos]
    q = _norm_rope(x[:, :nq], s["q_gamma"], cos, sin)
    k = _norm_rope(x[:, nq:nq + nkv], s["k_gamma"], cos, sin)
    page, row = s["table"][b, pos // P].long(), pos % P
    kp, ks = _plain_write(s["k"], s["k_scale"], k, page, row)
    vp, vs = _plain_write(s["v"], s["v_scale"], x[:, nq + nkv:], page, row)
    return _cache_out(q.to(s["qkv"].dtype), kp, vp, ks, vs)


def _gather(pages, scale, table):
    """The rows of every sequence in order: [B, nkv, blocks * P, 128] fp32."""
    x = pages[table.long()].float()
    if scale is not None:
        x = x * scale[table.long()][..., None, None]
    B, M, nkv, P, _ = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(B, nkv, M * P, HD)


def _plain_attention(s):
    c = s["case"]
    nq, nkv, B, T, N = c["nq"], c["nkv"], c["batch"], s["T"], s["max_q"]
    G = nq // nkv
    dev = s["q"].device
    n = (s["cu_q"][1:] - s["cu_q"][:-1]).long()
    i = torch.arange(N, device=dev)
    at = s["cu_q"][:-1].long()[:, None] + i                                    # token of (sequence, i)
    here = i[None, :] < n[:, None]
    tok = at.clamp(max=T - 1)
    q = s["q"][tok].float().view(B, N, nkv, G, HD).permute(0, 2, 3, 1, 4).reshape(B, nkv, G * N, HD)
    k, v = _gather(s["k"], s["k_scale"], s["table"]), _gather(s["v"], s["v_scale"], s["table"])
    L = k.shape[2]
    j = torch.arange(L, device=dev)
    base = s["kv_len"].long() - n
    seen = j[None, None, :] <= (base[:, None] + i)[:, :, None]                 # [B, N, L]
    if s["mask"] is not None:
        w = (j[None, :] - base[:, None]).clamp(0, N - 1)[:, None, :].expand(B, N, L)
        node = torch.gather(s["mask"][tok], 2, w) & (j[None, :] < s["kv_len"][:, None])[:, None, :]
        seen = torch.where((j[None, :] < base[:, None])[:, None, :], torch.ones_like(seen), node)
    p = torch.matmul(q, k.transpose(2, 3)).view(B, nkv, G, N, L).mul_(HD ** -0.5)
    p.masked_fill_(~seen[:, None, None], float("-inf"))
    m = p.amax(dim=-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    p.sub_(m).exp_()
    z = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p.view(B, nkv, G * N, L), v).view(B, nkv, G, N, HD) / torch.where(z > 0, z, torch.ones_like(z))
    out = torch.zeros(T, nq, HD, dtype=torch.float32, device=dev)
    out[at[here]] = o.permute(0, 3, 1, 2, 4).reshape(B, N, nq, HD)[here]
    if not c["lse"]:
        return {"out": out.to(s["q"].dtype)}
    lse = torch.full((T, nq), float("-inf"), device=dev)
    lse[at[here]] = (m + torch.log(z))[..., 0].permute(0, 3, 1, 2).reshape(B, N, nq)[here]
    return {"out": out.to(s["q"].dtype), "lse": lse}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------
def _e4m3(x):
    """float64 values rounded to e4m3 (half to even, largest 448, least step 2^-9)."""
    _, e = torch.frexp(x.abs().clamp(min=2.0 ** -40))
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def exact(case, seed):
    s = prepare(case, seed)
    before, new = _lens(case)
    nq, nkv, P, G = case["nq"], case["nkv"], case["page"], case["nq"] // case["nkv"]
    table = s["table"].cpu()
    f64 = torch.float64
    if case["op"] == "append":
        x = s["qkv"].to(f64).view(-1, nq + 2 * nkv, HD)
        pos = torch.cat([torch.arange(b, b + n) for b, n in zip(before, new)]).cuda()
        ang = torch.stack([s["cos"].to(f64)[pos], s["sin"].to(f64)[pos]])[:, :, None, :]

        def turned(y, g):
            y = y / torch.sqrt((y ** 2).sum(-1, keepdim=True) / HD + EPS) * g.to(f64)
            lo, hi = y.split(HD // 2, dim=-1)
            return torch.cat([lo * ang[0] - hi * ang[1], hi * ang[0] + lo * ang[1]], -1)

        def filled(pages, scale, rows):
            out = pages.to(f64)
            sc = None if scale is None else scale.to(f64)
            t = 0
            for b, (c0, n) in enumerate(zip(before, new)):
                p = c0
                while p < c0 + n:
                    r0 = p % P
                    r1 = min(P, r0 + c0 + n - p)
                    g, y = int(table[b, p // P]), rows[t:t + r1 - r0].transpose(0, 1)
                    if sc is not None:
                        top = y.abs().amax(dim=(1, 2))
                        e = torch.ceil(torch.log2(top / 448)).clamp(E_MIN, E_MAX)
                        e = torch.where(top > 448 * torch.exp2(e), e + 1, e)
                        e = torch.where(top <= 448 * torch.exp2(e - 1), e - 1, e)
                        now = torch.exp2(e) if r0 == 0 else torch.maximum(sc[g], torch.exp2(e))
                        if r0:
                            out[g, :, :r0] = _e4m3(out[g, :, :r0] * (sc[g] / now)[:, None, None])
                        y = _e4m3(y / now[:, None, None])
                        sc[g] = now
                    out[g, :, r0:r1] = y
                    t += r1 - r0
                    p += r1 - r0
            return out, sc

        k, ks = filled(s["k"], s["k_scale"], turned(x[:, nq:nq + nkv], s["k_gamma"]))
        v, vs = filled(s["v"], s["v_scale"], x[:, nq + nkv:])
        return _cache_out(turned(x[:, :nq], s["q_gamma"]), k, v, ks, vs)
    out = torch.empty(s["T"], nq, HD, dtype=f64, device="cuda")
    lse = torch.empty(s["T"], nq, dtype=f64, device="cuda")
    t = 0
    for b, (c0, n) in enumerate(zip(before, new)):
        L = c0 + n
        ids = s["table"][b, :-(-L // P)].long()
        bias = torch.zeros(n, L, dtype=f64, device="cuda")
        own_rows = (torch.ones(n, n, dtype=torch.bool, device="cuda").tril() if s["mask"] is None else s["mask"][t:t + n, :n])
        bias[:, c0:] = torch.where(own_rows, 0.0, float("-inf")).to(f64)
        for h in range(nkv):
            kk, vv = s["k"][ids, h].to(f64), s["v"][ids, h].to(f64)
            if s["k_scale"] is not None:
                kk, vv = kk * s["k_scale"][ids, h].to(f64)[:, None, None], vv * s["v_scale"][ids, h].to(f64)[:, None, None]
            kk, vv = kk.reshape(-1, HD)[:L], vv.reshape(-1, HD)[:L]
            for g in range(h * G, (h + 1) * G):
                w = s["q"][t:t + n, g].to(f64) @ kk.T / math.sqrt(HD) + bias
                lse[t:t + n, g] = torch.logsumexp(w, dim=1)
                out[t:t + n, g] = torch.exp(w - lse[t:t + n, g, None]) @ vv
        t += n
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}
