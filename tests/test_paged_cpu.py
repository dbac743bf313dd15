"""Paged cache operators without a GPU: refusals, argument blocks, and properties of the page scale on the 64-bit oracle."""
import ctypes as C

import pytest
import torch

import paged_oracle as O
from inferencehackathon_b200.ops import lib as K
from inferencehackathon_b200.ops import paged


def _append_args(**over):
    nq, nkv, P, B = 4, 2, 16, 3
    cos, sin = O.rope_tables(64)
    a = dict(qkv=torch.zeros(B, (nq + 2 * nkv) * 128), nq=nq, nkv=nkv, k_pages=torch.zeros(8, nkv, P, 128, dtype=torch.bfloat16),
             v_pages=torch.zeros(8, nkv, P, 128, dtype=torch.bfloat16), block_table=torch.zeros(B, 2, dtype=torch.int32),
             kv_len=torch.ones(B, dtype=torch.int32), cos_t=cos, sin_t=sin)
    a.update(over)
    return a


def _attn_args(**over):
    B = 3
    a = dict(q=torch.zeros(B, 4, 128), k_pages=torch.zeros(8, 2, 16, 128, dtype=torch.bfloat16),
             v_pages=torch.zeros(8, 2, 16, 128, dtype=torch.bfloat16), block_table=torch.zeros(B, 2, dtype=torch.int32),
             kv_len=torch.ones(B, dtype=torch.int32))
    a.update(over)
    return a


E4 = torch.float8_e4m3fn
COMMON = [
    (dict(k_pages=torch.zeros(8, 2, 24, 128, dtype=torch.bfloat16), v_pages=torch.zeros(8, 2, 24, 128, dtype=torch.bfloat16)), "page size"),
    (dict(k_pages=torch.zeros(8, 2, 16, 64, dtype=torch.bfloat16), v_pages=torch.zeros(8, 2, 16, 64, dtype=torch.bfloat16)), "pages must be"),
    (dict(v_pages=torch.zeros(9, 2, 16, 128, dtype=torch.bfloat16)), "alike"),
    (dict(k_pages=torch.zeros(8, 2, 16, 128), v_pages=torch.zeros(8, 2, 16, 128)), "bfloat16 or float8"),
    (dict(k_pages=torch.zeros(8, 2, 16, 128, dtype=E4), v_pages=torch.zeros(8, 2, 16, 128, dtype=E4)), "need k_scale"),
    (dict(k_pages=torch.zeros(8, 2, 16, 128, dtype=E4), v_pages=torch.zeros(8, 2, 16, 128, dtype=E4), k_scale=torch.ones(8, 2),
          v_scale=torch.ones(8, 3)), "page scales"),
    (dict(k_scale=torch.ones(8, 2), v_scale=torch.ones(8, 2)), "no scales"),
    (dict(k_pages=torch.zeros(8, 2, 16, 256, dtype=torch.bfloat16)[..., ::2], v_pages=torch.zeros(8, 2, 16, 128, dtype=torch.bfloat16)),
     "contiguous"),
    (dict(kv_len=torch.ones(3, dtype=torch.int64)), "kv_len"),
    (dict(kv_len=torch.ones(4, dtype=torch.int32), block_table=torch.zeros(4, 2, dtype=torch.int32)), "one token per sequence"),
    (dict(block_table=torch.zeros(3, 2, dtype=torch.int64)), "block_table"),
    (dict(block_table=torch.zeros(2, 2, dtype=torch.int32)), "block_table"),
    (dict(cu_q=torch.zeros(3, dtype=torch.int32)), "cu_q"),
    (dict(err=torch.zeros(1)), "err"),
]


@pytest.mark.parametrize("over,what", COMMON + [
    (dict(qkv=torch.zeros(3, 7 * 128)), "qkv must be"),
    (dict(qkv=torch.zeros(3, 8 * 128, dtype=torch.float16)), "float32 or bfloat16"),
    (dict(qkv=torch.zeros(1, 8 * 128).expand(3, -1)), "overlap"),
    (dict(nkv=1, nq=6), "KV heads"),
    (dict(cos_t=torch.zeros(64, 64, dtype=torch.float64)), "cos_t"),
    (dict(q_gamma=torch.ones(128)), "come together"),
    (dict(q_gamma=torch.ones(64), k_gamma=torch.ones(64)), "gammas"),
    (dict(positions=torch.zeros(3, dtype=torch.int64)), "positions"),
    (dict(q_out=torch.zeros(3, 5, 128)), "q_out"),
    (dict(q_out=torch.zeros(3, 4, 256)[..., ::2]), "q_out"),
    (dict(), "CUDA tensors"),
])
def test_append_refuses(over, what):
    with pytest.raises(ValueError, match=what):
        paged.paged_append(**_append_args(**over))


@pytest.mark.parametrize("over,what", COMMON + [
    (dict(q=torch.zeros(3, 5, 128)), "evenly"),
    (dict(q=torch.zeros(3, 4, 64)), "q must be"),
    (dict(q=torch.zeros(3, 4, 128, dtype=torch.float16)), "float32 or bfloat16"),
    (dict(q=torch.zeros(3, 4 * 128 + 4)[:, :512].unflatten(1, (4, 128))), "multiples of 8"),
    (dict(max_q=2), "max_q"),
    (dict(max_q=0), "max_q"),
    (dict(scale=0.0), "scale"),
    (dict(scale=float("nan")), "scale"),
    (dict(out=torch.zeros(3, 4, 128, dtype=torch.float16)), "out must be"),
    (dict(out=torch.zeros(1, 4, 128).expand(3, -1, -1)), "overlap"),
    (dict(lse=torch.zeros(3, 5)), "lse"),
    (dict(mask=torch.zeros(3, 1)), "mask"),
    (dict(mask=torch.zeros(2, 1, dtype=torch.bool)), "mask"),
    (dict(cu_q=torch.zeros(4, dtype=torch.int32), max_q=3, mask=torch.zeros(3, 2, dtype=torch.bool)), "mask"),
    (dict(), "CUDA tensors"),
])
def test_attention_refuses(over, what):
    with pytest.raises(ValueError, match=what):
        paged.paged_attention(**_attn_args(**over))


def test_c_entries_refuse_bad_blocks():
    """The C entry points check again, before anything is launched (no GPU needed: nothing is)."""
    lib = K.load()
    assert lib.ihb_paged_append(C.byref(K.IhbPagedAppend()), None) != 0
    a = K.IhbPagedAttn()
    assert lib.ihb_paged_attention(C.byref(a), None) != 0
    assert lib.ihb_paged_attention_scratch(C.byref(a)) == 0
    a.c = K.IhbPaged(k=16, v=16, n_pages=4, nkv=2, page=24, B=1, T=1, max_blocks=1, block_table=16, kv_len=16)
    a.q, a.out, a.nq, a.max_q, a.scratch = 16, 16, 4, 1, 16
    assert lib.ihb_paged_attention(C.byref(a), None) != 0                    # page size
    a.c.page, a.nq = 16, 5
    assert lib.ihb_paged_attention(C.byref(a), None) != 0                    # heads
    a.nq, a.c.T = 4, 2
    assert lib.ihb_paged_attention(C.byref(a), None) != 0                    # two tokens, one sequence, no cu_q


def test_a_page_filled_token_by_token_equals_one_filled_at_once():
    """Power-of-two scales: both ways give the same scale, and the same bytes but for values that become subnormal (then at
    most one step of 2^-9 apart)."""
    gen = torch.Generator().manual_seed(3)
    P, nq, nkv = 16, 2, 2
    qkv = torch.randn(P, (nq + 2 * nkv) * 128, generator=gen) * torch.exp2(torch.linspace(-6, 6, P))[:, None]
    cos, sin = O.rope_tables(P)
    table = torch.zeros(1, 1, dtype=torch.int32)
    blank = lambda: O.Pages(*(torch.zeros(1, nkv, P, 128) for _ in range(2)), *(torch.ones(1, nkv) for _ in range(2)))  # noqa: E731
    once, steps = blank(), blank()
    O.append(once, qkv, nq, nkv, table, [P], [0, P], cos, sin)
    for t in range(P):
        O.append(steps, qkv[t:t + 1], nq, nkv, table, [t + 1], [0, 1], cos, sin)
    assert torch.equal(once.ks, steps.ks) and torch.equal(once.vs, steps.vs)
    for a, b in ((once.k, steps.k), (once.v, steps.v)):
        normal = a.abs() >= 2.0 ** -6
        assert torch.equal(a[normal], b[normal])
        assert float((a - b).abs().max()) <= 2.0 ** -9


def test_oracle_rounding_is_torch_rounding():
    x = torch.cat([torch.linspace(-448, 448, 40001), torch.linspace(-0.05, 0.05, 40001)])
    assert torch.equal(O.e4m3_round(x.double()).float(), x.to(torch.float8_e4m3fn).float())


# ---- the cache's bookkeeping ------------------------------------------------------------------------------------------------
def _cache(n_pages=10, page=16, kv="fp8"):
    from inferencehackathon_b200.runtime.paged_kv import PagedKVCache
    return PagedKVCache(2, n_pages, 2, page, kv, device="cpu")


def test_pages_are_taken_and_given_back():
    c = _cache()
    c.add("a")
    c.add("b")
    b = c.extend({"a": 17, "b": 16})
    assert c.free_pages == 7 and b.max_q == 17 and b.n_tokens == 33 and b.cu_q.tolist() == [0, 17, 33]
    assert b.kv_len.tolist() == [17, 16] and b.block_table.shape == (2, 2) and b.block_table[1, 1] == -1
    b = c.extend({"b": 1, "a": 1})
    assert b.cu_q is None and b.kv_len.tolist() == [17, 18] and c.free_pages == 6
    c.truncate("a", 16)
    assert c.free_pages == 7 and c.length("a") == 16
    c.free("a")
    c.truncate("b", 0)
    assert c.free_pages == 10
    with pytest.raises(ValueError, match="cannot keep"):
        c.truncate("b", 1)
    with pytest.raises(ValueError, match="exists"):
        c.add("b")
    with pytest.raises(ValueError, match="no sequences"):
        c.extend({})
    with pytest.raises(ValueError, match="must be a token"):
        c.extend({"b": 0})


def test_a_full_pool_refuses_before_anything_changes():
    c = _cache(n_pages=3)
    c.add(1)
    c.add(2)
    c.extend({1: 20})
    with pytest.raises(RuntimeError, match="2 pages needed, 1 free"):
        c.extend({1: 13, 2: 1})
    assert c.free_pages == 1 and c.length(1) == 20 and c.length(2) == 0
    c.extend({1: 12, 2: 1})
    assert c.free_pages == 0


def test_a_forked_page_is_copied_when_it_is_written():
    c = _cache(n_pages=6)
    c.add("a")
    c.extend({"a": 20})
    c.k.view(torch.uint8).random_(0, 100)
    c.k_scale.uniform_(0.5, 2.0)
    c.fork("a", "b")
    c.fork("a", "d")
    shared = c.pages("a")
    assert c.pages("b") == shared and c.free_pages == 4
    c.extend({"b": 1})                                        # b writes into the partly filled page: its own copy
    assert c.pages("b")[0] == shared[0] and c.pages("b")[1] != shared[1] and c.free_pages == 3
    new = c.pages("b")[1]
    assert torch.equal(c.k[:, new].view(torch.uint8), c.k[:, shared[1]].view(torch.uint8)) and torch.equal(c.k_scale[:, new], c.k_scale[:, shared[1]])
    c.extend({"a": 1, "d": 1})                                # of the two that are left the first copies, the last keeps the page
    assert c.free_pages == 2 and c.pages("d")[1] == shared[1] and c.pages("a")[1] not in (shared[1], new)
    for q in "abd":
        c.free(q)
    assert c.free_pages == 6
    c.add("e")
    c.extend({"e": 32})
    c.fork("e", "f")
    c.truncate("f", 20)                                       # now inside a shared page
    c.extend({"f": 1})
    assert c.pages("f")[1] != c.pages("e")[1]


@pytest.mark.parametrize("kw", [dict(page=48), dict(kv="int8")])
def test_cache_refuses(kw):
    with pytest.raises(ValueError):
        _cache(**kw)


def test_packed_argument_blocks_are_the_structures():
    """Every field of the byte blocks that the entry points pack lies where the C structures have it."""
    def flat(st):
        for name, kind in st._fields_:
            v = getattr(st, name)
            yield from (flat(v) if isinstance(v, C.Structure) else [v])

    for block, kind in ((paged._APPEND, K.IhbPagedAppend), (paged._ATTN, K.IhbPagedAttn)):
        n = len([c for c in block.format if c.isalpha()])
        assert block.size == C.sizeof(kind)
        values = [i + 1 for i in range(n)]
        assert [int(v) for v in flat(kind.from_buffer_copy(block.pack(*values)))] == values
    assert list(flat(K.IhbPagedAttn.from_buffer_copy(paged._ATTN.pack(*values))))[-1] == n and paged._PTR.size == C.sizeof(C.c_void_p)


def test_more_query_heads_per_kv_head_than_the_work_split_counts_are_refused():
    a = _attn_args(q=torch.zeros(3, 2 * 257, 128))
    with pytest.raises(ValueError, match="256 query heads"):
        paged.paged_attention(a.pop("q"), **a)
    lib = K.load()
    c = K.IhbPaged(k=16, v=16, n_pages=4, nkv=1, page=16, B=1, T=1, max_blocks=1, block_table=16, kv_len=16)
    b = K.IhbPagedAttn(c=c, q=16, nq=257, out=16, max_q=1, scratch=16, q_stride_t=8, q_stride_h=8)
    assert lib.ihb_paged_attention(C.byref(b), None) != 0


def test_ragged_calls_name_their_longest_window():
    """With cu_q a forgotten max_q would leave rows of longer windows unwritten."""
    a = _attn_args(cu_q=torch.tensor([0, 1, 2, 3], dtype=torch.int32))
    with pytest.raises(ValueError, match="cu_q needs max_q"):
        paged.paged_attention(**a)
    for bound in (1, 3):
        with pytest.raises(ValueError, match="CUDA tensors"):            # all that it lacks
            paged.paged_attention(**a, max_q=bound)


def test_c_entry_refuses_masks_without_columns():
    lib = K.load()
    c = K.IhbPaged(k=16, v=16, n_pages=4, nkv=1, page=16, B=1, T=1, max_blocks=1, block_table=16, kv_len=16)
    for stride, cols in ((-1, 4), (4, 0), (0, -3)):
        b = K.IhbPagedAttn(c=c, q=16, nq=1, out=16, max_q=1, scratch=16, q_stride_t=8, q_stride_h=8, mask=16, mask_stride=stride, mask_cols=cols)
        assert lib.ihb_paged_attention(C.byref(b), None) != 0


def test_mask_views_pass_the_checks():
    """Shared, overlapping and sliced rows are masks like any other (what is left to refuse is the missing GPU)."""
    flat, wide = torch.ones(8, dtype=torch.bool), torch.ones(3, 9, dtype=torch.uint8)
    for mask in (flat.unfold(0, 3, 1)[:3], flat[:4].expand(3, -1), wide[:, 2:6], torch.ones(3, 1, dtype=torch.bool)):
        with pytest.raises(ValueError, match="CUDA tensors"):
            paged.paged_attention(**_attn_args(mask=mask))
    with pytest.raises(ValueError, match="contiguous rows"):
        paged.paged_attention(**_attn_args(mask=wide[:, ::2]))
