// Attention of a ragged batch over a paged KV cache: single decode tokens and short verify windows, head_dim 128, bf16 pages or
// e4m3 pages with one scale per (page, head). The contiguous, one-sequence siblings are attn.cu::flash_decode_kernel and
// window.cu::window_attn_mma_kernel.
//
// The rows of a (sequence, KV head) are its (token, query head) pairs, RT = 8 or 16 of them per tile. Scores are computed
// transposed, S^T = K Q^T with m16n8k16 (16 keys x 8 rows), and so is the output, O^T = V^T P^T: the large operand is the A operand
// of both products and a thread's fragments of it are contiguous bytes of the cache (the channel order inside a product is free,
// so a thread takes 16 neighbouring bytes), so K and V go from global memory to registers in 16-byte loads and never touch
// shared memory. With queries as the A operand (the usual way round) 8 query heads would waste half of every product.
//
// e4m3 pages: bytes become fp16 exactly; q is scaled per row by a power of two into fp16 (head and remainder for fp32
// queries: 22 bits); the K scale is a factor of the score, the V scale s_v goes into the exponent of the probability: with
// m the running maximum of score + log2 s_v, O = sum 2^(s + log2 s_v - m) v_bytes and l = sum 2^(s - m). The probability that
// meets the bytes is then at most 2^14 whatever the scales are, which is what fp16 holds.
//
// Work split: the 64-key units of all (sequence, head, tile) items are laid end to end and cut into equal ranges, one per CTA, so
// ragged batches and single long sequences load every SM the same. Lengths are read on the device. An item cut by a range end
// leaves one record (O, m, l) per piece, folded by a second kernel in a fixed order: results do not depend on timing.
#include "paged.cuh"

namespace ihb {

constexpr int PD_WARPS = 4;
constexpr int PD_UNIT = 64;                  // keys per unit: 16 per warp
constexpr int PD_REC = PG_HD + 4;            // record of a row: 128 channels, m, l, 2 pad
constexpr float PD_OFF = 6.f;                // log2 of what a probability is scaled by (fp16 keeps more small ones)
constexpr float PD_LAZY = 8.f;               // the running maximum may be passed by 2^8 before the accumulators are rescaled

template <bool F16>
__device__ __forceinline__ void pd_mma(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  if constexpr (F16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned pd_movt(unsigned x) {       // transpose of an 8x8 tile of 16-bit values held by a warp
  unsigned y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <bool F16>
__device__ __forceinline__ unsigned pd_pack(float lo, float hi) {
  if constexpr (F16) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&v);
  } else {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&v);
  }
}
template <bool F16>
__device__ __forceinline__ float2 pd_unpack(unsigned v) {
  if constexpr (F16) return __half22float2(*reinterpret_cast<const __half2*>(&v));
  else return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
// (x, y) -> packed heads and packed remainders
template <bool F16>
__device__ __forceinline__ void pd_split(float x, float y, unsigned& hi, unsigned& lo) {
  hi = pd_pack<F16>(x, y);
  const float2 h = pd_unpack<F16>(hi);
  lo = pd_pack<F16>(x - h.x, y - h.y);
}
__device__ __forceinline__ unsigned pd_cvt(unsigned pair) {     // two e4m3 bytes -> two fp16
  const __half2 h = cvt_e4m3x2(static_cast<unsigned short>(pair));
  return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ uint4 pd_ldg(const void* p) {        // cache rows are read once: no L1 allocation
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ float pd_ex2(float x) {
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ unsigned pd_word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// A page scale as a power of two's exponent, inside the range that append writes (a scale of 0 reads as the least one).
__device__ __forceinline__ float pd_log2_scale(float s) { return log2f(fminf(fmaxf(s, 8.673617379884035e-19f), 1.152921504606847e18f)); }

// ---- work items ------------------------------------------------------------------------------------------------------------
struct PdWork {
  int tiles, units, items;       // of one sequence: row tiles, units per item, items = nkv * tiles
  long long total;               // items * units
};
__device__ __forceinline__ PdWork pd_work(const IhbPaged& c, const PgSeq& s, int G, int RT) {
  PdWork w;
  w.tiles = (s.n * G + RT - 1) / RT;
  w.units = s.n > 0 ? (s.len + PD_UNIT - 1) / PD_UNIT : 0;
  w.items = w.units > 0 ? w.tiles * c.nkv : 0;
  w.total = static_cast<long long>(w.items) * w.units;
  return w;
}
__device__ __forceinline__ long long warp_incl_scan_ll(long long v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}
// Units of the whole batch (whole warp).
__device__ __forceinline__ long long pd_total(const IhbPaged& c, int G, int RT, int lane) {
  long long sum = 0;
  for (int b = lane; b < c.B; b += 32) sum += pd_work(c, pg_seq(c, b), G, RT).total;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}
// The sequence that holds unit u (whole warp, u < total); `before`: units ahead of it.
__device__ __forceinline__ int pd_find(const IhbPaged& c, int G, int RT, int lane, long long u, long long& before) {
  long long at = 0;
  for (int b0 = 0; b0 < c.B; b0 += 32) {
    long long t = 0;
    if (b0 + lane < c.B) t = pd_work(c, pg_seq(c, b0 + lane), G, RT).total;
    const long long incl = warp_incl_scan_ll(t, lane);
    const unsigned hit = __ballot_sync(0xffffffffu, at + incl > u);
    if (hit) {
      const int src = __ffs(hit) - 1;
      before = at + __shfl_sync(0xffffffffu, incl - t, src);
      return b0 + src;
    }
    at += __shfl_sync(0xffffffffu, incl, 31);
  }
  before = at;
  return c.B;
}
// Ranges: CTA i of `parts` takes units [i * total / parts, (i + 1) * total / parts).
__device__ __forceinline__ int pd_parts(long long total, int grid) { return static_cast<int>(total < grid ? total : grid); }
__device__ __forceinline__ long long pd_cut(long long total, int parts, int i) { return total * i / parts; }

__device__ __forceinline__ void pd_store(const IhbPagedAttn& a, int t, int h, int ch, float v) {
  const size_t o = static_cast<size_t>(t) * a.out_stride_t + static_cast<size_t>(h) * a.out_stride_h + ch;
  if (a.out_bf16) reinterpret_cast<__nv_bfloat16*>(a.out)[o] = __float2bfloat16(v);
  else reinterpret_cast<float*>(a.out)[o] = v;
}
// (m, l) of a finished row -> natural log of its denominator
template <bool KV8>
__device__ __forceinline__ float pd_lse(float m, float l) {
  return l > 0.f ? (m - (KV8 ? PD_OFF : 0.f) + log2f(l)) * 0.6931471805599453f : (l == 0.f ? -INFINITY : l);
}

// Does row i of the call's tokens (of a sequence with s.n) see key p?
__device__ __forceinline__ bool pd_sees(const IhbPagedAttn& a, const PgSeq& s, int i, int p) {
  if (i >= s.n || p >= s.len) return false;
  const int j = p - s.base;
  if (a.mask == nullptr) return j <= i;
  return j < 0 || (j < a.mask_stride && a.mask[static_cast<size_t>(s.t0 + i) * a.mask_stride + j] != 0);
}

template <int NT, bool KV8, bool QF32>
__global__ void __launch_bounds__(PD_WARPS * 32, NT == 1 ? 4 : (QF32 ? 2 : 3)) paged_rows_kernel(const __grid_constant__ IhbPagedAttn a, int grid) {
  constexpr int RT = 8 * NT;
  constexpr bool PSPLIT = QF32 || !KV8;      // probabilities as head + remainder: fp32 results, and bf16 would round them by 2^-9
  constexpr int KW = KV8 ? 2 : 4;            // 16-byte loads per key of a thread's 32 channels
  __shared__ __align__(16) float o_s[PD_WARPS][RT][PG_HD + 4];
  __shared__ float m_s[PD_WARPS][RT], l_s[PD_WARPS][RT];
  const IhbPaged& c = a.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const int G = a.nq / c.nkv;
  pdl_launch_dependents();                   // the folding kernel waits for this one's end; it may be scheduled from here on

  // entries without a cached row: zeros
  for (int b = blockIdx.x; b < c.B; b += grid) {
    const PgSeq s = pg_seq(c, b);
    if (s.len > 0 || s.n == 0) continue;
    for (int i = 0; i < s.n; ++i)
      for (int h = 0; h < a.nq; ++h) pd_store(a, s.t0 + i, h, tid, 0.f);
    if (a.lse != nullptr)
      for (int i = tid; i < s.n * a.nq; i += PD_WARPS * 32) a.lse[static_cast<size_t>(s.t0) * a.nq + i] = -INFINITY;
  }

  const long long total = pd_total(c, G, RT, lane);
  const int parts = pd_parts(total, grid);
  if (static_cast<int>(blockIdx.x) >= parts) return;
  long long u = pd_cut(total, parts, blockIdx.x);
  const long long u_end = pd_cut(total, parts, blockIdx.x + 1), u_first = u;
  long long before;
  int b = pd_find(c, G, RT, lane, u, before);
  PgSeq s = pg_seq(c, b);
  PdWork w = pd_work(c, s, G, RT);
  const int psh = __ffs(c.page) - 1;
  const float sm = a.scale * PG_LOG2E;

  while (u < u_end) {
    while (u - before >= w.total) {           // next sequence with work
      before += w.total;
      ++b;
      s = pg_seq(c, b);
      w = pd_work(c, s, G, RT);
    }
    const int item = static_cast<int>((u - before) / w.units), unit0 = static_cast<int>((u - before) % w.units);
    const int n_units = static_cast<int>(min(static_cast<long long>(w.units - unit0), u_end - u));
    const int kvh = item / w.tiles, row0 = (item % w.tiles) * RT;
    const int* table = c.block_table + static_cast<size_t>(b) * c.table_stride;

    // ---- Q^T fragments: row g of each group of 8, the channels that this thread takes of every key ----
    unsigned qh[NT][8][2], ql[QF32 ? NT : 1][8][2];
    float rowf[NT][2];                        // what a score of rows 2 t4, 2 t4 + 1 is multiplied by
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = row0 + nt * 8 + g, i = r / G;
      const bool ok = i < s.n;
      const size_t off = ok ? static_cast<size_t>(s.t0 + i) * a.q_stride_t + static_cast<size_t>(kvh * G + r % G) * a.q_stride_h : 0;
      float x[32];
#pragma unroll
      for (int j = 0; j < 4; ++j) {           // 8 neighbouring channels at a time
        const int ch = KV8 ? (j >> 1) * 64 + t4 * 16 + (j & 1) * 8 : j * 32 + t4 * 8;
        float4 lo = make_float4(0.f, 0.f, 0.f, 0.f), hi = lo;
        if (ok) {
          if (a.q_bf16) {
            const uint4 v = *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(a.q) + off + ch);
            lo = make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
            hi = make_float4(__uint_as_float(v.z << 16), __uint_as_float(v.z & 0xffff0000u), __uint_as_float(v.w << 16), __uint_as_float(v.w & 0xffff0000u));
          } else {
            const float4* f = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a.q) + off + ch);
            lo = f[0];
            hi = f[1];
          }
        }
        x[8 * j] = lo.x; x[8 * j + 1] = lo.y; x[8 * j + 2] = lo.z; x[8 * j + 3] = lo.w;
        x[8 * j + 4] = hi.x; x[8 * j + 5] = hi.y; x[8 * j + 6] = hi.z; x[8 * j + 7] = hi.w;
      }
      float f = 1.f;
      if constexpr (KV8) {                    // |q| of the row into [1, 2): exact, and fp16 then holds what bf16 does
        float mx = 0.f;
#pragma unroll
        for (int j = 0; j < 32; ++j) mx = fmaxf(mx, fabsf(x[j]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const int e = min(max(static_cast<int>(__float_as_uint(mx) >> 23) - 127, -100), 100);
        f = __uint_as_float(static_cast<unsigned>(127 + e) << 23);
        const float inv = __uint_as_float(static_cast<unsigned>(127 - e) << 23);
#pragma unroll
        for (int j = 0; j < 32; ++j) x[j] *= inv;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if constexpr (QF32) pd_split<KV8>(x[4 * k + 2 * h], x[4 * k + 2 * h + 1], qh[nt][k][h], ql[nt][k][h]);
          else qh[nt][k][h] = pd_pack<KV8>(x[4 * k + 2 * h], x[4 * k + 2 * h + 1]);
        }
      rowf[nt][0] = sm * __shfl_sync(0xffffffffu, f, (2 * t4) * 4);
      rowf[nt][1] = sm * __shfl_sync(0xffffffffu, f, (2 * t4 + 1) * 4);
    }

    float o[NT][8][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < 8; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.f;
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
    }
    // keys that any row of the tile sees lie below key_end; below key_all every row sees them
    const int i_last = min((row0 + RT - 1) / G, s.n - 1);
    const int seen_end = a.mask != nullptr ? s.len : min(s.len, s.base + i_last + 1);
    const int key_end = min(seen_end, (unit0 + n_units) * PD_UNIT);
    const int key_all = min(s.len, a.mask != nullptr ? s.base : s.base + row0 / G + 1);

    uint4 kr[2][KW], vr[4][KV8 ? 1 : 2];
    float ksc = 1.f, vsc = 1.f, ksn = 1.f, vsn = 1.f;
    int pg_next;                              // page of the step after the one whose rows are being loaded
    auto page_of = [&](int key) -> int {
      if (key >= key_end) return -2;
      const int p = table[key >> psh];
      return p;
    };
    auto load_k = [&](int key, int page) {
      const bool ok = key < key_end && page >= 0 && page < c.n_pages;
      const size_t hr = (static_cast<size_t>(ok ? page : 0) * c.nkv + kvh) * c.page + (ok ? (key & (c.page - 1)) : 0);
      const char* base = reinterpret_cast<const char*>(c.k) + hr * (KV8 ? PG_HD : 2 * PG_HD);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < KW; ++j)
          kr[h][j] = ok ? pd_ldg(base + (g + 8 * h) * (KV8 ? PG_HD : 2 * PG_HD) + j * 64 + t4 * 16) : make_uint4(0, 0, 0, 0);
      if constexpr (KV8) {
        const size_t si = static_cast<size_t>(ok ? page : 0) * c.nkv + kvh;
        ksn = ok ? c.k_scale[si] : 0.f;
        vsn = ok ? c.v_scale[si] : 0.f;
      }
    };
    auto load_v = [&](int key, int page) {
      const bool ok = key < key_end && page >= 0 && page < c.n_pages;
      const size_t hr = (static_cast<size_t>(ok ? page : 0) * c.nkv + kvh) * c.page + (ok ? (key & (c.page - 1)) : 0);
      const char* base = reinterpret_cast<const char*>(c.v) + hr * (KV8 ? PG_HD : 2 * PG_HD);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int kk = 2 * t4 + (i & 1) + 8 * (i >> 1);
        const bool in = ok && key + kk < s.len;   // rows behind the sequence may hold anything: 0 * NaN is NaN
#pragma unroll
        for (int j = 0; j < (KV8 ? 1 : 2); ++j)
          vr[i][j] = in ? pd_ldg(base + kk * (KV8 ? PG_HD : 2 * PG_HD) + j * 128 + g * 16) : make_uint4(0, 0, 0, 0);
      }
    };

    int key = unit0 * PD_UNIT + warp * 16;
    int page = page_of(key);
    load_k(key, page);
    load_v(key, page);
    pg_next = page_of(key + PD_UNIT);
    for (; key < key_end; key += PD_UNIT) {
      const bool bad_page = page < 0 || page >= c.n_pages;
      if (bad_page && lane == 0) set_error(c.err, ERR_BAD_ARGS);
      ksc = ksn;
      vsc = vsn;
      // ---- S^T: 16 keys x RT rows ----
      float d[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) d[nt][0] = d[nt][1] = d[nt][2] = d[nt][3] = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        unsigned af[4];
        if constexpr (KV8) {
          const unsigned w0 = pd_word(kr[0][k >> 2], k & 3), w1 = pd_word(kr[1][k >> 2], k & 3);
          af[0] = pd_cvt(w0 & 0xffffu); af[1] = pd_cvt(w1 & 0xffffu);
          af[2] = pd_cvt(w0 >> 16);     af[3] = pd_cvt(w1 >> 16);
        } else {
          af[0] = pd_word(kr[0][k >> 1], (k & 1) * 2);     af[1] = pd_word(kr[1][k >> 1], (k & 1) * 2);
          af[2] = pd_word(kr[0][k >> 1], (k & 1) * 2 + 1); af[3] = pd_word(kr[1][k >> 1], (k & 1) * 2 + 1);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          pd_mma<KV8>(d[nt], af, qh[nt][k][0], qh[nt][k][1]);
          if constexpr (QF32) pd_mma<KV8>(d[nt], af, ql[nt][k][0], ql[nt][k][1]);
        }
      }
      const int page_now = pg_next;
      load_k(key + PD_UNIT, page_now);        // the next step's K while this step's softmax and V product run
      pg_next = page_of(key + 2 * PD_UNIT);
      // ---- softmax: rows 2 t4, 2 t4 + 1, keys g, g + 8 ----
      const float ev = KV8 ? pd_log2_scale(vsc) : 0.f;
      const bool edge = bad_page || key + 16 > key_all;
      bool grow = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float f = KV8 ? rowf[nt][j & 1] * ksc : rowf[nt][j & 1];
          d[nt][j] = fmaf(d[nt][j], f, ev);
          if (edge && (bad_page || !pd_sees(a, s, (row0 + nt * 8 + 2 * t4 + (j & 1)) / G, key + g + 8 * (j >> 1)))) d[nt][j] = -INFINITY;
        }
        grow |= fmaxf(d[nt][0], d[nt][2]) > m[nt][0] + PD_LAZY || fmaxf(d[nt][1], d[nt][3]) > m[nt][1] + PD_LAZY;
      }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float mx = fmaxf(d[nt][r], d[nt][r + 2]);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float mn = fmaxf(m[nt][r], mx);
            const float f = m[nt][r] == -INFINITY ? 0.f : pd_ex2(m[nt][r] - mn);
            m[nt][r] = mn;
            l[nt][r] *= f;
#pragma unroll
            for (int j = 0; j < 8; ++j) { o[nt][j][r] *= f; o[nt][j][r + 2] *= f; }
          }
      }
      const float lf = KV8 ? pd_ex2(-ev) : 1.f;
      unsigned ph[NT][2], pl[PSPLIT ? NT : 1][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float mr = m[nt][j & 1] == -INFINITY ? 0.f : m[nt][j & 1];     // nothing seen yet: every score is -inf (or NaN)
          p[j] = pd_ex2(d[nt][j] - mr + (KV8 ? PD_OFF : 0.f));
        }
        l[nt][0] += (p[0] + p[2]) * lf;
        l[nt][1] += (p[1] + p[3]) * lf;
        if constexpr (PSPLIT) {
          unsigned h0, h1, r0, r1;
          pd_split<KV8>(p[0], p[1], h0, r0);
          pd_split<KV8>(p[2], p[3], h1, r1);
          ph[nt][0] = pd_movt(h0); ph[nt][1] = pd_movt(h1);
          pl[nt][0] = pd_movt(r0); pl[nt][1] = pd_movt(r1);
        } else {
          ph[nt][0] = pd_movt(pd_pack<KV8>(p[0], p[1]));
          ph[nt][1] = pd_movt(pd_pack<KV8>(p[2], p[3]));
        }
      }
      // ---- a value that is not finite in a row that not every query sees: those who see it get it, the others nothing ----
      if (key + 16 > key_all && key < seen_end) {
        bool odd = false;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < (KV8 ? 1 : 2); ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const unsigned x = pd_word(vr[i][j], q);
              if constexpr (KV8) odd |= ((((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0u);
              else odd |= (x & 0x7f80u) == 0x7f80u || (x & 0x7f800000u) == 0x7f800000u;
            }
        if (__any_sync(0xffffffffu, odd)) {
          for (int kk = 0; kk < 16; ++kk) {
            const int src = (lane & ~3) | ((kk & 7) >> 1), i = (kk & 1) + 2 * (kk >> 3);
#pragma unroll
            for (int j = 0; j < (KV8 ? 1 : 2); ++j)
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                unsigned mine = 0;
#pragma unroll
                for (int ii = 0; ii < 4; ++ii)
                  if (ii == i) mine = pd_word(vr[ii][j], q);
                const unsigned x = __shfl_sync(0xffffffffu, mine, src);
                float v[4];
                if constexpr (KV8) {
                  const float4 f = e4m3x4_to_float4(x);
                  v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
                } else {
                  v[0] = __uint_as_float(x << 16); v[1] = __uint_as_float(x & 0xffff0000u);
                  v[2] = v[3] = 0.f;
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                  for (int r = 0; r < 2; ++r) {
                    if (!pd_sees(a, s, (row0 + nt * 8 + 2 * t4 + r) / G, key + kk)) continue;
#pragma unroll
                    for (int e = 0; e < (KV8 ? 4 : 2); ++e) {
                      if (fabsf(v[e]) <= 3.4028235e38f) continue;     // finite
                      constexpr int M2 = KV8 ? 2 : 1;
                      const int mt = KV8 ? q * M2 + (e >> 1) : j * 4 + q;
#pragma unroll
                      for (int jj = 0; jj < 8; ++jj)
                        if (jj == mt) o[nt][jj][r + 2 * (e & 1)] += v[e];
                    }
                  }
              }
          }
          // and out of the product
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < (KV8 ? 1 : 2); ++j) {
              unsigned x[4] = {vr[i][j].x, vr[i][j].y, vr[i][j].z, vr[i][j].w};
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                if constexpr (KV8) {
#pragma unroll
                  for (int e = 0; e < 4; ++e)
                    if (((x[q] >> (8 * e)) & 0x7fu) == 0x7fu) x[q] &= ~(0xffu << (8 * e));
                } else {
                  if ((x[q] & 0x7f80u) == 0x7f80u) x[q] &= 0xffff0000u;
                  if ((x[q] & 0x7f800000u) == 0x7f800000u) x[q] &= 0x0000ffffu;
                }
              }
              vr[i][j] = make_uint4(x[0], x[1], x[2], x[3]);
            }
        }
      }
      // ---- O^T += V^T P^T: 8 tiles of 16 channels ----
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        unsigned af[4];
        if constexpr (KV8) {
          const unsigned sel = (j & 1) ? 0x7362u : 0x5140u;
          const unsigned x = __byte_perm(pd_word(vr[0][0], j >> 1), pd_word(vr[1][0], j >> 1), sel);
          const unsigned y = __byte_perm(pd_word(vr[2][0], j >> 1), pd_word(vr[3][0], j >> 1), sel);
          af[0] = pd_cvt(x & 0xffffu); af[1] = pd_cvt(x >> 16);
          af[2] = pd_cvt(y & 0xffffu); af[3] = pd_cvt(y >> 16);
        } else {
          const unsigned w0 = pd_word(vr[0][j >> 2], j & 3), w1 = pd_word(vr[1][j >> 2], j & 3);
          const unsigned w2 = pd_word(vr[2][j >> 2], j & 3), w3 = pd_word(vr[3][j >> 2], j & 3);
          af[0] = __byte_perm(w0, w1, 0x5410); af[1] = __byte_perm(w0, w1, 0x7632);
          af[2] = __byte_perm(w2, w3, 0x5410); af[3] = __byte_perm(w2, w3, 0x7632);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          pd_mma<KV8>(o[nt][j], af, ph[nt][0], ph[nt][1]);
          if constexpr (PSPLIT) pd_mma<KV8>(o[nt][j], af, pl[nt][0], pl[nt][1]);
        }
      }
      load_v(key + PD_UNIT, page_now);
      page = page_now;
    }

    // ---- the four warps' results ----
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float t = l[nt][r];
        t += __shfl_xor_sync(0xffffffffu, t, 4);
        t += __shfl_xor_sync(0xffffffffu, t, 8);
        t += __shfl_xor_sync(0xffffffffu, t, 16);
        const int row = nt * 8 + 2 * t4 + r;
        if (g == 0) { m_s[warp][row] = m[nt][r]; l_s[warp][row] = t; }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int ch = KV8 ? g * 16 + 2 * j : (j >> 2) * 64 + g * 8 + (j & 3) * 2;
          *reinterpret_cast<float2*>(&o_s[warp][row][ch]) = make_float2(o[nt][j][r], o[nt][j][r + 2]);
        }
      }
    __syncthreads();
    const bool whole = n_units == w.units;
    float* rec = reinterpret_cast<float*>(a.scratch) + (static_cast<size_t>(blockIdx.x) * 2 + (u == u_first ? 0 : 1)) * RT * PD_REC;
    for (int row = 0; row < RT; ++row) {
      float M = fmaxf(fmaxf(m_s[0][row], m_s[1][row]), fmaxf(m_s[2][row], m_s[3][row])), L = 0.f, acc = 0.f;
      if (M > -INFINITY) {
#pragma unroll
        for (int x = 0; x < PD_WARPS; ++x) {
          const float f = m_s[x][row] == -INFINITY ? 0.f : pd_ex2(m_s[x][row] - M);
          L += f * l_s[x][row];
          acc += f == 0.f ? 0.f : f * o_s[x][row][tid];
        }
      } else {                                 // nothing seen, or nothing but NaN
#pragma unroll
        for (int x = 0; x < PD_WARPS; ++x) { L += l_s[x][row]; acc += o_s[x][row][tid]; }
      }
      if (whole) {
        const int i = (row0 + row) / G;
        if (i < s.n) {
          const int hd = kvh * G + (row0 + row) % G;
          pd_store(a, s.t0 + i, hd, tid, L == 0.f ? acc * 0.f : acc / L);
          if (tid == 0 && a.lse != nullptr) a.lse[static_cast<size_t>(s.t0 + i) * a.nq + hd] = pd_lse<KV8>(M, L);
        }
      } else {
        rec[row * PD_REC + tid] = acc;
        if (tid == 0) { rec[row * PD_REC + PG_HD] = M; rec[row * PD_REC + PG_HD + 1] = L; }
      }
    }
    __syncthreads();
    u += n_units;
  }
}

// Folds the records of the items that a range end cut. Block i looks at the cut before range i: it owns the item if that cut is the
// first one inside it. 128 threads: one channel each.
template <bool KV8>
__global__ void __launch_bounds__(128) paged_fold_kernel(const __grid_constant__ IhbPagedAttn a, int grid, int RT) {
  const IhbPaged& c = a.c;
  const int tid = threadIdx.x, lane = tid & 31, G = a.nq / c.nkv;
  const long long total = pd_total(c, G, RT, lane);
  const int parts = pd_parts(total, grid), i0 = blockIdx.x + 1;
  if (i0 >= parts) { pdl_wait(); return; }
  const long long cut = pd_cut(total, parts, i0);
  long long before;
  const int b = pd_find(c, G, RT, lane, cut, before);
  const PgSeq s = pg_seq(c, b);
  const PdWork w = pd_work(c, s, G, RT);
  const int item = static_cast<int>((cut - before) / w.units);
  const long long lo = before + static_cast<long long>(item) * w.units, hi = lo + w.units;
  pdl_wait();
  if (cut == lo || pd_cut(total, parts, i0 - 1) > lo) return;   // not inside an item, or an earlier cut is
  int last = i0;                                                // ranges i0 - 1 .. last have a piece
  while (last + 1 < parts && pd_cut(total, parts, last + 1) < hi) ++last;
  const int kvh = item / w.tiles, row0 = (item % w.tiles) * RT;
  const float* recs = reinterpret_cast<const float*>(a.scratch);
  // the first range's piece is its last segment (slot 1 unless the range began inside this item or at its start)
  const int first_slot = pd_cut(total, parts, i0 - 1) == lo ? 0 : 1;
  for (int row = blockIdx.y; row < RT; row += gridDim.y) {
    const int i = (row0 + row) / G;
    if (i >= s.n) break;
    float M = -INFINITY;
    for (int x = i0 - 1; x <= last; ++x) M = fmaxf(M, recs[((static_cast<size_t>(x) * 2 + (x == i0 - 1 ? first_slot : 0)) * RT + row) * PD_REC + PG_HD]);
    float L = 0.f, acc = 0.f;
#pragma unroll 4
    for (int x = i0 - 1; x <= last; ++x) {
      const float* r = recs + ((static_cast<size_t>(x) * 2 + (x == i0 - 1 ? first_slot : 0)) * RT + row) * PD_REC;
      const float mx = r[PG_HD];
      const float f = M == -INFINITY ? 1.f : (mx == -INFINITY ? 0.f : pd_ex2(mx - M));
      const float v = r[tid];
      L += f * r[PG_HD + 1];
      acc += f == 0.f ? 0.f : f * v;
    }
    const int hd = kvh * G + (row0 + row) % G;
    pd_store(a, s.t0 + i, hd, tid, L == 0.f ? acc * 0.f : acc / L);
    if (tid == 0 && a.lse != nullptr) a.lse[static_cast<size_t>(s.t0 + i) * a.nq + hd] = pd_lse<KV8>(M, L);
  }
}

struct PdPlan {
  int nt, grid;
};
static PdPlan pd_plan(const IhbPagedAttn& a) {
  PdPlan p;
  const int G = a.nq / a.c.nkv;
  p.nt = static_cast<long long>(a.max_q) * G <= 8 ? 1 : 2;
  const bool f32 = !a.q_bf16;
  p.grid = 148 * (p.nt == 1 ? 4 : (f32 ? 2 : 3));             // what is resident at once
  return p;
}

template <int NT, bool KV8, bool QF32>
static cudaError_t pd_launch(const IhbPagedAttn& a, const PdPlan& p, cudaStream_t stream) {
  paged_rows_kernel<NT, KV8, QF32><<<p.grid, PD_WARPS * 32, 0, stream>>>(a, p.grid);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(p.grid - 1, 4);
  cfg.blockDim = dim3(128);
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_fold_kernel<KV8>, a, p.grid, 8 * NT);
}

}  // namespace ihb

using namespace ihb;

static bool paged_attn_ok(const IhbPagedAttn& a) {
  const IhbPaged& c = a.c;
  const bool page = c.page == 16 || c.page == 32 || c.page == 64 || c.page == 128;
  return page && c.k != nullptr && c.v != nullptr && (c.k_scale == nullptr) == (c.v_scale == nullptr) && c.n_pages > 0 && c.nkv > 0 &&
         c.B > 0 && c.T > 0 && c.max_blocks > 0 && c.block_table != nullptr && c.kv_len != nullptr && (c.cu_q != nullptr || c.B == c.T) &&
         a.q != nullptr && a.out != nullptr && a.nq > 0 && a.nq % c.nkv == 0 && a.max_q > 0 && (a.mask == nullptr || a.mask_stride >= 1) &&
         a.q_stride_t % 8 == 0 && a.q_stride_h % 8 == 0;
}

extern "C" size_t ihb_paged_attention_scratch(const IhbPagedAttn* a) {
  if (a->c.nkv < 1 || a->nq % a->c.nkv) return 0;
  const PdPlan p = pd_plan(*a);
  return static_cast<size_t>(p.grid) * 2 * 8 * p.nt * PD_REC * sizeof(float);
}

extern "C" int ihb_paged_attention(const IhbPagedAttn* p, cudaStream_t stream) {
  const IhbPagedAttn& a = *p;
  if (!paged_attn_ok(a) || a.scratch == nullptr) return cudaErrorInvalidValue;
  const PdPlan pl = pd_plan(a);
  const bool kv8 = a.c.k_scale != nullptr, f32 = !a.q_bf16;
  if (pl.nt == 1) {
    if (kv8) return f32 ? pd_launch<1, true, true>(a, pl, stream) : pd_launch<1, true, false>(a, pl, stream);
    return f32 ? pd_launch<1, false, true>(a, pl, stream) : pd_launch<1, false, false>(a, pl, stream);
  }
  if (kv8) return f32 ? pd_launch<2, true, true>(a, pl, stream) : pd_launch<2, true, false>(a, pl, stream);
  return f32 ? pd_launch<2, false, true>(a, pl, stream) : pd_launch<2, false, false>(a, pl, stream);
}
