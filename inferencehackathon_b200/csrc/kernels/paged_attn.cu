// Attention of a ragged batch over a paged KV cache: single decode tokens and short verify windows, head_dim 128, bf16 pages or
// e4m3 pages with one scale per (page, head). The contiguous, one-sequence siblings are attn.cu::flash_decode_kernel and
// window.cu::window_attn_mma_kernel.
//
// The rows of a (sequence, KV head) are its (token, query head) pairs, RT = 8 or 16 of them per tile. Scores are computed
// transposed, S^T = K Q^T with m16n8k16 (16 keys x 8 rows), and so is the output, O^T = V^T P^T: the large operand is the A operand
// of both products and a thread's fragments of it are contiguous bytes of the cache (the channel order inside a product is free,
// so a thread takes 16 neighbouring bytes). With queries as the A operand (the usual way round) 8 query heads would waste half of
// every product. Each warp walks its own keys, 16 per step (bf16 pages) or 32 (e4m3: two groups share the query fragments and the
// step's overhead: 75 -> 67 us at 64 sequences of 129 to 8191 keys), through a ring of asynchronous 16-byte copies in shared memory that
// only it reads: no barrier until the four warps' results are added at the end of an item.
//
// e4m3 pages: bytes become fp16 exactly; q is scaled per row by a power of two into fp16 (head and remainder for fp32
// queries: 22 bits); the K scale is a factor of the score, the V scale s_v goes into the exponent of the probability: with
// m the running maximum of score + log2 s_v, O = sum 2^(s + log2 s_v - m) v_bytes and l = sum 2^(s - m). The probability that
// meets the bytes is then at most 2^14 whatever the scales are, which is what fp16 holds.
//
// Work split: the 128-key units of all (sequence, head, tile) items are laid end to end and cut into equal ranges, one per CTA, so
// ragged batches and single long sequences load every SM the same. Lengths are read on the device. An item cut by a range end
// leaves one record (O, m, l) per piece, folded by a second kernel in a fixed order: results do not depend on timing. The folding
// kernel is launched with the first one and works out its pieces while that runs.
//
// Measured (64 query heads, 4 KV heads): 64 sequences of 129 to 8191 keys, e4m3 pages, 65 us, 66 % of the measured copy bandwidth; one
// sequence of 131071 keys 42 us, 49 %; bf16 pages of 16 tokens, 32 / 4 heads, fp32 queries, 24 sequences of up to 4096 keys, 29 us, 53 %.
// Bound by the latency of dependent instructions at 12 warps per SM (shared memory for the rings): over e4m3 pages, where a 16-byte chunk is eight
// conversions and two matrix instructions, 47 % of the issue slots and 28 % of the matrix pipe; over bf16 pages with fp32 queries 33 % and 20 %, with waits
// for pages and tables, the ring's loads and the barrier at an item's end beside it (the three-term products are not what bounds it).
#include "paged.cuh"
#include "paged_tiles.h"

namespace ihb {

constexpr int PD_WARPS = 4;
constexpr int PD_UNIT = 128;                 // keys per unit of the work split
constexpr float PD_NONE = 3.402823466e38f;   // OFF - running maximum before the first key: any finite score is above it

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
__device__ __forceinline__ unsigned pd_word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// ---- work items ------------------------------------------------------------------------------------------------------------
// An item costs its units and PD_START more (loading Q, filling the ring, adding the warps up; 64 sequences of e4m3 pages: 2 73 us, 3 68, 4 64,
// 6 66): ranges are cut on that cost, so a CTA
// with many short items gets fewer keys. Positions inside an item: [0, PD_START) start-up, then the units.
constexpr int PD_START = 4;

struct PdWork {
  int tiles, units, items;       // of one sequence: row tiles, units per item, items = nkv * tiles
  long long total;               // cost: items * (units + PD_START)
};
__device__ __forceinline__ PdWork pd_work(const IhbPaged& c, const PgSeq& s, int G, int RT) {
  PdWork w;
  w.tiles = (s.n * G + RT - 1) / RT;
  w.units = s.n > 0 ? (s.len + PD_UNIT - 1) / PD_UNIT : 0;
  w.items = w.units > 0 ? w.tiles * c.nkv : 0;
  w.total = static_cast<long long>(w.items) * (w.units + PD_START);
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
// Cost of the whole batch (whole warp).
__device__ __forceinline__ long long pd_total(const IhbPaged& c, int G, int RT, int lane) {
  long long sum = 0;
  for (int b = lane; b < c.B; b += 32) sum += pd_work(c, pg_seq(c, b), G, RT).total;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}
// The sequence that holds position u (whole warp, u < total); `before`: cost ahead of it.
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
// Ranges: the positions in `parts` pieces that differ by one at most, the longer ones first; CTA i takes [at(i), at(i + 1)).
__device__ __forceinline__ int pd_parts(long long total, int grid) { return static_cast<int>(total < grid ? total : grid); }
struct PdCuts {
  long long per, rem;
  __device__ __forceinline__ PdCuts(long long total, int parts) : per(pg_div(total, max(parts, 1))), rem(total - per * parts) {}
  __device__ __forceinline__ long long at(int i) const { return per * i + min(static_cast<long long>(i), rem); }
  __device__ __forceinline__ int of(long long p) const {               // the range that holds position p
    const long long edge = rem * (per + 1);
    return static_cast<int>(p < edge ? pg_div(p, per + 1) : rem + pg_div(p - edge, per));
  }
};

__device__ __forceinline__ void pd_store(const IhbPagedAttn& a, int t, int h, int ch, float v) {
  const size_t o = static_cast<size_t>(t) * a.out_stride_t + static_cast<size_t>(h) * a.out_stride_h + ch;
  if (a.out_bf16) reinterpret_cast<__nv_bfloat16*>(a.out)[o] = __float2bfloat16(v);
  else reinterpret_cast<float*>(a.out)[o] = v;
}
// Does row i of the call's tokens (of a sequence with s.n) see key p?
__device__ __forceinline__ bool pd_sees(const IhbPagedAttn& a, const PgSeq& s, int i, int p) {
  if (i >= s.n || p >= s.len) return false;
  const int j = p - s.base;
  if (a.mask == nullptr) return j <= i;
  return j < 0 || (j < a.mask_cols && a.mask[static_cast<size_t>(s.t0 + i) * a.mask_stride + j] != 0);
}

// Shared memory of a CTA: ST key steps per warp in flight (per group 16 rows of K, 16 of V, the page's scales), the Q fragments of the row
// tile; the four warps' results take the place of the steps at the end of an item.
template <int NT, bool KV8, int QT>
struct PdSmem {
  static constexpr int ROWB = KV8 ? PG_HD : 2 * PG_HD;
  static constexpr int KG = KV8 ? 2 : 1;               // groups of 16 keys per step: two share the query fragments and the step's overhead
  static constexpr int SUB = 2 * 16 * ROWB + 16, STEP = KG * SUB;
  // CTAs per SM that ring and registers leave room for (fp32 queries, 16 rows: with three, 168 registers, e4m3 pages spill: 95 us for 64 sequences of
  // 4096 keys, 82 with two)
  static constexpr int PER_SM = NT == 2 && QT > 1 ? 2 : 3;
  static constexpr int ST = PER_SM == 2 ? 3 : 2;
  static constexpr int QB = QT * NT * 8 * 32 * 8;
  static constexpr int STEPS = PD_WARPS * ST * STEP, OUT = PD_WARPS * 8 * NT * (PG_HD + 4) * 4;
  static constexpr int BYTES = QB + (STEPS > OUT ? STEPS : OUT);
};

__device__ __forceinline__ void pd_cp16(uint32_t dst, const void* src, bool ok) {       // zeros when !ok: src is not read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void pd_cp4(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(ok ? 4 : 0) : "memory");
}
__device__ __forceinline__ void pd_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void pd_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// 16-byte chunk `ch` of row r: the chunks that the eight lanes of one shared-memory phase read lie in different banks
__device__ __forceinline__ int pd_kswz(int r, int ch) { return ch ^ ((r & 1) << 2); }
__device__ __forceinline__ int pd_vswz(int r, int ch) { return ch ^ (((r >> 1) & 3) << 1); }

// QT / PT: 16-bit terms that a query element / a probability is split into.
template <int NT, bool KV8, int QT, int PT>
__global__ void __launch_bounds__(PD_WARPS * 32, PdSmem<NT, KV8, QT>::PER_SM) paged_rows_kernel(const __grid_constant__ IhbPagedAttn a, int grid) {
  using SM = PdSmem<NT, KV8, QT>;
  constexpr int RT = 8 * NT, ST = SM::ST, ROWB = SM::ROWB;
  extern __shared__ __align__(128) unsigned char pd_sm[];
  __shared__ float m_s[PD_WARPS][RT], l_s[PD_WARPS][RT], rowf_s[RT];
  uint2* qf = reinterpret_cast<uint2*>(pd_sm);                                   // [QT][NT][8][32]
  float (*o_s)[RT][PG_HD + 4] = reinterpret_cast<float (*)[RT][PG_HD + 4]>(pd_sm + SM::QB);
  const IhbPaged& c = a.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const int G = a.nq / c.nkv;
  unsigned char* ring = pd_sm + SM::QB + warp * ST * SM::STEP;
  pdl_launch_dependents();                   // the folding kernel waits for this one's end; it may be scheduled from here on

  // entries without a cached row: zeros
  for (int b = blockIdx.x; b < c.B; b += grid) {
    const PgSeq s = pg_seq(c, b);
    if (s.n > a.max_q && tid == 0) set_error(c.err, ERR_BAD_ARGS);      // more tokens than the caller planned for
    if (s.len > 0 || s.n == 0) continue;
    for (int i = 0; i < s.n; ++i)
      for (int h = 0; h < a.nq; ++h) pd_store(a, s.t0 + i, h, tid, 0.f);
    if (a.lse != nullptr)
      for (int i = tid; i < s.n * a.nq; i += PD_WARPS * 32) a.lse[static_cast<size_t>(s.t0) * a.nq + i] = -INFINITY;
  }

  const long long total = pd_total(c, G, RT, lane);
  const int parts = pd_parts(total, grid);
  if (static_cast<int>(blockIdx.x) >= parts) return;
  const PdCuts cuts(total, parts);
  long long u = cuts.at(blockIdx.x);
  const long long u_end = cuts.at(blockIdx.x + 1), u_first = u;
  long long before;
  int b = pd_find(c, G, RT, lane, u, before);
  PgSeq s = pg_seq(c, b);
  PdWork w = pd_work(c, s, G, RT);
  const int psh = __ffs(c.page) - 1;

  while (u < u_end) {
    while (u - before >= w.total) {           // next sequence with work
      before += w.total;
      ++b;
      s = pg_seq(c, b);
      w = pd_work(c, s, G, RT);
    }
    const int span = w.units + PD_START, item = static_cast<int>(pg_div(u - before, span));
    const int at = static_cast<int>(u - before - static_cast<long long>(item) * span);
    const int taken = static_cast<int>(min(static_cast<long long>(span - at), u_end - u));
    const int unit0 = max(at - PD_START, 0), n_units = at + taken - PD_START - unit0;
    if (n_units <= 0) {                       // only start-up cost of the item lies in this range
      u += taken;
      continue;
    }
    const int kvh = item / w.tiles, row0 = (item % w.tiles) * RT;
    const int* table = c.block_table + static_cast<size_t>(b) * c.table_stride;

    // keys that any row of the tile sees lie below key_end; below key_all every row sees them
    const int i_last = min((row0 + RT - 1) / G, s.n - 1);
    const int seen_end = a.mask != nullptr ? s.len : min(s.len, s.base + i_last + 1);
    const int key_end = min(seen_end, (unit0 + n_units) * PD_UNIT);
    const int key_all = min(s.len, a.mask != nullptr ? s.base : s.base + row0 / G + 1);

    auto page_of = [&](int key) -> int { return key < key_end ? table[key >> psh] : -1; };
    // lane's first chunk in the pages' rows: chunk `lane`, then every 32nd (two or four rows on)
    constexpr int CPR = ROWB / 16;            // chunks per row
    const int lr = lane / CPR, lc = lane % CPR;
    const size_t in_page = static_cast<size_t>(kvh) * c.page * ROWB + lane * 16;
    const char* k0 = reinterpret_cast<const char*>(c.k) + in_page;
    const char* v0 = reinterpret_cast<const char*>(c.v) + in_page;
    const unsigned page_bytes = static_cast<unsigned>(c.nkv * c.page) * ROWB;
    auto issue = [&](int key, int page, unsigned char* st) {             // the 16 keys from `key` on into one group of a step of the ring
      const bool ok = key < key_end && static_cast<unsigned>(page) < static_cast<unsigned>(c.n_pages);
      const unsigned pg = ok ? page : 0;
      const size_t off = static_cast<size_t>(pg) * page_bytes + (ok ? (key & (c.page - 1)) * ROWB : 0);
      const uint32_t kd = smem_u32(st), vd = kd + 16 * ROWB;
      const bool all = key + 16 <= s.len;     // rows behind the sequence may hold anything, and 0 * NaN is NaN: zeros instead
#pragma unroll
      for (int i = 0; i < ROWB / 32; ++i) {
        const int r = lr + i * (32 / CPR);
        pd_cp16(kd + r * ROWB + pd_kswz(r, lc) * 16, k0 + off + i * 512, ok);
        pd_cp16(vd + r * ROWB + pd_vswz(r, lc) * 16, v0 + off + i * 512, ok && (all || key + r < s.len));
      }
      if (KV8 && lane < 2) pd_cp4(kd + 32 * ROWB + lane * 4, (lane ? c.v_scale : c.k_scale) + static_cast<size_t>(pg) * c.nkv + kvh, ok);
      if (lane == 2) *reinterpret_cast<int*>(st + 32 * ROWB + 8) = ok || key >= key_end;
    };

    constexpr int KG = SM::KG, STRIDE = PD_WARPS * 16 * KG;            // keys between a warp's steps
    int key = unit0 * PD_UNIT + warp * 16 * KG;
    int page_next[KG];
#pragma unroll
    for (int kg = 0; kg < KG; ++kg) page_next[kg] = page_of(key + 16 * kg);
#pragma unroll
    for (int i = 0; i < ST - 1; ++i) {
#pragma unroll
      for (int kg = 0; kg < KG; ++kg) {
        const int page = page_next[kg];
        page_next[kg] = page_of(key + (i + 1) * STRIDE + 16 * kg);
        issue(key + i * STRIDE + 16 * kg, page, ring + i * SM::STEP + kg * SM::SUB);
      }
      pd_commit();
    }

    // ---- Q^T fragments, one group of 8 rows per warp: row g, the channels that lane t4 takes of every key ----
    if (warp < NT) {
      const int r = row0 + warp * 8 + g, i = r / G;
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
      if (t4 == 0) rowf_s[warp * 8 + g] = a.scale * PG_LOG2E * f;
#pragma unroll
      for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          unsigned q2[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float& y0 = x[4 * k + 2 * h];
            float& y1 = x[4 * k + 2 * h + 1];
            q2[h] = pd_pack<KV8>(y0, y1);
            const float2 v = pd_unpack<KV8>(q2[h]);
            y0 -= v.x;
            y1 -= v.y;
          }
          qf[((t * NT + warp) * 8 + k) * 32 + lane] = make_uint2(q2[0], q2[1]);
        }
    }
    __syncthreads();

    float o[NT][8][4];
    constexpr float OFF = KV8 ? PD_OFF : 0.f;
    float mo[NT][2], l[NT][2], rowf[NT][2];   // mo: OFF - running maximum
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < 8; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.f;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        mo[nt][r] = PD_NONE;
        l[nt][r] = 0.f;
        rowf[nt][r] = rowf_s[nt * 8 + 2 * t4 + r];
      }
    }

    int slot = 0;
    for (; key < key_end; key += STRIDE) {
      pd_wait<ST - 2>();                      // this step's copies have landed (those of the lane; the others' after the barrier)
      __syncwarp();
      {
        const int nslot = slot == 0 ? ST - 1 : slot - 1;                 // the step that was read last
#pragma unroll
        for (int kg = 0; kg < KG; ++kg) {
          const int page = page_next[kg];
          page_next[kg] = page_of(key + ST * STRIDE + 16 * kg);
          issue(key + (ST - 1) * STRIDE + 16 * kg, page, ring + nslot * SM::STEP + kg * SM::SUB);
        }
        pd_commit();
      }
      const unsigned char* st = ring + slot * SM::STEP;
      slot = slot == ST - 1 ? 0 : slot + 1;
      // ---- S^T: 16 keys x RT rows per group ----
      float d[KG][NT][4];
#pragma unroll
      for (int kg = 0; kg < KG; ++kg)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) d[kg][nt][0] = d[kg][nt][1] = d[kg][nt][2] = d[kg][nt][3] = 0.f;
#pragma unroll
      for (int k4 = 0; k4 < ROWB / 64; ++k4) {      // one 16-byte chunk of keys g and g + 8
        uint4 x0[KG], x1[KG];
#pragma unroll
        for (int kg = 0; kg < KG; ++kg) {
          x0[kg] = *reinterpret_cast<const uint4*>(st + kg * SM::SUB + g * ROWB + pd_kswz(g, k4 * 4 + t4) * 16);
          x1[kg] = *reinterpret_cast<const uint4*>(st + kg * SM::SUB + (g + 8) * ROWB + pd_kswz(g + 8, k4 * 4 + t4) * 16);
        }
#pragma unroll
        for (int kk = 0; kk < (KV8 ? 4 : 2); ++kk) {
          const int k = k4 * (KV8 ? 4 : 2) + kk;
          unsigned af[KG][4];
#pragma unroll
          for (int kg = 0; kg < KG; ++kg) {
            if constexpr (KV8) {
              pd_cvt4(pd_word(x0[kg], kk), af[kg][0], af[kg][2]);
              pd_cvt4(pd_word(x1[kg], kk), af[kg][1], af[kg][3]);
            } else {
              af[kg][0] = pd_word(x0[kg], 2 * kk);     af[kg][1] = pd_word(x1[kg], 2 * kk);
              af[kg][2] = pd_word(x0[kg], 2 * kk + 1); af[kg][3] = pd_word(x1[kg], 2 * kk + 1);
            }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int t = 0; t < QT; ++t) {
              const uint2 q2 = qf[((t * NT + nt) * 8 + k) * 32 + lane];
#pragma unroll
              for (int kg = 0; kg < KG; ++kg) pd_mma<KV8>(d[kg][nt], af[kg], q2.x, q2.y);
            }
        }
      }
      // ---- softmax: rows 2 t4, 2 t4 + 1, keys g, g + 8 of each group ----
      bool grow = false;
      float lf[KG];
#pragma unroll
      for (int kg = 0; kg < KG; ++kg) {
        const float2 sc = *reinterpret_cast<const float2*>(st + kg * SM::SUB + 32 * ROWB);
        const bool bad_page = *reinterpret_cast<const int*>(st + kg * SM::SUB + 32 * ROWB + 8) == 0;
        if (bad_page && lane == 0) set_error(c.err, ERR_BAD_ARGS);
        const float ev = KV8 ? pd_log2_scale(sc.y) : 0.f;
        lf[kg] = KV8 ? pd_ex2(-ev) : 1.f;
        const bool edge = bad_page || key + 16 * kg + 16 > key_all;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float (&x)[4] = d[kg][nt];
          const float f0 = KV8 ? rowf[nt][0] * sc.x : rowf[nt][0], f1 = KV8 ? rowf[nt][1] * sc.x : rowf[nt][1];
          x[0] = fmaf(x[0], f0, ev);
          x[1] = fmaf(x[1], f1, ev);
          x[2] = fmaf(x[2], f0, ev);
          x[3] = fmaf(x[3], f1, ev);
          if (edge)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (bad_page || !pd_sees(a, s, (row0 + nt * 8 + 2 * t4 + (j & 1)) / G, key + 16 * kg + g + 8 * (j >> 1))) x[j] = -INFINITY;
          grow |= fmaxf(x[0], x[2]) + mo[nt][0] > PD_LAZY + OFF || fmaxf(x[1], x[3]) + mo[nt][1] > PD_LAZY + OFF;
        }
      }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float mx = -INFINITY;
#pragma unroll
            for (int kg = 0; kg < KG; ++kg) mx = fmaxf(mx, fmaxf(d[kg][nt][r], d[kg][nt][r + 2]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            if (mx == -INFINITY) continue;
            const float was = mo[nt][r];
            mo[nt][r] = fminf(was, OFF - mx);
            const float f = was == PD_NONE ? 0.f : pd_ex2(mo[nt][r] - was);
            l[nt][r] *= f;
#pragma unroll
            for (int j = 0; j < 8; ++j) { o[nt][j][r] *= f; o[nt][j][r + 2] *= f; }
          }
      }
      unsigned ph[KG][NT][PT][2];
#pragma unroll
      for (int kg = 0; kg < KG; ++kg)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float p[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) p[j] = pd_ex2(d[kg][nt][j] + mo[nt][j & 1]);      // nothing seen yet: every score is -inf (or NaN), and so is the sum
          l[nt][0] += (p[0] + p[2]) * lf[kg];
          l[nt][1] += (p[1] + p[3]) * lf[kg];
#pragma unroll
          for (int t = 0; t < PT; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const unsigned x = pd_pack<KV8>(p[2 * h], p[2 * h + 1]);
              ph[kg][nt][t][h] = pd_movt(x);
              if (t + 1 < PT) {
                const float2 v = pd_unpack<KV8>(x);
                p[2 * h] -= v.x;
                p[2 * h + 1] -= v.y;
              }
            }
        }
      // ---- V rows 2 t4, 2 t4 + 1, + 8, + 9: 16 channels ----
#pragma unroll
      for (int kg = 0; kg < KG; ++kg) {
        const unsigned char* vst = st + kg * SM::SUB + 16 * ROWB;
        const int key0 = key + 16 * kg;
#pragma unroll
        for (int jv = 0; jv < (KV8 ? 1 : 2); ++jv) {
          uint4 vr[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = 2 * t4 + (i & 1) + 8 * (i >> 1);
            vr[i] = *reinterpret_cast<const uint4*>(vst + r * ROWB + pd_vswz(r, jv * 8 + g) * 16);
          }
          // a value that is not finite in a row that not every query sees: those who see it get it, the others nothing
          if (key0 + 16 > key_all) {
            bool odd = false;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const unsigned x = pd_word(vr[i], q);
                if constexpr (KV8) odd |= ((((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0u);
                else odd |= (x & 0x7f80u) == 0x7f80u || (x & 0x7f800000u) == 0x7f800000u;
              }
            if (__any_sync(0xffffffffu, odd)) {
              for (int kk = 0; kk < 16; ++kk) {
                const unsigned* xr = reinterpret_cast<const unsigned*>(vst + kk * ROWB + pd_vswz(kk, jv * 8 + g) * 16);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  const unsigned x = xr[q];
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
                      if (!pd_sees(a, s, (row0 + nt * 8 + 2 * t4 + r) / G, key0 + kk)) continue;
#pragma unroll
                      for (int e = 0; e < (KV8 ? 4 : 2); ++e)
                        if (!(fabsf(v[e]) <= 3.4028235e38f)) o[nt][KV8 ? 2 * q + (e >> 1) : jv * 4 + q][r + 2 * (e & 1)] += v[e];
                    }
                }
              }
#pragma unroll
              for (int i = 0; i < 4; ++i) {     // and out of the product
                unsigned x[4] = {vr[i].x, vr[i].y, vr[i].z, vr[i].w};
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
                vr[i] = make_uint4(x[0], x[1], x[2], x[3]);
              }
            }
          }
          // ---- O^T += V^T P^T: tiles of 16 channels ----
#pragma unroll
          for (int jj = 0; jj < (KV8 ? 8 : 4); ++jj) {
            const int j = KV8 ? jj : jv * 4 + jj;
            unsigned af[4];
            if constexpr (KV8) {
              const unsigned sel = (jj & 1) ? 0x7362u : 0x5140u;
              pd_cvt4(__byte_perm(pd_word(vr[0], jj >> 1), pd_word(vr[1], jj >> 1), sel), af[0], af[1]);
              pd_cvt4(__byte_perm(pd_word(vr[2], jj >> 1), pd_word(vr[3], jj >> 1), sel), af[2], af[3]);
            } else {
              const unsigned w0 = pd_word(vr[0], jj), w1 = pd_word(vr[1], jj), w2 = pd_word(vr[2], jj), w3 = pd_word(vr[3], jj);
              af[0] = __byte_perm(w0, w1, 0x5410); af[1] = __byte_perm(w0, w1, 0x7632);
              af[2] = __byte_perm(w2, w3, 0x5410); af[3] = __byte_perm(w2, w3, 0x7632);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              // fp32 queries: the matrix unit cuts its sums off, always towards zero, and over thousands of keys that adds up (110 K keys: 2.2e-6 of the
              // result, 4.8e-7 with a sum of each step's own and rounded additions; up to 5 % of the time)
              if constexpr (QT > 1) {
                float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int t = PT - 1; t >= 0; --t) pd_mma<KV8>(x, af, ph[kg][nt][t][0], ph[kg][nt][t][1]);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[nt][j][e] += x[e];
              } else {
#pragma unroll
                for (int t = 0; t < PT; ++t) pd_mma<KV8>(o[nt][j], af, ph[kg][nt][t][0], ph[kg][nt][t][1]);
              }
            }
          }
        }
      }
    }
    pd_wait<0>();
    __syncthreads();                           // every warp is done with its steps: their place takes the results

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
        if (g == 0) { m_s[warp][row] = mo[nt][r] == PD_NONE ? -INFINITY : OFF - mo[nt][r]; l_s[warp][row] = t; }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int ch = KV8 ? g * 16 + 2 * j : (j >> 2) * 64 + g * 8 + (j & 3) * 2;
          *reinterpret_cast<float2*>(&o_s[warp][row][ch]) = make_float2(o[nt][j][r], o[nt][j][r + 2]);
        }
      }
    __syncthreads();
    const bool whole = n_units == w.units;
    float* rec = reinterpret_cast<float*>(a.scratch) + (static_cast<size_t>(blockIdx.x) * 2 + (u == u_first ? 0 : 1)) * RT * PD_REC;
#pragma unroll
    for (int x = 0; x < RT / PD_WARPS; ++x) {   // a warp per row, four channels per lane
      const int row = x * PD_WARPS + warp, i = (row0 + row) / G;
      if (whole && i >= s.n) break;
      const float M = fmaxf(fmaxf(m_s[0][row], m_s[1][row]), fmaxf(m_s[2][row], m_s[3][row]));
      float L = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int y = 0; y < PD_WARPS; ++y) {      // M = -inf: nothing seen, or nothing but NaN
        const float f = M == -INFINITY ? 1.f : (m_s[y][row] == -INFINITY ? 0.f : pd_ex2(m_s[y][row] - M));
        L += f * l_s[y][row];
        if (f == 0.f) continue;
        const float4 v = *reinterpret_cast<const float4*>(&o_s[y][row][lane * 4]);
        acc.x += f * v.x; acc.y += f * v.y; acc.z += f * v.z; acc.w += f * v.w;
      }
      if (whole) {
        const int hd = kvh * G + (row0 + row) % G;
        const float inv = L == 0.f ? 0.f : 1.f / L;
        pd_store4(a, s.t0 + i, hd, lane * 4, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
        if (lane == 0 && a.lse != nullptr) a.lse[static_cast<size_t>(s.t0 + i) * a.nq + hd] = pd_lse<KV8>(M, L);
      } else {
        *reinterpret_cast<float4*>(rec + row * PD_REC + lane * 4) = acc;
        if (lane == 0) *reinterpret_cast<float2*>(rec + row * PD_REC + PG_HD) = make_float2(M, L);
      }
    }
    __syncthreads();
    u += taken;
  }
}

// Folds the records of the items that a range end cut. Block (item, group of rows); WPR warps share the pieces of a row, a lane
// holds four channels. All that depends on lengths alone is worked out while the main kernel still runs.
template <bool KV8, int WPR>
__global__ void __launch_bounds__(WPR == 1 ? 128 : WPR * 32) paged_fold_kernel(const __grid_constant__ IhbPagedAttn a, int grid, int RT) {
  __shared__ __align__(16) float red[WPR][PG_HD + 4];
  const IhbPaged& c = a.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = a.nq / c.nkv;
  // the item of this block: sequences in order, their items in order
  int left = blockIdx.x, b = -1;
  long long lo = 0, total = 0;
  for (int b0 = 0; b0 < c.B; b0 += 32) {
    PdWork w = {0, 0, 0, 0};
    if (b0 + lane < c.B) w = pd_work(c, pg_seq(c, b0 + lane), G, RT);
    const long long run = warp_incl_scan_ll(w.total, lane);
    if (b < 0) {
      const int incl = warp_incl_scan(w.items, lane);
      const unsigned hit = __ballot_sync(0xffffffffu, incl > left);
      if (hit) {
        const int src = __ffs(hit) - 1;
        b = b0 + src;
        left -= __shfl_sync(0xffffffffu, incl - w.items, src);
        lo = total + __shfl_sync(0xffffffffu, run - w.total, src);
      } else {
        left -= __shfl_sync(0xffffffffu, incl, 31);
      }
    }
    total += __shfl_sync(0xffffffffu, run, 31);
  }
  int first = 0, last = 0, row0 = 0, kvh = 0;
  size_t slot0 = 0;
  PgSeq s = {0, 0, 0, 0};
  if (b >= 0) {
    s = pg_seq(c, b);
    const PdWork w = pd_work(c, s, G, RT);
    lo += static_cast<long long>(left) * (w.units + PD_START);
    const long long hi = lo + w.units + PD_START, key0 = lo + PD_START;
    const PdCuts cuts(total, pd_parts(total, grid));
    first = cuts.of(key0);                                     // the range that holds the item's first unit
    last = cuts.of(hi - 1);                                    // the range that holds its last unit
    kvh = left / w.tiles;
    row0 = (left % w.tiles) * RT;
    slot0 = cuts.at(first) >= lo ? 0 : 1;         // the first piece is its range's last segment: slot 1, or 0 if the only one
  }
  pdl_wait();
  if (b < 0 || first == last) return;                          // one range had all of it and has written the result
  const int row = WPR == 1 ? blockIdx.y * 4 + warp : blockIdx.y, i = (row0 + row) / G;
  if (row >= RT || i >= s.n) return;
  const float* r0 = reinterpret_cast<const float*>(a.scratch) + ((static_cast<size_t>(first) * 2 + slot0) * RT + row) * PD_REC;
  const float* r1 = reinterpret_cast<const float*>(a.scratch) + (static_cast<size_t>(first) * 2 * RT + row) * PD_REC;   // slot 0 of the others
  const size_t step = static_cast<size_t>(2) * RT * PD_REC;
  const int n = last - first + 1;
  float M = -INFINITY;
  for (int x = lane; x < n; x += 32) M = fmaxf(M, (x == 0 ? r0 : r1 + x * step)[PG_HD]);
  M = warp_max(M);
  float L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int x = WPR == 1 ? 0 : warp; x < n; x += WPR) {
    const float* r = x == 0 ? r0 : r1 + x * step;
    const float2 ml = *reinterpret_cast<const float2*>(r + PG_HD);
    const float4 v = *reinterpret_cast<const float4*>(r + lane * 4);
    const float f = M == -INFINITY ? 1.f : (ml.x == -INFINITY ? 0.f : pd_ex2(ml.x - M));      // M = -inf: nothing seen, or only NaN
    L += f * ml.y;
    if (f != 0.f) { acc.x += f * v.x; acc.y += f * v.y; acc.z += f * v.z; acc.w += f * v.w; }
  }
  if (WPR > 1) {
    *reinterpret_cast<float4*>(&red[warp][lane * 4]) = acc;
    if (lane == 0) red[warp][PG_HD] = L;
    __syncthreads();
    if (warp) return;
#pragma unroll
    for (int x = 1; x < WPR; ++x) {
      const float4 v = *reinterpret_cast<const float4*>(&red[x][lane * 4]);
      acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
      L += red[x][PG_HD];
    }
  }
  const int hd = kvh * G + (row0 + row) % G;
  const float inv = L == 0.f ? 0.f : 1.f / L;
  pd_store4(a, s.t0 + i, hd, lane * 4, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
  if (lane == 0 && a.lse != nullptr) a.lse[static_cast<size_t>(s.t0 + i) * a.nq + hd] = pd_lse<KV8>(M, L);
}

struct PdPlan {
  int nt, per_sm, grid;
};
static PdPlan pd_plan(const IhbPagedAttn& a) {
  PdPlan p;
  const int G = a.nq / a.c.nkv;
  p.nt = static_cast<long long>(a.max_q) * G <= 8 ? 1 : 2;
  p.per_sm = p.nt == 2 && !a.q_bf16 ? 2 : 3;       // what is resident at once (PdSmem::PER_SM)
  p.grid = 148 * p.per_sm;
  return p;
}

template <int NT, bool KV8, int QT, int PT>
static cudaError_t pd_launch(const IhbPagedAttn& a, const PdPlan& p, cudaStream_t stream) {
  using SM = PdSmem<NT, KV8, QT>;
  cudaError_t e = cudaFuncSetAttribute(paged_rows_kernel<NT, KV8, QT, PT>, cudaFuncAttributeMaxDynamicSharedMemorySize, SM::BYTES);
  if (e != cudaSuccess) return e;
  paged_rows_kernel<NT, KV8, QT, PT><<<p.grid, PD_WARPS * 32, SM::BYTES, stream>>>(a, p.grid);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int G = a.nq / a.c.nkv, RT = 8 * NT;
  // items of the batch at most: by the longest window, and by the tokens of the call (a caller's bound of the window may be far above)
  const long long by_q = static_cast<long long>(a.c.B) * ((static_cast<long long>(a.max_q) * G + RT - 1) / RT);
  const long long by_t = static_cast<long long>(a.c.T) * G / RT + a.c.B;
  const long long items = (by_q < by_t ? by_q : by_t) * a.c.nkv;
  if (items > 0x7fffffffll) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  // few items: many pieces each, eight warps share a row's; many items: two or three pieces each, a warp takes a row
  const bool wide = items * 8 <= p.grid;
  cfg.gridDim = dim3(static_cast<unsigned>(items), wide ? RT : RT / 4);
  cfg.blockDim = dim3(wide ? 256 : 128);
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return wide ? cudaLaunchKernelEx(&cfg, paged_fold_kernel<KV8, 8>, a, p.grid, RT) : cudaLaunchKernelEx(&cfg, paged_fold_kernel<KV8, 1>, a, p.grid, RT);
}

}  // namespace ihb

using namespace ihb;

static bool paged_attn_ok(const IhbPagedAttn& a) {
  return paged_ok(a.c) && a.nq > 0 && a.nq % a.c.nkv == 0 && a.nq / a.c.nkv <= 256 &&
         a.q != nullptr && a.out != nullptr && a.max_q > 0 && (a.mask == nullptr || (a.mask_stride >= 0 && a.mask_cols >= 1)) &&
         a.q_stride_t % 8 == 0 && a.q_stride_h % 8 == 0;
}

// Which kernel. The tiles of paged_tiles.cu cost the same from 1 to 128 rows ((token, head) pairs of a sequence) and some 13 us more to
// start; here each 16 rows read the keys again. Measured, 32 / 4 heads, us here / there:
//   32 sequences of 2048 keys  32 rows 40 / 54 (bf16 pages 52 / 64)   64: 68 / 55 (89 / 65)   128: 121 / 58 (165 / 66)
//    8 sequences of 4096       32: 27 / 45 (33 / 47)                  64: 38 / 41 (49 / 49)   128:  61 / 43 ( 81 / 52)
//    1 sequence of 8192        32: 19 / 47 (21 / 45)                  64: 20 / 48 (23 / 46)   128:  26 / 50 ( 31 / 47)
//    4 sequences of 32768      32: 58 / 82 (101 / 104)                64: 99 / 84 (144 / 106) 128: 182 / 87 (291 / 108)
// so up to 32 rows they stay here, above 128 they go there, and between it is where the lines cross: with t sixteens of rows and W keys
// of all heads, 50 t W us a million here (bf16 pages 80), 180 W + 10 there (fitted to earlier times of the tiles: they are 5 to 15 % faster now over
// e4m3 pages, some windows are on the slower side of it). The lengths are on the device: W comes from the table's width,
// and a table much wider than its sequences gets the tiles earlier than it need: that costs time, not bits (over bf16 pages both keep two terms of P, over
// e4m3 pages P is fp16 in both). fp32 queries always stay: their precision has no tile form.
static bool use_tiles(const IhbPagedAttn& a) {
  const long long rows = static_cast<long long>(a.max_q) * (a.nq / a.c.nkv);
  if (!a.q_bf16 || rows <= 32) return false;
  if (rows > 128) return true;
  const double t = static_cast<double>((rows + 15) / 16), w = 1e-6 * a.c.B * a.c.nkv * a.c.max_blocks * a.c.page;
  return ((a.c.k_scale != nullptr ? 50. : 80.) * t - 180.) * w > 10.;
}

extern "C" size_t ihb_paged_attention_scratch(const IhbPagedAttn* a) {
  if (a->c.nkv < 1 || a->nq % a->c.nkv) return 0;
  if (use_tiles(*a)) return paged_tiles_scratch(*a);
  const PdPlan p = pd_plan(*a);
  return static_cast<size_t>(p.grid) * 2 * 8 * p.nt * PD_REC * sizeof(float);
}

extern "C" int ihb_paged_attention(const IhbPagedAttn* p, cudaStream_t stream) {
  const IhbPagedAttn& a = *p;
  if (!paged_attn_ok(a) || a.scratch == nullptr) return cudaErrorInvalidValue;
  if (use_tiles(a)) return paged_tiles_launch(a, stream);
  const PdPlan pl = pd_plan(a);
  const bool kv8 = a.c.k_scale != nullptr, f32 = !a.q_bf16;
  // terms of q / of the probabilities. e4m3 pages (fp16 products): bf16 queries are exact in one, fp32 ones take two (22 bits);
  // bf16 pages: probabilities in one term would be off by 2^-9, in two by 2^-17; fp32 in and out takes three of both
  if (pl.nt == 1) {
    if (kv8) return f32 ? pd_launch<1, true, 2, 2>(a, pl, stream) : pd_launch<1, true, 1, 1>(a, pl, stream);
    return f32 ? pd_launch<1, false, 3, 3>(a, pl, stream) : pd_launch<1, false, 1, 2>(a, pl, stream);
  }
  if (kv8) return f32 ? pd_launch<2, true, 2, 2>(a, pl, stream) : pd_launch<2, true, 1, 1>(a, pl, stream);
  return f32 ? pd_launch<2, false, 3, 3>(a, pl, stream) : pd_launch<2, false, 1, 2>(a, pl, stream);
}
