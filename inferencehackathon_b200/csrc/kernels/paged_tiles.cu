// Attention of prompt chunks and longer verify windows over a paged KV cache on the 5th-generation tensor cores (tcgen05, tensor
// memory), head_dim 128, bf16 pages or e4m3 pages with one scale per (page, head). paged_attn.cu has the single-token side, the
// formulas with the page scales and the C entry point.
//
// A CTA takes up to 256 rows ((token, query head) pairs of one sequence and KV head) as two tiles of 128 and walks key blocks of 128:
//   warps 0-3, 4-7   one softmax group per tile, a thread per row: scores from tensor memory, running maximum and sum in registers,
//                    probabilities (16 bits) back into tensor memory in the place of the scores
//   warps 8-11       loader: page lookups, 16-byte loads one block ahead in registers, e4m3 -> fp16, swizzled tiles in shared memory
//   warp 12          issues S = Q K^T (both operands in shared memory) and O += P V (P in tensor memory, V as an MN-major operand: the
//                    rows of the cache are used as they lie, no transpose)
// While one group computes its softmax the tensor cores work for the other. A sequence with at most 128 rows gives both groups the
// same rows: they take the even and the odd key blocks, and their results are added up at the end.
// The accumulators are rescaled only when a row's maximum has grown by more than 2^8 since the last time.
//
// Work split as in paged_attn.cu: items (sequence, KV head, pair of tiles) are laid end to end, with lengths that follow their causal
// key ranges, and cut into one equal range per SM; pieces of a cut item are folded by a second kernel.
#include "paged.cuh"
#include "paged_tiles.h"
#include "tc_common.cuh"

namespace ihb {

constexpr int PT_M = 128, PT_KB = 128;
constexpr int PT_THREADS = 512;
// Registers: 512 threads start with 128 each (all of the SM's); the loader and the issuer's group give theirs to the softmax groups, which
// then hold a row's 128 scores: 256 x 184 + 128 x 72 + 128 x 72 = 512 x 128.
constexpr int PT_REGS = 128, PT_REGS_SOFTMAX = 184, PT_REGS_LOAD = 72, PT_REGS_MMA = 72;
static_assert(256 * PT_REGS_SOFTMAX + 128 * PT_REGS_LOAD + 128 * PT_REGS_MMA <= PT_THREADS * PT_REGS, "more registers than the block has");
constexpr int PT_MMA_WARP = 12;
constexpr int PT_HALF = 16384;                 // 128 rows x 128 bytes: one swizzled half (64 channels) of a tile
constexpr int PT_TILE = 2 * PT_HALF;
constexpr int PT_HDR = 2048;                // barriers; m and l of the second group at 1024 and 1536
constexpr int PT_RAW = 128 * PG_HD;             // e4m3 bytes of a key block's K or V
template <bool KV8>
constexpr int pt_smem() { return 1024 + PT_HDR + 6 * PT_TILE + (KV8 ? 2 * PT_RAW : 0); }
constexpr int PT_MAX_GRID = 148;              // one CTA per SM
constexpr int PT_START = 256;                  // start-up cost of an item, in keys

constexpr int PT_SEGS = 4;
// A piece of an item: rows [row0, row0 + rows) of a sequence's KV head, key blocks [blk0, blk1) of nblk.
struct PtSeg {
  int b, kvh, row0, rows, blk0, blk1, nblk, first_in_range;
  int seen_end;                                // keys that any of the rows sees lie below it
  PgSeq s;
  int last;                                    // no segment: the end
};

struct PtHdr {
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t q_full[2], q_free, s_full[2], p_ready[2], pv_done[2], hand[2];
  uint32_t tmem;
  int abort_flag;
  int odd;                                     // V rows of the call's own tokens that are not finite were seen (set by the loader)
  uint64_t seg_full[PT_SEGS], seg_free[PT_SEGS];
  PtSeg seg[PT_SEGS];
};

// ---- work items ----------------------------------------------------------------------------------------------------------------
// Tile pair j of a sequence has the virtual length a + d * (j + 1): an arithmetic progression, so that positions are found in closed
// form; it is mapped onto the pair's key blocks proportionally.
struct PtWork {
  int tiles;
  long long a, d, head;                        // head: virtual length of one KV head's pairs
};
__device__ __forceinline__ PtWork pt_work(const IhbPagedAttn& p, const PgSeq& s, int G, int RT) {
  PtWork w;
  w.tiles = s.len > 0 ? (s.n * G + RT - 1) / RT : 0;
  if (p.mask != nullptr) {
    w.a = static_cast<long long>(s.len + PT_START) * G;
    w.d = 0;
  } else {
    w.a = static_cast<long long>(max(s.base, 0) + PT_START) * G;
    w.d = RT;
  }
  const long long t = w.tiles;
  w.head = t * w.a + w.d * (t * (t + 1) / 2);
  return w;
}
__device__ __forceinline__ long long pt_prefix(const PtWork& w, long long j) { return j * w.a + w.d * (j * (j + 1) / 2); }

// The segments of a CTA's range, in order.
struct PtIter {
  long long u, u_end, u0, before;
  int b;
  PgSeq s;
  PtWork w;
  __device__ __forceinline__ void start(const IhbPagedAttn& p, int G, int RT, long long total, long long before_, int b_, int grid) {
    u0 = u = total * blockIdx.x / grid;
    u_end = total * (blockIdx.x + 1) / grid;
    before = before_;
    b = b_;
    if (u < u_end) {
      s = pg_seq(p.c, b);
      w = pt_work(p, s, G, RT);
    }
  }
  // false at the end. A segment without a key block is only reported in the middle of an item (for the descriptor).
  __device__ __forceinline__ bool next(const IhbPagedAttn& p, int G, int RT, PtSeg& g) {
    while (u < u_end) {
      long long all = w.head * p.c.nkv;
      while (u - before >= all) {
        before += all;
        ++b;
        s = pg_seq(p.c, b);
        w = pt_work(p, s, G, RT);
        all = w.head * p.c.nkv;
      }
      const long long q = (u - before) % w.head;
      g.kvh = static_cast<int>((u - before) / w.head);
      long long j;
      if (w.d == 0) {
        j = q / w.a;
      } else {
        const double h = static_cast<double>(w.a) + 0.5 * static_cast<double>(w.d);
        j = static_cast<long long>((sqrt(h * h + 2.0 * static_cast<double>(w.d) * static_cast<double>(q)) - h) / static_cast<double>(w.d));
        j = min(max(j, 0ll), static_cast<long long>(w.tiles - 1));
        while (j > 0 && pt_prefix(w, j) > q) --j;
        while (j + 1 < w.tiles && pt_prefix(w, j + 1) <= q) ++j;
      }
      const long long lo = pt_prefix(w, j), len = w.a + w.d * (j + 1);
      const long long v0 = q - lo, v1 = min(len, v0 + (u_end - u));
      g.b = b;
      g.s = s;
      g.last = 0;
      g.row0 = static_cast<int>(j) * RT;
      g.rows = min(RT, s.n * G - g.row0);
      const int i_last = (g.row0 + g.rows - 1) / G;
      g.seen_end = p.mask != nullptr ? s.len : min(s.len, s.base + i_last + 1);
      g.nblk = max(1, (g.seen_end + PT_KB - 1) / PT_KB);
      g.blk0 = static_cast<int>(v0 * g.nblk / len);
      g.blk1 = static_cast<int>(v1 * g.nblk / len);
      g.first_in_range = u == u0;
      u += v1 - v0;
      if (g.blk0 < g.blk1 || g.blk0 > 0) return true;
    }
    return false;
  }
};

// What a CTA tells the folding kernel. cont: the CTA's first segment continues an item of the CTA before (1: without a block of its
// own, 2: with a piece in slot 0), ends: and ends it. tail: the CTA's last segment is the first piece of a cut item, in slot `slot`.
struct PtDesc {
  int cont, ends, tail, slot;
  int b, kvh, row0, rows;
};

__device__ __forceinline__ void pt_ld32(uint32_t t, float (&v)[32]) {
  uint32_t r[32];
  __syncwarp();                                // the lanes may come from a wait or a branch: the instruction wants them together
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,"
      "%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(t)
      : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
// Four of them in flight: pt_ld32_issue x 4, pt_wait_ld, pt_pin x 4 (ties the registers' first use to the wait).
__device__ __forceinline__ void pt_ld32_issue(uint32_t t, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,"
      "%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]),
        "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]),
        "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(t)
      : "memory");
}
__device__ __forceinline__ void pt_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pt_pin(float* v) {
  asm volatile(""
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]),
                 "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]),
                 "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]),
                 "+f"(v[31])
               :
               : "memory");
}
__device__ __forceinline__ void pt_st32(uint32_t t, const float (&v)[32]) {
  __syncwarp();
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
      "%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(t),
      "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]), "f"(v[11]),
      "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]), "f"(v[16]), "f"(v[17]), "f"(v[18]), "f"(v[19]), "f"(v[20]), "f"(v[21]), "f"(v[22]),
      "f"(v[23]), "f"(v[24]), "f"(v[25]), "f"(v[26]), "f"(v[27]), "f"(v[28]), "f"(v[29]), "f"(v[30]), "f"(v[31])
      : "memory");
}
__device__ __forceinline__ void pt_st16(uint32_t t, const unsigned (&v)[16]) {
  __syncwarp();
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(t), "r"(v[0]), "r"(v[1]),
      "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]),
      "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void pt_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void pt_regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void pt_regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
// D[tmem] += A[tmem] * B[shared]
__device__ __forceinline__ void pt_mma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(bdesc), "r"(idesc), "r"(acc)
      : "memory");
}
// Shared-memory descriptor of an MN-major operand, 128-byte swizzle: rows of 64 MN elements (128 bytes), one per K; the next 64 MN
// elements PT_HALF bytes on (leading offset), groups of 8 K 1024 bytes apart (stride offset).
__device__ __forceinline__ uint64_t pt_desc_mn(const void* tile) {
  uint64_t d = (static_cast<uint64_t>(smem_u32(tile)) >> 4) & 0x3FFFull;
  d |= static_cast<uint64_t>(PT_HALF >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= 1ull << 46;
  d |= 2ull << 61;
  return d;
}
// offset of a 16-byte chunk (8 channels) of row r in a swizzled tile
__device__ __forceinline__ int pt_at(int r, int ch) { return (ch >> 3) * PT_HALF + r * 128 + (((ch & 7) ^ (r & 7)) << 4); }

// Shared memory by 32-bit address: the aligned base is a computed pointer, which the compiler would access as generic memory.
__device__ __forceinline__ uint4 pt_lds(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ void pt_sts(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// Does a row see key p? vis: keys below it are seen; mrow: the row's mask over the call's tokens, or NULL.
__device__ __forceinline__ bool pt_sees(const IhbPagedAttn& a, const PgSeq& s, const unsigned char* mrow, int vis, int p) {
  if (p < vis) return true;
  return mrow != nullptr && p < s.len && p - s.base < a.mask_stride && mrow[p - s.base] != 0;
}
// One element of V as a float, for the rare correction of values that are not finite.
template <bool KV8>
__device__ __forceinline__ float pt_v_at(const IhbPaged& c, size_t row, int ch) {
  if constexpr (KV8) {
    const __half2 h = cvt_e4m3x2(reinterpret_cast<const uint8_t*>(c.v)[row * PG_HD + ch]);
    return __low2float(h);
  } else {
    return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(c.v)[row * PG_HD + ch]);
  }
}

template <bool KV8>
__global__ void __launch_bounds__(PT_THREADS, 1) paged_tiles_kernel(const __grid_constant__ IhbPagedAttn a, int grid, int rec_rows) {
  extern __shared__ uint8_t pt_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pt_raw) + 1023) & ~uintptr_t(1023));
  PtHdr& sh = *reinterpret_cast<PtHdr*>(smem);
  uint8_t* sq = smem + PT_HDR;
  uint8_t* sk = sq + 2 * PT_TILE;
  uint8_t* sv = sk + 2 * PT_TILE;
  uint8_t* raw = sv + 2 * PT_TILE;             // e4m3 pages: two batches of bytes on their way to the tiles
  constexpr int RT = 2 * PT_M;
  const IhbPaged& c = a.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = a.nq / c.nkv, psh = __ffs(c.page) - 1;
  PtDesc* descs = reinterpret_cast<PtDesc*>(a.scratch);
  float* recs = reinterpret_cast<float*>(reinterpret_cast<char*>(a.scratch) + PT_MAX_GRID * sizeof(PtDesc));
  pdl_launch_dependents();

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.k_full[i], 128); mbar_init(&sh.k_empty[i], 1);
      mbar_init(&sh.v_full[i], 128); mbar_init(&sh.v_empty[i], 1);
      mbar_init(&sh.q_full[i], 128); mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_ready[i], 128); mbar_init(&sh.pv_done[i], 1);
    }
    mbar_init(&sh.q_free, 1);
    mbar_init(&sh.hand[0], 128);
    mbar_init(&sh.hand[1], 128);
    for (int i = 0; i < PT_SEGS; ++i) { mbar_init(&sh.seg_full[i], 1); mbar_init(&sh.seg_free[i], 13); }
    sh.abort_flag = 0;
    sh.odd = 0;
    fence_mbar_init();
  }
  if (warp == PT_MMA_WARP) tmem_alloc(&sh.tmem, 512);
  // entries without a cached row: zeros
  for (int b = blockIdx.x; b < c.B; b += grid) {
    const PgSeq s = pg_seq(c, b);
    if (s.n > a.max_q && tid == 0) set_error(c.err, ERR_BAD_ARGS);
    if (s.len > 0) continue;
    for (int i = warp; i < s.n * a.nq; i += PT_THREADS / 32) {
      const size_t o = static_cast<size_t>(s.t0 + i / a.nq) * a.out_stride_t + static_cast<size_t>(i % a.nq) * a.out_stride_h + lane * 4;
      if (a.out_bf16) *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(a.out) + o) = make_uint2(0, 0);
      else *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out) + o) = make_float4(0.f, 0.f, 0.f, 0.f);
      if (lane == 0 && a.lse != nullptr) a.lse[static_cast<size_t>(s.t0) * a.nq + i] = -INFINITY;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  volatile int* abort_flag = &sh.abort_flag;
  // The next segment: every role reads the scheduler's records in order, and gives a record back (free_seg) when done with it.
  unsigned n_seg = 0;
  auto next_seg = [&]() -> const PtSeg* {
    if (!tc_wait(&sh.seg_full[n_seg % PT_SEGS], (n_seg / PT_SEGS) & 1u, abort_flag, c.err, ERR_MBAR_FULL_TIMEOUT)) return nullptr;
    const PtSeg* g = &sh.seg[n_seg % PT_SEGS];
    return g->last ? nullptr : g;
  };
  bool ok = true;

  if (warp < 8) {
    pt_regs_inc<PT_REGS_SOFTMAX>();
    // =============================== softmax groups ===============================================================================
    const int wg = warp >> 2, quarter = warp & 3, r_tile = quarter * 32 + lane;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t t_s = lane_base + wg * 128, t_o = lane_base + 256 + wg * 128;
    constexpr float OFF = KV8 ? PD_OFF : 0.f;
    unsigned n_blk = 0, n_hand = 0;            // blocks this group has been through, segments that both groups shared: barrier phases
    while (const PtSeg* gp = next_seg()) {
      const PtSeg& sg = *gp;
      const PgSeq& s = sg.s;
      const bool pair = sg.rows > PT_M;        // two tiles; else both groups have the same rows and every other key block
      const bool whole = sg.blk0 == 0 && sg.blk1 == sg.nblk;
      const int r = (pair ? wg * PT_M : 0) + r_tile;                    // row of the item
      const bool live = r < sg.rows;
      const int tok = live ? (sg.row0 + r) / G : 0, head = sg.kvh * G + (live ? (sg.row0 + r) % G : 0);
      const int vis = !live ? max(sg.seen_end, 0) : (a.mask != nullptr ? max(s.base, 0) : min(max(s.base + tok + 1, 0), s.len));   // keys [0, vis) are seen
      const unsigned char* mrow = a.mask != nullptr && live ? a.mask + static_cast<size_t>(s.t0 + tok) * a.mask_stride : nullptr;
      const int* table = c.block_table + static_cast<size_t>(sg.b) * c.table_stride;
      // ---- Q: one row per thread ----
      float rowf = a.scale * PG_LOG2E;
      if (ok && n_seg > 0) ok = tc_wait(&sh.q_free, (n_seg - 1) & 1u, abort_flag, c.err, ERR_TMEM_TIMEOUT);
      if (ok && n_hand > 0) ok = tc_wait(&sh.hand[1], (n_hand - 1) & 1u, abort_flag, c.err, ERR_TMEM_TIMEOUT);
      {
        const uint32_t dst = smem_u32(sq) + wg * PT_TILE;
        const size_t off = static_cast<size_t>(s.t0 + tok) * a.q_stride_t + static_cast<size_t>(head) * a.q_stride_h;
        uint4 v[16];
#pragma unroll
        for (int ch = 0; ch < 16; ++ch) {
          v[ch] = make_uint4(0, 0, 0, 0);
          if (live) v[ch] = *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(a.q) + off + ch * 8);
        }
        if constexpr (KV8) {                   // |q| of the row into [1, 2): a power of two, exact
          float mx = 0.f;
#pragma unroll
          for (int ch = 0; ch < 16; ++ch) {
            const unsigned x[4] = {v[ch].x, v[ch].y, v[ch].z, v[ch].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(x[e] << 16)), fabsf(__uint_as_float(x[e] & 0xffff0000u))));
          }
          const int e2 = min(max(static_cast<int>(__float_as_uint(mx) >> 23) - 127, -100), 100);
          rowf *= __uint_as_float(static_cast<unsigned>(127 + e2) << 23);
          const float inv = __uint_as_float(static_cast<unsigned>(127 - e2) << 23);
#pragma unroll
          for (int ch = 0; ch < 16; ++ch) {
            unsigned x[4] = {v[ch].x, v[ch].y, v[ch].z, v[ch].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = pd_pack<true>(__uint_as_float(x[e] << 16) * inv, __uint_as_float(x[e] & 0xffff0000u) * inv);
            v[ch] = make_uint4(x[0], x[1], x[2], x[3]);
          }
        }
#pragma unroll
        for (int ch = 0; ch < 16; ++ch) pt_sts(dst + pt_at(r_tile, ch), v[ch]);
        fence_proxy_async_smem();
        mbar_arrive(&sh.q_full[wg]);
      }
      // ---- page scales: lane i (0 .. 7) looks after the 16 keys i of a block, one block ahead ----
      const int step = pair ? 1 : 2;
      auto page_at = [&](int blk) -> int {
        const int key = blk * PT_KB + (lane & 7) * 16;
        return blk < sg.blk1 && key < sg.seen_end ? table[key >> psh] : 0;
      };
      auto scales_at = [&](int blk, int page, float& ks, float& vs) {
        const bool good = static_cast<unsigned>(page) < static_cast<unsigned>(c.n_pages);
        ks = good ? 1.f : -1.f;                // negative: not seen
        vs = 1.f;
        if (KV8 && good && blk < sg.blk1) {
          ks = fmaxf(c.k_scale[static_cast<size_t>(page) * c.nkv + sg.kvh], 1e-30f);      // (0 would turn a masked -inf into NaN)
          vs = c.v_scale[static_cast<size_t>(page) * c.nkv + sg.kvh];
        }
      };
      int blk = sg.blk0 + (pair ? 0 : wg);
      float ks_n, vs_n;
      scales_at(blk, page_at(blk), ks_n, vs_n);
      int page_n = page_at(blk + step);
      float m = -INFINITY, l = 0.f;
      bool have = false;                       // O holds something
      for (; blk < sg.blk1; blk += step) {
        const float ks_raw = ks_n, ev_l = KV8 ? pd_log2_scale(vs_n) : 0.f;          // of the lane's 16 keys
        scales_at(blk + step, page_n, ks_n, vs_n);
        page_n = page_at(blk + 2 * step);
        const int key0 = blk * PT_KB;
        const bool bad = __any_sync(0xffffffffu, ks_raw < 0.f);
        if (bad && lane == 0) set_error(c.err, ERR_BAD_ARGS);
        const bool edge = __any_sync(0xffffffffu, key0 + PT_KB > vis) || bad;
        unsigned seen[4] = {~0u, ~0u, ~0u, ~0u};      // bit e of word q: the row sees key q * 32 + e of the block
        if (edge) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int kc = key0 + q * 32, n = min(max(vis - kc, 0), 32);
            unsigned w = n == 32 ? ~0u : (1u << n) - 1u;
            if (mrow != nullptr && n < 32)
              for (int e = n; e < 32; ++e)
                if (pt_sees(a, s, mrow, vis, kc + e)) w |= 1u << e;
            if (bad) {
              if (__shfl_sync(0xffffffffu, ks_raw, 2 * q) < 0.f) w &= 0xffff0000u;
              if (__shfl_sync(0xffffffffu, ks_raw, 2 * q + 1) < 0.f) w &= 0x0000ffffu;
            }
            seen[q] = w;
          }
        }
        if (ok) ok = tc_wait(&sh.s_full[wg], n_blk & 1u, abort_flag, c.err, ERR_TMEM_TIMEOUT);
        tc_fence_after();
        __syncwarp();
        float v[PT_KB];
#pragma unroll
        for (int q = 0; q < 4; ++q) pt_ld32_issue(t_s + q * 32, v + q * 32);
        pt_wait_ld();
#pragma unroll
        for (int q = 0; q < 4; ++q) pt_pin(v + q * 32);
        if (edge) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!(seen[q] & (1u << e))) v[q * 32 + e] = -INFINITY;
        }
        // ---- maximum ----
        float mx = -INFINITY, kf[8], ev[8];    // factor of the scores and log2 of the V scale, per 16 keys
#pragma unroll
        for (int h = 0; h < 8; ++h) {
          kf[h] = KV8 ? __shfl_sync(0xffffffffu, ks_raw, h) * rowf : rowf;
          ev[h] = KV8 ? __shfl_sync(0xffffffffu, ev_l, h) : 0.f;
          float x0 = v[h * 16], x1 = v[h * 16 + 1];
#pragma unroll
          for (int e = 2; e < 16; e += 2) { x0 = fmaxf(x0, v[h * 16 + e]); x1 = fmaxf(x1, v[h * 16 + e + 1]); }
          x0 = fmaxf(x0, x1);
          if (KV8) mx = fmaxf(mx, fmaf(x0, kf[h], ev[h]));
          else mx = fmaxf(mx, x0);
        }
        if (!KV8) mx *= rowf;
        // ---- rescale when the maximum has grown enough ----
        if (__any_sync(0xffffffffu, mx > m + PD_LAZY)) {
          const float mn = fmaxf(m, mx), f = m == -INFINITY ? 0.f : pd_ex2(m - mn);
          m = mn;
          l *= f;
          if (have) {
            if (ok) ok = tc_wait(&sh.pv_done[wg], (n_blk - 1) & 1u, abort_flag, c.err, ERR_TMEM_TIMEOUT);
            tc_fence_after();
#pragma unroll 1
            for (int q = 0; q < 8; ++q) {
              float x[16];
              __syncwarp();
              tmem_ld16(t_o + q * 16, x);
              unsigned y[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) y[e] = __float_as_uint(x[e] * f);
              pt_st16(t_o + q * 16, y);
            }
          }
        }
        have = true;
        // ---- probabilities, in the place of the scores ----
        const float mo = OFF - (m == -INFINITY ? 0.f : m);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          unsigned pk[16];
#pragma unroll
          for (int h = 2 * q; h < 2 * q + 2; ++h) {
            const float add = KV8 ? ev[h] + mo : mo;
            float s0 = 0.f, s1 = 0.f;
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              float& x0 = v[h * 16 + e];
              float& x1 = v[h * 16 + e + 1];
              x0 = pd_ex2(fmaf(x0, kf[h], add));        // a masked score stays -inf: its factor is positive
              x1 = pd_ex2(fmaf(x1, kf[h], add));
              s0 += x0;
              s1 += x1;
              pk[(h & 1) * 8 + e / 2] = pd_pack<KV8>(x0, x1);
            }
            l += KV8 ? (s0 + s1) * pd_ex2(-ev[h]) : s0 + s1;
          }
          pt_st16(t_s + q * 16, pk);
        }
        pt_wait_st();
        tc_fence_before();
        mbar_arrive(&sh.p_ready[wg]);
        ++n_blk;
      }
      // ---- the result ----
      if (have && ok) ok = tc_wait(&sh.pv_done[wg], (n_blk - 1) & 1u, abort_flag, c.err, ERR_TMEM_TIMEOUT);
      tc_fence_after();
      float f0 = 1.f, f1 = 0.f;
      const uint32_t xs = smem_u32(sq) + r_tile * 512;                   // the row's place
      if (!pair) {                             // the second group hands its result over through the place of Q, which no product reads now
        float* xm = reinterpret_cast<float*>(smem + 1024);
        float* xl = reinterpret_cast<float*>(smem + 1536);
        if (ok) ok = tc_wait(&sh.q_free, n_seg & 1u, abort_flag, c.err, ERR_TMEM_TIMEOUT);
        if (wg == 1) {
          xm[r_tile] = m;
          xl[r_tile] = l;
          if (have) {
#pragma unroll 1
            for (int q = 0; q < 4; ++q) {
              float v[32];
              pt_ld32(t_o + q * 32, v);
#pragma unroll
              for (int e = 0; e < 8; ++e)
                pt_sts(xs + (((q * 8 + e) ^ (lane & 7)) << 4), make_uint4(__float_as_uint(v[4 * e]), __float_as_uint(v[4 * e + 1]), __float_as_uint(v[4 * e + 2]), __float_as_uint(v[4 * e + 3])));
            }
          }
        }
        if (wg == 1) mbar_arrive(&sh.hand[0]);
        else if (ok) ok = tc_wait(&sh.hand[0], n_hand & 1u, abort_flag, c.err, ERR_TMEM_TIMEOUT);
        if (wg == 0 && sg.blk1 - sg.blk0 > 1) {
          const float m1 = xm[r_tile], M = fmaxf(m, m1);
          f0 = M == -INFINITY ? 1.f : (m == -INFINITY ? 0.f : pd_ex2(m - M));       // M = -inf: nothing seen, or nothing but NaN
          f1 = M == -INFINITY ? 1.f : (m1 == -INFINITY ? 0.f : pd_ex2(m1 - M));
          l = l * f0 + xl[r_tile] * f1;
          m = M;
        }
      }
      if (pair || wg == 0) {
        const bool odd = *reinterpret_cast<volatile int*>(&sh.odd) != 0;
        const int slot = sg.first_in_range ? 0 : 1;
        const float inv = whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
        float* rec = recs + ((static_cast<size_t>(blockIdx.x) * 2 + slot) * rec_rows + r) * PD_REC;
#pragma unroll 1
        for (int q = 0; q < 4; ++q) {
          float v[32];
          pt_ld32(t_o + q * 32, v);
          if (f1 != 0.f) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const uint4 x = pt_lds(xs + (((q * 8 + e) ^ (lane & 7)) << 4));
              v[4 * e] = v[4 * e] * f0 + __uint_as_float(x.x) * f1;
              v[4 * e + 1] = v[4 * e + 1] * f0 + __uint_as_float(x.y) * f1;
              v[4 * e + 2] = v[4 * e + 2] * f0 + __uint_as_float(x.z) * f1;
              v[4 * e + 3] = v[4 * e + 3] * f0 + __uint_as_float(x.w) * f1;
            }
          } else if (f0 != 1.f) {
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] *= f0;
          }
          if (odd && live)                     // values that are not finite, left out of the products: added where they are seen
            for (int key = max(max(s.base, 0), sg.blk0 * PT_KB); key < min(sg.seen_end, sg.blk1 * PT_KB); ++key) {
              const int pg = table[key >> psh];
              if (!pt_sees(a, s, mrow, vis, key) || static_cast<unsigned>(pg) >= static_cast<unsigned>(c.n_pages)) continue;
              const size_t row = (static_cast<size_t>(pg) * c.nkv + sg.kvh) * c.page + (key & (c.page - 1));
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                const float x = pt_v_at<KV8>(c, row, q * 32 + e);
                if (!(fabsf(x) <= 3.4028235e38f)) v[e] += x;
              }
            }
          if (live && whole) {
            const size_t o = static_cast<size_t>(s.t0 + tok) * a.out_stride_t + static_cast<size_t>(head) * a.out_stride_h + q * 32;
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] *= inv;
            if (a.out_bf16) {
#pragma unroll
              for (int e = 0; e < 8; ++e)      // (strides of out are multiples of four elements)
                *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(a.out) + o + 4 * e) =
                    make_uint2(pd_pack<false>(v[4 * e], v[4 * e + 1]), pd_pack<false>(v[4 * e + 2], v[4 * e + 3]));
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out) + o + 4 * e) = make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
            }
          } else if (live && r < rec_rows) {
#pragma unroll
            for (int e = 0; e < 8; ++e) *reinterpret_cast<float4*>(rec + q * 32 + 4 * e) = make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
          }
        }
        if (live && whole && a.lse != nullptr) a.lse[static_cast<size_t>(s.t0 + tok) * a.nq + head] = pd_lse<KV8>(m, l);
        if (live && !whole && r < rec_rows) *reinterpret_cast<float2*>(rec + PG_HD) = make_float2(m, l);
      }
      tc_fence_before();
      if (!pair) {
        if (wg == 0) mbar_arrive(&sh.hand[1]);                           // the place of Q is free again
        ++n_hand;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.seg_free[n_seg % PT_SEGS]);
      ++n_seg;
    }
  } else if (warp < PT_MMA_WARP) {
    pt_regs_dec<PT_REGS_LOAD>();
    // =============================== loader ===========================================================================================
    // Batches: K, V, K, V ... of the key blocks, copied 16 bytes at a time by cp.async (rows that nobody sees: zeros). A thread works
    // on the chunks that it copied itself, so a batch needs no barrier among the loader's threads. Two batches are under way:
    // e4m3 bytes land in `raw` and go from there, as fp16, into the tile; bf16 rows land in the tile.
    const int lt = tid - 256;
    constexpr int CPR = KV8 ? 8 : 16, N = KV8 ? 8 : 16, RSTEP = 128 / CPR;      // chunks per row, chunks per thread, rows between them
    const int lrow = lt / CPR, lch = lt % CPR;
    unsigned gk = 0;                           // blocks so far
    while (const PtSeg* gp = next_seg()) {
      const int blk0 = gp->blk0, nb = 2 * (gp->blk1 - blk0), seen_end = gp->seen_end, base = gp->s.base;
      const int* table = c.block_table + static_cast<size_t>(gp->b) * c.table_stride;
      const size_t head_off = static_cast<size_t>(gp->kvh) * c.page * (PG_HD * (KV8 ? 1 : 2)) + lch * 16;
      const unsigned page_bytes = static_cast<unsigned>(c.nkv * c.page) * (PG_HD * (KV8 ? 1 : 2));
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.seg_free[n_seg % PT_SEGS]);
      ++n_seg;
      // pages of the block's eight groups of 16 keys: looked up while the block before is on its way, -1: nobody sees them
      int page[8];
      auto lookup = [&](int blk) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int key = blk * PT_KB + i * 16;
          page[i] = key < seen_end ? __ldg(table + (key >> psh)) : -1;
        }
      };
      auto issue = [&](int n) {                // batch n of the segment
        const int blk = blk0 + (n >> 1);
        const char* src0 = reinterpret_cast<const char*>((n & 1) ? c.v : c.k) + head_off;
        const unsigned g = gk + (n >> 1);
        const uint32_t dst = smem_u32(KV8 ? raw + (n & 1) * PT_RAW + lt * 16 : ((n & 1) ? sv : sk) + (g & 1) * PT_TILE + pt_at(lrow, lch));
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int key = blk * PT_KB + lrow + i * RSTEP, pg = page[KV8 ? i : i >> 1];
          const bool good = key < seen_end && static_cast<unsigned>(pg) < static_cast<unsigned>(c.n_pages);
          const char* src = src0 + (good ? static_cast<size_t>(pg) * page_bytes + (key & (c.page - 1)) * (PG_HD * (KV8 ? 1 : 2)) : 0);
          // (RSTEP is 16 or 8 rows: the swizzle of a thread's rows is the same)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + i * (KV8 ? 2048 : RSTEP * 128)), "l"(src), "r"(good ? 16 : 0));
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        if ((n & 1) && n + 1 < nb) lookup(blk + 1);
      };
      // what is not finite in rows of the call's own tokens (not every row sees them) is taken out; true: there was something
      auto clean = [&](uint4& y) -> bool {
        unsigned x[4] = {y.x, y.y, y.z, y.w};
        bool bad = false;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if constexpr (KV8) bad |= (((x[q] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0u;
          else bad |= (x[q] & 0x7f80u) == 0x7f80u || (x[q] & 0x7f800000u) == 0x7f800000u;
        }
        if (!bad) return false;
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
        y = make_uint4(x[0], x[1], x[2], x[3]);
        return true;
      };
      auto wait_empty = [&](int n) {
        const unsigned g = gk + (n >> 1);
        if (g >= 2 && ok) ok = tc_wait((n & 1) ? &sh.v_empty[g & 1] : &sh.k_empty[g & 1], ((g >> 1) & 1u) ^ 1u, abort_flag, c.err, ERR_MBAR_EMPTY_TIMEOUT);
      };
      auto finish = [&](int n) {               // batch n has landed
        const int blk = blk0 + (n >> 1);
        const unsigned g = gk + (n >> 1);
        const uint32_t dst = smem_u32((n & 1) ? sv : sk) + (g & 1) * PT_TILE;
        const bool window = (n & 1) && blk * PT_KB + PT_KB > base;
        bool hit = false;
        if constexpr (KV8) {
          const uint32_t src = smem_u32(raw) + (n & 1) * PT_RAW + lt * 16;
          // 16 bytes are two chunks of eight fp16; the halves of a row start with different ones: the eight lanes of a phase then write
          // to different banks. The swizzle of a thread's rows (16 apart) is the same.
          const int swap = lch >> 2;
          const uint32_t d0 = dst + pt_at(lrow, 2 * lch + swap), d1 = dst + pt_at(lrow, 2 * lch + 1 - swap);
          uint4 x[N];
#pragma unroll
          for (int i = 0; i < N; ++i) x[i] = pt_lds(src + i * 2048);
          if (window)
#pragma unroll
            for (int i = 0; i < N; ++i)
              if (blk * PT_KB + lrow + i * RSTEP >= base) hit |= clean(x[i]);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            uint4 lo, hi;
            pd_cvt4(x[i].x, lo.x, lo.y);
            pd_cvt4(x[i].y, lo.z, lo.w);
            pd_cvt4(x[i].z, hi.x, hi.y);
            pd_cvt4(x[i].w, hi.z, hi.w);
            pt_sts(d0 + i * RSTEP * 128, swap ? hi : lo);
            pt_sts(d1 + i * RSTEP * 128, swap ? lo : hi);
          }
        } else if (window) {
          for (int i = 0; i < N; ++i) {
            const uint32_t p = dst + pt_at(lrow, lch) + i * RSTEP * 128;
            uint4 x = pt_lds(p);
            if (blk * PT_KB + lrow + i * RSTEP >= base && clean(x)) { pt_sts(p, x); hit = true; }
          }
        }
        if (hit) *reinterpret_cast<volatile int*>(&sh.odd) = 1;
        fence_proxy_async_smem();
        mbar_arrive((n & 1) ? &sh.v_full[g & 1] : &sh.k_full[g & 1]);
      };
      lookup(blk0);
      if constexpr (KV8) {
        issue(0);
        issue(1);
        for (int n = 0; n < nb; ++n) {
          if (n + 1 < nb) asm volatile("cp.async.wait_group 1;" ::: "memory");
          else asm volatile("cp.async.wait_group 0;" ::: "memory");
          wait_empty(n);
          finish(n);
          if (n + 2 < nb) issue(n + 2);
        }
      } else {
        for (int n = 0; n < nb; ++n) {
          wait_empty(n);
          issue(n);
          if (n > 0) {
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            finish(n - 1);
          }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        finish(nb - 1);
      }
      gk += nb >> 1;
    }
  } else {
    pt_regs_dec<PT_REGS_MMA>();
    if (warp == PT_MMA_WARP && lane == 0) {
    // =============================== MMA issuer =========================================================================================
    constexpr uint32_t idesc = (1u << 4) | (KV8 ? 0u : ((1u << 7) | (1u << 10))) | (static_cast<uint32_t>(PT_KB >> 3) << 17) | (static_cast<uint32_t>(PT_M >> 4) << 24);
    constexpr uint32_t idesc_v = idesc | (1u << 16);                   // V: MN-major
    auto qk = [&](int w, unsigned gk) {
      tc_fence_after();
#pragma unroll
      for (int k = 0; k < 8; ++k)
        tc_mma<1>(tmem + w * 128, smem_desc_sw128(sq + w * PT_TILE + (k >> 2) * PT_HALF) + 2 * (k & 3),
                  smem_desc_sw128(sk + (gk & 1) * PT_TILE + (k >> 2) * PT_HALF) + 2 * (k & 3), idesc, k > 0);
      tc_commit(&sh.s_full[w]);
    };
    auto pv = [&](int w, unsigned gk, bool first) {
      tc_fence_after();
#pragma unroll
      for (int k = 0; k < 8; ++k)
        pt_mma_ts(tmem + 256 + w * 128, tmem + w * 128 + k * 8, pt_desc_mn(sv + (gk & 1) * PT_TILE) + k * (2048 >> 4), idesc_v, !first || k > 0);
      tc_commit(&sh.pv_done[w]);
    };
    unsigned gk = 0, n_p[2] = {0, 0};
    auto full = [&](uint64_t* bar, unsigned g) { return tc_wait(&bar[g & 1], (g >> 1) & 1u, abort_flag, c.err, ERR_MBAR_FULL_TIMEOUT); };
    while (const PtSeg* gp = ok ? next_seg() : nullptr) {
      const PtSeg& sg = *gp;
      const int nb = sg.blk1 - sg.blk0, ahead = sg.rows > PT_M ? 1 : 2;   // pair: both groups take block j; else group j & 1 does
      ok = tc_wait(&sh.q_full[0], n_seg & 1u, abort_flag, c.err, ERR_MBAR_FULL_TIMEOUT) &&
           tc_wait(&sh.q_full[1], n_seg & 1u, abort_flag, c.err, ERR_MBAR_FULL_TIMEOUT);
      for (int j = 0; j < min(ahead, nb) && ok; ++j) {
        ok = full(sh.k_full, gk + j);
        if (!ok) break;
        qk(j, gk + j);
        if (ahead == 1) qk(1, gk + j);
        tc_commit(&sh.k_empty[(gk + j) & 1]);
      }
      for (int j = 0; j < nb && ok; ++j, ++gk) {
        ok = full(sh.v_full, gk);
        for (int w = ahead == 1 ? 0 : (j & 1); ok && w < (ahead == 1 ? 2 : (j & 1) + 1); ++w) {
          const bool last = ahead == 2 || w == 1;
          ok = tc_wait(&sh.p_ready[w], n_p[w] & 1u, abort_flag, c.err, ERR_TMEM_TIMEOUT);
          if (!ok) break;
          ++n_p[w];
          pv(w, gk, j < ahead);
          if (last) tc_commit(&sh.v_empty[gk & 1]);
          if (j + ahead < nb) {
            if (ahead == 2 || w == 0) ok = full(sh.k_full, gk + ahead);
            if (!ok) break;
            qk(w, gk + ahead);
            if (last) tc_commit(&sh.k_empty[(gk + ahead) & 1]);
          }
        }
      }
      tc_commit(&sh.q_free);
      mbar_arrive(&sh.seg_free[n_seg % PT_SEGS]);
      ++n_seg;
    }
    } else if (warp == PT_MMA_WARP + 1) {
      // =============================== scheduler ==========================================================================================
      long long total = 0;
      for (int b = lane; b < c.B; b += 32) total += pt_work(a, pg_seq(c, b), G, RT).head * c.nkv;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
      const long long u = total * blockIdx.x / grid;
      long long at = 0, before = 0;
      int found = 0;
      for (int b0 = 0; b0 < c.B; b0 += 32) {   // the sequence in which this CTA's range begins
        long long t = 0;
        if (b0 + lane < c.B) t = pt_work(a, pg_seq(c, b0 + lane), G, RT).head * c.nkv;
        long long incl = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const long long v = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, at + incl > u);
        if (hit) {
          const int src = __ffs(hit) - 1;
          before = at + __shfl_sync(0xffffffffu, incl - t, src);
          found = b0 + src;
          break;
        }
        at += __shfl_sync(0xffffffffu, incl, 31);
      }
      if (lane == 0) {
        PtDesc desc = {0, 0, 0, 0, 0, 0, 0, 0};
        PtIter it;
        it.start(a, G, RT, total, before, found, grid);
        for (bool more = true; more && ok;) {
          PtSeg g;
          g.last = 0;
          more = it.next(a, G, RT, g);
          if (more) {
            if (g.blk0 > 0) {
              desc.cont = g.blk0 < g.blk1 ? 2 : 1;
              desc.ends = g.blk1 == g.nblk;
            }
            if (g.blk0 == g.blk1) continue;
            if (g.blk0 == 0 && g.blk1 < g.nblk) {
              desc.tail = 1; desc.slot = g.first_in_range ? 0 : 1; desc.b = g.b; desc.kvh = g.kvh; desc.row0 = g.row0; desc.rows = g.rows;
            }
          } else {
            g.last = 1;
            descs[blockIdx.x] = desc;
          }
          const unsigned i = n_seg % PT_SEGS;
          if (n_seg >= PT_SEGS) ok = tc_wait(&sh.seg_free[i], ((n_seg / PT_SEGS) & 1u) ^ 1u, abort_flag, c.err, ERR_MBAR_EMPTY_TIMEOUT);
          sh.seg[i] = g;
          mbar_arrive(&sh.seg_full[i]);
          ++n_seg;
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == PT_MMA_WARP) tmem_dealloc(tmem, 512);
}

// Folds the pieces of the item whose first piece CTA blockIdx.x left: the later ones are those of the following CTAs, slot 0.
template <bool KV8>
__global__ void __launch_bounds__(256) paged_tiles_fold_kernel(const __grid_constant__ IhbPagedAttn a, int grid, int rec_rows) {
  __shared__ int list[PT_MAX_GRID];
  __shared__ int n_s;
  const PtDesc* descs = reinterpret_cast<const PtDesc*>(a.scratch);
  const float* recs = reinterpret_cast<const float*>(reinterpret_cast<const char*>(a.scratch) + PT_MAX_GRID * sizeof(PtDesc));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = a.nq / a.c.nkv;
  pdl_wait();
  const PtDesc d = descs[blockIdx.x];
  if (!d.tail) return;
  if (warp == 0) {
    int n = 1;
    if (lane == 0) list[0] = blockIdx.x * 2 + d.slot;
    for (int y0 = blockIdx.x + 1; y0 < grid; y0 += 32) {
      PtDesc e = {0, 0, 0, 0, 0, 0, 0, 0};
      if (y0 + lane < grid) e = descs[y0 + lane];
      const unsigned stop = __ballot_sync(0xffffffffu, e.ends || e.cont == 0);
      const int upto = stop ? __ffs(stop) - 1 : 31;                    // (this lane included: the piece that ends the item)
      const unsigned mine = __ballot_sync(0xffffffffu, lane <= upto && e.cont == 2);
      if (lane <= upto && e.cont == 2) list[n + __popc(mine & ((1u << lane) - 1u))] = (y0 + lane) * 2;
      n += __popc(mine);
      if (stop) break;
    }
    if (lane == 0) n_s = n;
  }
  __syncthreads();
  const int n = n_s;
  const PgSeq s = pg_seq(a.c, d.b);
  for (int r = blockIdx.y * 8 + warp; r < min(d.rows, rec_rows); r += gridDim.y * 8) {
    float M = -INFINITY;
    for (int x = lane; x < n; x += 32) M = fmaxf(M, recs[(static_cast<size_t>(list[x]) * rec_rows + r) * PD_REC + PG_HD]);
    M = warp_max(M);
    float L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int x = 0; x < n; ++x) {
      const float* q = recs + (static_cast<size_t>(list[x]) * rec_rows + r) * PD_REC;
      const float2 ml = *reinterpret_cast<const float2*>(q + PG_HD);
      const float4 v = *reinterpret_cast<const float4*>(q + lane * 4);
      const float f = M == -INFINITY ? 1.f : (ml.x == -INFINITY ? 0.f : pd_ex2(ml.x - M));
      L += f * ml.y;
      if (f != 0.f) { acc.x += f * v.x; acc.y += f * v.y; acc.z += f * v.z; acc.w += f * v.w; }
    }
    const int tok = (d.row0 + r) / G, head = d.kvh * G + (d.row0 + r) % G;
    const float inv = L == 0.f ? 0.f : 1.f / L;
    pd_store4(a, s.t0 + tok, head, lane * 4, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
    if (lane == 0 && a.lse != nullptr) a.lse[static_cast<size_t>(s.t0 + tok) * a.nq + head] = pd_lse<KV8>(M, L);
  }
}

static int pt_rec_rows(const IhbPagedAttn& a) {
  const long long rows = static_cast<long long>(a.max_q) * (a.nq / a.c.nkv);
  return rows < 2 * PT_M ? static_cast<int>(rows) : 2 * PT_M;
}

size_t paged_tiles_scratch(const IhbPagedAttn& a) {
  return PT_MAX_GRID * sizeof(PtDesc) + static_cast<size_t>(PT_MAX_GRID) * 2 * pt_rec_rows(a) * PD_REC * sizeof(float);
}

template <bool KV8>
static cudaError_t pt_launch(const IhbPagedAttn& a, cudaStream_t stream) {
  const int grid = PT_MAX_GRID, rec_rows = pt_rec_rows(a);             // one CTA per SM
  static const int regs = [] {                 // the register split draws on what the block is launched with
    cudaFuncAttributes f;
    return cudaFuncGetAttributes(&f, paged_tiles_kernel<KV8>) == cudaSuccess ? f.numRegs : 0;
  }();
  if (regs < PT_REGS) return cudaErrorInvalidConfiguration;
  constexpr int bytes = pt_smem<KV8>();
  cudaError_t e = cudaFuncSetAttribute(paged_tiles_kernel<KV8>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return e;
  paged_tiles_kernel<KV8><<<grid, PT_THREADS, bytes, stream>>>(a, grid, rec_rows);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(grid, (rec_rows + 15) / 16);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_tiles_fold_kernel<KV8>, a, grid, rec_rows);
}

cudaError_t paged_tiles_launch(const IhbPagedAttn& a, cudaStream_t stream) {
  return a.c.k_scale != nullptr ? pt_launch<true>(a, stream) : pt_launch<false>(a, stream);
}

}  // namespace ihb
