// Attention of prompt chunks and longer verify windows over a paged KV cache on the 5th-generation tensor cores (tcgen05, tensor
// memory), head_dim 128, bf16 pages or e4m3 pages with one scale per (page, head). paged_attn.cu has the single-token side, the
// formulas with the page scales and the C entry point.
//
// A CTA takes up to 256 rows ((token, query head) pairs of one sequence and KV head) as two tiles of 128 and walks key blocks of 128:
//   warps 0-3, 4-7   one softmax group per tile, a thread per row: scores from tensor memory, running maximum and sum in registers,
//                    probabilities (16 bits) back into tensor memory in the place of the scores
//   warps 8-11       bring V: page lookups, 16-byte asynchronous copies, e4m3 -> fp16 on the way into the swizzled tile
//   warps 14, 15     bring K, and the page scales. e4m3 K needs no conversion: a bf16 query row, scaled by a power of two, is the sum of two
//                    e4m3 rows (8 significant bits: 4 + 4), so S = Qhi K^T + Qlo K^T runs on e4m3 products, which are twice as fast. What lies below
//                    2^-17 of a row's largest element is lost: 2^-8 of what that element's own rounding to bf16 was, and far below P's fp16
//   warps 12, 13     one issuer per tile (waits, fences and commits cost it more than the products' issue): S = Q K^T (both operands
//                    in shared memory) and O += P V (P in tensor memory, V as an MN-major operand: the rows of the cache are used as
//                    they lie, no transpose)
// Scores live in two halves of 64 keys: while a group computes the probabilities of one half the tensor cores multiply the other's
// with V and form the next block's scores in their place, so that the group does not wait for them (2048 tokens behind 14336 keys: 1160 us
// with whole blocks in turn, 1040 with halves, 990 with the masks out of the hot loop). A sequence with at most 128 rows gives both
// groups the same rows: they take the even and the odd key blocks, and their results are added up at the end.
// The accumulators are rescaled only when a row's maximum has grown by more than 2^8 since the last time.
//
// Work split as in paged_attn.cu: items (sequence, KV head, pair of tiles) are laid end to end, with lengths that follow their causal
// key ranges, and cut into one equal range per SM; pieces of a cut item are folded by a second kernel.
//
// Bound by the groups' latency: a half block is 512 cycles of the exponential unit per warp, two warps share the unit, and a half takes 2050
// cycles with loads from tensor memory, conversion, vote, store and hand-over. The tensor pipe is busy 40 % of the time. Per segment
// 5 us of set-up and result, most of what a batch of short windows costs.
#include "paged.cuh"
#include "paged_tiles.h"
#include "tc_common.cuh"

namespace ihb {

constexpr int PT_M = 128, PT_KB = 128;
constexpr int PT_THREADS = 512;
constexpr int PT_MMA_WARP = 12;
// Registers: 512 threads start with 128 each (all of the SM's); the others' groups give some to the softmax groups, where half a row's
// scores, the probabilities and what the scheduler wants to overlap do not fit 128 (measured: 3 %).
constexpr int PT_REGS = 128, PT_REGS_SOFTMAX = 168, PT_REGS_LOAD = 96, PT_REGS_MMA = 80;
static_assert(256 * PT_REGS_SOFTMAX + 128 * PT_REGS_LOAD + 128 * PT_REGS_MMA <= PT_THREADS * PT_REGS, "more registers than the block has");
constexpr int PT_HALF = 16384;                 // 128 rows x 128 bytes: one swizzled half (64 channels) of a tile
constexpr int PT_TILE = 2 * PT_HALF;
constexpr int PT_HDR = 3 * 1024;                  // barriers and segments; m and l of the second group at 1024 and 1536; page scales at 2048
constexpr int PT_RAW = 128 * PG_HD;             // e4m3 bytes of a key block's K or V
template <bool KV8>
constexpr int pt_smem() { return PT_HDR + 6 * PT_TILE + (KV8 ? 2 * PT_RAW : 0); }
constexpr int PT_MAX_GRID = 148;              // one CTA per SM
// Start-up cost of an item, in keys (a prompt of 4096 tokens, chunks of 4 sequences: 256 258 / 359 us, 384 221 / 360, 512 201 / 357,
// 768 200 / 354).
constexpr int PT_START = 512;
// A cut nearer than this to an end of its item, in keys, moves there: a short piece costs more (set-up, a record, its part in the fold) than the
// longer range. At most half a range, which bounds what one CTA can be given on top (token trees of 8 sequences 50 -> 44 us; a quarter 50).
constexpr int PT_SNAP = 1024;

constexpr int PT_SEGS = 4;
// A piece of an item: rows [row0, row0 + rows) of a sequence's KV head, key blocks [blk0, blk1) of nblk.
struct PtSeg {
  int b, kvh, row0, rows, blk0, blk1, nblk, first_in_range;
  int seen_end, all_see;                       // keys that any of the rows sees lie below the one, keys below the other are seen by all of them
  PgSeq s;
  int last;                                    // no segment: the end
};

template <bool KV8>
constexpr int pt_k_stages() { return KV8 ? 4 : 2; }             // of 16 / 32 KB
constexpr int PT_SC = 8;                       // blocks whose page scales are kept: more than are ever under way

struct PtHdr {
  uint64_t k_full[4], k_empty[2][4], v_full[2], v_empty[2][2];         // empty: [group that used it][stage]
  uint64_t q_full[2], q_free, s_full[4], p_ready[4], pv_done[4], hand[2];     // s_full .. pv_done: [group][half of the block]
  uint64_t drain[2];                           // an issuer's products are over (after a wait that ran out)
  uint32_t tmem;
  int abort_flag;
  int odd;                                     // V values that are not finite were met in keys that not every row sees (set by the loader)
  uint64_t seg_full[PT_SEGS], seg_free[PT_SEGS];
  PtSeg seg[PT_SEGS];
};

// First position of CTA i's range: `total` in PT_MAX_GRID parts that differ by one at most (a division by a constant).
__device__ __forceinline__ long long pt_cut(long long total, int i) {
  const long long per = total / PT_MAX_GRID;
  return per * i + min(static_cast<long long>(i), total - per * PT_MAX_GRID);
}

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
    w.a = static_cast<long long>(min(max(s.base, 0), s.len) + PT_START) * G;   // (a length that its table does not hold may be near 2^31)
    w.d = RT;
  }
  const long long t = w.tiles;
  w.head = t * w.a + w.d * (t * (t + 1) / 2);
  return w;
}
__device__ __forceinline__ long long pt_prefix(const PtWork& w, long long j) { return j * w.a + w.d * (j * (j + 1) / 2); }

// The segments of a CTA's range, in order.
struct PtIter {
  long long u, u_end, u0, before, snap;
  int b;
  PgSeq s;
  PtWork w;
  __device__ __forceinline__ void start(const IhbPagedAttn& p, int G, int RT, long long total, long long before_, int b_) {
    u0 = u = pt_cut(total, blockIdx.x);
    u_end = pt_cut(total, blockIdx.x + 1);
    snap = min(static_cast<long long>(PT_SNAP) * G, total / (2 * PT_MAX_GRID));
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
      g.kvh = static_cast<int>(pg_div(u - before, w.head));
      const long long q = u - before - g.kvh * w.head;
      long long j;
      if (w.d == 0) {
        j = pg_div(q, w.a);
      } else {
        const float h = static_cast<float>(w.a) + 0.5f * static_cast<float>(w.d), fq = static_cast<float>(q);    // the root that cancels nothing
        j = static_cast<long long>(__fdividef(2.f * fq, h + sqrtf(h * h + 2.f * static_cast<float>(w.d) * fq)));
        j = min(max(j, 0ll), static_cast<long long>(w.tiles - 1));
        while (j > 0 && pt_prefix(w, j) > q) --j;
        while (j + 1 < w.tiles && pt_prefix(w, j + 1) <= q) ++j;
      }
      const long long lo = pt_prefix(w, j), len = w.a + w.d * (j + 1);
      const long long p0 = q - lo, p1 = min(len, p0 + (u_end - u));
      // (a position is moved the same way by the CTA that ends there and by the one that begins)
      auto snapped = [&](long long v) { return v == len ? v : v < snap ? 0 : len - v < snap ? len : v; };
      const long long v0 = snapped(p0), v1 = snapped(p1);
      g.b = b;
      g.s = s;
      g.last = 0;
      g.row0 = static_cast<int>(j) * RT;
      g.rows = min(RT, s.n * G - g.row0);
      const int i_last = (g.row0 + g.rows - 1) / G;
      g.seen_end = p.mask != nullptr ? s.len : min(s.len, s.base + i_last + 1);
      g.all_see = max(0, p.mask != nullptr ? s.base : min(s.base + g.row0 / G + 1, s.len));
      g.nblk = max(1, (g.seen_end + PT_KB - 1) / PT_KB);
      g.blk0 = v0 == 0 ? 0 : static_cast<int>(pg_div(v0 * g.nblk, len));
      g.blk1 = v1 == len ? g.nblk : static_cast<int>(pg_div(v1 * g.nblk, len));
      g.first_in_range = u == u0;
      u += p1 - p0;
      if (g.blk0 < g.blk1 || (g.blk0 > 0 && v0 < len)) return true;
    }
    return false;
  }
};

// What a CTA tells the folding kernel. cont: the CTA's first segment continues an item of the CTA before (1: without a block of its
// own, 2: with a piece in slot 0; PT_LOST: one of the CTA's waits ran out, nothing it left may be used), ends: and ends it. tail: the CTA's
// last segment is the first piece of a cut item, in slot `slot`.
constexpr int PT_LOST = -1;
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
// Loads that are waited for later: pt_ld32_issue, pt_wait_ld, pt_pin (ties the registers' first use to the wait).
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
__device__ __forceinline__ void pt_st32(uint32_t t, const unsigned (&v)[32]) {
  __syncwarp();
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
      "%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(t),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
      "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]),
      "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
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
// Eight products (PT_PV: four), D[tmem] (+)= A B. PT_QK16: 16 channels each, both operands in shared memory (K-major, two swizzled halves); PT_QK8: e4m3, 32
// channels each, first Q's heads, then its remainders (a half further on) with the same K; PT_PV: 16 keys each, A in tensor memory (8
// columns per step), B in shared memory, MN-major. The issuing thread shares its scheduler with softmax warps, so the descriptors'
// high words are constants and a step costs one or two additions.
enum { PT_QK16, PT_QK8, PT_PV };
template <int KIND>
__device__ __forceinline__ void pt_mma8(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, uint32_t acc) {
  // high word: stride offset 1024 bytes, version 1, 128-byte swizzle
  if constexpr (KIND == PT_PV)
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t.reg .b32 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 b, {%2, %5};\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t"
        "add.u32 x, %1, 8;\n\tadd.u32 y, %2, 128;\n\tmov.b64 b, {y, %5};\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %3, 1;\n\t"
        "add.u32 x, %1, 16;\n\tadd.u32 y, %2, 256;\n\tmov.b64 b, {y, %5};\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %3, 1;\n\t"
        "add.u32 x, %1, 24;\n\tadd.u32 y, %2, 384;\n\tmov.b64 b, {y, %5};\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %3, 1;\n\t}"
        ::"r"(d), "r"(a), "r"(b_lo), "r"(idesc), "r"(acc), "n"(0x40004040)
        : "memory");
  else if constexpr (KIND == PT_QK8)
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t.reg .b32 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %3, p;\n\t"
        "add.u32 x, %1, 2;\n\tadd.u32 y, %2, 2;\n\tmov.b64 a, {x, %5};\n\tmov.b64 b, {y, %5};\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %3, 1;\n\t"
        "add.u32 x, %1, 4;\n\tadd.u32 y, %2, 4;\n\tmov.b64 a, {x, %5};\n\tmov.b64 b, {y, %5};\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %3, 1;\n\t"
        "add.u32 x, %1, 6;\n\tadd.u32 y, %2, 6;\n\tmov.b64 a, {x, %5};\n\tmov.b64 b, {y, %5};\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %3, 1;\n\t"
        "add.u32 x, %1, 1024;\n\tmov.b64 a, {x, %5};\n\tmov.b64 b, {%2, %5};\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %3, 1;\n\t"
        "add.u32 x, %1, 1026;\n\tadd.u32 y, %2, 2;\n\tmov.b64 a, {x, %5};\n\tmov.b64 b, {y, %5};\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %3, 1;\n\t"
        "add.u32 x, %1, 1028;\n\tadd.u32 y, %2, 4;\n\tmov.b64 a, {x, %5};\n\tmov.b64 b, {y, %5};\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %3, 1;\n\t"
        "add.u32 x, %1, 1030;\n\tadd.u32 y, %2, 6;\n\tmov.b64 a, {x, %5};\n\tmov.b64 b, {y, %5};\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %3, 1;\n\t}"
        ::"r"(d), "r"(a), "r"(b_lo), "r"(idesc), "r"(acc), "n"(0x40004040)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t.reg .b32 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t"
        "add.u32 x, %1, 2;\n\tadd.u32 y, %2, 2;\n\tmov.b64 a, {x, %5};\n\tmov.b64 b, {y, %5};\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t"
        "add.u32 x, %1, 4;\n\tadd.u32 y, %2, 4;\n\tmov.b64 a, {x, %5};\n\tmov.b64 b, {y, %5};\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t"
        "add.u32 x, %1, 6;\n\tadd.u32 y, %2, 6;\n\tmov.b64 a, {x, %5};\n\tmov.b64 b, {y, %5};\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t"
        "add.u32 x, %1, 1024;\n\tadd.u32 y, %2, 1024;\n\tmov.b64 a, {x, %5};\n\tmov.b64 b, {y, %5};\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t"
        "add.u32 x, %1, 1026;\n\tadd.u32 y, %2, 1026;\n\tmov.b64 a, {x, %5};\n\tmov.b64 b, {y, %5};\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t"
        "add.u32 x, %1, 1028;\n\tadd.u32 y, %2, 1028;\n\tmov.b64 a, {x, %5};\n\tmov.b64 b, {y, %5};\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t"
        "add.u32 x, %1, 1030;\n\tadd.u32 y, %2, 1030;\n\tmov.b64 a, {x, %5};\n\tmov.b64 b, {y, %5};\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t}"
        ::"r"(d), "r"(a), "r"(b_lo), "r"(idesc), "r"(acc), "n"(0x40004040)
        : "memory");
}
// Low words of the descriptors: start address; leading offset 16 bytes (K-major: unused) or PT_HALF (MN-major: rows of 64 MN elements, one
// per K, the next 64 a half further on; the stride offset is then that of 8 K).
__device__ __forceinline__ uint32_t pt_lo_k(uint32_t addr) { return ((addr >> 4) & 0x3FFFu) | (1u << 16); }
__device__ __forceinline__ uint32_t pt_lo_mn(uint32_t addr) { return ((addr >> 4) & 0x3FFFu) | (static_cast<uint32_t>(PT_HALF >> 4) << 16); }
// offset of a 16-byte chunk (8 channels) of row r in a swizzled tile
__device__ __forceinline__ int pt_at(int r, int ch) { return (ch >> 3) * PT_HALF + r * 128 + (((ch & 7) ^ (r & 7)) << 4); }

// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t pt_pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void pt_unpair(uint64_t v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t pt_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t pt_add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float pt_max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }
__device__ __forceinline__ void pt_mask32(float* v, unsigned seen) {
#pragma unroll
  for (int e = 0; e < 32; ++e)
    if (!(seen & (1u << e))) v[e] = -INFINITY;
}
// What one of NTH loader threads copies of a key block: RPT rows of one of its groups of 16 keys (one page: one lookup), COLS 16-byte chunks
// of each. A warp's copies cover whole rows.
template <bool KV8, int NTH>
struct PtRows {
  static constexpr int ROWB = KV8 ? PG_HD : 2 * PG_HD, TPG = NTH / 8, COLS = KV8 || TPG == 16 ? 1 : 2, CPT = ROWB / 16 / COLS, RPT = 16 * CPT / TPG;
  int grp, row, ch, key0, end, blk, psh, in_page;
  unsigned page_bytes;
  const char* src;
  const int* table;
  int page;                                    // of the next block's group, looked up while the block before is on its way
  __device__ __forceinline__ PtRows(const IhbPaged& c, int t, int psh_) : grp(t / TPG), row((t % TPG) / CPT * RPT), ch(t % CPT), psh(psh_), in_page(c.page - 1) {
    page_bytes = static_cast<unsigned>(c.nkv * c.page) * ROWB;
  }
  __device__ __forceinline__ void start(const IhbPaged& c, const void* base, const PtSeg& g) {
    key0 = g.blk0 * PT_KB + grp * 16;
    end = min(g.seen_end, g.blk1 * PT_KB);     // keys from here on: zeros
    blk = 0;
    src = reinterpret_cast<const char*>(base) + static_cast<size_t>(g.kvh) * c.page * ROWB + ch * 16;
    table = c.block_table + static_cast<size_t>(g.b) * c.table_stride;
    lookup();
  }
  __device__ __forceinline__ void lookup() {
    const int key = key0 + blk * PT_KB;
    page = key < end ? __ldg(table + (key >> psh)) : -1;
  }
  static __device__ __forceinline__ void copy(uint32_t d, const char* p, int n) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(p), "r"(n));
  }
  // Copies the next block. TILE: row r's chunk to its place in the swizzled tile at dst; else chunk i to dst + i * 2048 (the thread's own).
  template <bool TILE>
  __device__ __forceinline__ void issue(uint32_t dst, int n_pages) {
    const int key = key0 + blk * PT_KB + row;
    const bool good = static_cast<unsigned>(page) < static_cast<unsigned>(n_pages);
    const int live = good ? min(max(end - key, 0), RPT) : 0;
    const char* p = src + (good ? static_cast<size_t>(page) * page_bytes + (key & in_page) * ROWB : 0);
    const int r0 = grp * 16 + row;             // a multiple of 8: the swizzle of row r0 + i is that of i
    const uint32_t d = TILE ? dst + r0 * 128 + (ch << 4 & 127) + (ch >> 3) * PT_HALF : dst;
    if (live == RPT) {
#pragma unroll
      for (int i = 0; i < RPT; ++i)
#pragma unroll
        for (int c = 0; c < COLS; ++c) copy(TILE ? (d ^ ((i & 7) << 4)) + i * 128 + c * PT_HALF : d + i * 2048, p + i * ROWB + c * 128, 16);
    } else {
#pragma unroll 1
      for (int i = 0; i < RPT; ++i)
        for (int c = 0; c < COLS; ++c)
          copy(TILE ? (d ^ ((i & 7) << 4)) + i * 128 + c * PT_HALF : d + i * 2048, i < live ? p + i * ROWB + c * 128 : src, i < live ? 16 : 0);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    ++blk;
    lookup();
  }
};
// Takes what is not finite out of 16 bytes of V; true: there was something.
template <bool KV8>
__device__ __noinline__ bool pt_clean(uint4& y) {
  unsigned x[4] = {y.x, y.y, y.z, y.w};
  bool bad = false;
  for (int q = 0; q < 4; ++q) {
    if constexpr (KV8) {
      for (int e = 0; e < 4; ++e)
        if (((x[q] >> (8 * e)) & 0x7fu) == 0x7fu) { x[q] &= ~(0xffu << (8 * e)); bad = true; }
    } else {
      if ((x[q] & 0x7f80u) == 0x7f80u) { x[q] &= 0xffff0000u; bad = true; }
      if ((x[q] & 0x7f800000u) == 0x7f800000u) { x[q] &= 0x0000ffffu; bad = true; }
    }
  }
  y = make_uint4(x[0], x[1], x[2], x[3]);
  return bad;
}
// Bounded wait on a phase of an mbarrier; gives up when another role has. The clock is read only after a while of polling: the first
// read would cost more than most waits.
__device__ __forceinline__ bool pt_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, unsigned* err, unsigned code) {
  unsigned long long t0 = 0;
  for (unsigned spins = 1; !mbar_try_wait(bar, parity); ++spins) {
    if ((spins & 255u) == 0u) {
      if (*abort_flag) return false;
      const unsigned long long t = globaltimer_ns();
      if (t0 == 0) t0 = t;
      if (t - t0 > IHB_LOCAL_WAIT_NS) {
        *abort_flag = 1;
        set_error(err, code);
        return false;
      }
    }
  }
  return true;
}
// Shared memory by 32-bit address: the aligned base is a computed pointer, which the compiler would access as generic memory.
__device__ __forceinline__ uint4 pt_lds(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 pt_lds8(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ void pt_sts(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// Does a row see key p? vis: keys below it are seen; mrow: the row's mask over the call's tokens, or NULL.
__device__ __forceinline__ bool pt_sees(const IhbPagedAttn& a, const PgSeq& s, const unsigned char* mrow, int vis, int p) {
  if (p < vis) return true;
  return mrow != nullptr && p < s.len && p - s.base < a.mask_cols && mrow[p - s.base] != 0;
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

// P2 (bf16 pages): the probabilities go into the product as two bf16 terms, as those of paged_attn.cu do, and not as one.
template <bool KV8, bool P2>
__global__ void __launch_bounds__(PT_THREADS, 1) paged_tiles_kernel(const __grid_constant__ IhbPagedAttn a, int grid, int rec_rows) {
  extern __shared__ __align__(1024) uint8_t smem[];            // (checked below: the swizzle goes by address)
  PtHdr& sh = *reinterpret_cast<PtHdr*>(smem);
  uint8_t* sq = smem + PT_HDR;
  // per block and 16 keys: factor of the scores (negative: no such page), log2 of the V scale, 1 / V scale; .w of the first: a page is missing
  float4* sc = reinterpret_cast<float4*>(smem + 2048);         // [PT_SC][8]
  uint8_t* sk = sq + 2 * PT_TILE;
  uint8_t* sv = sk + 2 * PT_TILE;
  uint8_t* raw = sv + 2 * PT_TILE;             // e4m3 pages: the bytes of two V blocks on their way to the tiles
  constexpr int KS = pt_k_stages<KV8>(), K_BYTES = 2 * PT_TILE / KS;
  constexpr int RT = 2 * PT_M;
  const IhbPaged& c = a.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = a.nq / c.nkv, psh = __ffs(c.page) - 1;
  PtDesc* descs = reinterpret_cast<PtDesc*>(a.scratch);
  float* recs = reinterpret_cast<float*>(reinterpret_cast<char*>(a.scratch) + PT_MAX_GRID * sizeof(PtDesc));
  pdl_launch_dependents();

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.k_full[2 * i], 64); mbar_init(&sh.k_full[2 * i + 1], 64);
      for (int j = 0; j < 4; ++j) mbar_init(&sh.k_empty[i][j], 1);
      for (int j = 0; j < 2; ++j) mbar_init(&sh.v_empty[i][j], 1);
      mbar_init(&sh.v_full[i], 128);
      mbar_init(&sh.drain[i], 1);
      mbar_init(&sh.q_full[i], 128); mbar_init(&sh.s_full[2 * i], 2); mbar_init(&sh.s_full[2 * i + 1], 2);
      mbar_init(&sh.p_ready[2 * i], 128); mbar_init(&sh.p_ready[2 * i + 1], 128); mbar_init(&sh.pv_done[2 * i], 1); mbar_init(&sh.pv_done[2 * i + 1], 1);
    }
    mbar_init(&sh.q_free, 2);
    mbar_init(&sh.hand[0], 128);
    mbar_init(&sh.hand[1], 128);
    for (int i = 0; i < PT_SEGS; ++i) { mbar_init(&sh.seg_full[i], 1); mbar_init(&sh.seg_free[i], 16); }
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
  if (tid == 0 && (smem_u32(smem) & 1023u)) { set_error(c.err, ERR_BAD_ARGS); sh.abort_flag = 1; }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  volatile int* abort_flag = &sh.abort_flag;
  // The next segment: every role reads the scheduler's records in order, and gives a record back (free_seg) when done with it.
  unsigned n_seg = 0;
  auto next_seg = [&]() -> const PtSeg* {
    if (!pt_wait(&sh.seg_full[n_seg % PT_SEGS], (n_seg / PT_SEGS) & 1u, abort_flag, c.err, ERR_MBAR_FULL_TIMEOUT)) return nullptr;
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
    unsigned g0 = 0, n_blk = 0, n_hand = 0;            // blocks of earlier segments; blocks this group has been through, segments that both groups shared: barrier phases
    while (const PtSeg* gp = next_seg()) {
      const PtSeg& sg = *gp;
      const PgSeq& s = sg.s;
      const bool pair = sg.rows > PT_M;        // two tiles; else both groups have the same rows and every other key block
      const bool whole = sg.blk0 == 0 && sg.blk1 == sg.nblk;
      const int r = (pair ? wg * PT_M : 0) + r_tile;                    // row of the item
      const bool live = r < sg.rows;
      const int tok = live ? (sg.row0 + r) / G : 0, head = sg.kvh * G + (live ? (sg.row0 + r) % G : 0);
      const int vis = !live ? max(sg.seen_end, 0) : min(max(a.mask != nullptr ? s.base : s.base + tok + 1, 0), s.len);   // keys [0, vis) are seen
      const unsigned char* mrow = a.mask != nullptr && live ? a.mask + static_cast<size_t>(s.t0 + tok) * a.mask_stride : nullptr;
      const int* table = c.block_table + static_cast<size_t>(sg.b) * c.table_stride;
      // ---- Q: a warp brings its 32 rows, two at a time, 16 bytes per lane ----
      float rowf = fmaxf(a.scale * PG_LOG2E, 1.17549435e-38f);            // (never 0: times a masked -inf it would be NaN)
      if (ok && n_seg > 0) ok = pt_wait(&sh.q_free, (n_seg - 1) & 1u, abort_flag, c.err, ERR_TMEM_TIMEOUT);
      if (ok && n_hand > 0) ok = pt_wait(&sh.hand[1], (n_hand - 1) & 1u, abort_flag, c.err, ERR_TMEM_TIMEOUT);
      __syncwarp();
      {
        const uint32_t dst = smem_u32(sq) + wg * PT_TILE;
        const int ch = lane & 15, first = sg.row0 + (pair ? wg * PT_M : 0) + quarter * 32 + (lane >> 4), end = sg.row0 + sg.rows;    // rows of the sequence
        const __nv_bfloat16* qp = reinterpret_cast<const __nv_bfloat16*>(a.q) + static_cast<size_t>(s.t0 + first / G) * a.q_stride_t +
                                  static_cast<size_t>(sg.kvh * G) * a.q_stride_h + ch * 8;
        int h = first % G;
        // e4m3: the row's even 16 bytes in the tile's first half, the odd ones beside them in the second: what becomes of a pair of them,
        // 16 bytes of head and 16 of remainder, then has the same two places
        const uint32_t half = (KV8 ? ch & 1 : ch >> 3) * PT_HALF;
        const int pos = KV8 ? ch >> 1 : ch & 7;
#pragma unroll 4
        for (int i = 0; i < 16; ++i) {
          const int rt = quarter * 32 + 2 * i + (lane >> 4);
          const bool in = first + 2 * i < end;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + half + pt_at(rt, pos)), "l"(in ? qp + h * a.q_stride_h : a.q), "r"(in ? 16 : 0) : "memory");
          for (h += 2; h >= G; h -= G) qp += a.q_stride_t;               // two rows on
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
        if constexpr (KV8) {                   // |q| of the lane's row below 256 by a power of two, then an e4m3 head and an e4m3 remainder
          const uint32_t row = dst + r_tile * 128;
          unsigned mx2 = 0;                    // largest magnitudes of both halves: bf16 bits without the sign order like integers
#pragma unroll 4
          for (int p = 0; p < 16; ++p) {
            const uint4 v = pt_lds(row + (p & 1) * PT_HALF + (((p >> 1) ^ (lane & 7)) << 4));
            mx2 = __vmaxu2(mx2, __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)));
          }
          // A row with NaN (larger than anything) or an infinity (e4m3 has none) becomes NaN in all channels, and so do its scores: those that are seen
          const unsigned mx = max(mx2 & 0xffffu, mx2 >> 16), nan = mx < 0x7f80u ? 0u : 0x7f7f7f7fu;
          // (not below 2^-45, and the factor not below 2^-49: times the least page scale it is not 0, see above. Of a row below 2^-38 that loses 2^-55.)
          const int e2 = min(max(static_cast<int>(mx >> 7) - 127 - 7, -45), 100);
          rowf = fmaxf(rowf * __uint_as_float(static_cast<unsigned>(127 + e2) << 23), 1.7763568394002505e-15f);
          const float inv = __uint_as_float(static_cast<unsigned>(127 - e2) << 23);
#pragma unroll 2
          for (int p = 0; p < 8; ++p) {
            const uint32_t at = row + ((p ^ (lane & 7)) << 4);
            const uint4 v0 = pt_lds(at), v1 = pt_lds(at + PT_HALF);
            const unsigned x[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
            unsigned hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              unsigned h8[2], l8[2];
#pragma unroll
              for (int k = 0; k < 2; ++k) {    // through fp16, which holds the scaled bf16 values and the differences exactly
                const __half2 y = __floats2half2_rn(__uint_as_float(x[2 * e + k] << 16) * inv, __uint_as_float(x[2 * e + k] & 0xffff0000u) * inv);
                h8[k] = __nv_cvt_halfraw2_to_fp8x2(static_cast<__half2_raw>(y), __NV_SATFINITE, __NV_E4M3);
                const __half2 z = __hsub2(y, cvt_e4m3x2(static_cast<unsigned short>(h8[k])));
                l8[k] = __nv_cvt_halfraw2_to_fp8x2(static_cast<__half2_raw>(z), __NV_SATFINITE, __NV_E4M3);
              }
              hi[e] = h8[0] | h8[1] << 16 | nan;
              lo[e] = l8[0] | l8[1] << 16;
            }
            pt_sts(at, make_uint4(hi[0], hi[1], hi[2], hi[3]));
            pt_sts(at + PT_HALF, make_uint4(lo[0], lo[1], lo[2], lo[3]));
          }
        }
        fence_proxy_async_smem();
        mbar_arrive(&sh.q_full[wg]);
      }
      const int step = pair ? 1 : 2, blk_end = sg.blk1, blk_first = sg.blk0;
      float m = -INFINITY, l = 0.f;
      bool have = false;                       // O holds something
      for (int blk = blk_first + (pair ? 0 : wg); blk < blk_end; blk += step) {
        if (ok) ok = pt_wait(&sh.s_full[2 * wg], n_blk & 1u, abort_flag, c.err, ERR_TMEM_TIMEOUT);
        tc_fence_after();
        const float4* sb = sc + ((g0 + blk - blk_first) % PT_SC) * 8;
        const int key0 = blk * PT_KB;
        const bool bad = sb[0].w != 0.f;
        if (bad && lane == 0) set_error(c.err, ERR_BAD_ARGS);
        const bool edge = __any_sync(0xffffffffu, key0 + PT_KB > vis) || bad;
        // Half a block at a time, against the maximum so far: the probabilities are formed and held while this half's own maximum is
        // found; only when it is more than 2^8 above (the first keys, and rarely later) the accumulators are rescaled and the half is done
        // again. No pass for the maximum alone, and the first half's product with V runs under the second half's exponentials. The
        // loops stay short: unrolled over the row's 128 scores the hot code is several times the first instruction cache, and every
        // warp of the SM pays for it.
#pragma unroll 1
        for (int hf = 0; hf < 2; ++hf) {
          unsigned pk[32], pl[P2 ? 32 : 1];
          float sum;
          if (hf == 1) {
            if (ok) ok = pt_wait(&sh.s_full[2 * wg + 1], n_blk & 1u, abort_flag, c.err, ERR_TMEM_TIMEOUT);
            tc_fence_after();
          }
          // Keys that the row does not see: -infinity, written over their scores here. A branch with the masks between the loads and the arithmetic
          // below costs every half block 200 cycles of 1600, taken or not.
          if (edge) {
#pragma unroll 1
            for (int q = 2 * hf; q < 2 * hf + 2; ++q) {
              const int kc = key0 + q * 32, n = min(max(vis - kc, 0), 32);
              unsigned w = n == 32 ? ~0u : (1u << n) - 1u;               // bit e: the row sees key kc + e
              if (mrow != nullptr && n < 32 && kc < s.len) {             // (vis = base: the keys from there on are the call's tokens)
                unsigned char b[32];
                const int j0 = kc - s.base, j1 = min(min(a.mask_cols, s.n), s.len - s.base);
#pragma unroll
                for (int e = 0; e < 32; ++e) b[e] = j0 + e >= 0 && j0 + e < j1 ? mrow[j0 + e] : 0;       // all in flight at once
#pragma unroll
                for (int e = 0; e < 32; ++e)
                  if (b[e]) w |= 1u << e;
              }
              if (bad) {
                if (sb[2 * q].x < 0.f) w &= 0xffff0000u;
                if (sb[2 * q + 1].x < 0.f) w &= 0x0000ffffu;
              }
              float x[32];
              pt_ld32(t_s + q * 32, x);
              pt_mask32(x, w);
              unsigned y[32];
#pragma unroll
              for (int e = 0; e < 32; ++e) y[e] = __float_as_uint(x[e]);
              __syncwarp();
              pt_st32(t_s + q * 32, y);
            }
            pt_wait_st();
          }
          for (int turn = 0;; ++turn) {        // (a third turn would only come from scores beyond fp32's whole numbers, 2^24)
            float v[64];                       // (nothing but waits may stand between the loads and theirs: the registers fill behind the compiler's back)
            __syncwarp();
            pt_ld32_issue(t_s + hf * 64, v);
            pt_ld32_issue(t_s + hf * 64 + 32, v + 32);
            pt_wait_ld();
            pt_pin(v);
            pt_pin(v + 32);
            float mx = -INFINITY;
            const float mo = OFF - (m == -INFINITY ? 0.f : m);
            sum = 0.f;
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              float4 ke = make_float4(1.f, 0.f, 1.f, 0.f);
              if (KV8) ke = sb[hf * 4 + h];
              const float f = KV8 ? fabsf(ke.x) * rowf : rowf, add = KV8 ? ke.y + mo : mo;
              const uint64_t f2 = pt_pair(f, f), add2 = pt_pair(add, add);
              uint64_t s2 = 0;                 // (0.f, 0.f)
              float x = -INFINITY;
#pragma unroll
              for (int e = 0; e < 16; e += 2) {
                float p0, p1;
                pt_unpair(pt_fma2(pt_pair(v[h * 16 + e], v[h * 16 + e + 1]), f2, add2), p0, p1);      // a masked score stays -inf: f > 0
                x = pt_max3(x, p0, p1);
                p0 = pd_ex2(p0);
                p1 = pd_ex2(p1);
                s2 = pt_add2(s2, pt_pair(p0, p1));
                pk[h * 8 + e / 2] = pd_pack<KV8>(p0, p1);
                if constexpr (P2) {
                  const float2 r = pd_unpack<false>(pk[h * 8 + e / 2]);
                  pl[h * 8 + e / 2] = pd_pack<false>(p0 - r.x, p1 - r.y);
                }
              }
              mx = fmaxf(mx, x);
              float s0, s1;
              pt_unpair(s2, s0, s1);
              sum += KV8 ? (s0 + s1) * ke.z : s0 + s1;
            }
            mx -= mo;                          // this half's maximum of score + log2 of the V scale
            const bool grow = m == -INFINITY ? mx > -INFINITY : mx > m + PD_LAZY;
            if (!__any_sync(0xffffffffu, grow) || turn == 2) break;
            const float mn = fmaxf(m, mx), r = m == -INFINITY ? 0.f : pd_ex2(m - mn);
            m = mn;
            l *= r;
            if (have) {
              // the last product with V: the other half's, of this block or of the one before (a barrier per half: a wait must not lag two phases)
              if (ok) ok = pt_wait(&sh.pv_done[2 * wg + (hf ^ 1)], (n_blk - 1 + hf) & 1u, abort_flag, c.err, ERR_TMEM_TIMEOUT);
              tc_fence_after();
#pragma unroll 1
              for (int q = 0; q < 8; ++q) {
                float x[16];
                __syncwarp();
                tmem_ld16(t_o + q * 16, x);
                unsigned y[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) y[e] = __float_as_uint(x[e] * r);
                pt_st16(t_o + q * 16, y);
              }
            }
          }
          l += sum;
          have = true;
          pt_st32(t_s + hf * 64, pk);          // in the place of the scores
          if constexpr (P2) pt_st32(t_s + hf * 64 + 32, pl);
          pt_wait_st();
          tc_fence_before();
          mbar_arrive(&sh.p_ready[2 * wg + hf]);                         // (a barrier per half: both may be through before the issuer looks)
        }
        ++n_blk;
      }
      // ---- the result ----
      if (have && ok) ok = pt_wait(&sh.pv_done[2 * wg + 1], (n_blk - 1) & 1u, abort_flag, c.err, ERR_TMEM_TIMEOUT);
      tc_fence_after();
      float f0 = 1.f, f1 = 0.f;
      const uint32_t xs = smem_u32(sq) + r_tile * 512;                   // the row's place
      if (!pair) {                             // the second group hands its result over through the place of Q, which no product reads now
        float* xm = reinterpret_cast<float*>(smem + 1024);
        float* xl = reinterpret_cast<float*>(smem + 1536);
        if (ok) ok = pt_wait(&sh.q_free, n_seg & 1u, abort_flag, c.err, ERR_TMEM_TIMEOUT);
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
        else if (ok) ok = pt_wait(&sh.hand[0], n_hand & 1u, abort_flag, c.err, ERR_TMEM_TIMEOUT);
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
        // The stage, 256 bytes per row. A pair's: rows 0 to 15 and 16 to 31 in the two pieces of 4 KB that the warp's own queries have, nowhere else: the
        // group's other warps may be loading their next queries by now. Not a pair's: at the head of the row's handed-over 512 bytes (hand[1] orders it).
        const uint32_t stage = smem_u32(sq) + (pair ? wg * PT_TILE + quarter * 4096 : quarter * 16384);
        const int stage_row = pair ? 256 : 512, stage_gap = pair ? PT_HALF - 4096 : 0;
        const uint32_t mine = stage + lane * stage_row + (lane >> 4) * stage_gap;
        const bool wide_out = ((a.out_stride_t | a.out_stride_h) & 7) == 0;
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
            for (int key = max(sg.all_see, sg.blk0 * PT_KB); key < min(sg.seen_end, sg.blk1 * PT_KB); ++key) {
              const int pg = table[key >> psh];
              if (!pt_sees(a, s, mrow, vis, key) || static_cast<unsigned>(pg) >= static_cast<unsigned>(c.n_pages)) continue;
              const size_t row = (static_cast<size_t>(pg) * c.nkv + sg.kvh) * c.page + (key & (c.page - 1));
#pragma unroll 1
              for (int e = 0; e < 32; ++e) {
                const float x = pt_v_at<KV8>(c, row, q * 32 + e);
                if (!(fabsf(x) <= 3.4028235e38f)) {
#pragma unroll
                  for (int k = 0; k < 32; ++k)                           // (registers have no index; unrolled the other way it is 5 KB in the epilogue's path)
                    if (k == e) v[k] += x;
                }
              }
            }
          // into the row's 256 bytes of the stage, and out in whole rows when they are full
          if (whole) {
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] *= inv;
          }
          if (whole && a.out_bf16) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              pt_sts(mine + (((q * 4 + e) ^ (lane & 7)) << 4),
                     make_uint4(pd_pack<false>(v[8 * e], v[8 * e + 1]), pd_pack<false>(v[8 * e + 2], v[8 * e + 3]), pd_pack<false>(v[8 * e + 4], v[8 * e + 5]),
                                pd_pack<false>(v[8 * e + 6], v[8 * e + 7])));
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              pt_sts(mine + ((((q & 1) * 8 + e) ^ (lane & 7)) << 4),
                     make_uint4(__float_as_uint(v[4 * e]), __float_as_uint(v[4 * e + 1]), __float_as_uint(v[4 * e + 2]), __float_as_uint(v[4 * e + 3])));
          }
          if (whole && a.out_bf16 ? q != 3 : !(q & 1)) continue;
          __syncwarp();
          if (!whole) {                        // a piece: rows of the record
            const int ch = lane & 15, row = r - r_tile + quarter * 32 + (lane >> 4), n = min(sg.rows, rec_rows) - row;
            float* d = recs + ((static_cast<size_t>(blockIdx.x) * 2 + slot) * rec_rows + row) * PD_REC + (q >> 1) * 64 + ch * 4;
#pragma unroll 4
            for (int i = 0; i < 16; ++i) {
              const int rl = 2 * i + (lane >> 4);
              if (2 * i < n) *reinterpret_cast<uint4*>(d + 2 * i * PD_REC) = pt_lds(stage + rl * stage_row + (rl >> 4) * stage_gap + ((ch ^ (rl & 7)) << 4));
            }
            __syncwarp();
            continue;
          }
          const int ch = lane & 15, first = r - r_tile + quarter * 32 + (lane >> 4);                       // row of the item
          int h = (sg.row0 + first) % G;
          size_t o0 = static_cast<size_t>(s.t0 + (sg.row0 + first) / G) * a.out_stride_t + static_cast<size_t>(sg.kvh * G) * a.out_stride_h;
#pragma unroll 4
          for (int i = 0; i < 16; ++i) {
            const int rl = 2 * i + (lane >> 4), rr = first + 2 * i;
            const uint4 x = pt_lds(stage + rl * stage_row + (rl >> 4) * stage_gap + ((ch ^ (rl & 7)) << 4));
            const size_t o = o0 + static_cast<size_t>(h) * a.out_stride_h;
            for (h += 2; h >= G; h -= G) o0 += a.out_stride_t;           // two rows on
            if (rr >= sg.rows) continue;
            if (a.out_bf16) {                  // (out starts on 16 bytes, but its strides are multiples of four elements only)
              uint2* d = reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(a.out) + o + ch * 8);
              if (wide_out) {
                *reinterpret_cast<uint4*>(d) = x;
              } else {
                d[0] = make_uint2(x.x, x.y);
                d[1] = make_uint2(x.z, x.w);
              }
            } else {
              *reinterpret_cast<uint4*>(reinterpret_cast<float*>(a.out) + o + (q >> 1) * 64 + ch * 4) = x;
            }
          }
          __syncwarp();
        }
        if (live && whole && a.lse != nullptr) a.lse[static_cast<size_t>(s.t0 + tok) * a.nq + head] = pd_lse<KV8>(m, l);
        if (live && !whole && r < rec_rows)
          *reinterpret_cast<float2*>(recs + ((static_cast<size_t>(blockIdx.x) * 2 + slot) * rec_rows + r) * PD_REC + PG_HD) = make_float2(m, l);
      }
      tc_fence_before();
      if (!pair) {
        if (wg == 0) mbar_arrive(&sh.hand[1]);                           // the place of Q is free again
        ++n_hand;
      }
      g0 += blk_end - blk_first;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.seg_free[n_seg % PT_SEGS]);
      ++n_seg;
    }
  } else if (warp < PT_MMA_WARP) {
    pt_regs_dec<PT_REGS_LOAD>();
    // =============================== loader ===========================================================================================
    // V blocks, copied 16 bytes at a time by cp.async (rows that nobody sees: zeros). A thread works on the chunks that it copied itself, so a
    // block needs no barrier among the loader's threads. Two blocks are under way: e4m3 bytes land in `raw` and go from there, as fp16,
    // into the tile; bf16 rows land in the tile.
    const int lt = tid - 256;
    using Rows = PtRows<KV8, 128>;
    Rows rows(c, lt, psh);
    unsigned gk = 0;                           // blocks so far
    unsigned used = 0, turn = 0;               // bit (group, stage): the stage's last block was the group's; parity of how many were
    // The first warp also lays out the segments, one ahead of the one that it loads (the loader is ahead of the others).
    PtIter it;
    PtDesc desc = {0, 0, 0, 0, 0, 0, 0, 0};
    unsigned n_out = 0;
    bool more = true;
    if (warp == 8) {
      long long total = 0;
      for (int b = lane; b < c.B; b += 32) total += pt_work(a, pg_seq(c, b), G, RT).head * c.nkv;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
      const long long u = pt_cut(total, blockIdx.x);
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
      it.start(a, G, RT, total, before, found);
    }
    auto publish = [&]() {                     // the next segment with a key block, or the end
      while (more) {
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
        const unsigned i = n_out % PT_SEGS;
        if (n_out >= PT_SEGS && ok) ok = pt_wait(&sh.seg_free[i], ((n_out / PT_SEGS) & 1u) ^ 1u, abort_flag, c.err, ERR_MBAR_EMPTY_TIMEOUT);
        sh.seg[i] = g;
        mbar_arrive(&sh.seg_full[i]);
        ++n_out;
        break;
      }
    };
    if (tid == 256) publish();
    __syncwarp();
    while (const PtSeg* gp = next_seg()) {
      const int nb = gp->blk1 - gp->blk0, all_see = gp->all_see, first = gp->blk0 * PT_KB;
      rows.start(c, c.v, *gp);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.seg_free[n_seg % PT_SEGS]);
      ++n_seg;
      const bool both = gp->rows > PT_M;       // groups that use a block: both, or n & 1
      auto wait_empty = [&](int n) {
        const int st = (gk + n) & 1;
#pragma unroll
        for (int w = 0; w < 2; ++w) {          // who has had the stage's last block is waited for, who gets this one is noted
          const unsigned bit = 1u << (w * 2 + st);
          if ((used & bit) && ok) ok = pt_wait(&sh.v_empty[w][st], (turn & bit) ? 0u : 1u, abort_flag, c.err, ERR_MBAR_EMPTY_TIMEOUT);
          used &= ~bit;
          if (both || w == (n & 1)) {
            used |= bit;
            turn ^= bit;
          }
        }
      };
      auto finish = [&](int n) {               // block n has landed
        const unsigned g = gk + n;
        const int r0 = rows.grp * 16 + rows.row, key = first + n * PT_KB + r0;
        const uint32_t dst = smem_u32(sv) + (g & 1) * PT_TILE + r0 * 128;
        // keys that not every row sees: what is not finite is taken out here and added where it is seen
        const bool window = first + n * PT_KB + PT_KB > all_see;
        bool hit = false;
        if constexpr (KV8) {
          const uint32_t src = smem_u32(raw) + (n & 1) * PT_RAW + lt * 16;
          if (window)
#pragma unroll 1
            for (int i = 0; i < Rows::RPT; ++i)
              if (key + i >= all_see) {
                uint4 x = pt_lds(src + i * 2048);
                if (pt_clean<true>(x)) { pt_sts(src + i * 2048, x); hit = true; }
              }
          // 16 bytes are two chunks of eight fp16; the halves of a row start with different ones: the eight lanes of a phase then write
          // to different banks
          const int swap = rows.ch >> 2;
          const uint32_t d0 = dst + swap * PT_HALF + (((2 * rows.ch + swap) & 7) << 4), d1 = dst + swap * PT_HALF + (((2 * rows.ch + 1 - swap) & 7) << 4);
          uint2 x[Rows::RPT], y[Rows::RPT];
#pragma unroll
          for (int i = 0; i < Rows::RPT; ++i) {
            x[i] = pt_lds8(src + i * 2048 + swap * 8);
            y[i] = pt_lds8(src + i * 2048 + 8 - swap * 8);
          }
#pragma unroll
          for (int i = 0; i < Rows::RPT; ++i) {
            uint4 a0, a1;
            pd_cvt4(x[i].x, a0.x, a0.y);
            pd_cvt4(x[i].y, a0.z, a0.w);
            pd_cvt4(y[i].x, a1.x, a1.y);
            pd_cvt4(y[i].y, a1.z, a1.w);
            pt_sts((d0 ^ ((i & 7) << 4)) + i * 128, a0);
            pt_sts((d1 ^ ((i & 7) << 4)) + i * 128, a1);
          }
        } else if (window) {
#pragma unroll 1
          for (int i = 0; i < Rows::RPT; ++i)
            if (key + i >= all_see) {
              const uint32_t p = ((dst + (rows.ch >> 3) * PT_HALF + ((rows.ch & 7) << 4)) ^ ((i & 7) << 4)) + i * 128;
              uint4 x = pt_lds(p);
              if (pt_clean<false>(x)) { pt_sts(p, x); hit = true; }
            }
        }
        if (hit) *reinterpret_cast<volatile int*>(&sh.odd) = 1;
        fence_proxy_async_smem();
        mbar_arrive(&sh.v_full[g & 1]);
      };
      // e4m3: the bytes of block n + 2 are on their way while block n is converted; bf16: the rows of block n while block n - 1 is handed over
      constexpr int AHEAD = KV8 ? 2 : 0, LAG = KV8 ? 0 : 1;
#pragma unroll 1
      for (int n = -AHEAD; n < nb + LAG; ++n) {
        if (!KV8 && n < nb) wait_empty(n);
        const int f = n - LAG;
        if (KV8 && f >= 0) {
          if (n + 1 < nb) asm volatile("cp.async.wait_group 1;" ::: "memory");
          else asm volatile("cp.async.wait_group 0;" ::: "memory");
          wait_empty(f);
          finish(f);
        }
        if (n + AHEAD < nb) {
          if constexpr (KV8) rows.template issue<false>(smem_u32(raw) + ((n + AHEAD) & 1) * PT_RAW + lt * 16, c.n_pages);
          else rows.template issue<true>(smem_u32(sv) + ((gk + n) & 1) * PT_TILE, c.n_pages);
        }
        if (n == 0) {                          // the next segment, while this one's first blocks are on their way
          if (tid == 256) publish();
          __syncwarp();
        }
        if (!KV8 && f >= 0) {
          if (n < nb) asm volatile("cp.async.wait_group 1;" ::: "memory");
          else asm volatile("cp.async.wait_group 0;" ::: "memory");
          finish(f);
        }
      }
      gk += nb;
    }
  } else {
    pt_regs_dec<PT_REGS_MMA>();
    if (warp >= PT_MMA_WARP + 2) {
      // =============================== K and the page scales ==============================================================================
      constexpr int LAG = KS / 2;              // blocks under way
      const int lt = tid - (PT_MMA_WARP + 2) * 32;
      PtRows<KV8, 64> rows(c, lt, psh);
      unsigned gk = 0, used = 0, turn = 0;     // see the V loader
      while (const PtSeg* gp = next_seg()) {
        const int nb = gp->blk1 - gp->blk0, kvh = gp->kvh, first = gp->blk0 * PT_KB;
        const bool both = gp->rows > PT_M;
        rows.start(c, c.k, *gp);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.seg_free[n_seg % PT_SEGS]);
        ++n_seg;
        // lane i (0 .. 7) of warp 14 looks after the scales of the block's 16 keys i
        float ks = 1.f, vs = 1.f;
        auto page_at = [&](int n) {
          const int key = first + n * PT_KB + (lane & 7) * 16;
          return key < rows.end ? __ldg(rows.table + (key >> psh)) : 0;
        };
        int pg_next = page_at(0);
        auto load_scales = [&](int n) {
          const int key = first + n * PT_KB + (lane & 7) * 16, pg = pg_next;
          pg_next = page_at(n + 1);
          ks = vs = 1.f;
          if (key < rows.end) {
            if (static_cast<unsigned>(pg) >= static_cast<unsigned>(c.n_pages)) {
              ks = -1.f;
            } else if (KV8) {
              ks = fmaxf(__ldg(c.k_scale + static_cast<size_t>(pg) * c.nkv + kvh), 1e-30f);      // (0 would turn a masked -inf into NaN)
              vs = __ldg(c.v_scale + static_cast<size_t>(pg) * c.nkv + kvh);
            }
          }
        };
        auto store_scales = [&](int n) {
          const unsigned any = __ballot_sync(0xffffffffu, ks < 0.f);
          const float ev = KV8 ? pd_log2_scale(vs) : 0.f;
          if (lane < 8) sc[((gk + n) % PT_SC) * 8 + lane] = make_float4(ks, ev, KV8 ? pd_ex2(-ev) : 1.f, any ? 1.f : 0.f);
          if (any && lane == 0) set_error(c.err, ERR_BAD_ARGS);
        };
        auto finish = [&](int n) {
          fence_proxy_async_smem();
          mbar_arrive(&sh.k_full[(gk + n) % KS]);
        };
#pragma unroll 1
        for (int n = 0; n < nb + LAG; ++n) {
          const unsigned g = gk + n;
          if (n < nb) {
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              const unsigned bit = 1u << (w * 4 + g % KS);
              if ((used & bit) && ok) ok = pt_wait(&sh.k_empty[w][g % KS], (turn & bit) ? 0u : 1u, abort_flag, c.err, ERR_MBAR_EMPTY_TIMEOUT);
              used &= ~bit;
              if (both || w == (n & 1)) {
                used |= bit;
                turn ^= bit;
              }
            }
            rows.template issue<true>(smem_u32(sk) + (g % KS) * K_BYTES, c.n_pages);
          } else {
            asm volatile("cp.async.commit_group;" ::: "memory");       // (an empty group: the count below stays the same)
          }
          if (warp == PT_MMA_WARP + 2) {
            if (n > 0 && n <= nb) store_scales(n - 1);
            if (n < nb) load_scales(n);
          }
          if (n >= LAG) {
            asm volatile("cp.async.wait_group %0;" ::"n"(LAG) : "memory");
            finish(n - LAG);
          }
        }
        gk += nb;
      }
    } else
    if (lane == 0) {
    // =============================== MMA issuers ========================================================================================
    const int w = warp - PT_MMA_WARP;          // the group that this one works for
    constexpr uint32_t idesc = (1u << 4) | (KV8 ? 0u : ((1u << 7) | (1u << 10))) | (static_cast<uint32_t>(PT_M >> 4) << 24) | (static_cast<uint32_t>(PT_KB / 2 >> 3) << 17);
    constexpr uint32_t idesc_v = (idesc & ~(63u << 17)) | (static_cast<uint32_t>(PG_HD >> 3) << 17) | (1u << 16);      // V: MN-major
    const uint32_t q_lo = pt_lo_k(smem_u32(sq)), k_lo = pt_lo_k(smem_u32(sk)), v_lo = pt_lo_mn(smem_u32(sv));
    unsigned gk = 0, n_p = 0;                  // blocks so far; phase of the group's p_ready
    while (const PtSeg* gp = ok ? next_seg() : nullptr) {
      const int nb = gp->blk1 - gp->blk0, step = gp->rows > PT_M ? 1 : 2, first = step == 1 ? 0 : w;   // its blocks: all, or every other one
      mbar_arrive(&sh.seg_free[n_seg % PT_SEGS]);
      ok = pt_wait(&sh.q_full[w], n_seg & 1u, abort_flag, c.err, ERR_MBAR_FULL_TIMEOUT);
      tc_fence_after();
      // By halves of a block, two ahead: O += P V of a half as soon as its probabilities are there, then S of the next block's same half
      // into their place (products of one issuer run in order). The group meanwhile works on the other half.
      const int halves = 2 * ((nb - first + step - 1) / step);
#pragma unroll 1
      for (int t = 0; t < halves + 2 && ok; ++t) {
        const int hf = t & 1, j = first + (t >> 1) * step;
        if (t >= 2) {
          const unsigned g = gk + j - step;
          if (hf == 0) ok = pt_wait(&sh.v_full[g & 1], (g >> 1) & 1u, abort_flag, c.err, ERR_MBAR_FULL_TIMEOUT);
          if (ok) ok = pt_wait(&sh.p_ready[2 * w + hf], n_p, abort_flag, c.err, ERR_TMEM_TIMEOUT);
          if (!ok) break;
          tc_fence_after();
          pt_mma8<PT_PV>(tmem + 256 + w * 128, tmem + w * 128 + hf * 64, v_lo + (g & 1) * (PT_TILE >> 4) + hf * 512, idesc_v, t > 2);
          if constexpr (P2)
            pt_mma8<PT_PV>(tmem + 256 + w * 128, tmem + w * 128 + hf * 64 + 32, v_lo + (g & 1) * (PT_TILE >> 4) + hf * 512, idesc_v, 1);
          tc_commit(&sh.pv_done[2 * w + hf]);
          if (hf == 1) {
            n_p ^= 1u;
            tc_commit(&sh.v_empty[w][g & 1]);
          }
        }
        if (t < halves) {
          const unsigned g = gk + j;
          if (hf == 0) ok = pt_wait(&sh.k_full[g % KS], (g / KS) & 1u, abort_flag, c.err, ERR_MBAR_FULL_TIMEOUT);
          if (!ok) break;
          pt_mma8<KV8 ? PT_QK8 : PT_QK16>(tmem + w * 128 + hf * 64, q_lo + w * (PT_TILE >> 4), k_lo + (g % KS) * (K_BYTES >> 4) + hf * 512, idesc, 0);
          tc_commit(&sh.s_full[2 * w + hf]);
          mbar_arrive(&sh.s_full[2 * w + hf]); // hands on what the loader wrote beside the tile (the wait on k_full came before)
          if (hf == 1) tc_commit(&sh.k_empty[w][g % KS]);
        }
      }
      gk += nb;
      tc_commit(&sh.q_free);
      ++n_seg;
    }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {                           // products may be under way: what they use is given back after them
    if (tid == 0) descs[blockIdx.x].cont = PT_LOST;
    const int w = warp - PT_MMA_WARP;
    if ((w == 0 || w == 1) && lane == 0) {
      tc_commit(&sh.drain[w]);
      const unsigned long long t0 = globaltimer_ns();
      while (!mbar_try_wait(&sh.drain[w], 0) && globaltimer_ns() - t0 < IHB_LOCAL_WAIT_NS) {}
    }
    __syncthreads();
  }
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
  if (d.cont == PT_LOST) {
    // A wait of this CTA ran out, so its items are not all done: NaN for the call's tokens, so that no caller takes what the memory held for a result.
    const int t0 = a.c.cu_q != nullptr ? max(a.c.cu_q[0], 0) : 0, t1 = a.c.cu_q != nullptr ? min(a.c.cu_q[a.c.B], a.c.T) : a.c.T;
    const float nan = __uint_as_float(0x7fffffffu);
    for (int t = t0 + blockIdx.y; t < t1; t += gridDim.y)
      for (int h = warp; h < a.nq; h += 8) {
        pd_store4(a, t, h, lane * 4, make_float4(nan, nan, nan, nan));
        if (lane == 0 && a.lse != nullptr) a.lse[static_cast<size_t>(t) * a.nq + h] = nan;
      }
    return;
  }
  if (!d.tail) return;
  if (warp == 0) {
    int n = 1, lost = 0;
    if (lane == 0) list[0] = blockIdx.x * 2 + d.slot;
    for (int y0 = blockIdx.x + 1; y0 < grid; y0 += 32) {
      PtDesc e = {0, 0, 0, 0, 0, 0, 0, 0};
      if (y0 + lane < grid) e = descs[y0 + lane];
      const unsigned stop = __ballot_sync(0xffffffffu, e.ends || e.cont == 0 || e.cont == PT_LOST);
      const int upto = stop ? __ffs(stop) - 1 : 31;                    // (this lane included: the piece that ends the item)
      const unsigned mine = __ballot_sync(0xffffffffu, lane <= upto && e.cont == 2);
      if (lane <= upto && e.cont == 2) list[n + __popc(mine & ((1u << lane) - 1u))] = (y0 + lane) * 2;
      n += __popc(mine);
      lost = __any_sync(0xffffffffu, lane <= upto && e.cont == PT_LOST);
      if (stop) break;
    }
    if (lane == 0) n_s = lost ? 0 : n;
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
    if (n == 0) L = __uint_as_float(0x7fffffffu);                        // a piece is missing: NaN, as its CTA left for its own rows
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

template <bool KV8, bool P2>
static cudaError_t pt_launch(const IhbPagedAttn& a, cudaStream_t stream) {
  const int grid = PT_MAX_GRID, rec_rows = pt_rec_rows(a);             // one CTA per SM
  static_assert(sizeof(PtHdr) <= 1024, "header");
  static const int regs = [] {                 // the register split draws on what the block is launched with
    cudaFuncAttributes f;
    return cudaFuncGetAttributes(&f, paged_tiles_kernel<KV8, P2>) == cudaSuccess ? f.numRegs : 0;
  }();
  if (regs < PT_REGS) return cudaErrorInvalidConfiguration;
  constexpr int bytes = pt_smem<KV8>();
  cudaError_t e = cudaFuncSetAttribute(paged_tiles_kernel<KV8, P2>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return e;
  paged_tiles_kernel<KV8, P2><<<grid, PT_THREADS, bytes, stream>>>(a, grid, rec_rows);
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
  // Up to 128 rows the width of the block table chooses between this kernel and paged_attn.cu (use_tiles): both keep two terms of P over bf16 pages, so
  // that a wider table does not change the precision. Above, where every call comes here, a bf16 result takes one: that adds at most one more half
  // step of bf16 to the result's own (random inputs: 2.3e-3 from 64 bits against 1.65e-3), and the second product costs a sixth (prompt of 4096 tokens:
  // 200 us, 233 with two). An fp32 result always gets two.
  if (a.c.k_scale != nullptr) return pt_launch<true, false>(a, stream);
  const bool one = a.out_bf16 && static_cast<long long>(a.max_q) * (a.nq / a.c.nkv) > PT_M;
  return one ? pt_launch<false, false>(a, stream) : pt_launch<false, true>(a, stream);
}

}  // namespace ihb
