// Shared pieces of the paged KV cache kernels: the sequence a token or a work unit belongs to, page lookup, fp8 rows.
#pragma once
#include "common.cuh"
#include "api.h"

namespace ihb {

constexpr int PG_HD = 128;
constexpr float PG_LOG2E = 1.4426950408889634f;
constexpr int PG_EMIN = -60, PG_EMAX = 60;      // exponents a page scale may have: their differences stay inside fp32

// One sequence of the call: rows [0, len) of its cache, tokens [t0, t0 + n) of the call, the first of them at row base.
struct PgSeq {
  int len, n, t0, base;
};

__device__ __forceinline__ PgSeq pg_seq(const IhbPaged& c, int b) {
  PgSeq s;
  s.len = c.kv_len[b];
  if (c.cu_q != nullptr) {
    s.t0 = min(max(c.cu_q[b], 0), c.T);
    s.n = max(min(c.cu_q[b + 1], c.T) - s.t0, 0);
  } else {
    s.t0 = b;
    s.n = 1;
  }
  const long long cap = static_cast<long long>(c.max_blocks) * c.page;
  if (s.len > cap) {                              // longer than its block table: the rows that fit are seen
    s.base = s.len - s.n;
    s.len = static_cast<int>(cap);
    set_error(c.err, ERR_BAD_ARGS);
    return s;
  }
  s.len = max(s.len, 0);
  s.base = s.len - s.n;
  return s;
}

__device__ __forceinline__ int warp_incl_scan(int v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// Sequence of token t (whole warp): sequences are in token order, so it is the last one that starts at or before t. Empty
// sequences share their start with the next one. Returns -1 behind the last sequence.
__device__ __forceinline__ int pg_seq_of_token(const IhbPaged& c, int t, int lane) {
  if (c.cu_q == nullptr) return t < c.B ? t : -1;
  int before = 0;                                 // sequences that end at or before t
  for (int b0 = 0; b0 < c.B; b0 += 32) {
    const int b = b0 + lane;
    before += __popc(__ballot_sync(0xffffffffu, b < c.B && c.cu_q[min(b, c.B - 1) + 1] <= t));
  }
  return before < c.B && t >= c.cu_q[before] ? before : -1;
}

// What both entry points ask of a cache block before anything is launched. Rows of a sequence are counted in 32 bits.
static inline bool paged_ok(const IhbPaged& c) {
  const bool page = c.page == 16 || c.page == 32 || c.page == 64 || c.page == 128;
  return page && c.k != nullptr && c.v != nullptr && (c.k_scale == nullptr) == (c.v_scale == nullptr) && c.n_pages > 0 && c.nkv > 0 &&
         c.nkv <= 4096 && c.B > 0 && c.T > 0 && c.max_blocks > 0 && c.max_blocks <= (1 << 30) / c.page && c.block_table != nullptr &&
         c.kv_len != nullptr && (c.cu_q != nullptr || c.B == c.T);
}

// a / b for 0 <= a < 2^62, b > 0, a quotient below 2^40: two steps in fp32, each leaves 2^-21 of the quotient, and whole corrections. (A 64-bit
// division, and one in fp64, are subroutines of some hundred dependent instructions, and laying out a segment took eight.)
__device__ __forceinline__ long long pg_div(long long a, long long b) {
  const float fb = static_cast<float>(b);
  long long q = static_cast<long long>(__fdividef(static_cast<float>(a), fb));
  q += static_cast<long long>(__fdividef(static_cast<float>(a - q * b), fb));
  while (q * b > a) --q;
  while ((q + 1) * b <= a) ++q;
  return q;
}
// ---- attention ------------------------------------------------------------------------------------------------------------------
constexpr float PD_OFF = 6.f;                // e4m3 pages: log2 of what a probability is scaled by (fp16 keeps more small ones)
constexpr float PD_LAZY = 8.f;               // the running maximum may be passed by 2^8 before the accumulators are rescaled
constexpr int PD_REC = PG_HD + 4;            // record of a row in a cut item: 128 channels, m, l, 2 pad

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
__device__ __forceinline__ void pd_cvt4(unsigned w, unsigned& lo, unsigned& hi) {     // four e4m3 bytes -> two pairs of fp16
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
}
__device__ __forceinline__ float pd_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// log2 of a page scale inside the range that append writes (a scale of 0 reads as the least one): the exponent from the bits, exact
// for powers of two, and the logarithm of the mantissa for other scales (lg2.approx on [1, 2): within 2^-22).
__device__ __forceinline__ float pd_log2_scale(float s) {
  const unsigned u = __float_as_uint(fminf(fmaxf(s, 8.673617379884035e-19f), 1.152921504606847e18f));
  float f;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(f) : "f"(__uint_as_float((u & 0x7fffffu) | 0x3f800000u)));
  return static_cast<float>(static_cast<int>(u >> 23) - 127) + f;
}

__device__ __forceinline__ void pd_store4(const IhbPagedAttn& a, int t, int h, int ch, float4 v) {
  const size_t o = static_cast<size_t>(t) * a.out_stride_t + static_cast<size_t>(h) * a.out_stride_h + ch;
  if (a.out_bf16) *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(a.out) + o) = make_uint2(pd_pack<false>(v.x, v.y), pd_pack<false>(v.z, v.w));
  else *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out) + o) = v;
}
// (m, l) of a finished row -> natural log of its denominator
template <bool KV8>
__device__ __forceinline__ float pd_lse(float m, float l) {
  return l > 0.f ? (m - (KV8 ? PD_OFF : 0.f) + log2f(l)) * 0.6931471805599453f : (l == 0.f ? -INFINITY : l);
}

}  // namespace ihb
