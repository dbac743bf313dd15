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

__device__ __forceinline__ unsigned char pg_e4m3(float x) {
  return static_cast<unsigned char>(__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3));
}

}  // namespace ihb
