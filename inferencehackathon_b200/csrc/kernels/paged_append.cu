// Append to a paged KV cache: per-head QK RMSNorm (optional), NeoX RoPE, K / V rows into their pages, for a ragged batch of
// decode tokens and prompt chunks. The contiguous siblings are attn.cu::qk_norm_rope_kv_kernel (one token) and
// window.cu::qk_norm_rope_rows_kernel (one sequence).
//
// Scale of an e4m3 page = 2^e, e the least exponent with amax / 448 <= 2^e over the rows of the page (per head). A power of two
// costs nothing against amax / 448 itself (e4m3 is a floating format: the relative step does not depend on the scale, only
// the subnormal range loses up to one bit) and makes the running maximum exact: rows already in the page are moved to a larger scale by
// an exponent shift, so a page filled token by token holds the bytes of a page filled at once, subnormals apart. One
// block owns the rows that the call writes to one (page, head, K or V): the maximum needs no atomics and no second pass, the rows
// stay in registers between the maximum and the rounding.
#include "paged.cuh"

namespace ihb {

constexpr int PA_WARPS = 8;

template <bool BF16>
__device__ __forceinline__ float2 pa_load2(const void* p, size_t i) {
  if constexpr (BF16) {
    const unsigned r = *reinterpret_cast<const unsigned*>(reinterpret_cast<const __nv_bfloat16*>(p) + i);
    return make_float2(__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u));
  } else {
    return *reinterpret_cast<const float2*>(reinterpret_cast<const float*>(p) + i);
  }
}
__device__ __forceinline__ void pa_store2(void* p, bool bf16, size_t i, float x, float y) {
  if (bf16) *reinterpret_cast<__nv_bfloat162*>(reinterpret_cast<__nv_bfloat16*>(p) + i) = __floats2bfloat162_rn(x, y);
  else *reinterpret_cast<float2*>(reinterpret_cast<float*>(p) + i) = make_float2(x, y);
}

// One warp, one row of 128 channels: lane holds channels 2 lane, 2 lane + 1 (x) and the same + 64 (y): the pairs of the rotation.
struct PaRow {
  float2 x, y;
};
template <bool BF16>
__device__ __forceinline__ PaRow pa_load_row(const void* p, size_t i, int lane) {
  return {pa_load2<BF16>(p, i + 2 * lane), pa_load2<BF16>(p, i + 64 + 2 * lane)};
}
__device__ __forceinline__ void pa_norm_rope(PaRow& r, const float* __restrict__ gamma, float eps, float2 c, float2 s, int lane) {
  if (gamma != nullptr) {
    const float ss = warp_sum(r.x.x * r.x.x + r.x.y * r.x.y + r.y.x * r.y.x + r.y.y * r.y.y);
    const float rinv = rsqrtf(ss * (1.f / PG_HD) + eps);
    const float2 g0 = *reinterpret_cast<const float2*>(gamma + 2 * lane), g1 = *reinterpret_cast<const float2*>(gamma + 64 + 2 * lane);
    r.x.x *= rinv * g0.x; r.x.y *= rinv * g0.y;
    r.y.x *= rinv * g1.x; r.y.y *= rinv * g1.y;
  }
  const float2 a = r.x, b = r.y;
  r.x = make_float2(a.x * c.x - b.x * s.x, a.y * c.y - b.y * s.y);
  r.y = make_float2(b.x * c.x + a.x * s.x, b.y * c.y + a.y * s.y);
}

// Least e with amax <= 448 * 2^e (448 = 1.75 * 2^8), from the bits of amax >= 0, finite.
__device__ __forceinline__ int pa_exponent(float amax) {
  const unsigned u = __float_as_uint(amax);
  const int e = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, PG_EMIN), PG_EMAX);
}
__device__ __forceinline__ float pa_pow2(int e) { return __uint_as_float(static_cast<unsigned>(e + 127) << 23); }

// The sequence and page of segment `seg` (whole warp). A segment is the part of one page that the call writes. Returns false when
// there are fewer segments. first: row of the sequence at which the segment begins, rows: how many.
__device__ __forceinline__ bool pa_segment(const IhbPaged& c, int seg, int lane, PgSeq& s, int& b, int& first, int& rows) {
  const int sh = __ffs(c.page) - 1;
  int pg;
  if (c.cu_q == nullptr) {
    if (seg >= c.B) return false;
    b = seg;
    s = pg_seq(c, b);
    if (s.len < 1 || s.base >= s.len) return false;       // a padding entry, or one that its table does not hold
    pg = s.base >> sh;
  } else {
    bool found = false;
    int left = seg;
    for (int b0 = 0; b0 < c.B && !found; b0 += 32) {
      PgSeq t = {0, 0, 0, 0};
      if (b0 + lane < c.B) t = pg_seq(c, b0 + lane);
      const int lo = max(t.base, 0);
      const int cnt = (t.n > 0 && t.len > lo) ? ((t.len - 1) >> sh) - (lo >> sh) + 1 : 0;
      const int incl = warp_incl_scan(cnt, lane);
      const unsigned hit = __ballot_sync(0xffffffffu, incl > left);
      if (hit) {
        const int src = __ffs(hit) - 1;
        b = b0 + src;
        s.len = __shfl_sync(0xffffffffu, t.len, src);
        s.n = __shfl_sync(0xffffffffu, t.n, src);
        s.t0 = __shfl_sync(0xffffffffu, t.t0, src);
        s.base = __shfl_sync(0xffffffffu, t.base, src);
        left -= __shfl_sync(0xffffffffu, incl - cnt, src);
        found = true;
      } else {
        left -= __shfl_sync(0xffffffffu, incl, 31);
      }
    }
    if (!found) return false;
    pg = (max(s.base, 0) >> sh) + left;
  }
  first = max(max(s.base, 0), pg << sh);
  rows = min(s.len, (pg + 1) << sh) - first;
  return rows > 0;
}

// Blocks [0, kv_blocks): one (segment, KV head, K or V) each; RPW rows per warp cover the page. The others: HQ query heads of one
// token per warp.
template <bool BF16, bool KV8, int RPW>
__global__ void __launch_bounds__(PA_WARPS * 32) paged_append_kernel(const __grid_constant__ IhbPagedAppend a, int kv_blocks, int hq) {
  __shared__ float red[PA_WARPS];
  const IhbPaged& c = a.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nq = a.nq, nkv = c.nkv;
  if (static_cast<int>(blockIdx.x) >= kv_blocks) {
    const int groups = (nq + hq - 1) / hq;
    const long long w = static_cast<long long>(blockIdx.x - kv_blocks) * PA_WARPS + warp;
    const int t = static_cast<int>(w / groups), h0 = static_cast<int>(w % groups) * hq;
    if (t >= c.T) return;
    const int b = pg_seq_of_token(c, t, lane);
    if (b < 0) return;
    const PgSeq s = pg_seq(c, b);
    const int row = s.base + (t - s.t0);
    if (s.len < 1) return;                                  // padding entry
    const int pos = a.positions != nullptr ? a.positions[t] : row;
    if (row < 0 || pos < 0 || pos >= a.n_pos) {
      if (lane == 0) set_error(c.err, ERR_BAD_ARGS);
      return;
    }
    const float2 cs = *reinterpret_cast<const float2*>(a.cos_t + static_cast<size_t>(pos) * 64 + 2 * lane);
    const float2 sn = *reinterpret_cast<const float2*>(a.sin_t + static_cast<size_t>(pos) * 64 + 2 * lane);
    void* dst = a.q_out != nullptr ? a.q_out : a.qkv;
    const bool dbf = a.q_out != nullptr ? a.q_bf16 != 0 : BF16;
    const size_t src0 = static_cast<size_t>(t) * a.qkv_stride;
    const size_t dst0 = a.q_out != nullptr ? static_cast<size_t>(t) * a.q_stride : src0;
    for (int h = h0; h < min(nq, h0 + hq); h += 4) {        // four rows in flight
      PaRow r[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (h + i < min(nq, h0 + hq)) r[i] = pa_load_row<BF16>(a.qkv, src0 + static_cast<size_t>(h + i) * PG_HD, lane);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (h + i >= min(nq, h0 + hq)) break;
        pa_norm_rope(r[i], a.q_gamma, a.eps, cs, sn, lane);
        const size_t o = dst0 + static_cast<size_t>(h + i) * PG_HD + 2 * lane;
        pa_store2(dst, dbf, o, r[i].x.x, r[i].x.y);
        pa_store2(dst, dbf, o + 64, r[i].y.x, r[i].y.y);
      }
    }
    return;
  }
  const int seg = blockIdx.x / (2 * nkv), which = blockIdx.x % (2 * nkv);
  const int h = which >> 1;
  const bool is_v = which & 1;
  PgSeq s;
  int b, first, rows;
  if (!pa_segment(c, seg, lane, s, b, first, rows)) return;  // the same for every warp of the block
  const int page = c.block_table[static_cast<size_t>(b) * c.table_stride + first / c.page];
  if (page < 0 || page >= c.n_pages) {
    if (tid == 0) set_error(c.err, ERR_BAD_ARGS);
    return;
  }
  if (s.base < 0 && tid == 0) set_error(c.err, ERR_BAD_ARGS);
  const int r0 = first % c.page, tok0 = s.t0 + (first - s.base);
  const size_t head_row = (static_cast<size_t>(page) * nkv + h) * c.page;
  PaRow x[RPW];
  bool live[RPW];
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < RPW; ++i) {
    const int r = warp + PA_WARPS * i;
    live[i] = r < rows;
    if (live[i])
      x[i] = pa_load_row<BF16>(a.qkv, static_cast<size_t>(tok0 + r) * a.qkv_stride + static_cast<size_t>(nq + (is_v ? nkv : 0) + h) * PG_HD, lane);
  }
#pragma unroll
  for (int i = 0; i < RPW; ++i) {
    const int r = warp + PA_WARPS * i;
    if (!live[i]) continue;
    const int pos = a.positions != nullptr ? a.positions[tok0 + r] : first + r;
    if (pos < 0 || pos >= a.n_pos) {
      if (lane == 0) set_error(c.err, ERR_BAD_ARGS);
      live[i] = false;
      continue;
    }
    if (!is_v)
      pa_norm_rope(x[i], a.k_gamma, a.eps, *reinterpret_cast<const float2*>(a.cos_t + static_cast<size_t>(pos) * 64 + 2 * lane),
                   *reinterpret_cast<const float2*>(a.sin_t + static_cast<size_t>(pos) * 64 + 2 * lane), lane);
    if constexpr (KV8) {
      const float v[4] = {fabsf(x[i].x.x), fabsf(x[i].x.y), fabsf(x[i].y.x), fabsf(x[i].y.y)};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (v[j] <= 3.4028235e38f) amax = fmaxf(amax, v[j]);   // infinities saturate, NaN stays NaN: neither sets the scale
    }
  }
  if constexpr (!KV8) {
    __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(is_v ? c.v : c.k);
#pragma unroll
    for (int i = 0; i < RPW; ++i) {
      if (!live[i]) continue;
      const size_t o = (head_row + r0 + warp + PA_WARPS * i) * PG_HD + 2 * lane;
      pa_store2(dst, true, o, x[i].x.x, x[i].x.y);
      pa_store2(dst, true, o + 64, x[i].y.x, x[i].y.y);
    }
  } else {
    unsigned char* dst = reinterpret_cast<unsigned char*>(is_v ? c.v : c.k);
    float* sc = (is_v ? c.v_scale : c.k_scale) + static_cast<size_t>(page) * nkv + h;
    amax = warp_max(amax);
    if (lane == 0) red[warp] = amax;
    const float old = r0 > 0 ? *sc : 0.f;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < PA_WARPS; ++w) amax = fmaxf(amax, red[w]);
    const float now = fmaxf(old, pa_pow2(pa_exponent(amax)));
    const float inv = 1.f / now;
    if (r0 > 0 && now > old) {                                // rows of earlier calls move to the larger scale
      const float f = old * inv;
      uint2* rowp = reinterpret_cast<uint2*>(dst + head_row * PG_HD);
      for (int i = tid; i < r0 * (PG_HD / 8); i += PA_WARPS * 32) {
        const uint2 w = rowp[i];
        unsigned o[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float4 q = e4m3x4_to_float4(u ? w.y : w.x);
          o[u] = static_cast<unsigned>(__nv_cvt_float2_to_fp8x2(make_float2(q.x * f, q.y * f), __NV_SATFINITE, __NV_E4M3)) |
                 static_cast<unsigned>(__nv_cvt_float2_to_fp8x2(make_float2(q.z * f, q.w * f), __NV_SATFINITE, __NV_E4M3)) << 16;
        }
        rowp[i] = make_uint2(o[0], o[1]);
      }
    }
#pragma unroll
    for (int i = 0; i < RPW; ++i) {
      if (!live[i]) continue;
      unsigned char* o = dst + (head_row + r0 + warp + PA_WARPS * i) * PG_HD + 2 * lane;
      *reinterpret_cast<unsigned short*>(o) = __nv_cvt_float2_to_fp8x2(make_float2(x[i].x.x * inv, x[i].x.y * inv), __NV_SATFINITE, __NV_E4M3);
      *reinterpret_cast<unsigned short*>(o + 64) = __nv_cvt_float2_to_fp8x2(make_float2(x[i].y.x * inv, x[i].y.y * inv), __NV_SATFINITE, __NV_E4M3);
    }
    if (tid == 0) *sc = now;
  }
}

static bool paged_ok(const IhbPaged& c) {
  const bool page = c.page == 16 || c.page == 32 || c.page == 64 || c.page == 128;
  return page && c.k != nullptr && c.v != nullptr && (c.k_scale == nullptr) == (c.v_scale == nullptr) && c.n_pages > 0 && c.nkv > 0 &&
         c.B > 0 && c.T > 0 && c.max_blocks > 0 && c.block_table != nullptr && c.kv_len != nullptr && (c.cu_q != nullptr || c.B == c.T);
}

template <bool BF16, bool KV8>
static void paged_append_launch(const IhbPagedAppend& a, int grid, int kv_blocks, int hq, cudaStream_t stream) {
  switch (a.c.page) {
    case 16: paged_append_kernel<BF16, KV8, 2><<<grid, PA_WARPS * 32, 0, stream>>>(a, kv_blocks, hq); break;
    case 32: paged_append_kernel<BF16, KV8, 4><<<grid, PA_WARPS * 32, 0, stream>>>(a, kv_blocks, hq); break;
    case 64: paged_append_kernel<BF16, KV8, 8><<<grid, PA_WARPS * 32, 0, stream>>>(a, kv_blocks, hq); break;
    default: paged_append_kernel<BF16, KV8, 16><<<grid, PA_WARPS * 32, 0, stream>>>(a, kv_blocks, hq); break;
  }
}

}  // namespace ihb

using namespace ihb;

extern "C" int ihb_paged_append(const IhbPagedAppend* p, cudaStream_t stream) {
  const IhbPagedAppend& a = *p;
  const IhbPaged& c = a.c;
  if (!paged_ok(c) || a.qkv == nullptr || a.nq < 1 || a.n_pos < 1 || (a.q_gamma == nullptr) != (a.k_gamma == nullptr) ||
      a.qkv_stride % 2 || a.q_stride % 2)
    return cudaErrorInvalidValue;
  // pages that n tokens of a sequence touch: at most (n - 1) / page + 2, and no more than tokens
  long long segs = c.cu_q == nullptr ? c.B : static_cast<long long>(c.T) / c.page + 2ll * c.B;
  if (segs > c.T) segs = c.T;
  const long long kv_blocks = segs * 2 * c.nkv;
  // four heads per warp where that still leaves every SM a few blocks; one where tokens are few
  const int hq = static_cast<long long>(c.T) * a.nq >= 148ll * 8 * 16 ? 8 : 1;
  const long long q_warps = static_cast<long long>(c.T) * ((a.nq + hq - 1) / hq);
  const long long grid = kv_blocks + (q_warps + PA_WARPS - 1) / PA_WARPS;
  if (grid > 0x7fffffffll) return cudaErrorInvalidValue;
  const bool kv8 = c.k_scale != nullptr;
  if (a.qkv_bf16) {
    if (kv8) paged_append_launch<true, true>(a, static_cast<int>(grid), static_cast<int>(kv_blocks), hq, stream);
    else paged_append_launch<true, false>(a, static_cast<int>(grid), static_cast<int>(kv_blocks), hq, stream);
  } else {
    if (kv8) paged_append_launch<false, true>(a, static_cast<int>(grid), static_cast<int>(kv_blocks), hq, stream);
    else paged_append_launch<false, false>(a, static_cast<int>(grid), static_cast<int>(kv_blocks), hq, stream);
  }
  return cudaGetLastError();
}
