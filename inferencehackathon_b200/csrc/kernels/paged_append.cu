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

// Half a warp per row of 128 channels: lane c (0 .. 15) holds channels 4 c .. 4 c + 3 (x) and the same + 64 (y), the pairs of the
// rotation, in two loads of 16 (fp32) or 8 (bf16) bytes. With a warp per row the same work took twice the instructions.
struct PaRow {
  float x[4], y[4];
};
template <bool BF16>
__device__ __forceinline__ void pa_load4(const void* p, size_t i, float (&v)[4]) {
  if constexpr (BF16) {
    const uint2 r = *reinterpret_cast<const uint2*>(reinterpret_cast<const __nv_bfloat16*>(p) + i);
    v[0] = __uint_as_float(r.x << 16); v[1] = __uint_as_float(r.x & 0xffff0000u);
    v[2] = __uint_as_float(r.y << 16); v[3] = __uint_as_float(r.y & 0xffff0000u);
  } else {
    const float4 r = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
    v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w;
  }
}
__device__ __forceinline__ void pa_store4(void* p, bool bf16, size_t i, const float (&v)[4]) {
  if (bf16) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
    *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(p) + i) = make_uint2(*reinterpret_cast<const unsigned*>(&a), *reinterpret_cast<const unsigned*>(&b));
  } else {
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i) = make_float4(v[0], v[1], v[2], v[3]);
  }
}
template <bool BF16>
__device__ __forceinline__ void pa_load_row(PaRow& r, const void* p, size_t i, int c) {
  pa_load4<BF16>(p, i + 4 * c, r.x);
  pa_load4<BF16>(p, i + 64 + 4 * c, r.y);
}
// Norm (g: the lane's gammas, norm: whether there are any) and rotation of the two rows that a warp holds.
__device__ __forceinline__ void pa_norm_rope(PaRow& r, bool norm, const PaRow& g, float eps, const float (&cs)[4], const float (&sn)[4]) {
  if (norm) {
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) ss += r.x[j] * r.x[j] + r.y[j] * r.y[j];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float rinv = rsqrtf(ss * (1.f / PG_HD) + eps);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      r.x[j] *= rinv * g.x[j];
      r.y[j] *= rinv * g.y[j];
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float a = r.x[j], b = r.y[j];
    r.x[j] = a * cs[j] - b * sn[j];
    r.y[j] = b * cs[j] + a * sn[j];
  }
}

// K rows of e4m3 pages: in fp32 about one byte of a million falls on the wrong side of a tie, a whole step off. How far a value x of a rotated
// pair (x, y) may be from the exact one, in units of 2^-24: the norm's factor 10 |x| (a sum of 128 squares, 10 roundings deep, halved by the root; eps;
// rsqrtf 2 ulp), its products and the gammas' 2 M, the rotation's M + |x|, with M = |a c| + |b s| <= sqrt(x^2 + y^2) <= |x| + |y|, for any c and s.
// A row in which that decides the byte of a value, or the scale of the page, is done again in 64 bits: bytes and scales are those of
// exact arithmetic, whatever the call's size. 0.7 % of random rows are. (Decode step of 64 tokens, 4 heads: 5.7 us, 5.1 without; 8 K tokens: 71.5,
// 67.6 without, 90 with all rows in 64 bits.)
constexpr float PA_ULP = 5.9604645e-08f;                     // 2^-24
struct PaError {
  float x, y;                                                 // factors of |x| and |y|
  __device__ __forceinline__ explicit PaError(bool norm) : x((norm ? 15.f : 3.f) * PA_ULP), y((norm ? 4.f : 2.f) * PA_ULP) {}
};
// Rounded to odd (an inexact value has its last bit set): rounding that to e4m3 gives what rounding d itself gives.
__device__ __forceinline__ float pa_odd(double d) {
  const float f = __double2float_rn(d);
  if (!(fabsf(f) <= 3.4028235e38f) || static_cast<double>(f) == d) return f;
  return __uint_as_float(__float_as_uint(__double2float_rz(d)) | 1u);
}
template <bool BF16>
__device__ __forceinline__ PaRow pa_row64(const void* src, size_t at, const float* gamma, float eps, const float* cos_r, const float* sin_r, int c) {
  PaRow r, g = {};
  float cs[4], sn[4];
  pa_load_row<BF16>(r, src, at, c);
  pa_load4<false>(cos_r, 4 * c, cs);
  pa_load4<false>(sin_r, 4 * c, sn);
  double rinv = 1.;
  if (gamma != nullptr) {
    pa_load_row<false>(g, gamma, 0, c);
    double ss = 0.;
#pragma unroll
    for (int j = 0; j < 4; ++j) ss += static_cast<double>(r.x[j]) * r.x[j] + static_cast<double>(r.y[j]) * r.y[j];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const double v = ss * (1. / PG_HD) + static_cast<double>(eps);
    rinv = rsqrtf(static_cast<float>(v));                     // 2^-22; each of Newton's steps squares that
#pragma unroll
    for (int i = 0; i < 2; ++i) rinv += rinv * (0.5 - 0.5 * v * rinv * rinv);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const double a = gamma != nullptr ? r.x[j] * rinv * g.x[j] : r.x[j], b = gamma != nullptr ? r.y[j] * rinv * g.y[j] : r.y[j];
    r.x[j] = pa_odd(a * cs[j] - b * sn[j]);
    r.y[j] = pa_odd(b * cs[j] + a * sn[j]);
  }
  return r;
}

// Least e with amax <= 448 * 2^e (448 = 1.75 * 2^8), from the bits of amax >= 0, finite.
__device__ __forceinline__ int pa_exponent(float amax) {
  const unsigned u = __float_as_uint(amax);
  const int e = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, PG_EMIN), PG_EMAX);
}
__device__ __forceinline__ unsigned pa_e4m3x4(float x, float y, float z, float w, float f) {
  return static_cast<unsigned>(__nv_cvt_float2_to_fp8x2(make_float2(x * f, y * f), __NV_SATFINITE, __NV_E4M3)) |
         static_cast<unsigned>(__nv_cvt_float2_to_fp8x2(make_float2(z * f, w * f), __NV_SATFINITE, __NV_E4M3)) << 16;
}
// Does the error of a value decide its byte? inv: 1 / scale of the page.
__device__ __forceinline__ bool pa_unsure(const PaRow& r, const PaError& e, float inv) {
  bool any = false;
#pragma unroll
  for (int j = 0; j < 4; j += 2) {
    float lo[4], hi[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float x = r.x[j + i] * inv, y = r.y[j + i] * inv;
      const float dx = fabsf(x) * e.x + fabsf(y) * e.y, dy = fabsf(y) * e.x + fabsf(x) * e.y;
      lo[i] = x - dx; hi[i] = x + dx;
      lo[2 + i] = y - dy; hi[2 + i] = y + dy;
    }
    any |= pa_e4m3x4(lo[0], lo[1], lo[2], lo[3], 1.f) != pa_e4m3x4(hi[0], hi[1], hi[2], hi[3], 1.f);
  }
  return any;
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

// Blocks [0, kv_blocks): one (segment, KV head, K or V) each; 2 * RPW rows per warp cover the page. The others: hq query heads of one
// token per warp, two at a time.
template <bool BF16, bool KV8, int RPW>
__global__ void __launch_bounds__(PA_WARPS * 32, RPW == 1 ? 4 : RPW == 8 ? 2 : 3) paged_append_kernel(const __grid_constant__ IhbPagedAppend a, int kv_blocks, int hq) {
  __shared__ float red[PA_WARPS];
  const IhbPaged& c = a.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, half = lane >> 4, ch = lane & 15;
  const int nq = a.nq, nkv = c.nkv;
  if (static_cast<int>(blockIdx.x) >= kv_blocks) {
    // (launched for itself, this part runs beside the pages' part: it waits for that one only before it ends)
    struct AtEnd { __device__ ~AtEnd() { pdl_wait(); } } at_end;
    const int groups = (nq + hq - 1) / hq;
    const long long w = static_cast<long long>(blockIdx.x - kv_blocks) * PA_WARPS + warp;
    const int t = static_cast<int>(w / groups), h0 = static_cast<int>(w % groups) * hq, h1 = min(nq, h0 + hq);
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
    float cs[4], sn[4];
    pa_load4<false>(a.cos_t, static_cast<size_t>(pos) * 64 + 4 * ch, cs);
    pa_load4<false>(a.sin_t, static_cast<size_t>(pos) * 64 + 4 * ch, sn);
    const bool norm = a.q_gamma != nullptr;
    PaRow g = {};
    if (norm) pa_load_row<false>(g, a.q_gamma, 0, ch);
    void* dst = a.q_out != nullptr ? a.q_out : a.qkv;
    const bool dbf = a.q_out != nullptr ? a.q_bf16 != 0 : BF16;
    const size_t src0 = static_cast<size_t>(t) * a.qkv_stride;
    const size_t dst0 = a.q_out != nullptr ? static_cast<size_t>(t) * a.q_stride : src0;
    for (int h = h0; h < h1; h += 8) {                      // eight rows in flight
      PaRow r[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int hh = h + 2 * i + half;
        r[i] = {};
        if (hh < h1) pa_load_row<BF16>(r[i], a.qkv, src0 + static_cast<size_t>(hh) * PG_HD, ch);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int hh = h + 2 * i + half;
        if (h + 2 * i >= h1) break;
        pa_norm_rope(r[i], norm, g, a.eps, cs, sn);
        if (hh >= h1) continue;
        const size_t o = dst0 + static_cast<size_t>(hh) * PG_HD + 4 * ch;
        pa_store4(dst, dbf, o, r[i].x);
        pa_store4(dst, dbf, o + 64, r[i].y);
      }
    }
    return;
  }
  pdl_launch_dependents();
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
  const bool norm = a.k_gamma != nullptr && !is_v;
  PaRow x[RPW], g = {};
  if (norm) pa_load_row<false>(g, a.k_gamma, 0, ch);
  unsigned live = 0;                                         // bit i: row 2 (warp + PA_WARPS i) + half is written
  float amax = 0.f;
  auto take_amax = [&](const PaRow& v) {                     // infinities saturate, NaN stays NaN: neither sets the scale
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float s = fabsf(v.x[j]), t = fabsf(v.y[j]);
      if (s <= 3.4028235e38f) amax = fmaxf(amax, s);
      if (t <= 3.4028235e38f) amax = fmaxf(amax, t);
    }
  };
#pragma unroll
  for (int i = 0; i < RPW; ++i) {
    const int r = 2 * (warp + PA_WARPS * i) + half;
    x[i] = {};
    if (r < rows) {
      live |= 1u << i;
      pa_load_row<BF16>(x[i], a.qkv, static_cast<size_t>(tok0 + r) * a.qkv_stride + static_cast<size_t>(nq + (is_v ? nkv : 0) + h) * PG_HD, ch);
    }
  }
#pragma unroll
  for (int i = 0; i < RPW; ++i) {
    const int r = 2 * (warp + PA_WARPS * i) + half;
    if (2 * (warp + PA_WARPS * i) >= rows) break;            // (the same for the whole warp: the norm is a warp's work)
    float cs[4] = {}, sn[4] = {};
    if (r < rows) {
      const int pos = a.positions != nullptr ? a.positions[tok0 + r] : first + r;
      if (pos < 0 || pos >= a.n_pos) {
        if (ch == 0) set_error(c.err, ERR_BAD_ARGS);
        live &= ~(1u << i);
      } else if (!is_v) {
        pa_load4<false>(a.cos_t, static_cast<size_t>(pos) * 64 + 4 * ch, cs);
        pa_load4<false>(a.sin_t, static_cast<size_t>(pos) * 64 + 4 * ch, sn);
      }
    }
    if (!is_v) pa_norm_rope(x[i], norm, g, a.eps, cs, sn);
    if (KV8 && (live >> i & 1)) take_amax(x[i]);
  }
  if constexpr (!KV8) {
    void* dst = is_v ? c.v : c.k;
#pragma unroll
    for (int i = 0; i < RPW; ++i) {
      if (!(live >> i & 1)) continue;
      const size_t o = (head_row + r0 + 2 * (warp + PA_WARPS * i) + half) * PG_HD + 4 * ch;
      pa_store4(dst, true, o, x[i].x);
      pa_store4(dst, true, o + 64, x[i].y);
    }
  } else {
    unsigned char* dst = reinterpret_cast<unsigned char*>(is_v ? c.v : c.k);
    float* sc = (is_v ? c.v_scale : c.k_scale) + static_cast<size_t>(page) * nkv + h;
    const float old = r0 > 0 ? *sc : 0.f;
    auto block_amax = [&]() {
      amax = warp_max(amax);
      if (lane == 0) red[warp] = amax;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < PA_WARPS; ++w) amax = fmaxf(amax, red[w]);
    };
    auto move = [&](float now) {                              // rows of earlier calls move to a larger scale
      if (r0 == 0 || !(now > old)) return;
      const float f = old / now;
      uint2* rowp = reinterpret_cast<uint2*>(dst + head_row * PG_HD);
      for (int i = tid; i < r0 * (PG_HD / 8); i += PA_WARPS * 32) {
        const uint2 w = rowp[i];
        const float4 p = e4m3x4_to_float4(w.x), q = e4m3x4_to_float4(w.y);
        rowp[i] = make_uint2(pa_e4m3x4(p.x, p.y, p.z, p.w, f), pa_e4m3x4(q.x, q.y, q.z, q.w, f));
      }
    };
    auto put = [&](int i, const PaRow& v, float inv) {
      unsigned char* o = dst + (head_row + r0 + 2 * (warp + PA_WARPS * i) + half) * PG_HD + 4 * ch;
      *reinterpret_cast<unsigned*>(o) = pa_e4m3x4(v.x[0], v.x[1], v.x[2], v.x[3], inv);
      *reinterpret_cast<unsigned*>(o + 64) = pa_e4m3x4(v.y[0], v.y[1], v.y[2], v.y[3], inv);
    };
    auto row64 = [&](int i) {                                 // (whole warp; a dead half does row 0 of the call's part along, and drops it)
      const int r = live >> i & 1 ? 2 * (warp + PA_WARPS * i) + half : 0;
      const int pos = live >> i & 1 ? (a.positions != nullptr ? a.positions[tok0 + r] : first + r) : 0;
      return pa_row64<BF16>(a.qkv, static_cast<size_t>(tok0 + r) * a.qkv_stride + static_cast<size_t>(nq + h) * PG_HD, a.k_gamma, a.eps,
                            a.cos_t + static_cast<size_t>(pos) * 64, a.sin_t + static_cast<size_t>(pos) * 64, ch);
    };
    block_amax();
    const PaError e(norm);
    const float d = (e.x + e.y) * amax;
    float now;
    unsigned again = 0;                                       // rows to be done in 64 bits, the same for the warp. Behind everything else: the rows in registers
                                                              // need not outlive a call, which costs a block its place on the SM
    if (is_v || pa_exponent(amax - d) == pa_exponent(amax + d)) {
      now = fmaxf(old, pa_pow2(pa_exponent(amax)));
      const float inv = 1.f / now;
      move(now);
#pragma unroll
      for (int i = 0; i < RPW; ++i) {
        if (live >> i & 1) put(i, x[i], inv);
        if (!is_v && __any_sync(0xffffffffu, (live >> i & 1) && pa_unsure(x[i], e, inv))) again |= 1u << i;
      }
    } else {                                                  // one page of 250 thousand, the same for the whole block
      amax = 0.f;
#pragma unroll 1
      for (int i = 0; i < RPW && 2 * (warp + PA_WARPS * i) < rows; ++i) {
        const PaRow v = row64(i);
        if (live >> i & 1) take_amax(v);
        again |= 1u << i;
      }
      __syncthreads();                                        // (red has been read)
      block_amax();
      now = fmaxf(old, pa_pow2(pa_exponent(amax)));
      move(now);
    }
#pragma unroll 1
    for (; again; again &= again - 1) {
      const int i = __ffs(again) - 1;
      const PaRow v = row64(i);
      if (live >> i & 1) put(i, v, 1.f / now);
    }
    if (tid == 0) *sc = now;
  }
}

template <bool BF16, bool KV8>
static void paged_append_launch(const IhbPagedAppend& a, int grid, int kv_blocks, int hq, cudaStream_t stream) {
  // Large pages hold many rows per thread between the maximum and the rounding: 120 registers for 128-token pages, which leaves the query
  // rows, most of the traffic, too few warps per SM. Where there are many they get a launch of their own at 64 registers, which need
  // not wait for the pages' part (8 K tokens of 64 / 4 heads: 97 us in one launch, 72 in two one after the other).
  const bool apart = hq == 16 && a.c.page >= 64;
  const int blocks = apart ? kv_blocks : grid;
  switch (a.c.page) {
    case 16: paged_append_kernel<BF16, KV8, 1><<<blocks, PA_WARPS * 32, 0, stream>>>(a, kv_blocks, hq); break;
    case 32: paged_append_kernel<BF16, KV8, 2><<<blocks, PA_WARPS * 32, 0, stream>>>(a, kv_blocks, hq); break;
    case 64: paged_append_kernel<BF16, KV8, 4><<<blocks, PA_WARPS * 32, 0, stream>>>(a, kv_blocks, hq); break;
    default: paged_append_kernel<BF16, KV8, 8><<<blocks, PA_WARPS * 32, 0, stream>>>(a, kv_blocks, hq); break;
  }
  if (!apart) return;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(grid - kv_blocks);
  cfg.blockDim = dim3(PA_WARPS * 32);
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, paged_append_kernel<BF16, KV8, 1>, a, 0, hq);
}

}  // namespace ihb

using namespace ihb;

extern "C" int ihb_paged_append(const IhbPagedAppend* p, cudaStream_t stream) {
  const IhbPagedAppend& a = *p;
  const IhbPaged& c = a.c;
  if (!paged_ok(c) || a.qkv == nullptr || a.nq < 1 || a.n_pos < 1 || (a.q_gamma == nullptr) != (a.k_gamma == nullptr) ||
      a.qkv_stride % 8 || a.q_stride % 8)
    return cudaErrorInvalidValue;
  // pages that n tokens of a sequence touch: at most (n - 1) / page + 2, and no more than tokens
  long long segs = c.cu_q == nullptr ? c.B : static_cast<long long>(c.T) / c.page + 2ll * c.B;
  if (segs > c.T) segs = c.T;
  const long long kv_blocks = segs * 2 * c.nkv;
  // heads per warp: eight (one round of loads) or sixteen where that still leaves every SM blocks to choose from; two where tokens are few
  const long long pairs = static_cast<long long>(c.T) * a.nq;
  const int hq = pairs >= 148ll * 64 * 16 ? 16 : pairs >= 148ll * 8 * 16 ? 8 : 2;
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
