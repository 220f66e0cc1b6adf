// The paged 8-bit key/value cache: writing new tokens and following the
// hypotheses of a beam search.
//
// A page holds `page` tokens; for each head its codes are page * D contiguous
// bytes of e4m3 under one scale 2^e. For values A let need(A) be the smallest
// integer e >= -126 with max |A| <= 448 * 2^e. Tokens X written to a page that
// holds codes c at 2^e0 give
//   e = max(e0, need(X)),  c <- e4m3(c 2^(e0 - e)),  new = e4m3(x 2^-e),
// and e = need(X) where the page holds no token yet. A power of two costs an
// e4m3 value nothing (its precision is relative), makes the change of scale
// exact but for codes that become subnormal, and lets attention apply the
// scale without a rounding. Infinities take the largest code; a NaN is stored
// as zero and recorded in the error word, so a cache holds finite values only.
#include "common.cuh"
#include "decode.h"

namespace pkc {

namespace {

// two floats -> two e4m3 codes (the first in the low byte), to nearest even,
// saturating
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 from_e4m3x2(uint32_t w) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)w));
  return __half22float2(*reinterpret_cast<__half2*>(&r));
}
__device__ __forceinline__ float exp2i(int e) {  // 2^e, e in [-126, 127]; 0 below
  return e < -126 ? 0.f : __int_as_float((e + 127) << 23);
}
__device__ __forceinline__ int exponent_of(float x) { return ((__float_as_int(x) >> 23) & 255) - 127; }

// need() of a largest value (finite, >= 0): 448 = 1.75 * 2^8
__device__ __forceinline__ int need_exp(float most) {
  const int bits = __float_as_int(most);
  const int e = (bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
  return e < -126 ? -126 : e;
}

// rescale eight codes by f
__device__ __forceinline__ uint2 rescale8(uint2 c, float f) {
  uint32_t w[2] = {c.x, c.y};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float2 a = from_e4m3x2(w[i] & 0xffffu), b = from_e4m3x2(w[i] >> 16);
    w[i] = to_e4m3x2(a.x * f, a.y * f) | to_e4m3x2(b.x * f, b.y * f) << 16;
  }
  return make_uint2(w[0], w[1]);
}

// One group of T threads (a warp or a CTA) writes one page's new tokens of one
// head, keys or values: D / 8 vectors of 8 values a token.
template <typename H, int T>
__global__ void __launch_bounds__(128) k_kv8_append(const Kv8AppendArgs a, int width, long long units) {
  constexpr int kGroups = 128 / T;
  __shared__ float s_max[4];
  const long long unit = (long long)blockIdx.x * kGroups + threadIdx.x / T;
  const int lane = threadIdx.x % T;
  pdl_wait();
  pdl_trigger();
  if (unit >= units) return;
  const Kv8& c = a.c;
  const int D = c.head_dim, vec = D / 8;
  const int x = (int)(unit % 2);  // 0 keys, 1 values
  long long rest = unit / 2;
  const int h = (int)(rest % c.n_kv_heads);
  rest /= c.n_kv_heads;
  const int w = (int)(rest % width), s = (int)(rest / width);
  const int r0 = a.new_off[s], n = a.new_off[s + 1] - r0, len = a.lens[s];
  if (n == 0) return;
  if (r0 < 0 || n < 0 || n > a.max_new || r0 > a.rows - n || len < n || len > (long long)c.table_ld * c.page) {
    if (lane == 0) report_error(a.err, DEV_ERR_BAD_SHAPE);
    return;
  }
  const int base = len - n, pg = base / c.page + w;  // tokens before, this unit's page
  if ((long long)pg * c.page >= len) return;
  const int id = c.table[(long long)s * c.table_ld + pg];
  if (id < 0 || id >= c.n_pages) {
    if (lane == 0) report_error(a.err, DEV_ERR_BAD_SHAPE);
    return;
  }
  const int t0 = max(base - pg * c.page, 0), t1 = min(len - pg * c.page, c.page);  // new tokens of the page
  const long long ld = x ? a.ldv : a.ldk;
  const H* src = reinterpret_cast<const H*>(x ? a.v : a.k) + (long long)(r0 + pg * c.page + t0 - base) * ld + h * D;
  const long long ph = (long long)id * c.n_kv_heads + h;
  uint8_t* dst = (x ? c.v : c.k) + ph * c.page * D;
  float* scale = (x ? c.v_scale : c.k_scale) + ph;

  // ---- the largest new value
  float most = 0.f;
  bool nan = false;
  for (int i = lane; i < (t1 - t0) * vec; i += T) {
    const uint4 raw = *reinterpret_cast<const uint4*>(src + (long long)(i / vec) * ld + i % vec * 8);
    const H* y = reinterpret_cast<const H*>(&raw);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float f = fabsf(from_h(y[k]));
      nan |= f != f;
      if (f < INFINITY) most = fmaxf(most, f);
    }
  }
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, k));
  if constexpr (T > 32) {
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = most;
    __syncthreads();
    most = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
  }
  if (nan) report_error(a.err, DEV_ERR_NONFINITE);
  const int need = need_exp(most);
  const int e0 = t0 > 0 ? exponent_of(*scale) : -127;
  const int e = max(e0, need);
  // ---- the page's older codes, where the scale grew
  if (t0 > 0 && e > e0) {
    const float f = exp2i(e0 - e);
    for (int i = lane; i < t0 * vec; i += T) {
      uint2* p = reinterpret_cast<uint2*>(dst + i * 8);
      *p = rescale8(*p, f);
    }
  }
  // every lane has read the scale
  if constexpr (T > 32)
    __syncthreads();
  else
    __syncwarp();
  if (lane == 0) *scale = exp2i(e);
  // ---- the new tokens
  const float f = exp2i(-e);
  for (int i = lane; i < (t1 - t0) * vec; i += T) {
    const uint4 raw = *reinterpret_cast<const uint4*>(src + (long long)(i / vec) * ld + i % vec * 8);
    const H* y = reinterpret_cast<const H*>(&raw);
    float z[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float v = from_h(y[k]);
      z[k] = v == v ? v * f : 0.f;
    }
    *reinterpret_cast<uint2*>(dst + (t0 * vec + i) * 8) =
        make_uint2(to_e4m3x2(z[0], z[1]) | to_e4m3x2(z[2], z[3]) << 16, to_e4m3x2(z[4], z[5]) | to_e4m3x2(z[6], z[7]) << 16);
  }
}

// Each item's K sequences follow their parents, in place: entries of the block
// table for full pages, contents and scales for the page that is being filled
// (which stays its sequence's own). A thread reads one 16-byte column of all
// the pages that it has to before it writes any of them.
template <int KM>
__global__ void __launch_bounds__(256) k_kv8_reorder(const Kv8 c, const int* parent, const int* lens, int K, int* err) {
  __shared__ int s_parent[KM], s_page[KM], s_ok;
  const int b = blockIdx.y;
  if (threadIdx.x == 0) s_ok = 1;
  pdl_wait();
  pdl_trigger();
  __syncthreads();
  const int len = lens[(long long)b * K], full = len / c.page, part = len % c.page;
  if (threadIdx.x < K) {
    const int k = threadIdx.x, p = parent[(long long)b * K + k];
    bool ok = p >= 0 && p < K && len >= 0 && lens[(long long)b * K + k] == len && len <= (long long)c.table_ld * c.page;
    int id = 0;
    if (ok && part > 0) {
      id = c.table[((long long)b * K + k) * c.table_ld + full];
      ok = id >= 0 && id < c.n_pages;
    }
    s_parent[k] = p;
    s_page[k] = id;
    if (!ok) s_ok = 0;
  }
  __syncthreads();
  if (threadIdx.x < K && part > 0)
    for (int k = 0; k < threadIdx.x; ++k)
      if (s_page[k] == s_page[threadIdx.x]) s_ok = 0;  // two sequences cannot fill one page
  __syncthreads();
  if (!s_ok) {
    if (threadIdx.x == 0) report_error(err, DEV_ERR_BAD_SHAPE);
    return;
  }
  if (blockIdx.x == 0) {
    // block table: full pages
    for (int i = threadIdx.x; i < full; i += 256) {
      int* t = c.table + (long long)b * K * c.table_ld + i;
      int v[KM];
#pragma unroll
      for (int k = 0; k < KM; ++k)
        if (k < K && s_parent[k] != k) v[k] = t[(long long)s_parent[k] * c.table_ld];
#pragma unroll
      for (int k = 0; k < KM; ++k)
        if (k < K && s_parent[k] != k) t[(long long)k * c.table_ld] = v[k];
    }
    return;
  }
  if (part == 0) return;
  const int h = (blockIdx.x - 1) >> 1;
  uint8_t* pool = (blockIdx.x - 1) & 1 ? c.v : c.k;
  float* scale = (blockIdx.x - 1) & 1 ? c.v_scale : c.k_scale;
  const long long slice = (long long)c.page * c.head_dim;
  for (int i = threadIdx.x; i < part * c.head_dim / 16; i += 256) {
    uint4 v[KM];
#pragma unroll
    for (int k = 0; k < KM; ++k)
      if (k < K && s_parent[k] != k)
        v[k] = *reinterpret_cast<const uint4*>(pool + ((long long)s_page[s_parent[k]] * c.n_kv_heads + h) * slice + 16 * i);
#pragma unroll
    for (int k = 0; k < KM; ++k)
      if (k < K && s_parent[k] != k)
        *reinterpret_cast<uint4*>(pool + ((long long)s_page[k] * c.n_kv_heads + h) * slice + 16 * i) = v[k];
  }
  if (threadIdx.x == 0) {
    float v[KM];
#pragma unroll
    for (int k = 0; k < KM; ++k)
      if (k < K) v[k] = scale[(long long)s_page[s_parent[k]] * c.n_kv_heads + h];
#pragma unroll
    for (int k = 0; k < KM; ++k)
      if (k < K) scale[(long long)s_page[k] * c.n_kv_heads + h] = v[k];
  }
}

template <typename H>
cudaError_t append_h(const Kv8AppendArgs& a, cudaStream_t st) {
  const int width = (a.max_new + a.c.page - 2) / a.c.page + 1;  // pages that a sequence's new tokens may touch
  const long long units = (long long)a.n_seqs * width * a.c.n_kv_heads * 2;
  if (units > 0x7fffffffLL) return cudaErrorInvalidValue;
  if (a.max_new <= 4)
    return launch_pdl(k_kv8_append<H, 32>, dim3((unsigned)((units + 3) / 4)), dim3(128), 0, st, a, width, units);
  return launch_pdl(k_kv8_append<H, 128>, dim3((unsigned)units), dim3(128), 0, st, a, width, units);
}

}  // namespace

cudaError_t kv8_append_launch(const Kv8AppendArgs& a, bool bf16, cudaStream_t st) {
  if (a.n_seqs <= 0 || a.max_new <= 0) return cudaSuccess;
  return bf16 ? append_h<__nv_bfloat16>(a, st) : append_h<__half>(a, st);
}

cudaError_t kv8_reorder_launch(const Kv8& c, const int* parent, const int* lens, int B, int K, int* err,
                               cudaStream_t st) {
  if (B <= 0) return cudaSuccess;
  const dim3 grid(1 + 2 * c.n_kv_heads, B), block(256);
  if (K <= 4) return launch_pdl(k_kv8_reorder<4>, grid, block, 0, st, c, parent, lens, K, err);
  if (K <= 8) return launch_pdl(k_kv8_reorder<8>, grid, block, 0, st, c, parent, lens, K, err);
  if (K <= 16) return launch_pdl(k_kv8_reorder<16>, grid, block, 0, st, c, parent, lens, K, err);
  return launch_pdl(k_kv8_reorder<32>, grid, block, 0, st, c, parent, lens, K, err);
}

}  // namespace pkc
