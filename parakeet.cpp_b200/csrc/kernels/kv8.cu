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

// What a page's new tokens are for one sequence, checked against the sizes of
// the call.
struct PageShare {
  int t0, t1;       // its tokens t0 .. t1 - 1 are new; 0 .. t0 - 1 are old
  long long row;    // row of token t0 among the new ones
  int id;           // the page
  bool on;
};
__device__ __forceinline__ PageShare page_share(const Kv8AppendArgs& a, int s, int w, bool report) {
  const Kv8& c = a.c;
  PageShare p{0, 0, 0, 0, false};
  const int r0 = a.new_off[s], n = a.new_off[s + 1] - r0, len = a.lens[s];
  if (n == 0) return p;
  if (r0 < 0 || n < 0 || n > a.max_new || r0 > a.rows - n || len < n || len > (long long)c.table_ld * c.page) {
    if (report) report_error(a.err, DEV_ERR_BAD_SHAPE);
    return p;
  }
  const int base = len - n, pg = base / c.page + w;  // tokens before, this share's page
  if ((long long)pg * c.page >= len) return p;
  p.id = c.table[(long long)s * c.table_ld + pg];
  if (p.id < 0 || p.id >= c.n_pages) {
    if (report) report_error(a.err, DEV_ERR_BAD_SHAPE);
    return p;
  }
  p.t0 = max(base - pg * c.page, 0);
  p.t1 = min(len - pg * c.page, c.page);
  p.row = (long long)r0 + (pg * c.page + p.t0 - base);
  p.on = true;
  return p;
}

// The magnitudes of 16-bit floats order as unsigned integers, a NaN above the
// infinity above the finite values: running maximum of two of them at a time.
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t look8(uint4 raw, uint32_t most) {
  most = max_u16x2(most, raw.x & 0x7fff7fffu);
  most = max_u16x2(most, raw.y & 0x7fff7fffu);
  most = max_u16x2(most, raw.z & 0x7fff7fffu);
  return max_u16x2(most, raw.w & 0x7fff7fffu);
}
template <typename H>
__device__ __forceinline__ float value16(uint32_t bits) {
  if constexpr (is_bf16<H>::value)
    return __uint_as_float(bits << 16);
  else
    return __half2float(__ushort_as_half((unsigned short)bits));
}
// the bits of infinity
template <typename H>
__device__ __forceinline__ uint32_t inf16() { return is_bf16<H>::value ? 0x7f80u : 0x7c00u; }
// largest finite magnitude of eight values where some are not finite, and
// whether one is a NaN
template <typename H>
__device__ __noinline__ uint32_t finite8(uint4 raw, uint32_t most, bool* nan) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  for (int k = 0; k < 8; ++k) {
    const uint32_t u = (w[k / 2] >> (16 * (k & 1))) & 0x7fffu;
    if (u > inf16<H>()) *nan = true;
    if (u < inf16<H>() && u > most) most = u;
  }
  return most;
}
// eight values times f as codes (f a power of two: exact before the rounding,
// but for what is far below the codes); a NaN is 0
template <typename H, bool NANS>
__device__ __forceinline__ uint2 code8(uint4 raw, float f) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  uint32_t o[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float lo = value16<H>(w[k] & 0xffffu), hi = value16<H>(w[k] >> 16);
    if (NANS) {
      lo = lo == lo ? lo : 0.f;
      hi = hi == hi ? hi : 0.f;
    }
    o[k] = to_e4m3x2(lo * f, hi * f);
  }
  return make_uint2(o[0] | o[1] << 16, o[2] | o[3] << 16);
}

// Few new tokens (a decoder step): a warp writes one page's of one head, keys
// or values. Bound by the chain of reads that leads to the page.
template <typename H>
__global__ void __launch_bounds__(128) k_kv8_append_few(const Kv8AppendArgs a, int width, long long units) {
  const long long unit = (long long)blockIdx.x * 4 + threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  pdl_wait();
  pdl_trigger();
  if (unit >= units) return;
  const Kv8& c = a.c;
  const int D = c.head_dim, vec = D / 8;
  const int x = (int)(unit % 2);  // 0 keys, 1 values
  long long rest = unit / 2;
  const int h = (int)(rest % c.n_kv_heads);
  rest /= c.n_kv_heads;
  const PageShare p = page_share(a, (int)(rest / width), (int)(rest % width), lane == 0);
  if (!p.on) return;
  const long long ld = x ? a.ldv : a.ldk;
  const H* src = reinterpret_cast<const H*>(x ? a.v : a.k) + p.row * ld + h * D;
  const long long ph = (long long)p.id * c.n_kv_heads + h;
  uint8_t* dst = (x ? c.v : c.k) + ph * c.page * D;
  float* scale = (x ? c.v_scale : c.k_scale) + ph;
  const int n_vec = (p.t1 - p.t0) * vec;
  const int e0 = p.t0 > 0 ? exponent_of(*scale) : -127;
  auto value = [&](int i) { return *reinterpret_cast<const uint4*>(src + (long long)(i / vec) * ld + i % vec * 8); };
  uint32_t most = 0;
  for (int i = lane; i < n_vec; i += 32) most = look8(value(i), most);
  most = __reduce_max_sync(0xffffffffu, max(most & 0xffffu, most >> 16));
  const bool special = most >= inf16<H>();
  if (special) {
    bool nan = false;
    most = 0;
    for (int i = lane; i < n_vec; i += 32) most = finite8<H>(value(i), most, &nan);
    if (nan) report_error(a.err, DEV_ERR_NONFINITE);
    most = __reduce_max_sync(0xffffffffu, most);
  }
  const int e = max(e0, need_exp(value16<H>(most)));
  if (p.t0 > 0 && e > e0) {  // the page's older codes, where the scale grew
    const float f = exp2i(e0 - e);
    for (int i = lane; i < p.t0 * vec; i += 32) {
      uint2* q = reinterpret_cast<uint2*>(dst + i * 8);
      *q = rescale8(*q, f);
    }
  }
  __syncwarp();  // every lane has read the scale
  if (lane == 0) *scale = exp2i(e);
  const float f = exp2i(-e);
  for (int i = lane; i < n_vec; i += 32)
    *reinterpret_cast<uint2*>(dst + (p.t0 * vec + i) * 8) = code8<H, true>(value(i), f);
}

// Many new tokens (a prompt): eight warps write one page's of eight heads (keys
// and values counted apart), WPH warps a head where a head's page is more than
// 4096 values. NV vectors of it stay in each lane's registers between the
// search for the largest value and the rounding, so every value is read once,
// and neighbouring heads of a row at the same time: a CTA for each head, whose
// reads are 128 bytes apart from the next ones' by a whole row, reached half
// the copy rate. 64 sequences of 1 to 1024 tokens, 8 heads of 64, pages of 64:
// 24 us for 97 MB, 62% of the copy rate (41 us a CTA a head with two reads; 47
// us with maxima and checks in f32: the arithmetic on each value counts). The
// grid is that of the longest sequence, so half of its CTAs have no page here;
// 36 bytes a thread are spilled.
template <typename H, int NV, int WPH>
__global__ void __launch_bounds__(256, 3) k_kv8_append(const Kv8AppendArgs a, int width, int passes) {
  __shared__ uint32_t s_max[2][8];
  const Kv8& c = a.c;
  const int D = c.head_dim, sh = D == 128 ? 4 : 3, vec = D / 8;
  const int warp = threadIdx.x >> 5;
  const int rest = blockIdx.x / passes;
  const int unit = blockIdx.x % passes * (8 / WPH) + warp / WPH;  // 0 .. Hkv - 1 keys, then values
  pdl_wait();
  pdl_trigger();
  const PageShare p = page_share(a, rest / width, rest % width, threadIdx.x == 0);
  if (!p.on) return;
  const bool have = unit < 2 * c.n_kv_heads;
  const int x = have && unit >= c.n_kv_heads, h = have ? unit - x * c.n_kv_heads : 0;
  const long long ld = x ? a.ldv : a.ldk;
  const H* src = reinterpret_cast<const H*>(x ? a.v : a.k) + p.row * ld + h * D;
  const long long ph = (long long)p.id * c.n_kv_heads + h;
  uint8_t* dst = (x ? c.v : c.k) + ph * c.page * D;
  float* scale = (x ? c.v_scale : c.k_scale) + ph;
  const int n_vec = have ? (p.t1 - p.t0) * vec : 0;
  const int lane = threadIdx.x % (32 * WPH);  // of the head's threads
  uint4 raw[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int i = j * 32 * WPH + lane;
    raw[j] = make_uint4(0, 0, 0, 0);
    if (i < n_vec) raw[j] = *reinterpret_cast<const uint4*>(src + (long long)(i >> sh) * ld + (i & (vec - 1)) * 8);
  }
  const int e0 = p.t0 > 0 ? exponent_of(*scale) : -127;
  // over the head's threads (which passes every thread's reading of the scale)
  auto joined = [&](uint32_t most, int k) -> uint32_t {
    most = __reduce_max_sync(0xffffffffu, most);
    if constexpr (WPH > 1) {
      if ((threadIdx.x & 31) == 0) s_max[k][warp] = most;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < WPH; ++w) most = max(most, s_max[k][warp / WPH * WPH + w]);
    }
    return most;
  };
  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < NV; ++j) most = look8(raw[j], most);
  most = joined(max(most & 0xffffu, most >> 16), 0);
  const bool special = __syncthreads_or(most >= inf16<H>());
  if (special) {
    bool nan = false;
    most = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) most = finite8<H>(raw[j], most, &nan);
    if (nan) report_error(a.err, DEV_ERR_NONFINITE);
    most = joined(most, 1);
  }
  if (!have) return;
  const int e = max(e0, need_exp(value16<H>(most)));
  if (p.t0 > 0 && e > e0) {  // the page's older codes, where the scale grew
    const float f = exp2i(e0 - e);
    for (int i = lane; i < p.t0 * vec; i += 32 * WPH) {
      uint2* q = reinterpret_cast<uint2*>(dst + i * 8);
      *q = rescale8(*q, f);
    }
  }
  if (lane == 0) *scale = exp2i(e);
  const float f = exp2i(-e);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int i = j * 32 * WPH + lane;
    if (i < n_vec)
      *reinterpret_cast<uint2*>(dst + (p.t0 * vec + i) * 8) = special ? code8<H, true>(raw[j], f) : code8<H, false>(raw[j], f);
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
  const int width = (int)(((long long)a.max_new + a.c.page - 2) / a.c.page) + 1;  // pages that a sequence's new tokens may touch
  const long long units = (long long)a.n_seqs * width * a.c.n_kv_heads * 2;
  if (units > 0x7fffffffLL) return cudaErrorInvalidValue;
  if (a.max_new <= 4)
    return launch_pdl(k_kv8_append_few<H>, dim3((unsigned)((units + 3) / 4)), dim3(128), 0, st, a, width, units);
  auto many = [&](auto kern, int wph) {
    const int passes = (2 * a.c.n_kv_heads * wph + 7) / 8;
    return launch_pdl(kern, dim3((unsigned)((long long)a.n_seqs * width * passes)), dim3(256), 0, st, a, width, passes);
  };
  switch (a.c.page * a.c.head_dim / 1024) {
    case 1: return many(k_kv8_append<H, 4, 1>, 1);
    case 2: return many(k_kv8_append<H, 8, 1>, 1);
    case 4: return many(k_kv8_append<H, 16, 1>, 1);
    case 8: return many(k_kv8_append<H, 16, 2>, 2);
    default: return many(k_kv8_append<H, 16, 4>, 4);
  }
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
