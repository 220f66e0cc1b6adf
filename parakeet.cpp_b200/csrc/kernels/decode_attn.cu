// Attention of a few query rows over keys and values of another length: a
// decoder step's cross attention over the encoder's states (16-bit rows) and
// its self attention over the paged 8-bit cache.
//
//   s_ij = scale q_i . k_j,  p = softmax_j(s),  o_i = sum_j p_ij v_j
//
// Such a call reads every key and value once for at most a few rows, so it is
// bound by memory: one CTA takes up to 16 rows (tokens x heads of one shared
// key head) of one item and one part of its keys; its warps walk tiles of WT
// keys on their own, each with its own ring of tiles in shared memory (filled
// by cp.async two tiles ahead, no barrier but the warp's own) and its own
// running maximum and sum. Parts are joined by k_attn_join when there is more
// than one.
//
// Fragments are 16-byte reads of the tile as it lies in memory: the order of
// the contraction is free as long as both operands share it, so a thread of
// mma.m16n8k16 that owns key n = lane / 4 takes 16 contiguous bytes of that
// key's row and the query fragments are loaded in the same order; for P V it
// takes 16 contiguous bytes of each of its four keys' value rows, whose
// elements belong to different 8-column tiles of the product. No transposition
// lies between the copy and the product.
//
// 8-bit codes become f16 exactly (cvt e4m3x2 -> f16x2). A tile lies in one
// page, so its two scales are scalars: the key scale goes into the softmax's
// factor, the value scale (a power of two) multiplies the tile's product in
// f32, where it cannot under- or overflow as it could in f16 probabilities.
// bf16 queries are brought to f16 with a power of two for each row (their 8
// bits fit f16's 11), which the softmax's factor takes back.
#include "common.cuh"
#include "decode.h"
#include "per_device.h"

namespace pkc {

namespace {

constexpr int kRows = 16;
constexpr int kStages = 3;  // tiles in a warp's ring
constexpr int kSms = 148;

template <typename M>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (is_bf16<M>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// two e4m3 codes (the low or high half of w) -> f16x2
__device__ __forceinline__ uint32_t e4m3_lo(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t e4m3_hi(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(w));
  return r;
}

// One item's share of a call, checked against the sizes that the host knows.
struct Item {
  int q0, n, len, kv0;
  bool ok;
};
template <bool Q8>
__device__ __forceinline__ Item load_item(const DecodeAttnArgs& a, int b) {
  Item it;
  it.q0 = a.q_off[b];
  it.n = a.q_off[b + 1] - it.q0;
  it.len = a.kv_len[b];
  it.kv0 = Q8 ? 0 : a.kv_off[b];
  it.ok = it.q0 >= 0 && it.n >= 0 && it.n <= a.max_q && it.q0 <= a.q_rows - it.n && it.len >= 0 && it.len <= a.max_kv;
  if (Q8)
    it.ok = it.ok && it.n <= it.len;
  else
    it.ok = it.ok && it.kv0 >= 0 && it.kv0 <= a.kv_rows - it.len;
  return it;
}

// keys that row i (token i of n) sees
template <bool Q8>
__device__ __forceinline__ int visible(const Item& it, int i) {
  return Q8 ? it.len - it.n + i + 1 : it.len;
}

// index of the 16-row block of partials
__device__ __forceinline__ long long part_at(const DecodeAttnArgs& a, int row_tiles, int b, int h, int rt) {
  return ((long long)b * a.n_kv_heads + h) * row_tiles + rt;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Where 16-byte chunk ch of row r of a tile lies. The reads below take, at a
// time, four chunks of two neighbouring rows (keys) or two chunks of rows 0, 2,
// 4, 6 of eight (values): these permutations give each such set eight
// different chunk columns of 128 bytes.
template <int RB>
__device__ __forceinline__ int key_at(int r, int ch) {
  return RB == 64 ? r * 64 + ch * 16 : r * RB + (ch ^ ((r & 1) << 2)) * 16;
}
template <int RB>
__device__ __forceinline__ int value_at(int r, int ch) {
  return RB == 64 ? (r ^ ((r >> 2) & 1)) * 64 + (ch ^ (r & 2)) * 16 : r * RB + (ch ^ (r & 6)) * 16;
}

// Shared memory of a CTA of W warps: the rings, then each stage's two scales;
// the join of the warps reuses the rings.
template <int RB, int WT>
struct RowsLayout {
  static constexpr int kTile = WT * RB;  // keys or values of a tile
  static constexpr int kStage = 2 * kTile;
  static constexpr int kWarp = kStages * kStage + kStages * 16;  // + {key scale, value scale}
};

// H: type of q and out; Q8: 8-bit cache, else keys and values of type H; W
// warps share the CTA's part of the keys.
template <typename H, bool Q8, int D, int WT, int W>
__global__ void __launch_bounds__(32 * W, 8 / W) k_attn_rows(const DecodeAttnArgs a, int row_tiles, int n_split) {
  using M = typename std::conditional<Q8, __half, H>::type;  // type of the products
  constexpr int RB = Q8 ? D : 2 * D;                         // bytes of a row
  constexpr int KC = RB / 64;                                // 16-byte reads of a key row, per thread
  constexpr int VW = RB / 32;                                // 32-bit words of a value row, per thread
  constexpr int NT = D / 8;                                  // 8-column tiles of the output
  using L = RowsLayout<RB, WT>;
  extern __shared__ __align__(128) uint8_t smem[];

  const int G = a.n_heads / a.n_kv_heads;
  const int split = blockIdx.x % n_split;
  int rest = blockIdx.x / n_split;
  const int rt = rest % row_tiles;
  rest /= row_tiles;
  const int h = rest % a.n_kv_heads, b = rest / a.n_kv_heads;
  const int warp = W == 1 ? 0 : threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  pdl_wait();
  pdl_trigger();
  const Item it = load_item<Q8>(a, b);
  if (!it.ok) {
    if (threadIdx.x == 0) report_error(a.err, DEV_ERR_BAD_SHAPE);
    return;
  }
  const int rows = it.n * G;
  if (rt * kRows >= rows) return;

  // ---- this warp's tiles: t_begin + warp, + W, ...
  // the last row's last key ends the walk
  const int last = min(rows, (rt + 1) * kRows) - 1;
  const int vmax = max(0, visible<Q8>(it, last / G));
  const int n_tiles = (vmax + WT - 1) / WT;
  const int per = (n_tiles + n_split - 1) / n_split;
  const int t0 = split * per + warp, t_end = min(n_tiles, (split + 1) * per);
  const int cnt = t0 < t_end ? (t_end - t0 + W - 1) / W : 0;
  uint8_t* ring = smem + warp * L::kWarp;
  const uint32_t ring_s = smem_u32(ring);
  const uint8_t* kbase = nullptr;
  const uint8_t* vbase = nullptr;
  if constexpr (!Q8) {
    kbase = reinterpret_cast<const uint8_t*>(reinterpret_cast<const H*>(a.k) + (long long)it.kv0 * a.ldk + h * D);
    vbase = reinterpret_cast<const uint8_t*>(reinterpret_cast<const H*>(a.v) + (long long)it.kv0 * a.ldv + h * D);
  }
  auto page_of = [&](int i) -> int {  // page of the warp's i-th tile
    if constexpr (!Q8) return 0;
    if (i >= cnt) return 0;
    return a.cache.table[(long long)b * a.cache.table_ld + (t0 + W * i) * WT / a.cache.page];
  };
  // copy the warp's i-th tile; rows that no query row sees become zeros (a NaN
  // there would survive a probability of zero)
  auto issue = [&](int i, int id) {
    if (i < cnt) {
      const int k0 = (t0 + W * i) * WT, left = vmax - k0;
      const uint32_t dst = ring_s + (i % kStages) * L::kStage;
      const uint8_t *kp = kbase, *vp = vbase;
      long long kst = RB, vst = RB;
      bool on = true;
      if constexpr (Q8) {
        const Kv8& cc = a.cache;
        on = id >= 0 && id < cc.n_pages;
        const long long ph = (long long)(on ? id : 0) * cc.n_kv_heads + h;
        kp = cc.k + (ph * cc.page + k0 % cc.page) * D;
        vp = cc.v + (ph * cc.page + k0 % cc.page) * D;
        const uint32_t sc = ring_s + kStages * L::kStage + (i % kStages) * 16;
        if (on) {
          if (lane < 2) cp_async4(sc + 4 * lane, (lane ? cc.v_scale : cc.k_scale) + ph);
        } else if (lane == 0) {
          // the keys of a page that is none are not seen
          report_error(a.err, DEV_ERR_BAD_SHAPE);
          *reinterpret_cast<float*>(ring + kStages * L::kStage + (i % kStages) * 16) = -1.f;
        }
      } else {
        kst = a.ldk * 2;
        vst = a.ldv * 2;
        kp += k0 * kst;
        vp += k0 * vst;
      }
#pragma unroll
      for (int j = 0; j < L::kTile / 512; ++j) {
        const int q = j * 32 + lane, r = q / (RB / 16), ch = q % (RB / 16);
        const bool in = on && r < left;
        cp_async16(dst + key_at<RB>(r, ch), kp + (in ? r : 0) * kst + ch * 16, in ? 16 : 0);
      }
#pragma unroll
      for (int j = 0; j < L::kTile / 512; ++j) {
        const int q = j * 32 + lane, r = q / (RB / 16), ch = q % (RB / 16);
        const bool in = on && r < left;
        cp_async16(dst + L::kTile + value_at<RB>(r, ch), vp + (in ? r : 0) * vst + ch * 16, in ? 16 : 0);
      }
    }
    cp_commit();
  };
  int id_next;
  {
    int ids[kStages];
#pragma unroll
    for (int i = 0; i < kStages; ++i) ids[i] = page_of(i);
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue(i, ids[i]);
    id_next = ids[kStages - 1];
  }

  // ---- queries: rows g and g + 8 of the tile, in the key loads' order
  uint32_t qf[D / 16][4];
  float rs[2];
  int vis[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = rt * kRows + g + 8 * e;
    const bool on = r < rows;
    const int i = on ? r / G : 0, hd = h * G + (on ? r % G : 0);
    vis[e] = on ? visible<Q8>(it, i) : 0;
    const H* qp = reinterpret_cast<const H*>(a.q) + (long long)(it.q0 + i) * a.ldq + hd * D;
    rs[e] = a.scale_log2;
    uint4 w[D / 32];
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      const int col = Q8 ? (j >> 1) * 64 + c * 16 + (j & 1) * 8 : j * 32 + c * 8;
      w[j] = on ? *reinterpret_cast<const uint4*>(qp + col) : make_uint4(0, 0, 0, 0);
    }
    if constexpr (Q8 && is_bf16<H>::value) {
      float m = 0.f;
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        const H* x = reinterpret_cast<const H*>(&w[j]);
#pragma unroll
        for (int k = 0; k < 8; ++k) m = fmaxf(m, fabsf(from_h(x[k])));
      }
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
      // 2^-x, x the exponent of the row's largest value (rows of zeros or
      // infinities as they are)
      const int x = ((__float_as_int(m) >> 23) & 255) - 127;
      const float f = m > 0.f && x < 127 && x > -126 ? __int_as_float((127 - x) << 23) : 1.f;
      rs[e] /= f;
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        H* y = reinterpret_cast<H*>(&w[j]);
        uint32_t o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = pack2<__half>(from_h(y[2 * k]) * f, from_h(y[2 * k + 1]) * f);
        w[j] = make_uint4(o[0], o[1], o[2], o[3]);
      }
    }
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      qf[2 * j][e] = w[j].x;
      qf[2 * j][2 + e] = w[j].y;
      qf[2 * j + 1][e] = w[j].z;
      qf[2 * j + 1][2 + e] = w[j].w;
    }
  }
  float o[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

  for (int i = 0; i < cnt; ++i) {
    cp_wait<kStages - 2>();
    __syncwarp();
    issue(i + kStages - 1, id_next);
    id_next = page_of(i + kStages);
    const int k0 = (t0 + W * i) * WT;
    const uint8_t* kt = ring + (i % kStages) * L::kStage;
    const uint8_t* vt = kt + L::kTile;
    float ks = 1.f, vs = 1.f;
    if constexpr (Q8) {
      const float* sc = reinterpret_cast<const float*>(ring + kStages * L::kStage + (i % kStages) * 16);
      ks = sc[0];
      vs = sc[1];
      if (ks < 0.f) continue;
    }
    // ---- scores
    float s[WT / 8][4];
#pragma unroll
    for (int i = 0; i < WT / 8; ++i) {
      s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
      for (int j = 0; j < KC; ++j) {
        const uint4 kr = *reinterpret_cast<const uint4*>(kt + key_at<RB>(8 * i + g, 4 * j + c));
        const uint32_t w[4] = {kr.x, kr.y, kr.z, kr.w};
        if constexpr (Q8) {
#pragma unroll
          for (int u = 0; u < 4; ++u) mma16816<M>(s[i], qf[4 * j + u], e4m3_lo(w[u]), e4m3_hi(w[u]));
        } else {
          mma16816<M>(s[i], qf[2 * j], w[0], w[1]);
          mma16816<M>(s[i], qf[2 * j + 1], w[2], w[3]);
        }
      }
    }
    // ---- running softmax in the log2 domain
    float mt[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < WT / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = k0 + 8 * i + 2 * c + (e & 1);
        s[i][e] = key < vis[e >> 1] ? s[i][e] * (rs[e >> 1] * ks) : -INFINITY;
        mt[e >> 1] = fmaxf(mt[e >> 1], s[i][e]);
      }
    float mu[2], alpha[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      mt[e] = fmaxf(mt[e], __shfl_xor_sync(0xffffffffu, mt[e], 1));
      mt[e] = fmaxf(mt[e], __shfl_xor_sync(0xffffffffu, mt[e], 2));
      const float mn = fmaxf(m[e], mt[e]);
      mu[e] = mn == -INFINITY ? 0.f : mn;
      alpha[e] = ex2_approx(m[e] - mu[e]);
      m[e] = mn;
      l[e] *= alpha[e];
    }
    if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] *= alpha[e >> 1];
    }
    uint32_t pf[WT / 16][4];
#pragma unroll
    for (int i = 0; i < WT / 8; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[i][e] = ex2_approx(s[i][e] - mu[e >> 1]);
        l[e >> 1] += s[i][e];
      }
      // probabilities in the products' type: at most half a step off each
      pf[i >> 1][2 * (i & 1)] = pack2<M>(s[i][0], s[i][1]);
      pf[i >> 1][2 * (i & 1) + 1] = pack2<M>(s[i][2], s[i][3]);
    }
    // ---- values: keys 16 i + {0, 1, 8, 9} + 2 c
    uint32_t vr[WT / 4][VW];
#pragma unroll
    for (int i = 0; i < WT / 4; ++i) {
      const int r = 16 * (i >> 2) + 2 * c + (i & 1) + 8 * ((i >> 1) & 1);
      if constexpr (VW == 2) {
        const uint2 x = *reinterpret_cast<const uint2*>(vt + value_at<RB>(r, g >> 1) + (g & 1) * 8);
        vr[i][0] = x.x;
        vr[i][1] = x.y;
      } else {
#pragma unroll
        for (int j = 0; j < VW / 4; ++j) {
          const uint4 x = *reinterpret_cast<const uint4*>(vt + value_at<RB>(r, 8 * j + g));
          vr[i][4 * j] = x.x;
          vr[i][4 * j + 1] = x.y;
          vr[i][4 * j + 2] = x.z;
          vr[i][4 * j + 3] = x.w;
        }
      }
    }
    if constexpr (Q8) {
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        float acc[4][4];
#pragma unroll
        for (int x = 0; x < 4; ++x) acc[x][0] = acc[x][1] = acc[x][2] = acc[x][3] = 0.f;
#pragma unroll
        for (int i = 0; i < WT / 16; ++i) {
          const uint32_t a0 = vr[4 * i][w], a1 = vr[4 * i + 1][w], a2 = vr[4 * i + 2][w], a3 = vr[4 * i + 3][w];
          const uint32_t p0 = __byte_perm(a0, a1, 0x5140), p1 = __byte_perm(a2, a3, 0x5140);
          const uint32_t p2 = __byte_perm(a0, a1, 0x7362), p3 = __byte_perm(a2, a3, 0x7362);
          mma16816<M>(acc[0], pf[i], e4m3_lo(p0), e4m3_lo(p1));
          mma16816<M>(acc[1], pf[i], e4m3_hi(p0), e4m3_hi(p1));
          mma16816<M>(acc[2], pf[i], e4m3_lo(p2), e4m3_lo(p3));
          mma16816<M>(acc[3], pf[i], e4m3_hi(p2), e4m3_hi(p3));
        }
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[4 * w + x][e] = fmaf(acc[x][e], vs, o[4 * w + x][e]);
      }
    } else {
#pragma unroll
      for (int w = 0; w < VW; ++w)
#pragma unroll
        for (int i = 0; i < WT / 16; ++i) {
          const uint32_t a0 = vr[4 * i][w], a1 = vr[4 * i + 1][w], a2 = vr[4 * i + 2][w], a3 = vr[4 * i + 3][w];
          mma16816<M>(o[2 * w], pf[i], __byte_perm(a0, a1, 0x5410), __byte_perm(a2, a3, 0x5410));
          mma16816<M>(o[2 * w + 1], pf[i], __byte_perm(a0, a1, 0x7632), __byte_perm(a2, a3, 0x7632));
        }
    }
  }

  // ---- what this warp holds of rows g (e = 0) and g + 8: four columns at a time
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
  }
  auto each = [&](auto&& f) {
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int n = 0; n < 2; ++n)  // column 2 c + n of the 8-column tiles
#pragma unroll
        for (int i = 0; i < NT; i += 4) {
          const int dim = Q8 ? (2 * c + n) * (D / 8) + i : (i >> 3) * 64 + (2 * c + n) * 8 + (i & 7);
          const int x = 2 * e + n;
          f(e, dim, make_float4(o[i][x], o[i + 1][x], o[i + 2][x], o[i + 3][x]));
        }
  };
  const int valid = min(kRows, rows - rt * kRows);
  float* po = a.ws + (part_at(a, row_tiles, b, h, rt) * n_split + split) * (kRows * (D + 2));
  auto store_out = [&](int r, int dim, float4 v) {
    const int row = rt * kRows + r;
    H* op = reinterpret_cast<H*>(a.out) + (long long)(it.q0 + row / G) * a.ldo + (h * G + row % G) * D + dim;
    *reinterpret_cast<uint2*>(op) = make_uint2(pack2<H>(v.x, v.y), pack2<H>(v.z, v.w));
  };
  if constexpr (W == 1) {
    if (n_split == 1) {
      float inv[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) inv[e] = l[e] == 0.f ? 0.f : 1.f / l[e];  // no key seen: zeros
      each([&](int e, int dim, float4 v) {
        if (g + 8 * e < valid)
          store_out(g + 8 * e, dim, make_float4(v.x * inv[e], v.y * inv[e], v.z * inv[e], v.w * inv[e]));
      });
    } else {
      each([&](int e, int dim, float4 v) {
        if (g + 8 * e < valid) *reinterpret_cast<float4*>(po + (g + 8 * e) * D + dim) = v;
      });
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (c == 0 && g + 8 * e < valid)
          *reinterpret_cast<float2*>(po + kRows * D + 2 * (g + 8 * e)) = make_float2(m[e], l[e]);
    }
  } else {
    // ---- join the warps, in the rings' memory
    cp_wait<0>();
    __syncthreads();
    constexpr int LD = D + 4;
    float* s_o = reinterpret_cast<float*>(smem);          // [W][kRows][LD]
    float* s_ml = s_o + W * kRows * LD;                   // [W][kRows][2]
    static_assert((W * kRows * (LD + 2)) * 4 <= W * L::kWarp, "the join fits the rings");
    each([&](int e, int dim, float4 v) {
      *reinterpret_cast<float4*>(s_o + (warp * kRows + g + 8 * e) * LD + dim) = v;
    });
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (c == 0)
        *reinterpret_cast<float2*>(s_ml + (warp * kRows + g + 8 * e) * 2) = make_float2(m[e], l[e]);
    __syncthreads();
    for (int idx = threadIdx.x; idx < valid * (D / 4); idx += 32 * W) {
      const int r = idx / (D / 4), d4 = idx % (D / 4) * 4;
      float mm = -INFINITY;
#pragma unroll
      for (int w = 0; w < W; ++w) mm = fmaxf(mm, s_ml[(w * kRows + r) * 2]);
      const float base = mm == -INFINITY ? 0.f : mm;
      float ll = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float f = ex2_approx(s_ml[(w * kRows + r) * 2] - base);
        ll += s_ml[(w * kRows + r) * 2 + 1] * f;
        const float4 v = *reinterpret_cast<const float4*>(s_o + (w * kRows + r) * LD + d4);
        x[0] = fmaf(v.x, f, x[0]);
        x[1] = fmaf(v.y, f, x[1]);
        x[2] = fmaf(v.z, f, x[2]);
        x[3] = fmaf(v.w, f, x[3]);
      }
      if (n_split == 1) {
        const float inv = ll == 0.f ? 0.f : 1.f / ll;
        store_out(r, d4, make_float4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv));
      } else {
        *reinterpret_cast<float4*>(po + r * D + d4) = make_float4(x[0], x[1], x[2], x[3]);
        if (d4 == 0) *reinterpret_cast<float2*>(po + kRows * D + 2 * r) = make_float2(mm, ll);
      }
    }
  }
}

// Joins the parts of one 16-row block: o = sum_s o_s 2^(m_s - m) / sum_s l_s 2^(m_s - m).
template <typename H, bool Q8, int D>
__global__ void __launch_bounds__(kRows * D / 4) k_attn_join(const DecodeAttnArgs a, int row_tiles, int n_split) {
  const int G = a.n_heads / a.n_kv_heads;
  int rest = blockIdx.x;
  const int rt = rest % row_tiles;
  rest /= row_tiles;
  const int h = rest % a.n_kv_heads, b = rest / a.n_kv_heads;
  pdl_wait();
  pdl_trigger();
  const Item it = load_item<Q8>(a, b);
  if (!it.ok) return;
  const int rows = it.n * G, r = threadIdx.x / (D / 4), d4 = threadIdx.x % (D / 4) * 4, row = rt * kRows + r;
  if (row >= rows) return;
  const float* p = a.ws + part_at(a, row_tiles, b, h, rt) * n_split * (kRows * (D + 2));
  float m = -INFINITY, l = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < n_split; ++s, p += kRows * (D + 2)) {
    const float ms = p[kRows * D + 2 * r], ls = p[kRows * D + 2 * r + 1];
    if (ls == 0.f) continue;  // a part without keys
    const float4 v = *reinterpret_cast<const float4*>(p + r * D + d4);
    const float mn = fmaxf(m, ms), f0 = ex2_approx(m - mn), f1 = ex2_approx(ms - mn);
    l = l * f0 + ls * f1;
    x[0] = x[0] * f0 + v.x * f1;
    x[1] = x[1] * f0 + v.y * f1;
    x[2] = x[2] * f0 + v.z * f1;
    x[3] = x[3] * f0 + v.w * f1;
    m = mn;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  H* op = reinterpret_cast<H*>(a.out) + (long long)(it.q0 + row / G) * a.ldo + (h * G + row % G) * D + d4;
  *reinterpret_cast<uint2*>(op) = make_uint2(pack2<H>(x[0] * inv, x[1] * inv), pack2<H>(x[2] * inv, x[3] * inv));
}

// How a call is cut: `warps` a CTA and parts of each item's keys.
//  - Many blocks of rows: a warp takes one alone (CTAs of one warp, no join).
//  - Else four warps share a part, and the keys are cut into as many parts as
//    give about six CTAs an SM (lengths differ; two run at a time), of at
//    least 128 keys.
struct Plan {
  int warps, n_split;
};
Plan plan_rows(long long blocks, int max_kv) {
  if (blocks >= 8LL * kSms) return {1, 1};
  const long long want = (6LL * kSms + blocks - 1) / blocks;
  const long long most = (max_kv + 127) / 128;
  const long long n = want < most ? want : most;
  return {4, n < 1 ? 1 : n > 64 ? 64 : (int)n};
}

long long row_blocks(int n_items, int max_q, int n_heads, int n_kv_heads, int* row_tiles) {
  *row_tiles = (int)(((long long)max_q * (n_heads / n_kv_heads) + kRows - 1) / kRows);
  return (long long)n_items * n_kv_heads * *row_tiles;
}

template <typename H, bool Q8, int D, int WT, int W>
cudaError_t launch_w(const DecodeAttnArgs& a, long long blocks, int rt, int n_split, cudaStream_t st) {
  auto kern = k_attn_rows<H, Q8, D, WT, W>;
  constexpr int smem = W * RowsLayout<Q8 ? D : 2 * D, WT>::kWarp;
  static PerDevice once;
  int unused = 0;
  const cudaError_t e = per_device(once, &unused, [&](int, int&) {
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  });
  if (e != cudaSuccess) return e;
  return launch_pdl(kern, dim3((unsigned)(blocks * n_split)), dim3(32 * W), smem, st, a, rt, n_split);
}

template <typename H, bool Q8, int D, int WT>
cudaError_t launch_rows(const DecodeAttnArgs& a, cudaStream_t st) {
  int rt = 0;
  const long long blocks = row_blocks(a.n_items, a.max_q, a.n_heads, a.n_kv_heads, &rt);
  const Plan p = plan_rows(blocks, a.max_kv);
  if (blocks * p.n_split > 0x7fffffffLL) return cudaErrorInvalidValue;
  const cudaError_t e = p.warps == 1 ? launch_w<H, Q8, D, WT, 1>(a, blocks, rt, p.n_split, st)
                                     : launch_w<H, Q8, D, WT, 4>(a, blocks, rt, p.n_split, st);
  if (e != cudaSuccess || p.n_split == 1) return e;
  return launch_pdl(k_attn_join<H, Q8, D>, dim3((unsigned)blocks), dim3(kRows * D / 4), 0, st, a, rt, p.n_split);
}

template <typename H>
cudaError_t launch_h(const DecodeAttnArgs& a, cudaStream_t st) {
  if (a.cache.k) {
    if (a.head_dim == 128)
      return a.cache.page == 16 ? launch_rows<H, true, 128, 16>(a, st) : launch_rows<H, true, 128, 32>(a, st);
    return a.cache.page == 16 ? launch_rows<H, true, 64, 16>(a, st) : launch_rows<H, true, 64, 32>(a, st);
  }
  return a.head_dim == 128 ? launch_rows<H, false, 128, 16>(a, st) : launch_rows<H, false, 64, 16>(a, st);
}

}  // namespace

size_t decode_attn_ws_bytes(int n_items, int max_q, int max_kv, int n_heads, int n_kv_heads, int head_dim, bool q8) {
  int rt = 0;
  const long long blocks = row_blocks(n_items, max_q, n_heads, n_kv_heads, &rt);
  if (blocks <= 0) return 0;
  const int n_split = plan_rows(blocks, max_kv).n_split;
  return n_split == 1 ? 0 : (size_t)blocks * n_split * kRows * (head_dim + 2) * sizeof(float);
}

cudaError_t decode_attn_launch(const DecodeAttnArgs& a, bool bf16, cudaStream_t st) {
  if (a.n_items <= 0 || a.max_q <= 0) return cudaSuccess;
  return bf16 ? launch_h<__nv_bfloat16>(a, st) : launch_h<__half>(a, st);
}

}  // namespace pkc
