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
// by cp.async ahead of its use, no barrier but the warp's own) and its own
// running maximum and sum. Parts are joined by k_attn_join when there is more
// than one.
//
// The products are taken transposed, S^T = K Q^T and O^T = V^T P^T: keys and
// then output columns fill the 16 rows of mma.m16n8k16 and the few query rows
// its 8 columns, so eight rows cost half of what 16 do (rows as the 16-row
// side: 850 instructions a tile of 32 keys of 128 8-bit columns instead of 510,
// and twice the accumulators). P^T goes from the accumulator's layout to the operand's by
// movmatrix.
//
// Fragments are 16-byte reads of the tile as it lies in memory: the order of
// the contraction is free as long as both operands share it, so a thread that
// owns key lane / 4 takes 16 contiguous bytes of that key's row and the query
// fragments are loaded in the same order; for V^T it takes 16 contiguous bytes
// of each of its four keys' value rows, whose elements belong to different
// rows of the product's tiles. No transposition lies between the copy and the
// product.
//
// 8-bit codes become f16 exactly (cvt e4m3x2 -> f16x2). A tile lies in one
// page, so its two scales are scalars. The key scale goes into the softmax's
// factor. The value scale, a power of two, goes into the exponent of the
// probabilities as the difference to a reference exponent in which the output
// is kept, as long as the page is at most 2^4 below it (the reference rises
// with the pages); values of a page further below would lose bits of their f16
// probabilities and take a product of their own, scaled in f32. bf16 queries
// are brought to f16 with a power of two for each row (their 8 bits fit f16's
// 11), which the softmax's factor takes back.
//
// Measured (copy rate 6539 GB/s): 512 sequences of 1 to 448 tokens, 8 heads of
// 128, pages of 32: 46 us for 230 MB, 77% of it; 8 sequences of 9001 to 131071
// tokens, 2 key heads for 16: 57 us for 265 MB, 71%; cross attention of 64 x 8
// rows over 25 to 437 frames, 8 heads of 128: 17 us for 70 MB, 63%; one row
// over 437 frames: 4.8 us. What is left is latency: the chain item -> table ->
// codes at the start of each block of rows, and 40% of the issue slots.
#include "common.cuh"
#include "decode.h"
#include "decode_common.cuh"
#include "per_device.h"

namespace pkc {

namespace {

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

// 8x8 matrix of 16-bit elements, transposed across the warp
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
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

// from the shared memory of a CTA of the cluster
__device__ __forceinline__ float2 ld_cluster2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
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
//
// Two tiles a ring and 168 registers let twelve warps run on an SM, which is
// what hides the latencies here (against three tiles and eight warps: a step of
// 512 short sequences 49 instead of 53 us, 8 long ones 60 instead of 68 us);
// with two blocks of rows the registers leave eight, and three tiles.
template <int RB, int WT, int NB>
struct RowsLayout {
  static constexpr int kStages = NB == 1 ? 2 : 3;
  static constexpr int kTile = WT * RB;  // keys or values of a tile
  static constexpr int kStage = 2 * kTile;
  static constexpr int kWarp = kStages * kStage + kStages * 16;  // + {key scale, value scale}
};

// H: type of q and out; Q8: 8-bit cache, else keys and values of type H; W
// warps share the CTA's part of the keys; NB blocks of 8 query rows.
template <typename H, bool Q8, int D, int WT, int W, int NB>
__global__ void __launch_bounds__(32 * W, NB == 1 ? 12 / W : 8 / W) k_attn_rows(const DecodeAttnArgs a, int row_tiles, int n_split, int clustered) {
  using M = typename std::conditional<Q8, __half, H>::type;  // type of the products
  constexpr int RB = Q8 ? D : 2 * D;                         // bytes of a row
  constexpr int KC = RB / 64;                                // 16-byte reads of a key row, per thread
  constexpr int VW = RB / 32;                                // 32-bit words of a value row, per thread
  constexpr int MT = D / 16;                                 // 16-row tiles of the output
  constexpr int R = 8 * NB;                                  // query rows
  using L = RowsLayout<RB, WT, NB>;
  constexpr int kStages = L::kStages;
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
  const int rows = it.n * G, row0 = rt * R;
  if (row0 >= rows) return;

  // ---- this warp's tiles: t0, t0 + W, ...
  // the last row's last key ends the walk
  const int last = min(rows, row0 + R) - 1;
  const int vmax = max(0, visible<Q8>(it, last / G));
  const int vmin = Q8 ? visible<Q8>(it, row0 / G) : vmax;  // every row sees these
  const int n_tiles = (vmax + WT - 1) / WT;
  const int per = (n_tiles + n_split - 1) / n_split;
  const int t0 = split * per + warp, t_end = min(n_tiles, (split + 1) * per);
  const int cnt = t0 < t_end ? (t_end - t0 + W - 1) / W : 0;
  uint8_t* ring = smem + warp * L::kWarp;
  const uint32_t ring_s = smem_u32(ring);
  // this lane's 16 bytes of a tile: chunk `ch` of rows r0, r0 + RS, ...
  constexpr int RS = 512 / RB;
  const int r0 = lane / (RB / 16), ch = lane % (RB / 16);
  const uint32_t kd0 = key_at<RB>(r0, ch), vd0 = L::kTile + value_at<RB>(r0, ch);
  const uint8_t *lane_k, *lane_v;  // 8-bit: of page 0 of this head; else of the item's first row
  long long k_row = RB, v_row = RB;
  int shift = 0;  // of a page in tokens
  const int* table = nullptr;
  long long page_bytes = 0;
  if constexpr (Q8) {
    const Kv8& cc = a.cache;
    shift = __ffs(cc.page) - 1;
    table = cc.table + (long long)b * cc.table_ld;
    page_bytes = ((long long)cc.n_kv_heads << shift) * D;
    lane_k = cc.k + ((long long)h << shift) * D + lane * 16;
    lane_v = cc.v + ((long long)h << shift) * D + lane * 16;
  } else {
    k_row = a.ldk * 2;
    v_row = a.ldv * 2;
    lane_k = reinterpret_cast<const uint8_t*>(reinterpret_cast<const H*>(a.k) + (long long)(it.kv0 + r0) * a.ldk + h * D) + ch * 16;
    lane_v = reinterpret_cast<const uint8_t*>(reinterpret_cast<const H*>(a.v) + (long long)(it.kv0 + r0) * a.ldv + h * D) + ch * 16;
  }
  auto page_of = [&](int i) -> int {  // page of the warp's i-th tile
    if constexpr (!Q8) return 0;
    return i < cnt ? table[((t0 + W * i) * WT) >> shift] : 0;
  };
  // copy the warp's i-th tile; rows that no query row sees become zeros (a NaN
  // there would survive a probability of zero)
  auto issue = [&](int i, int id) {
    if (i < cnt) {
      const int k0 = (t0 + W * i) * WT, left = vmax - k0;
      const uint32_t dst = ring_s + (i % kStages) * L::kStage;
      const uint8_t *kp, *vp;
      bool on = true;
      if constexpr (Q8) {
        const Kv8& cc = a.cache;
        on = (unsigned)id < (unsigned)cc.n_pages;
        const long long at = (long long)(on ? id : 0) * page_bytes + (k0 & (cc.page - 1)) * D;
        kp = lane_k + at;
        vp = lane_v + at;
        const uint32_t sc = kStages * L::kStage + (i % kStages) * 16;
        if (on) {
          if (lane < 2) cp_async4(ring_s + sc + 4 * lane, (lane ? cc.v_scale : cc.k_scale) + (long long)id * cc.n_kv_heads + h);
        } else if (lane == 0) {
          // the keys of a page that is none are not seen
          report_error(a.err, DEV_ERR_BAD_SHAPE);
          *reinterpret_cast<float*>(ring + sc) = -1.f;
        }
      } else {
        kp = lane_k + k0 * k_row;
        vp = lane_v + k0 * v_row;
      }
      // (the permutation of a value row's chunks changes with j alone)
      constexpr int VX = RB == 64 ? 0 : RB == 128 ? 4 : 6;
      if (left >= WT && on) {
#pragma unroll
        for (int j = 0; j < WT / RS; ++j) cp_async16(dst + kd0 + j * 512, kp + (Q8 ? j * 512 : j * RS * k_row), 16);
#pragma unroll
        for (int j = 0; j < WT / RS; ++j)
          cp_async16(dst + (vd0 ^ (((j * RS) & VX) * 16)) + j * 512, vp + (Q8 ? j * 512 : j * RS * v_row), 16);
      } else {
#pragma unroll
        for (int j = 0; j < WT / RS; ++j) {
          const bool in = on && r0 + j * RS < left;  // (rows that are not read start nowhere else than the item's first)
          cp_async16(dst + kd0 + j * 512, in ? kp + j * RS * k_row : lane_k - (Q8 ? 0 : r0 * k_row), in ? 16 : 0);
          cp_async16(dst + (vd0 ^ (((j * RS) & VX) * 16)) + j * 512, in ? vp + j * RS * v_row : lane_v - (Q8 ? 0 : r0 * v_row),
                     in ? 16 : 0);
        }
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

  // ---- queries: row g of each block of 8, in the key reads' order
  uint32_t qf[NB][D / 16][2];
  float rs[NB][2];  // softmax factors and visible keys of rows 2 c and 2 c + 1
  int vis[NB][2];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int r = row0 + nb * 8 + g;
    const bool on = r < rows;
    const int i = on ? r / G : 0, hd = h * G + (on ? r % G : 0);
    const H* qp = reinterpret_cast<const H*>(a.q) + (long long)(it.q0 + i) * a.ldq + hd * D;
    float factor = fabsf(a.scale_log2);
    uint4 w[D / 32];
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      const int col = Q8 ? (j >> 1) * 64 + c * 16 + (j & 1) * 8 : j * 32 + c * 8;
      w[j] = on ? *reinterpret_cast<const uint4*>(qp + col) : make_uint4(0, 0, 0, 0);
      if (a.scale_log2 < 0.f) {  // the factor stays positive: the largest product has the largest score
        w[j].x ^= 0x80008000u;
        w[j].y ^= 0x80008000u;
        w[j].z ^= 0x80008000u;
        w[j].w ^= 0x80008000u;
      }
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
      factor /= f;
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
      qf[nb][2 * j][0] = w[j].x;
      qf[nb][2 * j][1] = w[j].y;
      qf[nb][2 * j + 1][0] = w[j].z;
      qf[nb][2 * j + 1][1] = w[j].w;
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      rs[nb][x] = __shfl_sync(0xffffffffu, factor, 8 * c + 4 * x);
      const int rr = row0 + nb * 8 + 2 * c + x;
      vis[nb][x] = rr < rows ? visible<Q8>(it, rr / G) : 0;
    }
  }

  float o[NB][MT][4];
  float m[NB][2], l[NB][2];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
    for (int i = 0; i < MT; ++i) o[nb][i][0] = o[nb][i][1] = o[nb][i][2] = o[nb][i][3] = 0.f;
    m[nb][0] = m[nb][1] = -INFINITY;
    l[nb][0] = l[nb][1] = 0.f;
  }
  float ref = -1000.f;  // the output is kept in units of 2^ref (8-bit cache)

  for (int i = 0; i < cnt; ++i) {
    cp_wait<kStages - 2>();
    __syncwarp();
    issue(i + kStages - 1, id_next);
    id_next = page_of(i + kStages);
    const int k0 = (t0 + W * i) * WT;
    const uint8_t* kt = ring + (i % kStages) * L::kStage;
    const uint8_t* vt = kt + L::kTile;
    float ks = 1.f, vs = 1.f, dv = 0.f;
    bool apart = false;
    if constexpr (Q8) {
      const float2 sc = *reinterpret_cast<const float2*>(ring + kStages * L::kStage + (i % kStages) * 16);
      ks = sc.x;
      vs = sc.y;
      if (ks < 0.f) continue;
      const float ev = (float)((__float_as_int(vs) >> 23) - 127);
      if (ev > ref) {
        if (ref > -1000.f) {
          const float f = ex2_approx(ref - ev);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int j = 0; j < MT; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[nb][j][e] *= f;
        }
        ref = ev;
      }
      dv = ev - ref;
      apart = dv < -4.f;
      if (apart) dv = 0.f;
    }
    // ---- scores: keys 16 t + g (and + 8) by rows 2 c, 2 c + 1
    float s[NB][WT / 16][4];
#pragma unroll
    for (int t = 0; t < WT / 16; ++t) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) s[nb][t][0] = s[nb][t][1] = s[nb][t][2] = s[nb][t][3] = 0.f;
#pragma unroll
      for (int j = 0; j < KC; ++j) {
        const uint4 ka = *reinterpret_cast<const uint4*>(kt + key_at<RB>(16 * t + g, 4 * j + c));
        const uint4 kb = *reinterpret_cast<const uint4*>(kt + key_at<RB>(16 * t + 8 + g, 4 * j + c));
        const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
        if constexpr (Q8) {
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const uint32_t f[4] = {e4m3_lo(wa[u]), e4m3_lo(wb[u]), e4m3_hi(wa[u]), e4m3_hi(wb[u])};
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) mma16816<M>(s[nb][t], f, qf[nb][4 * j + u][0], qf[nb][4 * j + u][1]);
          }
        } else {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t f[4] = {wa[2 * u], wb[2 * u], wa[2 * u + 1], wb[2 * u + 1]};
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) mma16816<M>(s[nb][t], f, qf[nb][2 * j + u][0], qf[nb][2 * j + u][1]);
          }
        }
      }
    }
    // ---- running softmax in the log2 domain
    const bool partial = k0 + WT > vmin;  // some row does not see every key of the tile
    if (partial) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int t = 0; t < WT / 16; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (k0 + 16 * t + g + 8 * (e >> 1) >= vis[nb][e & 1]) s[nb][t][e] = -INFINITY;
    }
    uint32_t pf[NB][WT / 16][2];
    float mu[NB][2], alpha[NB][2];
    bool moved = false;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float mt[2] = {s[nb][0][0], s[nb][0][1]};
#pragma unroll
      for (int t = 0; t < WT / 16; ++t) {
        mt[0] = fmaxf(mt[0], fmaxf(s[nb][t][0], s[nb][t][2]));
        mt[1] = fmaxf(mt[1], fmaxf(s[nb][t][1], s[nb][t][3]));
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int k = 4; k < 32; k <<= 1) mt[x] = fmaxf(mt[x], __shfl_xor_sync(0xffffffffu, mt[x], k));
        const float mn = fmaxf(m[nb][x], mt[x] * (rs[nb][x] * ks));  // (a NaN of no key and no factor is passed over)
        mu[nb][x] = mn == -INFINITY ? 0.f : mn;
        alpha[nb][x] = ex2_approx(m[nb][x] - mu[nb][x]);
        m[nb][x] = mn;
        moved |= alpha[nb][x] != 1.f;
      }
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        l[nb][0] *= alpha[nb][0];
        l[nb][1] *= alpha[nb][1];
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[nb][j][e] *= alpha[nb][e & 1];
      }
    }
    const float back = Q8 ? ex2_approx(-dv) : 1.f;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const float f0 = rs[nb][0] * ks, f1 = rs[nb][1] * ks, z0 = dv - mu[nb][0], z1 = dv - mu[nb][1];
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int t = 0; t < WT / 16; ++t) {
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) p[e] = ex2_approx(fmaf(s[nb][t][e], e & 1 ? f1 : f0, e & 1 ? z1 : z0));
        if (partial) {  // (zero also where the factor is zero)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (k0 + 16 * t + g + 8 * (e >> 1) >= vis[nb][e & 1]) p[e] = 0.f;
        }
        sum[0] += p[0] + p[2];
        sum[1] += p[1] + p[3];
        // probabilities in the products' type: at most half a step off each
        pf[nb][t][0] = movmatrix(pack2<M>(p[0], p[1]));
        pf[nb][t][1] = movmatrix(pack2<M>(p[2], p[3]));
      }
      l[nb][0] = fmaf(sum[0], back, l[nb][0]);
      l[nb][1] = fmaf(sum[1], back, l[nb][1]);
    }
    // ---- values: keys 16 t + {0, 1, 8, 9} + 2 c; word w of a row holds the
    // columns of output tile w (16-bit) or tiles 2 w, 2 w + 1 (8-bit)
    constexpr int VC = VW == 2 ? 2 : 4;  // words of one read
#pragma unroll
    for (int j = 0; j < VW / VC; ++j) {
      uint32_t vr[WT / 4][VC];
#pragma unroll
      for (int k = 0; k < WT / 4; ++k) {
        const int r = 16 * (k >> 2) + 2 * c + (k & 1) + 8 * ((k >> 1) & 1);
        if constexpr (VC == 2) {
          const uint2 x = *reinterpret_cast<const uint2*>(vt + value_at<RB>(r, g >> 1) + (g & 1) * 8);
          vr[k][0] = x.x;
          vr[k][1] = x.y;
        } else {
          const uint4 x = *reinterpret_cast<const uint4*>(vt + value_at<RB>(r, 8 * j + g));
          vr[k][0] = x.x;
          vr[k][1] = x.y;
          vr[k][2] = x.z;
          vr[k][3] = x.w;
        }
      }
      auto product = [&](float (&acc)[NB][4], int w, int half, int t) {
        const uint32_t a0 = vr[4 * t][w], a1 = vr[4 * t + 1][w], a2 = vr[4 * t + 2][w], a3 = vr[4 * t + 3][w];
        uint32_t f[4];
        if constexpr (Q8) {
          const uint32_t sel = half ? 0x7362 : 0x5140;
          const uint32_t lo = __byte_perm(a0, a1, sel), hi = __byte_perm(a2, a3, sel);
          f[0] = e4m3_lo(lo);
          f[1] = e4m3_hi(lo);
          f[2] = e4m3_lo(hi);
          f[3] = e4m3_hi(hi);
        } else {
          f[0] = __byte_perm(a0, a1, 0x5410);
          f[1] = __byte_perm(a0, a1, 0x7632);
          f[2] = __byte_perm(a2, a3, 0x5410);
          f[3] = __byte_perm(a2, a3, 0x7632);
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) mma16816<M>(acc[nb], f, pf[nb][t][0], pf[nb][t][1]);
      };
      constexpr int HV = Q8 ? 2 : 1;
      if (!apart) {
#pragma unroll
        for (int w = 0; w < VC; ++w)
#pragma unroll
          for (int half = 0; half < HV; ++half) {
            const int tile = (j * VC + w) * HV + half;
            float acc[NB][4];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[nb][e] = o[nb][tile][e];
#pragma unroll
            for (int t = 0; t < WT / 16; ++t) product(acc, w, half, t);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[nb][tile][e] = acc[nb][e];
          }
      } else if constexpr (Q8) {
        const float f = ex2_approx((float)((__float_as_int(vs) >> 23) - 127) - ref);
#pragma unroll
        for (int w = 0; w < VC; ++w)
#pragma unroll
          for (int half = 0; half < HV; ++half) {
            const int tile = (j * VC + w) * HV + half;
            float acc[NB][4] = {};
#pragma unroll
            for (int t = 0; t < WT / 16; ++t) product(acc, w, half, t);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[nb][tile][e] = fmaf(acc[nb][e], f, o[nb][tile][e]);
          }
      }
    }
  }
  if constexpr (Q8) {
    const float f = ref > -1000.f ? ex2_approx(ref) : 0.f;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nb][j][e] *= f;
  }

  // ---- what this warp holds: rows 2 c and 2 c + 1 of each block of 8, four
  // neighbouring columns at a time
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int k = 4; k < 32; k <<= 1) l[nb][x] += __shfl_xor_sync(0xffffffffu, l[nb][x], k);
  auto each = [&](auto&& f) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int i = 0; i < MT; i += 2) {
          const int dim = Q8 ? g * (D / 8) + 2 * i : (i >> 2) * 64 + g * 8 + 2 * (i & 3);
          f(nb, x, dim, make_float4(o[nb][i][x], o[nb][i][2 + x], o[nb][i + 1][x], o[nb][i + 1][2 + x]));
        }
  };
  const int valid = min(R, rows - row0);
  float* po = a.ws + (part_at(a, row_tiles, b, h, rt) * n_split + split) * (R * (D + 2));
  auto store_out = [&](int r, int dim, float4 v) {
    const int row = row0 + r;
    H* op = reinterpret_cast<H*>(a.out) + (long long)(it.q0 + row / G) * a.ldo + (h * G + row % G) * D + dim;
    *reinterpret_cast<uint2*>(op) = make_uint2(pack2<H>(v.x, v.y), pack2<H>(v.z, v.w));
  };
  if constexpr (W == 1) {  // (alone with its rows)
    each([&](int nb, int x, int dim, float4 v) {
      const int r = nb * 8 + 2 * c + x;
      const float inv = l[nb][x] == 0.f ? 0.f : 1.f / l[nb][x];  // no key seen: zeros
      if (r < valid) store_out(r, dim, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
    });
  } else {
    // ---- join the warps, in the rings' memory
    cp_wait<0>();
    __syncthreads();
    constexpr int LD = D + 4;
    float* s_o = reinterpret_cast<float*>(smem);  // [W][R][LD]
    float* s_ml = s_o + W * R * LD;               // [W][R][2]
    float* s_p = s_ml + W * R * 2;                // [R][LD] this CTA's sums, then [R][2]
    each([&](int nb, int x, int dim, float4 v) {
      *reinterpret_cast<float4*>(s_o + (warp * R + nb * 8 + 2 * c + x) * LD + dim) = v;
    });
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int x = 0; x < 2; ++x)
        if (g == 0)
          *reinterpret_cast<float2*>(s_ml + (warp * R + nb * 8 + 2 * c + x) * 2) = make_float2(m[nb][x], l[nb][x]);
    __syncthreads();
    for (int idx = threadIdx.x; idx < valid * (D / 4); idx += 32 * W) {
      const int r = idx / (D / 4), d4 = idx % (D / 4) * 4;
      float mm = -INFINITY;
#pragma unroll
      for (int w = 0; w < W; ++w) mm = fmaxf(mm, s_ml[(w * R + r) * 2]);
      const float base = mm == -INFINITY ? 0.f : mm;
      float ll = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float f = ex2_approx(s_ml[(w * R + r) * 2] - base);
        ll += s_ml[(w * R + r) * 2 + 1] * f;
        const float4 v = *reinterpret_cast<const float4*>(s_o + (w * R + r) * LD + d4);
        x[0] = fmaf(v.x, f, x[0]);
        x[1] = fmaf(v.y, f, x[1]);
        x[2] = fmaf(v.z, f, x[2]);
        x[3] = fmaf(v.w, f, x[3]);
      }
      if (n_split == 1) {
        const float inv = ll == 0.f ? 0.f : 1.f / ll;
        store_out(r, d4, make_float4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv));
      } else {
        float* to = clustered ? s_p + r * LD : po + r * D;
        *reinterpret_cast<float4*>(to + d4) = make_float4(x[0], x[1], x[2], x[3]);
        if (d4 == 0) *reinterpret_cast<float2*>(clustered ? s_p + R * LD + 2 * r : po + R * D + 2 * r) = make_float2(mm, ll);
      }
    }
    if (clustered) {
      // ---- the parts are the CTAs of a cluster: join them through distributed
      // shared memory, four columns a thread
      cluster_sync();
      const uint32_t base_s = smem_u32(s_p), ml_s = smem_u32(s_p + R * LD);
      for (int idx = split * 32 * W + threadIdx.x; idx < valid * (D / 4); idx += n_split * 32 * W) {
        const int r = idx / (D / 4), d4 = idx % (D / 4) * 4;
        float mm = -INFINITY;
        for (int s = 0; s < n_split; ++s) mm = fmaxf(mm, ld_cluster2(mapa_shared(ml_s + 8 * r, s)).x);
        const float base = mm == -INFINITY ? 0.f : mm;
        float ll = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < n_split; ++s) {
          const float2 ml = ld_cluster2(mapa_shared(ml_s + 8 * r, s));
          const float4 v = ld_cluster4(mapa_shared(base_s + (r * LD + d4) * 4, s));
          const float f = ex2_approx(ml.x - base);
          ll = fmaf(ml.y, f, ll);
          x[0] = fmaf(v.x, f, x[0]);
          x[1] = fmaf(v.y, f, x[1]);
          x[2] = fmaf(v.z, f, x[2]);
          x[3] = fmaf(v.w, f, x[3]);
        }
        const float inv = ll == 0.f ? 0.f : 1.f / ll;
        store_out(r, d4, make_float4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv));
      }
      cluster_sync();  // every part has been read
    }
  }
}

// Joins the parts of a row: o = sum_s o_s 2^(m_s - m) / sum_s l_s 2^(m_s - m).
// P warps a row, each taking every P-th part (a part is a read that depends on
// nothing): four for the few rows of k_attn_rows, whose parts are many, one for
// the 128-row tiles.
template <typename H, bool Q8, int D, int R, int P>
__global__ void __launch_bounds__(128) k_attn_join(const DecodeAttnArgs a, int row_tiles, int n_split) {
  __shared__ float s_x[4][D], s_l[4];
  constexpr int RC = 4 / P;  // rows of a CTA
  const int G = a.n_heads / a.n_kv_heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = blockIdx.x % (R / RC) * RC + warp / P;
  int rest = blockIdx.x / (R / RC);
  const int rt = rest % row_tiles;
  rest /= row_tiles;
  const int h = rest % a.n_kv_heads, b = rest / a.n_kv_heads;
  pdl_wait();
  pdl_trigger();
  const Item it = load_item<Q8>(a, b);
  if (!it.ok) return;
  const int row = rt * R + r;
  if (row >= it.n * G) return;
  constexpr int PS = R * (D + 2);  // floats of a part
  const float* p = a.ws + part_at(a, row_tiles, b, h, rt) * n_split * PS;
  // the largest maximum (n_split <= 64: two parts a lane)
  float m = -INFINITY;
  for (int s = lane; s < n_split; s += 32) m = fmaxf(m, p[s * PS + R * D + 2 * r]);
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
  const float base = m == -INFINITY ? 0.f : m;
  constexpr int V = D / 32;  // columns of a lane
  float x[V] = {}, l = 0.f;
#pragma unroll 4
  for (int s = warp % P; s < n_split; s += P) {
    const float2 ml = *reinterpret_cast<const float2*>(p + s * PS + R * D + 2 * r);
    if (ml.x == -INFINITY && ml.y == 0.f) continue;  // a part without keys leaves its sums unwritten
    const float f = ex2_approx(ml.x - base);
    l = fmaf(ml.y, f, l);
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = fmaf(p[s * PS + r * D + V * lane + v], f, x[v]);
  }
  if constexpr (P > 1) {
#pragma unroll
    for (int v = 0; v < V; ++v) s_x[warp][V * lane + v] = x[v];
    if (lane == 0) s_l[warp] = l;
    __syncthreads();
    if (warp > 0) return;
    l = (s_l[0] + s_l[1]) + (s_l[2] + s_l[3]);
#pragma unroll
    for (int v = 0; v < V; ++v)
      x[v] = (s_x[0][V * lane + v] + s_x[1][V * lane + v]) + (s_x[2][V * lane + v] + s_x[3][V * lane + v]);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  H* op = reinterpret_cast<H*>(a.out) + (long long)(it.q0 + row / G) * a.ldo + (h * G + row % G) * D + V * lane;
#pragma unroll
  for (int v = 0; v < V; v += 2) *reinterpret_cast<uint32_t*>(op + v) = pack2<H>(x[v] * inv, x[v + 1] * inv);
}

// How a call is cut. (tiles: false for what the tcgen05 kernel cannot describe,
// which then needs no workspace either.)
//  - Items of many rows (few_rows below): tiles of 128 rows on tcgen05
//    (decode_attn_tc.cu), the keys in parts where there are few tiles.
//  - Blocks of 8 rows, or of 16 where an item has more: they share one read of
//    the keys.
//  - Eight to 16 warps run on an SM, by their registers. Many blocks: a warp
//    takes one alone (CTAs of one warp, no join); fewer: four warps share one.
//  - Still fewer: the keys are cut into parts of at least 128, one for each CTA
//    of a cluster, which joins them: one launch and no workspace.
//  - Where that leaves SMs without work and the parts are long, into more
//    parts, about six CTAs an SM (lengths differ; three run at a time), joined
//    by a second kernel.
//  - Parts of less than 1024 keys, and one item's, which has one length: no more
//    of them than run at a time, since a round of short ones is mostly their
//    starts (64 sequences of 4 new tokens over 300, 16 heads of 64 for 4: one
//    part 8 us, three 21; 16 clips of one row over 2000 keys, 8 heads of 128:
//    three parts 24 us, six 28). Two that fill a little more than one round are
//    kept down to 512 keys (32 clips of 4 rows over 200 to 1500, 8 heads of 64:
//    18 us, one part 21).
struct Plan {
  int rows, warps, n_split;  // warps 0: the tcgen05 kernel
  bool clustered;            // the parts are joined in a cluster
  long long row_tiles, blocks;
};
// Blocks of a call whose bounds may be loose; more than a grid has count as
// 2^31, which is refused where the call is launched.
long long count_blocks(int n_items, int n_kv_heads, long long row_tiles) {
  const double n = (double)n_items * n_kv_heads * (double)row_tiles;
  return n < (double)(1LL << 31) ? (long long)n_items * n_kv_heads * row_tiles : 1LL << 31;
}
// Parts of the keys for the tcgen05 kernel, of at least 256 keys; 2 * kSms CTAs
// run at a time.
//  - One item: the number that ends first, in tiles one after another, the start
//    and the end of a part counted as six. 256 new tokens over 16384, 16 heads
//    of 64 for 4: nine parts in one round 57 us, 19 in a little over two 74 us.
//  - Several, whose lengths may differ: one round of CTAs, or two of parts of at
//    least 512 keys over the 8-bit cache, whose tiles cost more (the 8-bit chunk
//    180 us with one, 174 with two); one where that leaves the second mostly
//    empty (three items of 8192, 8 heads for one: 48 instead of 62 us).
int tile_parts(int n_items, long long blocks, int max_kv, bool q8) {
  constexpr long long slots = 2LL * kSms;
  const int tiles = max_kv / 64 + 1, most = max_kv / 256 < 1 ? 1 : max_kv / 256 > 64 ? 64 : max_kv / 256;
  if (n_items == 1) {
    int best = 1;
    long long least = 0;
    for (int n = 1; n <= most; ++n) {
      const long long cost = (blocks * n + slots - 1) / slots * ((tiles + n - 1) / n + 6);
      if (n == 1 || cost < least) best = n, least = cost;
    }
    return best;
  }
  if (blocks <= 0) return 1;
  const long long fill = q8 ? 2 * slots : slots;
  long long n = fill / blocks;
  if (n < 4) n = (fill + blocks - 1) / blocks;
  if (n > most) n = most;
  if (blocks * n > slots && n > max_kv / 512) n = max_kv / 512;
  if (4 * blocks <= slots && blocks * n > slots && 4 * blocks * n < 7 * slots) n = slots / blocks;
  return n < 1 ? 1 : (int)n;
}

// Whether an item's rows for one key head are few, blocks of 16 of which read
// the keys again, rather than a tile of 128 with its longer start:
//  - up to 32;
//  - up to 64 where the blocks have little to do, 2^22 keys x columns in all, or
//    2^24 over the 8-bit cache, whose tiles cost more (one clip of 36 rows over
//    500 keys, 8 heads of 64: 6 us, tiles 9; 4 clips over 1500: 16 and 14 us.
//    16 new tokens of 32 heads for 8 of 128 over 4000 cached ones: 15 us, tiles
//    21; over 60000: 107 and 89 us);
//  - over at most 2048 cached tokens up to 48, or 64 of 64 columns (128
//    sequences of 100 to 1500, 36 to 64 rows of 64 columns: 54 to 67 us, tiles
//    87 to 90; 200 of 36 rows of 128 columns 85 and 120 us).
bool few_rows(long long rows, int n_items, int max_kv, int n_kv_heads, int head_dim, bool q8) {
  if (rows <= 32) return true;
  if (rows > 64) return false;
  const double work = (double)n_items * n_kv_heads * ((rows + 15) / 16) * max_kv * head_dim;
  return work <= (q8 ? 1 << 24 : 1 << 22) || (q8 && max_kv <= 2048 && (rows <= 48 || head_dim == 64));
}

Plan plan_rows(int n_items, int max_q, int max_kv, int n_heads, int n_kv_heads, int head_dim, bool q8,
               bool tiles_ok = true) {
  Plan p;
  const long long rows = (long long)max_q * (n_heads / n_kv_heads);
  if (tiles_ok && !few_rows(rows, n_items, max_kv, n_kv_heads, head_dim, q8)) {
    p.rows = kTileRows;
    p.row_tiles = (rows + p.rows - 1) / p.rows;
    p.blocks = count_blocks(n_items, n_kv_heads, p.row_tiles);
    p.warps = 0;
    p.clustered = false;
    p.n_split = tile_parts(n_items, p.blocks, max_kv, q8);
    return p;
  }
  p.rows = rows <= 8 ? 8 : 16;
  p.row_tiles = (rows + p.rows - 1) / p.rows;
  p.blocks = count_blocks(n_items, n_kv_heads, p.row_tiles);
  // warps that run at a time; rounds of CTAs of w warps over tiles of keys, the
  // start and the end of a CTA counted as five tiles
  const int warps_sm = head_dim == 128 ? (p.rows == 8 ? 12 : 8) : p.rows == 8 ? 16 : q8 ? 8 : 12;
  const long long slots = (long long)warps_sm * kSms, tiles = max_kv / (q8 ? 32 : 16) + 1;
  auto cost = [&](int w) { return (p.blocks * w + slots - 1) / slots * ((tiles + w - 1) / w + 5); };
  p.warps = p.blocks > 6 * kSms || (4 * p.blocks > slots && cost(1) < cost(4)) ? 1 : 4;
  p.n_split = 1;
  p.clustered = false;
  if (p.warps == 4 && tiles_ok && p.blocks > 0) {
    const long long most = ((long long)max_kv + 127) / 128, want = 6LL * kSms / p.blocks, round = slots / 4 / p.blocks;
    const long long n0 = want < most ? want : most;
    p.clustered = n0 <= 8 || max_kv <= 8 * 1024;
    long long n = p.clustered && n0 > 8 ? 8 : n0 > 64 ? 64 : n0;
    const bool brief = max_kv < 1024 * n && (round > 1 || max_kv < 512 * n);
    if ((n_items == 1 || brief) && n > round) n = round;
    p.n_split = n < 1 ? 1 : (int)n;
    p.clustered = p.clustered && p.n_split > 1;
  }
  return p;
}

template <typename H, bool Q8, int D, int WT, int W, int NB>
cudaError_t launch_w(const DecodeAttnArgs& a, const Plan& p, cudaStream_t st) {
  auto kern = k_attn_rows<H, Q8, D, WT, W, NB>;
  // the rings, and in their place the join of the warps
  constexpr int rings = W * RowsLayout<Q8 ? D : 2 * D, WT, NB>::kWarp, join = (W + 1) * 8 * NB * (D + 6) * 4;
  constexpr int smem = W > 1 && join > rings ? join : rings;
  static PerDevice once;
  int unused = 0;
  cudaError_t e = per_device(once, &unused, [&](int, int&) {
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  });
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.blocks * p.n_split));
  cfg.blockDim = dim3(32 * W);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = p.n_split;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = p.clustered ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, kern, a, (int)p.row_tiles, p.n_split, p.clustered ? 1 : 0);
  if (e != cudaSuccess || p.n_split == 1 || p.clustered) return e;
  return launch_pdl(k_attn_join<H, Q8, D, 8 * NB, 4>, dim3((unsigned)(p.blocks * 8 * NB)), dim3(128), 0, st, a,
                    (int)p.row_tiles, p.n_split);
}

template <typename H, bool Q8, int D, int WT>
cudaError_t launch_rows(const DecodeAttnArgs& a, cudaStream_t st) {
  const Plan p = plan_rows(a.n_items, a.max_q, a.max_kv, a.n_heads, a.n_kv_heads, D, Q8, attn_tiles_fit(a));
  if (p.blocks * p.n_split * p.rows > 0x7fffffffLL) return cudaErrorInvalidValue;
  if (p.warps == 0) {
    const cudaError_t e = attn_tiles_launch(a, is_bf16<H>::value, (int)p.row_tiles, p.n_split, st);
    if (e != cudaSuccess || p.n_split == 1) return e;
    return launch_pdl(k_attn_join<H, Q8, D, kTileRows, 1>, dim3((unsigned)(p.blocks * (kTileRows / 4))), dim3(128), 0, st, a,
                      (int)p.row_tiles, p.n_split);
  }
  if (p.rows == 8)
    return p.warps == 1 ? launch_w<H, Q8, D, WT, 1, 1>(a, p, st) : launch_w<H, Q8, D, WT, 4, 1>(a, p, st);
  return p.warps == 1 ? launch_w<H, Q8, D, WT, 1, 2>(a, p, st) : launch_w<H, Q8, D, WT, 4, 2>(a, p, st);
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
  const Plan p = plan_rows(n_items, max_q, max_kv, n_heads, n_kv_heads, head_dim, q8);
  return p.n_split == 1 || p.clustered ? 0 : (size_t)p.blocks * p.n_split * p.rows * (head_dim + 2) * sizeof(float);
}

cudaError_t decode_attn_launch(const DecodeAttnArgs& a, bool bf16, cudaStream_t st) {
  if (a.n_items <= 0 || a.max_q <= 0) return cudaSuccess;
  return bf16 ? launch_h<__nv_bfloat16>(a, st) : launch_h<__half>(a, st);
}

}  // namespace pkc
