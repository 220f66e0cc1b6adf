// Attention of many query rows over keys and values of another length on the
// 5th-generation tensor cores: rescoring, prompts, chunks of a prompt. The
// operators and their masks are those of decode_attn.cu.
//
// One CTA takes 128 query rows (tokens x heads of one shared key head: one
// TMEM lane each) of one item and one part of its keys, in tiles of 64 keys:
//   S = Q K^T  (tcgen05.mma, f32 in tensor memory), p = exp2(c S - m),
//   O += P V   (P in 16 bits in tensor memory, over the S that it came from).
// Two CTAs share an SM (half of the tensor memory each): while one's softmax
// runs, the other's products do. A row is a thread, so its maximum and sum
// need no exchange; the maximum that the exponentials use moves only when it
// is exceeded by more than 2^8, and only then is O rescaled.
//
// Tensor memory (256 columns x 128 lanes): S of even and odd tiles at 0 and 64
// (the first 32 columns of each become that tile's P), O at 128.
// Shared memory: Q (written by the softmax warps, in the 128-byte swizzle that
// the products read), a ring of four 64-row tiles K0 K1 V0 K2 V1 ... in the
// order of their use.
//
// 16-bit keys and values come by TMA. Rows behind an item's last key belong to
// others: their scores are masked, and their values, which a zero probability
// would not silence if they are not numbers, are zeroed in the last tile.
//
// The 8-bit cache's codes are turned into f16 by four warps that write the same
// ring: exactly, with the value scale taken in as a power of two relative to a
// reference 2^ref in which O is kept. f16 holds e4m3 codes times 2^-15 .. 2^7
// exactly, so ref stands while the pages stay in that range of it; else it
// moves to the tile's largest scale and O is multiplied. A tile of several
// small pages that are further apart than that takes them one after another,
// each under its own reference (16 keys of one product step lie in one page).
// A page more than 2^80 below the largest one so far (all zeros, as a rule:
// their scale is 2^-126) counts as zeros and moves nothing. So O stays finite
// however far ref falls: with weights up to 2^8, 2^30 keys and codes up to 448 it
// is below 2^47 in units of the largest scale, and below 2^127 in those of ref.
//
// Measured: 64 x 130 to 384 rows over 250 to 1500 keys, 8 heads of 128: 104 us,
// 570 TFLOP/s, at 1965 MHz; 120 us on end, where the power cap holds 1645 MHz.
// A tile takes a CTA 1450 cycles beside the other CTA's; the products alone are
// 640 for each of the two (a step of 64 columns reads 6 KB of shared memory, 48
// cycles, for 32 of products), and about 10,000 cycles a CTA lie before its
// first and behind its last tile. 8 x 100 to 256 new tokens
// over 300 to 16384 cached ones, 16 heads of 64 for 4, pages of 64: 174 us, 300
// TFLOP/s: a tile takes a CTA 2400 cycles and more, of which its softmax warps
// work 1860 (96 registers, of which 56 to 64 bytes are spilled, beside converting
// warps that use a third of the issue slots) and wait the rest; 53% of the issue
// slots are used. Two row tiles a CTA under one conversion took 186 us (16-bit
// keys: 135 instead of 104), three converting warps and 128 registers 169 us but
// up to 19% more with 128 columns.
#include "common.cuh"
#include "decode.h"
#include "decode_common.cuh"
#include "gemm.h"
#include "per_device.h"

namespace pkc {

namespace {

constexpr int QM = kTileRows;
constexpr int KN = 64;
constexpr int SOFT_WARPS = 4;
constexpr int CVT_WARPS = 4;
constexpr float kRescaleLog2 = 8.0f;
constexpr float kTiny = 1e-38f;  // the least softmax factor: a masked score (-inf) times zero is not a number
constexpr uint32_t TM_O = 128, TM_COLS = 256;

constexpr int MAX_RING = 4;  // 64-row tiles of keys or values
enum : int {
  B_QREADY = 0, B_RFULL = 1, B_REMPTY = B_RFULL + MAX_RING, B_SFULL = B_REMPTY + MAX_RING, B_PFULL = B_SFULL + 2,
  B_PVDONE = B_PFULL + 2, B_INFO = B_PVDONE + 2, B_FINAL = B_INFO + MAX_RING, N_BARS = B_FINAL + 1
};

// What the converting warps tell the softmax about a tile.
struct TileInfo {
  float4 head;    // the largest key scale (of a tile in one page: its own, negative: a page that is none), what O is
                  // multiplied by before the tile is added (see move_by), the exponent that O is kept under behind the tile,
                  // parts (1, or the tile's pages)
  float4 ks;      // several pages: key scale of each 16 keys over the largest; negative: a page that is none
  float grow[4];  // and, where it has parts, what O is multiplied by before each
};

// Two CTAs have 113 KB each: with the converting warps' raw codes the ring of
// 128-column tiles has three places instead of four.
template <bool Q8, int D>
struct TilesLayout {
  static constexpr int KB = D / 64;
  static constexpr int RING = Q8 && D == 128 ? 3 : 4;
  static constexpr int RAW = D == 128 ? 1 : 2;               // a converting warp's tiles whose codes are on their way
  static constexpr int ROWS = KN / (CVT_WARPS / 2);          // of a tile, for each of them
  static constexpr int RAW_BYTES = ROWS * D + 256;           // their codes, then two scales a lane
  static constexpr int Q_BYTES = QM * D * 2;
  static constexpr int T_BYTES = KB * KN * 128;
  static constexpr int OFF_RING = Q_BYTES;
  static constexpr int OFF_RAW = OFF_RING + RING * T_BYTES;
  static constexpr int OFF_FACTOR = OFF_RAW + (Q8 ? CVT_WARPS * RAW * RAW_BYTES : 0);  // [QM] softmax factors
  static constexpr int OFF_INFO = OFF_FACTOR + QM * 4;                     // [RING] TileInfo
  static constexpr int OFF_BAR = OFF_INFO + RING * 64;
  static constexpr int OFF_SLOT = OFF_BAR + N_BARS * 8;
  static constexpr int SMEM = OFF_SLOT + 16 + 1024;  // + alignment slack
  static_assert(2 * (SMEM + 1024) <= 228 * 1024, "two CTAs share an SM");
};
static_assert(sizeof(TileInfo) <= 64, "the layout gives it 64 bytes");

// place of a tile in the ring's order K0 K1 V0 K2 V1 ... K(n-1) V(n-2) V(n-1)
__device__ __forceinline__ int at_k(int t) { return t < 2 ? t : 2 * t - 1; }
__device__ __forceinline__ int at_v(int t, int n) { return t < n - 2 ? 2 * t + 2 : t == n - 1 ? 2 * n - 1 : 2 * n - 2; }

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint64_t fadd2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

constexpr int kFarBelow = 80;  // exponents; see above
constexpr int kNoPage = -1000;

__device__ __forceinline__ float pow2i(int e) {  // 2^e for e <= 127; 0 below 2^-126
  return e < -126 ? 0.f : __int_as_float((e + 127) << 23);
}
// What O is multiplied by when its reference moves: 2^e, or -2^(e + 126) for
// 2^e below 2^-126 (a page 2^80 above the largest so far, which may be 2^80
// above the reference, still leaves that one's values their bits).
__device__ __forceinline__ float move_by(int e) { return e < -126 ? -pow2i(e + 126) : pow2i(e); }

template <typename H, bool Q8, int D>
__global__ void __launch_bounds__(32 * (1 + SOFT_WARPS + (Q8 ? CVT_WARPS : 1)), 2)
    k_attn_tiles(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const DecodeAttnArgs a,
                 int row_tiles, int n_split) {
  using M = typename std::conditional<Q8, __half, H>::type;
  using L = TilesLayout<Q8, D>;
  constexpr int RING = L::RING;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + L::OFF_BAR);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + L::OFF_SLOT);
  float* s_factor = reinterpret_cast<float*>(sm + L::OFF_FACTOR);
  const uint32_t sbase = smem_u32(sm);
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  auto info = [&](int t) { return reinterpret_cast<TileInfo*>(sm + L::OFF_INFO + (t % RING) * 64); };

  const int G = a.n_heads / a.n_kv_heads;
  const int split = blockIdx.x % n_split;
  int rest = blockIdx.x / n_split;
  const int rt = rest % row_tiles;
  rest /= row_tiles;
  const int h = rest % a.n_kv_heads, b = rest / a.n_kv_heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  const Item it = load_item<Q8>(a, b);
  if (!it.ok) {
    if (threadIdx.x == 0) report_error(a.err, DEV_ERR_BAD_SHAPE);
    return;
  }
  const int rows = it.n * G, row0 = rt * QM;
  if (row0 >= rows) return;
  const int valid = min(QM, rows - row0);
  const int vmax = max(0, visible<Q8>(it, (row0 + valid - 1) / G));  // keys that some row sees
  const int vmin = Q8 ? visible<Q8>(it, row0 / G) : vmax;            // keys that every row sees
  const int n_all = (vmax + KN - 1) / KN, per = (n_all + n_split - 1) / n_split;
  const int t0 = split * per;
  const int nT = max(0, min(n_all, t0 + per) - t0);  // this CTA's tiles: t0, t0 + 1, ...

  constexpr int LOAD_WARP = 1 + SOFT_WARPS;  // TMA producer, or the first converting warp
  // 16-bit keys and values: load n of the ring's order K0 K1 V0 K2 V1 ...
  int n_load = 0, k_load = 0, v_load = 0;
  auto load_next = [&](uint32_t leader) {
    if constexpr (!Q8) {
      const int s = n_load % RING;
      const bool is_k = k_load < nT && n_load == at_k(k_load);
      const int t = is_k ? k_load++ : v_load++;
      const CUtensorMap* map = is_k ? &tm_k : &tm_v;
      mbar_arrive_expect_tx_if(leader, bar(B_RFULL + s), L::T_BYTES);
#pragma unroll
      for (int kb = 0; kb < L::KB; ++kb)
        tma_load_2d_if(leader, sbase + L::OFF_RING + s * L::T_BYTES + kb * KN * 128, map, bar(B_RFULL + s),
                       h * D + kb * 64, it.kv0 + (t0 + t) * KN);
      ++n_load;
    }
  };
  uint32_t load_leader = 0;
  if (warp == LOAD_WARP) {
    if (lane < N_BARS) {
      const int i = lane;
      const bool soft = i == B_QREADY || i == B_PFULL || i == B_PFULL + 1;
      const bool full = i >= B_RFULL && i < B_RFULL + MAX_RING;
      mbar_init(bar(i), soft ? SOFT_WARPS : full && Q8 ? CVT_WARPS / 2 : 1);
    }
    static_assert(N_BARS <= 32, "a lane each");
    fence_barrier_init();
    __syncwarp();
    // the first loads need not wait for the other warps
    load_leader = elect_one();
    if constexpr (!Q8)
      while (n_load < min(RING, 2 * nT)) load_next(load_leader);
  }
  if (warp == 0) {
    tmem_alloc(smem_u32(tmem_slot), TM_COLS);
    tmem_relinquish();
  }
  // ---- softmax warps: 32 rows of Q each, D / 8 lanes a row, asked for before
  // the wait for the tensor memory (and all of them before the first is stored)
  constexpr int CH = D / 8, RP = 32 / CH;
  const int ch = lane % CH;
  const bool soft_warp = warp >= 1 && warp <= SOFT_WARPS;
  uint4 qw[32 / RP];
  // row, head of the group and token of this lane's first row; the next are RP
  // rows on each
  const int r_lane = 32 * (warp & 3) + lane / CH;
  const int i_first = (row0 + r_lane) / G, g_first = (row0 + r_lane) % G;
  const int i_step = RP / G, g_step = RP % G;
  if (soft_warp) {
    int i = i_first, gh = g_first;
#pragma unroll
    for (int j = 0; j < 32 / RP; ++j) {
      qw[j] = make_uint4(0, 0, 0, 0);
      if (r_lane + j * RP < valid)
        qw[j] = *reinterpret_cast<const uint4*>(reinterpret_cast<const H*>(a.q) + (long long)(it.q0 + i) * a.ldq +
                                                (h * G + gh) * D + ch * 8);
      i += i_step;
      gh += g_step;
      if (gh >= G) gh -= G, ++i;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // (not before this block has its tensor memory: a dependent kernel's block
  // may take all of the SM's and then wait for this kernel's end)
  pdl_trigger();
  const uint32_t tmem = *tmem_slot;
  auto wwait = [&](int i, uint32_t parity) -> bool {
    return __all_sync(0xffffffffu, mbar_wait(bar(i), parity, a.err, DEV_ERR_TIMEOUT_ATTN)) != 0;
  };
  // pages: tokens of a page, pages in a tile, keys of one in it
  const int page = Q8 ? a.cache.page : KN, np = Q8 && page < KN ? KN / page : 1;

  if (warp == 0) {
    // ------------------------------------------------------------------ MMA issuer
    if (nT > 0) {
      const uint32_t leader = elect_one();
      constexpr int fmt = is_bf16<M>::value ? 1 : 0;
      constexpr uint32_t id_s = idesc_f16(QM, KN, fmt);
      constexpr uint32_t id_pv = idesc_f16(QM, D, fmt) | (1u << 16);  // B (V) MN-major
      const uint64_t dq = smem_desc_sw128(sbase);
      auto ring_wait = [&](int n) -> bool {
        if (!wwait(B_RFULL + n % RING, (uint32_t)(n / RING) & 1u)) return false;
        tc_fence_after();
        return true;
      };
      auto ring_addr = [&](int n) { return sbase + L::OFF_RING + (n % RING) * L::T_BYTES; };
      auto s_mma = [&](int t) -> bool {
        const int n = at_k(t);
        if (!ring_wait(n)) return false;
        const uint64_t dk = smem_desc_sw128(ring_addr(n));
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_f16_if(leader, tmem + 64u * (uint32_t)(t & 1), dq + (uint64_t)(((kk >> 2) * QM * 128 + (kk & 3) * 32) >> 4),
                      dk + (uint64_t)(((kk >> 2) * KN * 128 + (kk & 3) * 32) >> 4), id_s, kk > 0 ? 1u : 0u);
        umma_commit_if(leader, bar(B_REMPTY + n % RING));
        umma_commit_if(leader, bar(B_SFULL + (t & 1)));
        return true;
      };
      bool ok = wwait(B_QREADY, 0);
      tc_fence_after();
      ok = ok && s_mma(0) && (nT < 2 || s_mma(1));
      uint32_t pf = 0;  // completed phases of the two PFULL barriers, as parities
      for (int t = 0; t < nT && ok; ++t) {
        const int n = at_v(t, nT), buf = t & 1;
        if (!(ok = ring_wait(n))) break;
        if constexpr (!Q8) {
          const int left = vmax - (t0 + t) * KN;
          if (left < KN) {
            uint8_t* vt = sm + L::OFF_RING + (n % RING) * L::T_BYTES;
#pragma unroll
            for (int kb = 0; kb < L::KB; ++kb)
              for (int at = left * 128 + lane * 16; at < KN * 128; at += 512)
                *reinterpret_cast<uint4*>(vt + kb * KN * 128 + at) = make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();
            __syncwarp();
          }
        }
        const uint64_t dv = smem_desc_sw128_mn(ring_addr(n), KN * 128, 1024);
        const uint32_t pa = tmem + 64u * (uint32_t)buf;
        const int parts = Q8 ? (int)info(t)->head.w : 1;
        const int part_shift = parts == 1 ? 2 : parts == 2 ? 1 : 0;  // of 16-key steps
        for (int j = 0; j < parts && ok; ++j) {
          ok = wwait(B_PFULL + buf, (pf >> buf) & 1u);
          pf ^= 1u << buf;
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < KN / 16; ++kk)
            if (kk >> part_shift == j)
              umma_f16_ts_if(leader, tmem + TM_O, pa + 8u * kk, dv + (uint64_t)((kk * 16 * 128) >> 4), id_pv,
                             (t > 0 || kk > 0) ? 1u : 0u);
          if (j == parts - 1) umma_commit_if(leader, bar(B_REMPTY + n % RING));
          umma_commit_if(leader, bar(B_PVDONE + buf));
        }
        if (ok && t + 2 < nT) ok = s_mma(t + 2);
      }
      // every issued product has completed before the tensor memory goes
      umma_commit_if(leader, bar(B_FINAL));
      wwait(B_FINAL, 0);
    }
  } else if (warp <= SOFT_WARPS) {
    // ---------------------------------------------------------------- softmax warps
    const int q = warp & 3;  // TMEM lane quarter
    const int i = 32 * q + lane;
    const uint32_t trow = tmem + ((uint32_t)(32 * q) << 16);
    // ---- this warp's 32 rows of Q into the operand's layout
#pragma unroll
    for (int j = 0; j < 32 / RP; ++j) {
      const int r = 32 * q + j * RP + lane / CH;
      uint4 w = qw[j];
      if (a.scale_log2 < 0.f) {  // the factor stays positive: the largest product has the largest score
        w.x ^= 0x80008000u;
        w.y ^= 0x80008000u;
        w.z ^= 0x80008000u;
        w.w ^= 0x80008000u;
      }
      float factor = fabsf(a.scale_log2);
      if constexpr (Q8 && is_bf16<H>::value) {
        // to f16 with a power of two for the row (see decode_attn.cu)
        const H* x = reinterpret_cast<const H*>(&w);
        float m = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) m = fmaxf(m, fabsf(from_h(x[k])));
#pragma unroll
        for (int k = CH / 2; k > 0; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
        const int e = ((__float_as_int(m) >> 23) & 255) - 127;
        const float f = m > 0.f && e < 127 && e > -126 ? __int_as_float((127 - e) << 23) : 1.f;
        factor /= f;
        uint32_t o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = pack2<__half>(from_h(x[2 * k]) * f, from_h(x[2 * k + 1]) * f);
        w = make_uint4(o[0], o[1], o[2], o[3]);
      }
      if (ch == 0) s_factor[r] = factor;
      *reinterpret_cast<uint4*>(sm + (ch >> 3) * QM * 128 + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = w;
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(B_QREADY));

    // (over the 8-bit cache together with a key scale: the one may be as small
    // as the other is large)
    const float rs = Q8 ? s_factor[i] : fmaxf(s_factor[i], kTiny);
    const int vis = i < valid ? visible<Q8>(it, (row0 + i) / G) : 0;
    float m_used = -INFINITY, lsum = 0.f, ref = 0.f;
    bool ok = true;
    uint32_t pvw = 0;        // PVDONE phases: parity to wait for next, per buffer
    int pv_buf = -1;         // buffer of the last part handed to the MMA warp
    uint32_t pv_par = 0;
    // O of the parts so far is complete
    auto o_settled = [&]() -> bool {
      if (pv_buf < 0) return true;
      if (!wwait(B_PVDONE + pv_buf, pv_par)) return false;
      tc_fence_after();
      return true;
    };
    auto scale_o = [&](float f, float g) {
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tmem_ld32(trow + TM_O + 32u * c, o);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f * g);
        tmem_st32(trow + TM_O + 32u * c, o);
      }
      tmem_st_wait();
    };
    for (int t = 0; t < nT && ok; ++t) {
      const int buf = t & 1, k0 = (t0 + t) * KN;
      if (!(ok = wwait(B_SFULL + buf, (uint32_t)(t >> 1) & 1u))) break;
      tc_fence_after();
      float4 ti = make_float4(1.f, 1.f, 0.f, 1.f), ks4 = ti;
      if constexpr (Q8) {
        if (!(ok = wwait(B_INFO + t % RING, (uint32_t)(t / RING) & 1u))) break;
        ti = info(t)->head;
        if (np > 1) ks4 = info(t)->ks;
      }
      float x[KN];
      {
        uint32_t s0[32], s1[32];
        tmem_ld32(trow + 64u * buf, s0);
        tmem_ld32(trow + 64u * buf + 32u, s1);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          x[j] = __uint_as_float(s0[j]);
          x[32 + j] = __uint_as_float(s1[j]);
        }
      }
      float c = rs;
      if constexpr (Q8) {
        c = fmaxf(c * fabsf(ti.x), kTiny);
        if (np > 1) {
#pragma unroll
          for (int j = 0; j < KN; ++j) x[j] *= fabsf(j < 16 ? ks4.x : j < 32 ? ks4.y : j < 48 ? ks4.z : ks4.w);
        }
      }
      if (k0 + KN > vmin) {
#pragma unroll
        for (int j = 0; j < KN; ++j)
          if (k0 + j >= vis) x[j] = -INFINITY;
      }
      if constexpr (Q8) {
        // pages that are none are not seen
        if (np == 1) {
          if (ti.x < 0.f) {
#pragma unroll
            for (int j = 0; j < KN; ++j) x[j] = -INFINITY;
          }
        } else if (fminf(fminf(ks4.x, ks4.y), fminf(ks4.z, ks4.w)) < 0.f) {
#pragma unroll
          for (int j = 0; j < KN; ++j)
            if ((j < 16 ? ks4.x : j < 32 ? ks4.y : j < 48 ? ks4.z : ks4.w) < 0.f) x[j] = -INFINITY;
        }
      }
      // (three-way maxima; a NaN is passed over here and makes its weight one)
      float mx[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        mx[k] = max3(x[k], x[4 + k], x[8 + k]);
#pragma unroll
        for (int j = 12; j < KN - 4; j += 8) mx[k] = max3(mx[k], x[j + k], x[j + 4 + k]);
        mx[k] = fmaxf(mx[k], x[KN - 4 + k]);
      }
      const float mt = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]) * c;
      float alpha = 1.f;
      if (mt > m_used + kRescaleLog2) {
        alpha = ex2_approx(m_used - mt);
        m_used = mt;
        lsum *= alpha;
      }
      const float mu = m_used == -INFINITY ? 0.f : m_used;
      uint32_t pk[KN / 2];
      uint64_t sum[4] = {0, 0, 0, 0};
      const uint64_t c2 = f2_pack(c, c), mu2 = f2_pack(-mu, -mu);
#pragma unroll
      for (int j = 0; j < KN / 2; ++j) {
        const float2 y = f2_unpack(ffma2(f2_pack(x[2 * j], x[2 * j + 1]), c2, mu2));
        const float p0 = ex2_approx(y.x), p1 = ex2_approx(y.y);
        sum[j & 3] = fadd2(sum[j & 3], f2_pack(p0, p1));
        pk[j] = pack2<M>(p0, p1);
      }
      const float2 total = f2_unpack(fadd2(fadd2(sum[0], sum[1]), fadd2(sum[2], sum[3])));
      lsum += total.x + total.y;
      tmem_st32(trow + 64u * buf, pk);
      // ---- O: the row's maximum moved, or the reference of the values did
      const int parts = Q8 ? (int)ti.w : 1;
#pragma unroll 1
      for (int j = 0; j < parts && ok; ++j) {
        const float move = Q8 ? (j == 0 ? ti.y : info(t)->grow[j]) : 1.f;
        const float f = j == 0 ? alpha * fabsf(move) : fabsf(move);
        const bool scale = pv_buf >= 0 && __any_sync(0xffffffffu, f != 1.f);
        // (a part that is not the tile's first also waits because its arrival
        // below must not count for the part before)
        if ((scale || j > 0) && !(ok = o_settled())) break;
        if (scale) scale_o(f, Q8 && move < 0.f ? 0x1p-126f : 1.f);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_PFULL + buf));
        pv_buf = buf;
        pv_par = (pvw >> buf) & 1u;
        pvw ^= 1u << buf;
      }
      if constexpr (Q8) ref = ti.z;
    }
    // (without a tile nothing above has waited for the other warps' rows of Q,
    // which lie where this one's output goes)
    if (ok) ok = nT > 0 ? o_settled() : wwait(B_QREADY, 0);
    // ---- O / l, through this warp's rows of the Q tile (every product that
    // reads Q is done), stored as whole rows; or the part's sums
    if (ok) {
      const float back = Q8 && nT > 0 ? pow2i((int)ref) : 1.f;
      if (n_split == 1) {
        // (1 / l and 2^ref apart: their product may be too small for all of its bits)
        const float inv = lsum == 0.f ? 0.f : 1.f / lsum;  // no key seen: zeros
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          if (nT > 0) {
            tmem_ld32(trow + TM_O + 32u * c, o);
            tmem_ld_wait();
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w[e] = lsum == 0.f ? 0u : pack2<H>(__uint_as_float(o[8 * k + 2 * e]) * inv * back,
                                                 __uint_as_float(o[8 * k + 2 * e + 1]) * inv * back);
            *reinterpret_cast<uint4*>(sm + i * (D * 2) + (((4 * c + k) ^ (i & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 32 / RP; ++j) {
          const int r = r_lane + j * RP;
          qw[j] = *reinterpret_cast<const uint4*>(sm + r * (D * 2) + ((ch ^ (r & 7)) << 4));
        }
        int i = i_first, gh = g_first;
#pragma unroll
        for (int j = 0; j < 32 / RP; ++j) {
          if (r_lane + j * RP < valid)
            *reinterpret_cast<uint4*>(reinterpret_cast<H*>(a.out) + (long long)(it.q0 + i) * a.ldo + (h * G + gh) * D +
                                      ch * 8) = qw[j];
          i += i_step;
          gh += g_step;
          if (gh >= G) gh -= G, ++i;
        }
      } else {
        float* po = a.ws + (part_at(a, row_tiles, b, h, rt) * n_split + split) * (QM * (D + 2));
#pragma unroll 1
        for (int c = 0; c < D / 32 && nT > 0; ++c) {
          uint32_t o[32];
          tmem_ld32(trow + TM_O + 32u * c, o);
          tmem_ld_wait();
          if (i < valid) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<float4*>(po + i * D + 32 * c + e) =
                  make_float4(__uint_as_float(o[e]) * back, __uint_as_float(o[e + 1]) * back,
                              __uint_as_float(o[e + 2]) * back, __uint_as_float(o[e + 3]) * back);
          }
        }
        if (i < valid) *reinterpret_cast<float2*>(po + QM * D + 2 * i) = make_float2(m_used, lsum);
      }
    }
  } else if constexpr (!Q8) {
    // ------------------------------------------------------------------ TMA producer
    while (n_load < 2 * nT) {
      if (!wwait(B_REMPTY + n_load % RING, ((uint32_t)(n_load / RING) & 1u) ^ 1u)) break;
      load_next(load_leader);
    }
    if (n_load < 2 * nT) {
      // a consumer gave up: every copy in flight lands before the CTA exits
      for (int m = n_load - RING; m < n_load; ++m)
        if (m >= 0) mbar_wait(bar(B_RFULL + m % RING), (uint32_t)(m / RING) & 1u, nullptr, 0);
    }
  } else {
    // ------------------------------------------------------------ 8-bit converters
    // Two warps turn the keys, 32 of a tile's 64 rows each, two the values,
    // which also keep the account of the pages' scales.
    if constexpr (Q8) {
      const Kv8& cc = a.cache;
      const int w = warp - LOAD_WARP;
      const bool values = w >= CVT_WARPS / 2;
      constexpr int ROWS = L::ROWS, LR = D / 16, RI = 32 / LR, IT = ROWS / RI;  // lanes a row, rows an iteration, iterations
      constexpr int RAW = L::RAW;
      const int ch = lane % LR;
      const int row_first = ROWS * (w % (CVT_WARPS / 2)) + lane / LR;  // this lane's rows of a tile: it, + RI, ...
      const int shift = __ffs(page) - 1;                               // of a page in tokens
      // a lane's own codes and scales, copied RAW tiles ahead of their use
      uint8_t* raw = sm + L::OFF_RAW + w * RAW * L::RAW_BYTES + lane * 16;
      uint8_t* raw_sc = sm + L::OFF_RAW + w * RAW * L::RAW_BYTES + ROWS * D + lane * 8;
      // (a tile in one page: every lane knows that page; else lane j the tile's page j)
      const bool one = np == 1;
      const int my_page = one ? 0 : lane << shift, n_pages = cc.n_pages;
      const int* table = cc.table + (long long)b * cc.table_ld;
      auto page_id = [&](int t) -> int {
        const int key = (t0 + t) * KN + my_page;
        return (one || lane < np) && t < nT && key < vmax ? table[key >> shift] : -1;
      };
      auto is_page = [&](int id) { return (unsigned)id < (unsigned)n_pages; };
      // this lane's first codes of page 0 of this head; bytes from page to page
      const long long page_bytes = ((long long)cc.n_kv_heads << shift) * D;
      const uint8_t* const base = (values ? cc.v : cc.k) + ((long long)h << shift) * D + ch * 16;
      // ask for a tile's codes, and for the scales
      auto ask = [&](int t, int ids) {
        if (t < nT) {
          uint8_t* sc = raw_sc + (t % RAW) * L::RAW_BYTES;
          const uint32_t dst = smem_u32(raw) + (t % RAW) * L::RAW_BYTES;
          const int key0 = (t0 + t) * KN;
          const bool on = is_page(ids);
          if (values) {
            if (on) {
              const long long ph = (long long)ids * cc.n_kv_heads + h;
              cp_async4(smem_u32(sc), cc.k_scale + ph);
              cp_async4(smem_u32(sc) + 4, cc.v_scale + ph);
            } else {
              *reinterpret_cast<float2*>(sc) = make_float2(-1.f, 1.f);
            }
          }
          if (one && key0 + KN <= vmax && on) {  // a whole tile of one page
            const uint8_t* src = base + (long long)ids * page_bytes + ((key0 & (page - 1)) + row_first) * D;
#pragma unroll
            for (int j = 0; j < IT; ++j) cp_async16(dst + j * 512, src + j * (RI * D), 16);
          } else {
#pragma unroll
            for (int j = 0; j < IT; ++j) {
              const int r = row_first + j * RI, key = key0 + r;
              const int id = __shfl_sync(0xffffffffu, ids, r >> shift);
              const bool in = key < vmax && is_page(id);
              cp_async16(dst + j * 512, base + (in ? id * page_bytes + (key & (page - 1)) * D : 0), in ? 16 : 0);
            }
          }
        }
        cp_commit();
      };
      const int c0 = (2 * ch) & 7, flip = (ch >> 2) & 1;
      int ref = 0, most = kNoPage;  // the reference, the largest exponent of a page so far
      bool ok = true;
      int id_next = page_id(0);
#pragma unroll
      for (int t = 0; t < RAW; ++t) {
        const int id = id_next;
        id_next = page_id(t + 1);
        ask(t, id);
      }
#pragma unroll 1
      for (int t = 0; t < nT && ok; ++t) {
        cp_wait<RAW - 1>();
        uint4 codes[IT];
        const uint8_t* from = raw + (t % RAW) * L::RAW_BYTES;
#pragma unroll
        for (int j = 0; j < IT; ++j) codes[j] = *reinterpret_cast<const uint4*>(from + j * 512);
        const float2 sc = *reinterpret_cast<const float2*>(raw_sc + (t % RAW) * L::RAW_BYTES);
        {
          const int id = id_next;
          id_next = page_id(t + RAW + 1);
          ask(t + RAW, id);
        }
        int dv = 0;  // exponent of the values' factor, lane j: of the tile's page j
        if (values) {
          // ---- the tile's scales
          const float ks = sc.x;
          const int ev = ((__float_as_int(sc.y) >> 23) & 255) - 127;
          const bool in = one || (lane < np && (t0 + t) * KN + my_page < vmax);
          const bool none = in && ks < 0.f;
          if (none) report_error(a.err, DEV_ERR_BAD_SHAPE);
          float grow = 1.f;  // of part j in lane j
          int parts = 1;
          if (one) {
            if (none) {  // no values
            } else if (most - ev > kFarBelow) {
              dv = kNoPage;  // its values times 0
            } else {
              if (most != kNoPage && ev - ref <= 7 && ev - ref >= -15) {
                dv = ev - ref;
              } else {
                grow = most != kNoPage ? move_by(ref - ev) : 1.f;
                ref = ev;
              }
              most = max(most, ev);
            }
          } else {
            // the largest exponent of the pages before lane j's
            int before_j = in && !none ? ev : kNoPage;
#pragma unroll
            for (int k = 1; k < KN / 16; k <<= 1) {
              const int y = __shfl_up_sync(0xffffffffu, before_j, k);
              if (lane >= k) before_j = max(before_j, y);
            }
            before_j = __shfl_up_sync(0xffffffffu, before_j, 1);
            before_j = lane == 0 ? most : max(before_j, most);
            const bool far = in && !none && before_j - ev > kFarBelow;
            const bool counts = in && !none && !far;
            const int mx = __reduce_max_sync(0xffffffffu, counts ? ev : kNoPage);
            const int mn = __reduce_min_sync(0xffffffffu, counts ? ev : 1000);
            if (far) dv = kNoPage;
            if (mx == kNoPage) {  // no values
            } else if (most != kNoPage && mx - ref <= 7 && mn - ref >= -15) {
              if (counts) dv = ev - ref;
            } else if (mx - mn <= 15) {
              grow = most != kNoPage ? move_by(ref - mx) : 1.f;
              ref = mx;
              if (counts) dv = ev - ref;
            } else {
              // each counting page under its own reference; from which one O
              // comes to it: the last counting page before, or the tile before
              parts = np;
              const uint32_t have = __ballot_sync(0xffffffffu, counts);
              const uint32_t before = have & ((1u << lane) - 1u);
              const int last = 31 - __clz(have);
              const int prev = __shfl_sync(0xffffffffu, ev, before ? 31 - __clz(before) : 0);
              grow = !counts ? 1.f : before ? move_by(prev - ev) : most != kNoPage ? move_by(ref - ev) : 1.f;
              ref = __shfl_sync(0xffffffffu, ev, last);
            }
            most = max(most, mx);
          }
          if (w == CVT_WARPS / 2) {
            // (info t - RING was read before P V of t - 3, which had to be done
            // for the place of values t - 1, or of keys t - 1 before it)
            TileInfo* ti = info(t);
            float ks_most = ks;
            if (!one) {
              const int j = lane < 4 ? (lane * 16) >> shift : 0;
              const int ek = ((__float_as_int(ks) >> 23) & 255) - 127;
              const int ek_most = __reduce_max_sync(0xffffffffu, in && !none ? ek : kNoPage);
              const float over = none ? -1.f : in ? pow2i(ek - ek_most) : 1.f;  // (keys behind the last are masked)
              const float over_j = __shfl_sync(0xffffffffu, over, j);
              if (lane < 4) {
                reinterpret_cast<float*>(&ti->ks)[lane] = over_j;
                ti->grow[lane] = grow;
              }
              ks_most = ek_most == kNoPage ? 1.f : pow2i(ek_most);
              __syncwarp();
            }
            if (lane == 0) {
              ti->head = make_float4(ks_most, grow, (float)ref, (float)parts);
              mbar_arrive(bar(B_INFO + t % RING));
            }
          }
        }
        // ---- codes to f16 into the ring: 16-byte chunks 2 ch and 2 ch + 1 of
        // the row (the other one first in the second half of the row: fewer
        // bank conflicts), times 2^dv of the row's page
        const int n = values ? at_v(t, nT) : at_k(t), place = n % RING;
        if (!(ok = wwait(B_REMPTY + place, ((uint32_t)(n / RING) & 1u) ^ 1u))) break;
        uint8_t* tile = sm + L::OFF_RING + place * L::T_BYTES + (ch >> 2) * KN * 128 + row_first * 128;
        const bool scaled = one ? dv != 0 : __any_sync(0xffffffffu, dv != 0);
#pragma unroll
        for (int j = 0; j < IT; ++j) {
          const int r = row_first + j * RI;
          const uint32_t cw[4] = {codes[j].x, codes[j].y, codes[j].z, codes[j].w};
          uint32_t f[8];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t"
                "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
                : "=r"(f[2 * e]), "=r"(f[2 * e + 1])
                : "r"(cw[e]));
          if (scaled) {
            const __half2 m = __float2half2_rn(pow2i(one ? dv : __shfl_sync(0xffffffffu, dv, r >> shift)));
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              __half2 y = __hmul2(*reinterpret_cast<__half2*>(&f[e]), m);
              f[e] = *reinterpret_cast<uint32_t*>(&y);
            }
          }
          const uint4 lo = make_uint4(f[0], f[1], f[2], f[3]), hi = make_uint4(f[4], f[5], f[6], f[7]);
          uint8_t* row = tile + j * RI * 128;
          *reinterpret_cast<uint4*>(row + (((c0 + flip) ^ (r & 7)) << 4)) = flip ? hi : lo;
          *reinterpret_cast<uint4*>(row + (((c0 + 1 - flip) ^ (r & 7)) << 4)) = flip ? lo : hi;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_RFULL + place));
      }
      cp_wait<0>();
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, TM_COLS);
}

template <typename H, bool Q8, int D>
cudaError_t launch_tiles(const DecodeAttnArgs& a, int row_tiles, int n_split, cudaStream_t st) {
  auto kern = k_attn_tiles<H, Q8, D>;
  constexpr int smem = TilesLayout<Q8, D>::SMEM;
  static PerDevice once;
  int unused = 0;
  const cudaError_t e = per_device(once, &unused, [&](int, int&) {
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  });
  if (e != cudaSuccess) return e;
  CUtensorMap tk{}, tv{};
  if constexpr (!Q8) {
    const int cols = a.n_kv_heads * D;
    const bool bf = is_bf16<H>::value;
    if (!make_tmap_kmajor(&tk, a.k, a.kv_rows, cols, (int)a.ldk, KN, bf) ||
        !make_tmap_kmajor(&tv, a.v, a.kv_rows, cols, (int)a.ldv, KN, bf))
      return cudaErrorInvalidValue;
  }
  const long long grid = (long long)a.n_items * a.n_kv_heads * row_tiles * n_split;
  if (grid > 0x7fffffffLL) return cudaErrorInvalidValue;
  return launch_pdl(kern, dim3((unsigned)grid), dim3(32 * (1 + SOFT_WARPS + (Q8 ? CVT_WARPS : 1))), smem, st, tk, tv, a,
                    row_tiles, n_split);
}

template <typename H>
cudaError_t launch_tiles_h(const DecodeAttnArgs& a, int row_tiles, int n_split, cudaStream_t st) {
  if (a.cache.k)
    return a.head_dim == 128 ? launch_tiles<H, true, 128>(a, row_tiles, n_split, st)
                             : launch_tiles<H, true, 64>(a, row_tiles, n_split, st);
  return a.head_dim == 128 ? launch_tiles<H, false, 128>(a, row_tiles, n_split, st)
                           : launch_tiles<H, false, 64>(a, row_tiles, n_split, st);
}

}  // namespace

// A tensor map needs rows, and its stride as an int.
bool attn_tiles_fit(const DecodeAttnArgs& a) {
  return a.cache.k || (a.kv_rows > 0 && a.ldk <= 0x7fffffffLL && a.ldv <= 0x7fffffffLL);
}

cudaError_t attn_tiles_launch(const DecodeAttnArgs& a, bool bf16, int row_tiles, int n_split, cudaStream_t st) {
  return bf16 ? launch_tiles_h<__nv_bfloat16>(a, row_tiles, n_split, st)
              : launch_tiles_h<__half>(a, row_tiles, n_split, st);
}

}  // namespace pkc
