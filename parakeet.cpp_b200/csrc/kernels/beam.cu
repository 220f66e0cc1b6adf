// Beam search: the selection of the next hypotheses over beams and vocabulary,
// and the reordering of states that follow them.
//
// Selection. Item b has K hypotheses with scores cum and a row of V logits
// each: score(beam, v) = cum[beam] + x_v - log sum_u exp(x_u). The K best of
// the K * V continuations are taken, ties to the lowest beam * V + v. A
// finished hypothesis offers itself alone (its end token, score unchanged); a
// row whose sum is not finite (NaN, +inf, or nothing but -inf) and a score
// that is NaN offer -inf.
//
// Within a row the order is that of the logits, so each CTA reads its row (or
// its part of one) once from memory and keeps the K largest as keys (ordered
// value bits over the inverted index); only between rows do the sums matter.
// Those are kept in f64, and the scores are compared in f64: two hypotheses a few f32 steps apart come out in the order
// of their exact scores. A cluster holds one item: its CTAs put their lists
// into the first one's shared memory, which joins them, so there is one launch
// and no workspace.
//
// The K largest: the first pass leaves each thread's largest value; each warp
// sorts its lanes' and takes the K-th, a value that K elements reach; the
// largest of these bounds leaves a few dozen candidates, which the second pass
// (out of the L1 cache) gathers and which are put in order by counting. Where
// ties leave too many of them, the keys are taken one after another.
//
// Measured: 64 items of 8 rows of 8193 f32 logits 14 us (17 MB, 19% of the copy
// rate), one item of 4 rows of 1025 5.6 us. Bound by the chain load -> sum ->
// bound -> gather -> order -> cluster barrier -> K choices, 9 us for one item of
// 8 rows, of which all CTAs run at once. Blocks of 8192 elements in registers
// with all threads' maxima counted against each other took 120 us; the choice
// by counting all K * K candidates 3 us more.
#include "common.cuh"
#include "decode.h"

namespace pkc {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kCap = 512;  // candidates at most
constexpr int kMaxCluster = 8;

// Larger keys for larger values, and for the lower index among equal values.
__device__ __forceinline__ unsigned long long make_key(float x, unsigned int idx) {
  unsigned int u = __float_as_uint(x);
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)u << 32) | (0xffffffffu - idx);
}
__device__ __forceinline__ float key_value(unsigned long long k) {
  const unsigned int u = (unsigned int)(k >> 32);
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}
__device__ __forceinline__ int key_index(unsigned long long k) { return (int)(0xffffffffu - (unsigned int)k); }

// A thread's share of row[v0 .. v1): f(values, first index, how many, index
// step) for VE elements at a time, missing ones -inf. Which thread takes which
// element, and so the order of the sums, goes by the index alone and is the
// same for every row of a call: equal rows have equal sums, to the bit, and tie.
// Aligned: every row of the call starts on 16 bytes (v0 a multiple of VE).
template <typename T, bool ALIGNED, typename F>
__device__ __forceinline__ void each_group(const T* row, int v0, int v1, F&& f) {
  constexpr int VE = 16 / sizeof(T);
  auto value = [](T x) -> float {
    if constexpr (sizeof(T) == 4)
      return x;
    else
      return from_h(x);
  };
  if constexpr (ALIGNED) {
#pragma unroll 4
    for (int v = v0 + threadIdx.x * VE; v < v1; v += kThreads * VE) {
      float x[VE];
      const int n = min(VE, v1 - v);
      if (n == VE) {
        const uint4 raw = *reinterpret_cast<const uint4*>(row + v);
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          if constexpr (sizeof(T) == 4) {
            x[e] = __uint_as_float(w[e]);
          } else {
            const uint32_t u = e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xffffu;
            x[e] = is_bf16<T>::value ? __uint_as_float(u << 16) : __half2float(__ushort_as_half((unsigned short)u));
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < VE; ++e) x[e] = e < n ? value(row[v + e]) : -INFINITY;
      }
      f(x, v, n, 1);
    }
  } else {
#pragma unroll 2
    for (int v = v0 + threadIdx.x; v < v1; v += kThreads * VE) {
      float x[VE];
      const int n = min(VE, (v1 - v + kThreads - 1) / kThreads);
#pragma unroll
      for (int e = 0; e < VE; ++e) x[e] = e < n ? value(row[v + e * kThreads]) : -INFINITY;
      f(x, v, n, kThreads);
    }
  }
}

// What one part of one row gives: its K largest logits, in order, and the sum
// of its exponentials.
struct Part {
  unsigned long long key[kMaxBeams];
  double sum;  // of exp(x - max); NaN where the part holds a NaN or +inf
  float max;
  int n;       // keys
};

struct SelectShared {
  Part part[kMaxBeams];  // in the cluster's first CTA: those of [row][part of it]
  Part mine;
  unsigned long long list[kCap];
  unsigned long long best[kMaxBeams];
  double sum[kWarps];
  float max[kWarps], bound[kWarps];
  int count;
};

__device__ __forceinline__ unsigned int ordered(float x) {
  const unsigned int u = __float_as_uint(x);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float unordered(unsigned int u) {
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}
__device__ __forceinline__ unsigned long long ordered(double x) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(x);
  return (u >> 63) ? ~u : (u | (1ull << 63));
}

// The n keys of list into the K largest in order (all keys differ): each key's
// place is the number of larger ones. Four threads count for a key where there
// are few.
__device__ void order_list(const unsigned long long* list, int n, int K, unsigned long long* out) {
  const int share = n <= kThreads / 4 ? 4 : 1, first = threadIdx.x % share;
  for (int base = 0; base < n; base += kThreads / share) {
    const int i = base + threadIdx.x / share;
    const unsigned long long k = i < n ? list[i] : ~0ull;
    int at = 0;
#pragma unroll 8
    for (int j = first; j < n; j += share) at += list[j] > k;
    if (share == 4) {
      at += __shfl_xor_sync(0xffffffffu, at, 1);
      at += __shfl_xor_sync(0xffffffffu, at, 2);
    }
    if (i < n && first == 0 && at < K) out[at] = k;
  }
}

// K-th largest of the warp's 32 values (bitonic sort, descending)
__device__ __forceinline__ float warp_kth(float v, int K) {
  unsigned int x = ordered(v);
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      const unsigned int y = __shfl_xor_sync(0xffffffffu, x, j);
      const bool up = ((lane & k) == 0) == ((lane & j) == 0);  // this lane keeps the larger
      x = up ? max(x, y) : min(x, y);
    }
  return unordered(__shfl_sync(0xffffffffu, x, K - 1));
}

// exp(x - base) for base >= x: the special-function unit's error, 2^-22, and
// 2^-24 of the exponent
__device__ __forceinline__ float exp_below(float x, float base) { return ex2_approx((x - base) * 1.44269504f); }

template <typename T, bool ALIGNED>
__device__ void scan_part(SelectShared& sh, const T* row, int v0, int v1, int K) {
  constexpr int VE = 16 / sizeof(T);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Part& out = sh.mine;
  // ---- pass 1: the largest value and the sum (a NaN or +inf makes it NaN)
  constexpr float kLowest = -3.402823466e38f;
  float tmax = kLowest;
  double tsum = 0.0;
  each_group<T, ALIGNED>(row, v0, v1, [&](const float (&x)[VE], int, int, int) {
    float m = x[0];
#pragma unroll
    for (int e = 1; e < VE; ++e) m = fmaxf(m, x[e]);
    if (m > tmax) {
      tsum *= (double)exp_below(tmax, m);
      tmax = m;
    }
    // each term into f64: next to the row's largest term a sum in f32 would
    // lose what tells two rows apart
    double s0 = 0.0, s1 = 0.0;
#pragma unroll
    for (int e = 0; e < VE; e += 2) {
      s0 += (double)exp_below(x[e], tmax);
      s1 += (double)exp_below(x[e + 1], tmax);
    }
    tsum += s0 + s1;
  });
  const float kth = warp_kth(tmax == kLowest ? -INFINITY : tmax, K);
  float m = tmax;
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
  double s = tsum * (double)exp_below(tmax, m);
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
  if (lane == 0) {
    sh.bound[warp] = kth;
    sh.max[warp] = m;
    sh.sum[warp] = s;
  }
  if (tid == 0) sh.count = 0;
  __syncthreads();
  float bound = sh.bound[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) bound = fmaxf(bound, sh.bound[w]);
  // ---- pass 2: what reaches the bound (few threads hold any)
  if (tmax >= bound || bound == -INFINITY) each_group<T, ALIGNED>(row, v0, v1, [&](const float (&x)[VE], int v, int n, int step) {
    float m = x[0];
#pragma unroll
    for (int e = 1; e < VE; ++e) m = fmaxf(m, x[e]);
    if (m >= bound) {
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (e < n && x[e] >= bound) {
          const int at = atomicAdd(&sh.count, 1);
          if (at < kCap) sh.list[at] = make_key(x[e], v + e * step);
        }
    }
  });
  __syncthreads();
  const int n = sh.count;
  if (n <= kCap) {
    order_list(sh.list, n, K, out.key);
  } else {
    // too many equal values: the keys one after another, each the largest
    // below the one before
    unsigned long long before = ~0ull;
    for (int j = 0; j < K; ++j) {
      unsigned long long best = 0;
      each_group<T, ALIGNED>(row, v0, v1, [&](const float (&x)[VE], int v, int cnt, int step) {
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const unsigned long long k = make_key(x[e], v + e * step);
          if (e < cnt && x[e] == x[e] && k < before && k > best) best = k;
        }
      });
#pragma unroll
      for (int k = 16; k > 0; k >>= 1) {
        const unsigned long long y = __shfl_xor_sync(0xffffffffu, best, k);
        best = y > best ? y : best;
      }
      if (lane == 0) sh.best[warp] = best;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWarps; ++w) best = sh.best[w] > best ? sh.best[w] : best;
      if (tid == 0) out.key[j] = best;
      before = best;
      __syncthreads();
    }
  }
  if (tid == 0) {
    m = sh.max[0];
    for (int w = 1; w < kWarps; ++w) m = fmaxf(m, sh.max[w]);
    s = 0.0;
    for (int w = 0; w < kWarps; ++w) s += sh.sum[w] * (double)exp_below(sh.max[w], m);
    out.sum = s;
    out.max = m;
    out.n = min(n, K);
  }
  __syncthreads();
}

// chunks: parts of a row (CTA r takes part r % chunks of rows r / chunks, + C / chunks, ...)
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kThreads, 4) k_beam_select(const BeamSelectArgs a, int chunks) {
  __shared__ SelectShared sh;
  uint32_t C;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(C));
  const int rank = (int)cluster_ctarank(), b = blockIdx.x / (int)C, tid = threadIdx.x;
  const int K = a.K, lanes = (int)C / chunks;  // rows that the cluster scans at a time
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // this CTA runs
  pdl_wait();
  pdl_trigger();
  bool started = false;
  const int chunk = rank % chunks, per = ((a.V + chunks - 1) / chunks + 7) / 8 * 8;
  for (int beam = rank / chunks; beam < K; beam += lanes) {
    const T* row = reinterpret_cast<const T*>(a.logits) + (long long)(b * (long long)K + beam) * a.ld;
    scan_part<T, ALIGNED>(sh, row, min(a.V, chunk * per), min(a.V, (chunk + 1) * per), K);
    // to the first CTA's part [beam][chunk], word by word
    if (!started) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // all of them run
    started = true;
    const uint32_t dst = mapa_shared(smem_u32(&sh.part[beam * chunks + chunk]), 0);
    const uint32_t* src = reinterpret_cast<const uint32_t*>(&sh.mine);
    if (tid < (int)(sizeof(Part) / 4))
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(dst + 4 * tid), "r"(src[tid]) : "memory");
    __syncthreads();
  }
  if (!started) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  cluster_sync();  // every part has arrived
  if (rank != 0 || tid >= 32) return;
  // ---- the first warp takes the K best off the heads of the lists, a lane a
  // list (K * chunks <= 32); the lowest lane among equal scores has the lowest
  // beam and, of a row's parts, the lowest tokens
  const int beam = tid / chunks;
  const bool on = beam < K;
  const Part* rows = &sh.part[on ? beam * chunks : 0];
  float m = -INFINITY;
  for (int ch = 0; ch < chunks; ++ch) m = fmaxf(m, rows[ch].max);
  double s = 0.0;
  for (int ch = 0; ch < chunks; ++ch) s += rows[ch].sum * (double)exp_below(rows[ch].max, m);
  const float cum = on ? a.cum[(long long)b * K + beam] : -INFINITY;
  const bool fin = on && a.finished && a.finished[(long long)b * K + beam];
  // 0: a live row; 1: finished, its end token, then the lowest others; 2: one
  // that offers nothing, its lowest tokens
  const int kind = cum != cum || cum == -INFINITY ? 2 : fin ? 1 : s > 0.0 && isfinite(s) && isfinite(m) ? 0 : 2;
  const double lse = (double)m + log(s);
  const Part& mine = sh.part[on ? tid : 0];
  const bool lists = on && (kind == 0 || tid % chunks == 0);
  const int len = !lists ? 0 : kind == 0 ? mine.n : min(a.V, K);
  int j = 0, tok = -1;
  unsigned long long head = 0;  // ordered bits of the score; 0: the list is empty
  auto next = [&]() {
    head = 0;
    if (j >= len) return;
    double sc = -INFINITY;
    if (kind == 0) {
      const unsigned long long k = mine.key[j];
      tok = key_index(k);
      sc = (double)cum + ((double)key_value(k) - lse);
    } else {
      tok = kind == 2 ? j : j == 0 ? a.eos : j - 1 < a.eos ? j - 1 : j;
      if (kind == 1 && j == 0) sc = (double)cum;
    }
    head = ordered(sc);
    ++j;
  };
  next();
  float score = 0.f;
  int parent = 0, token = 0, done = 0;  // of place tid
  for (int place = 0; place < K; ++place) {
    const unsigned int hi = (unsigned int)(head >> 32), top = __reduce_max_sync(0xffffffffu, hi);
    const unsigned int lo = hi == top ? (unsigned int)head : 0u, low = __reduce_max_sync(0xffffffffu, lo);
    const int from = __ffs(__ballot_sync(0xffffffffu, hi == top && lo == low && head != 0)) - 1;
    const unsigned long long best = ((unsigned long long)top << 32) | low;
    const int t = __shfl_sync(0xffffffffu, tok, from), f = __shfl_sync(0xffffffffu, (int)fin, from);
    if (tid == place) {
      const double sc = __longlong_as_double((long long)((best >> 63) ? (best & ~(1ull << 63)) : ~best));
      score = (float)sc;
      parent = from / chunks;
      token = t;
      done = t == a.eos || f;
    }
    if (tid == from) next();
  }
  // (cum and finished, which these may be, have been read)
  if (tid < K) {
    const long long o = (long long)b * K + tid;
    a.score[o] = score;
    a.parent[o] = parent;
    a.token[o] = token;
    if (a.finished_out) a.finished_out[o] = (uint8_t)done;
  }
}

// state[o][b * K + k] <- state[o][b * K + parent[b, k]], in place: a thread
// reads one column of every row that moves before it writes any of them.
//
// Registers are held to what lets four CTAs run on an SM where a thread's
// column fits (K <= 8: 8 blocks of 512 rows of 200 KB 132 us, 177 us with two).
template <typename V, int KM>
__global__ void __launch_bounds__(256, KM <= 8 ? 4 : KM <= 16 ? 2 : 1) k_beam_reorder(const BeamReorderArgs a) {
  __shared__ int s_parent[KM];
  const int b = blockIdx.y, K = a.K;
  pdl_wait();
  pdl_trigger();
  if (threadIdx.x < K) {
    int p = a.parent[(long long)b * K + threadIdx.x];
    if (p < 0 || p >= K) {
      report_error(a.err, DEV_ERR_BAD_SHAPE);
      p = threadIdx.x;
    }
    s_parent[threadIdx.x] = p;
  }
  __syncthreads();
  long long bytes = a.row_bytes;
  if (a.lens) {
    const long long live = a.lens[b] > 0 ? a.lens[b] * a.unit_bytes : 0;
    bytes = live < bytes ? live : bytes;
  }
  const long long cols = bytes / (long long)sizeof(V), tail = bytes % (long long)sizeof(V);
  uint8_t* base = a.state + (long long)blockIdx.z * a.outer_stride + (long long)b * K * a.row_stride;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < cols; i += gridDim.x * 256LL) {
    V v[KM];
#pragma unroll
    for (int k = 0; k < KM; ++k)
      if (k < K && s_parent[k] != k)
        v[k] = *reinterpret_cast<const V*>(base + s_parent[k] * a.row_stride + i * (long long)sizeof(V));
#pragma unroll
    for (int k = 0; k < KM; ++k)
      if (k < K && s_parent[k] != k) *reinterpret_cast<V*>(base + k * a.row_stride + i * (long long)sizeof(V)) = v[k];
  }
  if (blockIdx.x == 0 && threadIdx.x < tail) {
    const long long at = cols * (long long)sizeof(V) + threadIdx.x;
    uint8_t v[KM];
#pragma unroll
    for (int k = 0; k < KM; ++k)
      if (k < K) v[k] = base[s_parent[k] * a.row_stride + at];
#pragma unroll
    for (int k = 0; k < KM; ++k)
      if (k < K && s_parent[k] != k) base[k * a.row_stride + at] = v[k];
  }
}

template <typename V>
cudaError_t reorder_v(const BeamReorderArgs& a, cudaStream_t st) {
  const long long cols = a.row_bytes / (long long)sizeof(V);
  const long long gx = (cols + 255) / 256;
  const dim3 grid((unsigned)(gx < 1 ? 1 : gx > 4096 ? 4096 : gx), a.B, a.n_outer), block(256);
  if (a.K <= 4) return launch_pdl(k_beam_reorder<V, 4>, grid, block, 0, st, a);
  if (a.K <= 8) return launch_pdl(k_beam_reorder<V, 8>, grid, block, 0, st, a);
  if (a.K <= 16) return launch_pdl(k_beam_reorder<V, 16>, grid, block, 0, st, a);
  return launch_pdl(k_beam_reorder<V, 32>, grid, block, 0, st, a);
}

template <typename T, bool ALIGNED>
cudaError_t select_t(const BeamSelectArgs& a, cudaStream_t st) {
  // CTAs of an item: a row each, or parts of a row where there are few rows
  // and the parts are not short
  int chunks = 1;
  while (a.K * chunks * 2 <= kMaxCluster && a.V >= chunks * 2 * 2048) chunks *= 2;
  const int C = a.K * chunks < kMaxCluster ? a.K * chunks : kMaxCluster / chunks * chunks;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.B * C));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, k_beam_select<T, ALIGNED>, a, chunks);
}

}  // namespace

cudaError_t beam_select_launch(const BeamSelectArgs& a, int dtype, cudaStream_t st) {
  if (a.B <= 0) return cudaSuccess;
  const bool al = (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0 && a.ld % (dtype == 2 ? 4 : 8) == 0;
  if (dtype == 0) return al ? select_t<__half, true>(a, st) : select_t<__half, false>(a, st);
  if (dtype == 1) return al ? select_t<__nv_bfloat16, true>(a, st) : select_t<__nv_bfloat16, false>(a, st);
  return al ? select_t<float, true>(a, st) : select_t<float, false>(a, st);
}

cudaError_t beam_reorder_launch(const BeamReorderArgs& a, cudaStream_t st) {
  if (a.B <= 0 || a.n_outer <= 0 || a.row_bytes <= 0) return cudaSuccess;
  const unsigned long long al = (unsigned long long)reinterpret_cast<uintptr_t>(a.state) | (unsigned long long)a.row_stride |
                                (unsigned long long)a.outer_stride;
  if (al % 16 == 0) return reorder_v<uint4>(a, st);
  if (al % 4 == 0) return reorder_v<uint32_t>(a, st);
  if (al % 2 == 0) return reorder_v<uint16_t>(a, st);
  return reorder_v<uint8_t>(a, st);
}

}  // namespace pkc
