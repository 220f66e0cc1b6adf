// Beam search: the selection of the next hypotheses over beams and vocabulary,
// and the reordering of states that follow them.
//
// Selection. Item b has K hypotheses with scores cum and a row of V logits
// each: score(beam, v) = cum[beam] + x_v - log sum_u exp(x_u). The K best of
// the K * V continuations are taken, ties to the lowest beam * V + v. A
// finished hypothesis offers itself alone (its end token, score unchanged); a
// row whose sum is not finite (NaN, +inf, or nothing but -inf) and a
// hypothesis whose score is not finite offer -inf.
//
// Within a row the order is that of the logits, so each CTA reads its row (or
// its part of one) once from memory and keeps the K largest as keys (ordered
// value bits over the inverted index); only between rows do the sums matter.
// Those are kept in f64 (of exponentials in f32, good to 2^-22, so their
// logarithm is too), and the scores are compared in f64: two hypotheses more
// than 2^-20 apart come out in the order of their exact scores, which at -1000
// is a 64th of an f32 step. A cluster holds one item: its CTAs put their lists
// into the first one's shared memory, which joins them, so there is one launch
// and no workspace.
//
// The K largest: the first pass leaves each thread's largest value; each warp
// sorts its lanes'. K elements reach a warp's K-th, and the least of four warps'
// (K / 4)-th: the largest of these bounds leaves about 2 K candidates, which the
// second pass (out of the L1 cache) gathers and which are put in order by
// counting. (With the first bound alone they were 120 for K = 16 and 700 for
// K = 32.) Where ties leave too many, those above the bound and the first of the
// equal ones are taken.
//
// Measured: 64 items of 8 rows of 8193 f32 logits 12.2 us (17 MB, 21% of the copy
// rate), one item of 4 rows of 1025 5.1 us. Bound by the chain load -> sum ->
// bound -> gather -> order -> cluster barrier -> K choices, 5.5 us for one item of
// 8 rows of 1025, and the start of 512 CTAs in clusters, 8.6 us for 64 such items.
// Blocks of 8192 elements in registers with all threads' maxima counted against
// each other took 120 us; the choice by counting all K * K candidates 3 us more.
#include "common.cuh"
#include "decode.h"
#include "per_device.h"

namespace pkc {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kCap = 1024;  // candidates at most

// Larger keys for larger values, and for the lower index among equal values
// (-0 + 0 is +0: the zeros are equal).
__device__ __forceinline__ unsigned long long make_key(float x, unsigned int idx) {
  unsigned int u = __float_as_uint(x + 0.f);
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)u << 32) | (0xffffffffu - idx);
}
__device__ __forceinline__ float key_value(unsigned long long k) {
  const unsigned int u = (unsigned int)(k >> 32);
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}
__device__ __forceinline__ int key_index(unsigned long long k) { return (int)(0xffffffffu - (unsigned int)k); }

template <typename T>
__device__ __forceinline__ float to_float(T x) {
  if constexpr (sizeof(T) == 4)
    return x;
  else
    return from_h(x);
}

// A thread's share of row[v0 .. v1), every kThreads-th element: f(values, first
// index, how many) for VE of them at a time, missing ones -inf. Which thread
// takes which element, and so the order of the sums, goes by the index alone:
// equal rows have equal sums, to the bit, and tie, however they are aligned.
// Reads of single elements, 16 on their way at a time: 3 of 16 rows of 50736 f32
// logits 22 us; reads of 16 bytes, of which the registers hold fewer ahead, 33 us.
template <typename T, typename F>
__device__ __forceinline__ void each_group(const T* row, int v0, int v1, F&& f) {
  constexpr int VE = 16 / sizeof(T);
  constexpr int U = 16 / VE, STEP = kThreads * VE;  // 16 reads on their way
  for (int v4 = v0 + threadIdx.x; v4 < v1; v4 += U * STEP) {
    float x[U][VE];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const int v = v4 + u * STEP + e * kThreads;
        x[u][e] = v < v1 ? to_float(row[v]) : -INFINITY;
      }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = v4 + u * STEP;
      if (v >= v1) break;
      f(x[u], v, min(VE, (v1 - v + kThreads - 1) / kThreads));
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
  float max[kWarps], bound[kWarps], fourth[kWarps];
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

// The warp's 32 values in order (bitonic sort, descending)
__device__ __forceinline__ float warp_sort(float v) {
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
  return unordered(x);
}

// exp(x - base) for base >= x: the special-function unit's error, 2^-22, and
// 2^-24 of the exponent
__device__ __forceinline__ float exp_below(float x, float base) { return ex2_approx((x - base) * 1.44269504f); }

template <typename T>
__device__ void scan_part(SelectShared& sh, const T* row, int v0, int v1, int K) {
  constexpr int VE = 16 / sizeof(T);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Part& out = sh.mine;
  // ---- pass 1: the largest value and the sum (a NaN or +inf makes it NaN)
  constexpr float kLowest = -3.402823466e38f;
  float tmax = kLowest;
  double part[4] = {0.0, 0.0, 0.0, 0.0};  // (four sums: an addition in f64 takes long)
  each_group<T>(row, v0, v1, [&](const float (&x)[VE], int, int) {
    float m = x[0];
#pragma unroll
    for (int e = 1; e < VE; ++e) m = fmaxf(m, x[e]);
    if (m > tmax) {
      const double f = (double)exp_below(tmax, m);
#pragma unroll
      for (int e = 0; e < 4; ++e) part[e] *= f;
      tmax = m;
    }
    // each term into f64: next to the row's largest term a sum in f32 would
    // lose what tells two rows apart
#pragma unroll
    for (int e = 0; e < VE; ++e) part[e & 3] += (double)exp_below(x[e], tmax);
  });
  const double tsum = (part[0] + part[1]) + (part[2] + part[3]);
  const float sorted = warp_sort(tmax == kLowest ? -INFINITY : tmax);
  const float kth = __shfl_sync(0xffffffffu, sorted, K - 1), fourth = __shfl_sync(0xffffffffu, sorted, (K + 3) / 4 - 1);
  float m = tmax;
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
  double s = tsum * (double)exp_below(tmax, m);
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
  if (lane == 0) {
    sh.bound[warp] = kth;
    sh.fourth[warp] = fourth;
    sh.max[warp] = m;
    sh.sum[warp] = s;
  }
  if (tid == 0) sh.count = 0;
  __syncthreads();
  // a value that K elements reach: K of one warp, or a quarter of K (rounded up)
  // of each of four warps
  float bound;
  {
    const float of_one = sh.bound[lane % kWarps], of_four = sh.fourth[lane % kWarps];
    int above = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) above += sh.fourth[w] > of_four;
    const unsigned int one = __reduce_max_sync(0xffffffffu, ordered(of_one));
    const unsigned int four = __reduce_min_sync(0xffffffffu, above < 4 ? ordered(of_four) : 0xffffffffu);
    bound = unordered(max(one, four));
  }
  // ---- pass 2: what reaches the bound (few threads hold any), no more than the
  // list holds
  if (tmax >= bound || bound == -INFINITY) each_group<T>(row, v0, v1, [&](const float (&x)[VE], int v, int n) {
    float m = x[0];
#pragma unroll
    for (int e = 1; e < VE; ++e) m = fmaxf(m, x[e]);
    if (m >= bound && *(volatile int*)&sh.count <= kCap) {
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (e < n && x[e] >= bound) {
          const int at = atomicAdd(&sh.count, 1);
          if (at < kCap) sh.list[at] = make_key(x[e], v + e * kThreads);
        }
    }
  });
  __syncthreads();
  int n = sh.count;
  if (n > kCap) {
    // many equal ones, as where a mask leaves few tokens: what is above the
    // bound, then the first of those that equal it
    __syncthreads();
    if (tid == 0) sh.count = 0;
    __syncthreads();
    each_group<T>(row, v0, v1, [&](const float (&x)[VE], int v, int cnt) {
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (e < cnt && x[e] > bound && *(volatile int*)&sh.count <= kCap) {
          const int at = atomicAdd(&sh.count, 1);
          if (at < kCap) sh.list[at] = make_key(x[e], v + e * kThreads);
        }
    });
    __syncthreads();
    n = sh.count;
    for (int base = v0; n < K && base < v1; base += kThreads) {
      __syncthreads();
      if (base + tid < v1) {
        const float x = to_float(row[base + tid]);
        if (x == bound) sh.list[atomicAdd(&sh.count, 1)] = make_key(x, base + tid);
      }
      __syncthreads();
      n = sh.count;
    }
  }
  if (n <= kCap) {
    order_list(sh.list, n, K, out.key);
  } else {
    // still too many: the keys one after another, each the largest below the
    // one before
    unsigned long long before = ~0ull;
    for (int j = 0; j < K; ++j) {
      unsigned long long best = 0;
      each_group<T>(row, v0, v1, [&](const float (&x)[VE], int v, int cnt) {
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const unsigned long long k = make_key(x[e], v + e * kThreads);
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
template <typename T>
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
    scan_part<T>(sh, row, min(a.V, chunk * per), min(a.V, (chunk + 1) * per), K);
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
  if (rank != 0) return;
  // ---- the scores of all K * chunks <= 32 lists, a lane a list, warps sharing
  // the places: list[place][lane], ordered bits, 0 where the list has ended
  static_assert(kCap >= 32 * kMaxBeams, "the scores lie where the candidates were");
  const int lane = tid & 31, beam = lane / chunks;
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
  const int kind = !isfinite(cum) ? 2 : fin ? 1 : s > 0.0 && isfinite(s) && isfinite(m) ? 0 : 2;
  const double lse = (double)m + log(s);
  const Part& mine = sh.part[on ? lane : 0];
  const bool lists = on && (kind == 0 || lane % chunks == 0);
  const int len = !lists ? 0 : kind == 0 ? mine.n : min(a.V, K);
  for (int j = tid >> 5; j < K; j += kWarps) {
    double sc = -INFINITY;
    if (kind == 0 && j < len) sc = (double)cum + ((double)key_value(mine.key[j]) - lse);
    if (kind == 1 && j == 0) sc = (double)cum;
    sh.list[j * 32 + lane] = j < len ? ordered(sc + 0.0) : 0;  // (+ 0: the zeros are equal)
  }
  __syncthreads();  // (cum and finished, which the outputs may be, have been read)
  if (tid >= 32) return;
  // ---- the first warp takes the K best off the lists' heads; the lowest lane
  // among equal scores has the lowest beam and, of a row's parts, the lowest
  // tokens. (Scores worked out as their lists' heads moved on: 1.2 us more for
  // K = 8, 2.6 us for K = 16.)
  unsigned long long head = sh.list[lane], best = 0;
  int at = 0, list = 0, entry = 0;  // list, entry: of place lane
  for (int place = 0; place < K; ++place) {
    const unsigned int hi = (unsigned int)(head >> 32), top = __reduce_max_sync(0xffffffffu, hi);
    const unsigned int lo = hi == top ? (unsigned int)head : 0u, low = __reduce_max_sync(0xffffffffu, lo);
    const int from = __ffs(__ballot_sync(0xffffffffu, hi == top && lo == low)) - 1;
    const int e = __shfl_sync(0xffffffffu, at, from);
    if (lane == place) {
      best = ((unsigned long long)top << 32) | low;
      list = from;
      entry = e;
    }
    if (lane == from) {
      ++at;
      head = at < K ? sh.list[at * 32 + lane] : 0;
    }
  }
  const int from_kind = __shfl_sync(0xffffffffu, kind, list), from_fin = __shfl_sync(0xffffffffu, (int)fin, list);
  if (lane < K) {
    const int token = from_kind == 0   ? key_index(sh.part[list].key[entry])
                : from_kind == 2 ? entry
                : entry == 0     ? a.eos
                                 : (entry - 1 < a.eos ? entry - 1 : entry);
    const long long o = (long long)b * K + lane;
    a.score[o] = (float)__longlong_as_double((long long)((best >> 63) ? (best & ~(1ull << 63)) : ~best));
    a.parent[o] = list / chunks;
    a.token[o] = token;
    if (a.finished_out) a.finished_out[o] = (uint8_t)(token == a.eos || from_fin);
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
    const int len = a.lens[b];
    if (len < 0 && threadIdx.x == 0) report_error(a.err, DEV_ERR_BAD_SHAPE);
    const long long live = len > 0 ? len * a.unit_bytes : 0;
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

template <typename T>
cudaError_t select_t(const BeamSelectArgs& a, cudaStream_t st) {
  // CTAs of an item: a row each, or, where all rows together leave SMs without
  // work, parts of at least 2048 elements of each. More than eight CTAs (which
  // only some devices' clusters allow) where there are few items: 3 of 16 rows
  // of 50736 logits 20 us, 34 with eight.
  const long long rows = (long long)a.B * a.K;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  static PerDevice once;
  int largest = 0;
  const cudaError_t ae = per_device(once, &largest, [&](int, int& v) {
    cudaError_t e = cudaFuncSetAttribute(k_beam_select<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    at[0].val.clusterDim.x = 16;
    cfg.gridDim = dim3(16);
    cfg.numAttrs = 1;
    int n = 0;
    e = cudaOccupancyMaxActiveClusters(&n, k_beam_select<T>, &cfg);
    v = e == cudaSuccess && n > 0 ? 16 : 8;
    if (e != cudaSuccess) cudaGetLastError();
    return cudaSuccess;
  });
  if (ae != cudaSuccess) return ae;
  const int most = rows < 2 * 148 ? largest : 8;
  int chunks = most / a.K;
  if (chunks > a.V / 2048) chunks = a.V / 2048;
  if (chunks > 2 * 148 / rows) chunks = (int)(2 * 148 / rows);
  if (chunks < 1) chunks = 1;
  const int C = a.K * chunks < most ? a.K * chunks : most / chunks * chunks;
  at[0].val.clusterDim.x = C;
  cfg.gridDim = dim3((unsigned)(a.B * C));
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, k_beam_select<T>, a, chunks);
}

}  // namespace

cudaError_t beam_select_launch(const BeamSelectArgs& a, int dtype, cudaStream_t st) {
  if (a.B <= 0) return cudaSuccess;
  if (dtype == 0) return select_t<__half>(a, st);
  if (dtype == 1) return select_t<__nv_bfloat16>(a, st);
  return select_t<float>(a, st);
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
