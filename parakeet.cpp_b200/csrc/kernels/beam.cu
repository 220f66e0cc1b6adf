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
// its part of one) once and keeps the K largest as keys (ordered value bits
// over the inverted index); only between rows do the sums matter. Those are
// kept in f64 from groups of f32 exponentials, and the scores are compared in
// f64: two hypotheses a few f32 steps apart come out in the order of their
// exact scores. A cluster holds one item: its first CTA joins the rows' lists
// through distributed shared memory, so there is one launch and no workspace.
#include "common.cuh"
#include "decode.h"
#include "per_device.h"

namespace pkc {

namespace {

constexpr int kThreads = 256;
constexpr int kPer = 32;                    // elements of a block, per thread
constexpr int kBlock = kThreads * kPer;     // elements that are looked at together
constexpr int kCap = kMaxBeams * kPer + kMaxBeams;  // candidates of one block at most, see gather
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

template <typename T>
__device__ __forceinline__ float load_f(const T* p);
template <>
__device__ __forceinline__ float load_f<float>(const float* p) { return *p; }
template <>
__device__ __forceinline__ float load_f<__half>(const __half* p) { return __half2float(*p); }
template <>
__device__ __forceinline__ float load_f<__nv_bfloat16>(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// What one part of one row gives: its K largest logits, in order, and the sum
// of its exponentials.
struct Part {
  unsigned long long key[kMaxBeams];
  double sum;  // of exp(x - max); NaN where the part holds a NaN
  float max;
  int n;       // keys
};

struct SelectShared {
  Part part[kMaxBeams];  // this CTA's rows (one part each)
  unsigned long long list[kCap];
  unsigned long long best[kThreads];
  double sum[kThreads / 32];
  float max[kThreads / 32];
  int count, nan;
  unsigned long long thr;
};

// The n keys of sh.list into the K largest in order (all keys differ): each
// key's place is the number of larger ones.
__device__ void order_list(const unsigned long long* list, int n, int K, unsigned long long* out) {
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const unsigned long long k = list[i];
    int at = 0;
    for (int j = 0; j < n && at < K; ++j) at += list[j] > k;
    if (at < K) out[at] = k;
  }
}

template <typename T>
__device__ void scan_part(SelectShared& sh, Part& out, const T* row, int v0, int v1, int K) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  float tmax = -INFINITY;
  double tsum = 0.0;
  bool nan = false;
  int have = 0;  // keys in out so far
  for (int blk = v0; blk < v1; blk += kBlock) {
    float x[kPer];
    unsigned long long best = 0;
    float bmax = -INFINITY;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int v = blk + i * kThreads + tid;
      x[i] = v < v1 ? load_f<T>(row + v) : -INFINITY;
      nan |= x[i] != x[i];
      if (x[i] != x[i]) x[i] = -INFINITY;
      bmax = fmaxf(bmax, x[i]);
    }
    if (bmax > tmax) {
      tsum *= (double)expf(tmax - bmax);
      tmax = bmax;
    }
    const float base = tmax == -INFINITY ? 0.f : tmax;
#pragma unroll
    for (int i = 0; i < kPer; i += 4)
      tsum += (double)((expf(x[i] - base) + expf(x[i + 1] - base)) + (expf(x[i + 2] - base) + expf(x[i + 3] - base)));
    // first index of the thread's largest value
#pragma unroll
    for (int i = kPer - 1; i >= 0; --i) {
      const int v = blk + i * kThreads + tid;
      if (v < v1 && x[i] == bmax) best = make_key(x[i], v);
    }
    // ---- a bound that K keys reach: the K-th largest of the threads' largest
    sh.best[tid] = best;
    if (tid == 0) sh.count = 0, sh.thr = 1;
    __syncthreads();
    {
      int at = 0;
      for (int j = 0; j < kThreads; ++j) at += sh.best[j] > best;
      if (at == K - 1 && best) sh.thr = best;
    }
    __syncthreads();
    // ---- gather: at most K threads hold a key at or above it
    unsigned long long thr = sh.thr;
    if (have == K && out.key[K - 1] > thr) thr = out.key[K - 1];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int v = blk + i * kThreads + tid;
      if (v < v1) {
        const unsigned long long k = make_key(x[i], v);
        if (k >= thr) sh.list[atomicAdd(&sh.count, 1)] = k;
      }
    }
    if (tid < have) sh.list[atomicAdd(&sh.count, 1)] = out.key[tid];
    __syncthreads();
    const int n = sh.count;
    order_list(sh.list, n, K, out.key);
    have = min(n, K);
    __syncthreads();
  }
  // ---- join the sums
  float m = tmax;
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
  if (lane == 0) sh.max[warp] = m;
  if (tid == 0) sh.nan = 0;
  __syncthreads();
  m = sh.max[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) m = fmaxf(m, sh.max[w]);
  if (nan) sh.nan = 1;
  double s = tmax == -INFINITY ? 0.0 : tsum * (double)expf(tmax - m);
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
  if (lane == 0) sh.sum[warp] = s;
  __syncthreads();
  if (tid == 0) {
    s = 0.0;
    for (int w = 0; w < kThreads / 32; ++w) s += sh.sum[w];
    out.sum = sh.nan ? (double)NAN : s;
    out.max = m;
    out.n = have;
  }
  __syncthreads();
}

// chunks: parts of a row (CTA r takes part r % chunks of rows r / chunks, + C / chunks, ...)
template <typename T>
__global__ void __launch_bounds__(kThreads) k_beam_select(const BeamSelectArgs a, int chunks) {
  extern __shared__ __align__(16) uint8_t smem[];
  SelectShared& sh = *reinterpret_cast<SelectShared*>(smem);
  uint32_t C;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(C));
  const int rank = (int)cluster_ctarank(), b = blockIdx.x / (int)C, tid = threadIdx.x;
  const int K = a.K, lanes = (int)C / chunks;  // rows that the cluster scans at a time
  pdl_wait();
  pdl_trigger();
  const int chunk = rank % chunks, per = (a.V + chunks - 1) / chunks;
  int slot = 0;
  for (int beam = rank / chunks; beam < K; beam += lanes, ++slot) {
    const T* row = reinterpret_cast<const T*>(a.logits) + (long long)(b * (long long)K + beam) * a.ld;
    scan_part<T>(sh, sh.part[slot], row, chunk * per, min(a.V, (chunk + 1) * per), K);
  }
  cluster_sync();
  if (rank == 0) {
    // ---- candidates of every row: (score, beam * V + token)
    long long* c_at = reinterpret_cast<long long*>(smem + sizeof(SelectShared));
    double* cs = reinterpret_cast<double*>(c_at + kMaxBeams * (kMaxBeams + 1));
    __shared__ int s_n;
    __shared__ double s_lse[kMaxBeams];
    __shared__ int s_kind[kMaxBeams];  // 0 live, 1 finished, 2 none
    if (tid == 0) s_n = 0;
    auto remote = [&](int beam, int ch) -> const Part* {
      const uint32_t local = smem_u32(&sh.part[beam / lanes]);
      const uint32_t addr = mapa_shared(local, (uint32_t)(beam % lanes * chunks + ch));
      uint64_t g;
      asm("cvta.shared::cluster.u64 %0, %1;" : "=l"(g) : "l"((uint64_t)addr));
      return reinterpret_cast<const Part*>(g);
    };
    if (tid < K) {
      float m = -INFINITY;
      for (int ch = 0; ch < chunks; ++ch) m = fmaxf(m, remote(tid, ch)->max);
      double s = 0.0;
      for (int ch = 0; ch < chunks; ++ch) {
        const Part* p = remote(tid, ch);
        // a part of -inf alone adds nothing
        if (p->max != -INFINITY || p->sum != p->sum) s += p->sum * (double)expf(p->max - m);
      }
      const float cum = a.cum[(long long)b * K + tid];
      const bool fin = a.finished && a.finished[(long long)b * K + tid];
      s_kind[tid] = cum != cum || cum == -INFINITY ? 2 : fin ? 1 : isfinite(s) && isfinite(m) ? 0 : 2;
      s_lse[tid] = (double)m + log(s);
    }
    __syncthreads();
    // each row's K best of its parts' lists (one candidate a thread and step)
    for (int i = tid; i < K * (K + 1); i += kThreads) {
      const int beam = i / (K + 1), j = i % (K + 1);
      const int kind = s_kind[beam];
      double sc = -INFINITY;
      long long at = -1;
      if (kind == 0) {
        // j-th of the parts' merged lists: found by its place
        int need = j;
        unsigned long long pick = 0;
        if (j < K) {
          int head[kMaxCluster];
          for (int ch = 0; ch < chunks; ++ch) head[ch] = 0;
          for (; need >= 0; --need) {
            pick = 0;
            int from = 0;
            for (int ch = 0; ch < chunks; ++ch) {
              const Part* p = remote(beam, ch);
              if (head[ch] < p->n && p->key[head[ch]] > pick) pick = p->key[head[ch]], from = ch;
            }
            ++head[from];
          }
        }
        if (pick) {
          at = (long long)beam * a.V + key_index(pick);
          sc = (double)a.cum[(long long)b * K + beam] + ((double)key_value(pick) - s_lse[beam]);
        }
      } else if (kind == 1) {
        // the end token first, then the lowest of the others
        const int v = j == 0 ? a.eos : (j - 1 < a.eos ? j - 1 : j);
        if (v < a.V) {
          at = (long long)beam * a.V + v;
          sc = j == 0 ? (double)a.cum[(long long)b * K + beam] : -INFINITY;
        }
      } else if (j < a.V) {
        at = (long long)beam * a.V + j;
      }
      cs[i] = sc;
      c_at[i] = at;
    }
    __syncthreads();
    const int n = K * (K + 1);
    for (int i = tid; i < n; i += kThreads) {
      if (c_at[i] < 0) continue;
      int place = 0;
      for (int j = 0; j < n && place < K; ++j)
        place += c_at[j] >= 0 && (cs[j] > cs[i] || (cs[j] == cs[i] && c_at[j] < c_at[i]));
      if (place < K) {
        const int beam = (int)(c_at[i] / a.V), tok = (int)(c_at[i] - (long long)beam * a.V);
        const long long o = (long long)b * K + place;
        a.score[o] = (float)cs[i];
        a.parent[o] = beam;
        a.token[o] = tok;
        if (a.finished_out) sh.best[place] = (tok == a.eos || s_kind[beam] == 1 || (a.finished && a.finished[(long long)b * K + beam])) ? 1 : 0;
      }
    }
    __syncthreads();  // the flags read above may be the ones written here
    if (a.finished_out && tid < K) a.finished_out[(long long)b * K + tid] = (uint8_t)sh.best[tid];
  }
  cluster_sync();  // the parts are read until here
}

// state[o][b * K + k] <- state[o][b * K + parent[b, k]], in place: a thread
// reads one column of every row that moves before it writes any of them.
template <typename V, int KM>
__global__ void __launch_bounds__(256) k_beam_reorder(const BeamReorderArgs a) {
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

template <typename T>
cudaError_t select_t(const BeamSelectArgs& a, cudaStream_t st) {
  auto kern = k_beam_select<T>;
  static PerDevice once;
  int unused = 0;
  constexpr int smem = sizeof(SelectShared) + kMaxBeams * (kMaxBeams + 1) * 16;
  const cudaError_t ae = per_device(once, &unused, [&](int, int&) {
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  });
  if (ae != cudaSuccess) return ae;
  // CTAs of an item: a row each, or parts of a row where there are few rows
  // and the parts are not short
  int chunks = 1;
  while (a.K * chunks * 2 <= kMaxCluster && a.V >= chunks * 2 * 2048) chunks *= 2;
  const int C = a.K * chunks < kMaxCluster ? a.K * chunks : kMaxCluster / chunks * chunks;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.B * C));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, a, chunks);
}

}  // namespace

cudaError_t beam_select_launch(const BeamSelectArgs& a, int dtype, cudaStream_t st) {
  if (a.B <= 0) return cudaSuccess;
  return dtype == 0 ? select_t<__half>(a, st) : dtype == 1 ? select_t<__nv_bfloat16>(a, st) : select_t<float>(a, st);
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
