// C-ABI entry points of the attention decoder's kernels: cross attention, the
// 8-bit key/value cache, beam selection and state reordering. Each checks what
// the host can know, launches on the caller's stream and returns.
#include <cuda_runtime.h>

#include <cmath>
#include <initializer_list>
#include <string>

#include "../../include/pkc.h"
#include "kernels/decode.h"
#include "status.hpp"

namespace {

// Runs an entry point's body; nothing may leave it as a C++ exception.
template <typename F>
pkc_status guarded(const char* what, F&& body) noexcept {
  try {
    return body();
  } catch (...) {
    try {
      return pkc::set_thread_error(PKC_ERR_INTERNAL, std::string(what) + ": host error");
    } catch (...) {
      return PKC_ERR_INTERNAL;
    }
  }
}

constexpr float kLog2e = 1.4426950408889634f;
// keys of one item: places of keys are ints, and rounded up to tiles
constexpr int kMaxKeys = 1 << 30;

pkc_status bad(const char* what, const char* why) {
  return pkc::set_thread_error(PKC_ERR_ARG, std::string(what) + ": " + why);
}

bool aligned(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// The stream and the given memory belong to the current device; arrays of
// 32-bit numbers are aligned. NULLs are passed over.
pkc_status check_device(const char* what, void* stream, std::initializer_list<const void*> ints,
                        std::initializer_list<const void*> more) {
  for (const void* p : ints)
    if (!aligned(p, 4)) return bad(what, "an array of 32-bit numbers is not aligned");
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return pkc::set_thread_error(PKC_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (st && st != cudaStreamLegacy && st != cudaStreamPerThread) {
    // (a capturing stream must not be asked for its device: that ends the capture)
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(st, &cap) != cudaSuccess) {
      cudaGetLastError();
      return bad(what, "invalid stream");
    }
    int sdev = dev;
    if (cap == cudaStreamCaptureStatusNone && cudaStreamGetDevice(st, &sdev) != cudaSuccess) {
      cudaGetLastError();
      return bad(what, "invalid stream");
    }
    if (sdev != dev) return bad(what, "the stream belongs to another device than the current one");
  }
  for (const auto* list : {&ints, &more})
    for (const void* p : *list) {
      if (!p) continue;
      cudaPointerAttributes at;
      if (cudaPointerGetAttributes(&at, p) != cudaSuccess) {
        cudaGetLastError();
        return bad(what, "a pointer is not device memory");
      }
      if (at.type != cudaMemoryTypeManaged && (at.type != cudaMemoryTypeDevice || at.device != dev))
        return bad(what, "memory of the host or of another device than the current one");
    }
  return PKC_OK;
}

pkc_status launched(const char* what, cudaError_t e) {
  if (e == cudaSuccess) return PKC_OK;
  cudaGetLastError();
  return pkc::set_thread_error(PKC_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

// nullptr, or what is wrong with a cache
const char* cache_fault(const pkc_kv8_cache* c) {
  if (!c) return "cache is NULL";
  if (!c->k || !c->v || !c->k_scale || !c->v_scale || !c->table) return "a cache pointer is NULL";
  if (c->page != 16 && c->page != 32 && c->page != 64 && c->page != 128) return "page must be 16, 32, 64 or 128";
  if (c->head_dim != 64 && c->head_dim != 128) return "head_dim must be 64 or 128";
  if (c->n_pages <= 0 || c->n_kv_heads <= 0 || c->table_ld <= 0) return "a size of the cache is not positive";
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4) ||
      !aligned(c->table, 4))
    return "the cache's codes must be 16-byte aligned";
  return nullptr;
}

pkc::Kv8 kv8_of(const pkc_kv8_cache* c) {
  return pkc::Kv8{static_cast<uint8_t*>(c->k), static_cast<uint8_t*>(c->v), c->k_scale, c->v_scale, c->table,
                  c->n_pages, c->page, c->n_kv_heads, c->head_dim, c->table_ld};
}

// row strides of 16-bit rows of `row` elements
const char* rows_fault(const void* p, long long ld, long long row, const char* why) {
  return !aligned(p, 16) || ld % 8 != 0 || ld < row ? why : nullptr;
}

}  // namespace

extern "C" size_t pkc_cross_attention_workspace(int B, int max_q, int max_kv, int n_heads, int n_kv_heads,
                                                int head_dim) {
  if (B <= 0 || max_q <= 0 || max_kv < 0 || n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads || head_dim <= 0)
    return 0;
  return pkc::decode_attn_ws_bytes(B, max_q, max_kv, n_heads, n_kv_heads, head_dim, false);
}

extern "C" pkc_status pkc_cross_attention(const void* q, long long ldq, const int* q_off, int max_q, int q_rows,
                                          const void* k, long long ldk, const void* v, long long ldv,
                                          const int* kv_off, const int* kv_len, int max_kv, int kv_rows, int B,
                                          int n_heads, int n_kv_heads, int head_dim, float scale, int dtype, void* out,
                                          long long ldo, void* workspace, size_t workspace_bytes, int* err,
                                          void* stream) {
  const char* what = "pkc_cross_attention";
  return guarded(what, [&]() -> pkc_status {
    if (B < 0 || q_rows < 0 || kv_rows < 0 || max_q < 0 || max_kv < 0) return bad(what, "a size is negative");
    if (max_kv > kMaxKeys) return bad(what, "max_kv is more than 2^30");
    if (dtype != 0 && dtype != 1) return bad(what, "dtype must be 0 (f16) or 1 (bf16)");
    if (head_dim != 64 && head_dim != 128) return bad(what, "head_dim must be 64 or 128");
    if (n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads)
      return bad(what, "n_heads must be a positive multiple of n_kv_heads");
    if (!std::isfinite(scale * kLog2e)) return bad(what, "scale must be finite, and its product with log2(e)");
    if (B == 0 || max_q == 0 || q_rows == 0) return PKC_OK;
    if (!q || !q_off || !kv_off || !kv_len || !out || ((!k || !v) && kv_rows > 0)) return bad(what, "a pointer is NULL");
    const long long qr = (long long)n_heads * head_dim, kr = (long long)n_kv_heads * head_dim;
    const char* why = rows_fault(q, ldq, qr, "q rows must be 16-byte aligned and not overlap");
    if (!why) why = rows_fault(out, ldo, qr, "out rows must be 16-byte aligned and not overlap");
    if (!why && kv_rows > 0) why = rows_fault(k, ldk, kr, "k rows must be 16-byte aligned and not overlap");
    if (!why && kv_rows > 0) why = rows_fault(v, ldv, kr, "v rows must be 16-byte aligned and not overlap");
    if (why) return bad(what, why);
    const size_t need = pkc::decode_attn_ws_bytes(B, max_q, max_kv, n_heads, n_kv_heads, head_dim, false);
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
      return bad(what, "the workspace is missing, too small or not 16-byte aligned");
    const pkc_status ds = check_device(what, stream, {q_off, kv_off, kv_len, err},
                                       {q, out, kv_rows > 0 ? k : nullptr, kv_rows > 0 ? v : nullptr,
                                        need > 0 ? workspace : nullptr});
    if (ds != PKC_OK) return ds;
    pkc::DecodeAttnArgs a{};
    a.q = q; a.ldq = ldq; a.q_off = q_off; a.max_q = max_q; a.q_rows = q_rows;
    a.k = k; a.v = v; a.ldk = ldk; a.ldv = ldv; a.kv_off = kv_off; a.kv_len = kv_len;
    a.max_kv = max_kv; a.kv_rows = kv_rows;
    a.n_items = B; a.n_heads = n_heads; a.n_kv_heads = n_kv_heads; a.head_dim = head_dim;
    a.scale_log2 = scale * kLog2e;
    a.out = out; a.ldo = ldo; a.ws = static_cast<float*>(workspace); a.err = err;
    return launched(what, pkc::decode_attn_launch(a, dtype == 1, reinterpret_cast<cudaStream_t>(stream)));
  });
}

extern "C" pkc_status pkc_kv8_append(const pkc_kv8_cache* cache, const void* k, long long ldk, const void* v,
                                     long long ldv, const int* new_off, const int* lens, int n_seqs, int rows,
                                     int max_new, int dtype, int* err, void* stream) {
  const char* what = "pkc_kv8_append";
  return guarded(what, [&]() -> pkc_status {
    if (const char* why = cache_fault(cache)) return bad(what, why);
    if (n_seqs < 0 || rows < 0 || max_new < 0) return bad(what, "a size is negative");
    if (dtype != 0 && dtype != 1) return bad(what, "dtype must be 0 (f16) or 1 (bf16)");
    if (n_seqs == 0 || rows == 0 || max_new == 0) return PKC_OK;
    if (!k || !v || !new_off || !lens) return bad(what, "a pointer is NULL");
    const long long row = (long long)cache->n_kv_heads * cache->head_dim;
    const char* why = rows_fault(k, ldk, row, "k rows must be 16-byte aligned and not overlap");
    if (!why) why = rows_fault(v, ldv, row, "v rows must be 16-byte aligned and not overlap");
    if (why) return bad(what, why);
    const pkc_status ds = check_device(what, stream, {new_off, lens, cache->table, cache->k_scale, cache->v_scale, err},
                                       {k, v, cache->k, cache->v});
    if (ds != PKC_OK) return ds;
    // (no sequence has more new tokens than there are, or than its pages hold)
    const long long holds = (long long)cache->table_ld * cache->page;
    int most = max_new < rows ? max_new : rows;
    if (most > holds) most = (int)holds;
    pkc::Kv8AppendArgs a{kv8_of(cache), k, v, ldk, ldv, new_off, lens, n_seqs, rows, most, err};
    return launched(what, pkc::kv8_append_launch(a, dtype == 1, reinterpret_cast<cudaStream_t>(stream)));
  });
}

extern "C" size_t pkc_kv8_attention_workspace(const pkc_kv8_cache* cache, int n_seqs, int max_q, int max_len,
                                              int n_heads) {
  if (cache_fault(cache) || n_seqs <= 0 || max_q <= 0 || max_len < 0 || n_heads <= 0 || n_heads % cache->n_kv_heads)
    return 0;
  return pkc::decode_attn_ws_bytes(n_seqs, max_q, max_len, n_heads, cache->n_kv_heads, cache->head_dim, true);
}

extern "C" pkc_status pkc_kv8_attention(const pkc_kv8_cache* cache, const void* q, long long ldq, const int* q_off,
                                        int max_q, int q_rows, const int* lens, int max_len, int n_seqs, int n_heads,
                                        float scale, int dtype, void* out, long long ldo, void* workspace,
                                        size_t workspace_bytes, int* err, void* stream) {
  const char* what = "pkc_kv8_attention";
  return guarded(what, [&]() -> pkc_status {
    if (const char* why = cache_fault(cache)) return bad(what, why);
    if (n_seqs < 0 || q_rows < 0 || max_q < 0 || max_len < 0) return bad(what, "a size is negative");
    if (max_len > kMaxKeys || max_len > (long long)cache->table_ld * cache->page)
      return bad(what, "max_len is more than 2^30 or beyond the block table");
    if (dtype != 0 && dtype != 1) return bad(what, "dtype must be 0 (f16) or 1 (bf16)");
    if (n_heads <= 0 || n_heads % cache->n_kv_heads)
      return bad(what, "n_heads must be a positive multiple of n_kv_heads");
    if (!std::isfinite(scale * kLog2e)) return bad(what, "scale must be finite, and its product with log2(e)");
    if (n_seqs == 0 || max_q == 0 || q_rows == 0) return PKC_OK;
    if (!q || !q_off || !lens || !out) return bad(what, "a pointer is NULL");
    const long long qr = (long long)n_heads * cache->head_dim;
    const char* why = rows_fault(q, ldq, qr, "q rows must be 16-byte aligned and not overlap");
    if (!why) why = rows_fault(out, ldo, qr, "out rows must be 16-byte aligned and not overlap");
    if (why) return bad(what, why);
    const size_t need =
        pkc::decode_attn_ws_bytes(n_seqs, max_q, max_len, n_heads, cache->n_kv_heads, cache->head_dim, true);
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
      return bad(what, "the workspace is missing, too small or not 16-byte aligned");
    const pkc_status ds = check_device(what, stream, {q_off, lens, cache->table, cache->k_scale, cache->v_scale, err},
                                       {q, out, cache->k, cache->v, need > 0 ? workspace : nullptr});
    if (ds != PKC_OK) return ds;
    pkc::DecodeAttnArgs a{};
    a.q = q; a.ldq = ldq; a.q_off = q_off; a.max_q = max_q; a.q_rows = q_rows;
    a.kv_len = lens; a.max_kv = max_len; a.cache = kv8_of(cache);
    a.n_items = n_seqs; a.n_heads = n_heads; a.n_kv_heads = cache->n_kv_heads; a.head_dim = cache->head_dim;
    a.scale_log2 = scale * kLog2e;
    a.out = out; a.ldo = ldo; a.ws = static_cast<float*>(workspace); a.err = err;
    return launched(what, pkc::decode_attn_launch(a, dtype == 1, reinterpret_cast<cudaStream_t>(stream)));
  });
}

extern "C" pkc_status pkc_kv8_reorder(const pkc_kv8_cache* cache, const int* parent, const int* lens, int B, int K,
                                      int* err, void* stream) {
  const char* what = "pkc_kv8_reorder";
  return guarded(what, [&]() -> pkc_status {
    if (const char* why = cache_fault(cache)) return bad(what, why);
    if (B < 0 || B > 65535 || K <= 0 || K > pkc::kMaxBeams)
      return bad(what, "B must be in [0, 65535] and K in [1, 32]");
    if (B == 0) return PKC_OK;
    if (!parent || !lens) return bad(what, "a pointer is NULL");
    const pkc_status ds = check_device(what, stream, {parent, lens, cache->table, cache->k_scale, cache->v_scale, err},
                                       {cache->k, cache->v});
    if (ds != PKC_OK) return ds;
    return launched(what, pkc::kv8_reorder_launch(kv8_of(cache), parent, lens, B, K, err,
                                                  reinterpret_cast<cudaStream_t>(stream)));
  });
}

extern "C" pkc_status pkc_beam_select(const void* logits, long long ld, int dtype, const float* cum,
                                      const uint8_t* finished, int B, int K, int V, int eos, float* score, int* parent,
                                      int* token, uint8_t* finished_out, void* stream) {
  const char* what = "pkc_beam_select";
  return guarded(what, [&]() -> pkc_status {
    if (B < 0 || B > (1 << 24) || K <= 0 || K > pkc::kMaxBeams)
      return bad(what, "B must be in [0, 2^24] and K in [1, 32]");
    if (V <= 0 || V > (1 << 30) || eos < 0 || eos >= V || ld < V) return bad(what, "bad V, eos or ld");
    if (dtype < 0 || dtype > 2) return bad(what, "dtype must be 0 (f16), 1 (bf16) or 2 (f32)");
    if (B == 0) return PKC_OK;
    if (!logits || !cum || !score || !parent || !token) return bad(what, "a pointer is NULL");
    if (!aligned(logits, dtype == 2 ? 4 : 2)) return bad(what, "logits are not aligned to their type");
    const pkc_status ds = check_device(what, stream, {cum, score, parent, token}, {logits, finished, finished_out});
    if (ds != PKC_OK) return ds;
    pkc::BeamSelectArgs a{logits, ld, cum, finished, B, K, V, eos, score, parent, token, finished_out};
    return launched(what, pkc::beam_select_launch(a, dtype, reinterpret_cast<cudaStream_t>(stream)));
  });
}

extern "C" pkc_status pkc_beam_reorder(void* state, const int* parent, int B, int K, long long row_bytes,
                                       long long row_stride, int n_outer, long long outer_stride, const int* lens,
                                       long long unit_bytes, int* err, void* stream) {
  const char* what = "pkc_beam_reorder";
  return guarded(what, [&]() -> pkc_status {
    if (B < 0 || B > 65535 || K <= 0 || K > pkc::kMaxBeams || n_outer < 0 || n_outer > 65535)
      return bad(what, "B and n_outer must be in [0, 65535] and K in [1, 32]");
    if (row_bytes < 0 || row_stride < row_bytes || (lens && (unit_bytes < 0 || unit_bytes > (1LL << 31))))
      return bad(what, "bad row_bytes, row_stride or unit_bytes");
    // (a quotient: the product may pass 64 bits)
    if (n_outer > 1 && B > 0 && outer_stride / ((long long)B * K) < row_stride)
      return bad(what, "blocks overlap: outer_stride is less than B * K * row_stride");
    if (B == 0 || n_outer == 0 || row_bytes == 0) return PKC_OK;
    if (!state || !parent) return bad(what, "a pointer is NULL");
    const pkc_status ds = check_device(what, stream, {parent, lens, err}, {state});
    if (ds != PKC_OK) return ds;
    pkc::BeamReorderArgs a{static_cast<uint8_t*>(state), parent, B, K, n_outer, n_outer > 1 ? outer_stride : 0,
                           row_stride, row_bytes, lens, lens ? unit_bytes : 0, err};
    return launched(what, pkc::beam_reorder_launch(a, reinterpret_cast<cudaStream_t>(stream)));
  });
}
