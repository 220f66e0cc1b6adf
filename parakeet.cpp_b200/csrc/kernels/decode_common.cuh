// What the kernels of the decoder's attention share: the items of a call and
// the partial results of parts of their keys.
#pragma once
#include "common.cuh"
#include "decode.h"

namespace pkc {

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

// index of a block of rows
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

// 128 query rows a CTA on tcgen05 (decode_attn_tc.cu); the call's keys in
// n_split parts, joined by k_attn_join.
constexpr int kTileRows = 128;
bool attn_tiles_fit(const DecodeAttnArgs& a);
cudaError_t attn_tiles_launch(const DecodeAttnArgs& a, bool bf16, int row_tiles, int n_split, cudaStream_t st);

}  // namespace pkc
