// Host interface of the attention decoder's kernels: cross attention over the
// encoder's states, the 8-bit key/value cache (append, attention, reordering)
// and beam search's selection and state reordering. Device pointers; every
// launcher is asynchronous on its stream and allocates nothing.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace pkc {

// The paged 8-bit cache (pkc_kv8_cache): e4m3 codes [n_pages][Hkv][page][D]
// and one f32 power-of-two scale for each (page, head).
struct Kv8 {
  uint8_t* k;
  uint8_t* v;
  float* k_scale;
  float* v_scale;
  int* table;  // [n_seqs][table_ld] page of each block of tokens
  int n_pages, page, n_kv_heads, head_dim, table_ld;
};

// One attention call of packed query rows over keys and values of another
// length: 16-bit rows (cross attention) or the 8-bit cache (cache.k != null).
struct DecodeAttnArgs {
  const void* q;  // [q_rows, H, D], row stride ldq elements
  long long ldq;
  const int* q_off;  // [n_items + 1]
  int max_q, q_rows;
  const void* k;  // [kv_rows, Hkv, D], row strides ldk / ldv
  const void* v;
  long long ldk, ldv;
  const int* kv_off;  // [n_items] first row
  const int* kv_len;  // [n_items] keys (8-bit cache: tokens, the new ones included)
  int max_kv, kv_rows;
  Kv8 cache;
  int n_items, n_heads, n_kv_heads, head_dim;
  float scale_log2;  // scale * log2(e)
  void* out;         // [q_rows, H, D], row stride ldo
  long long ldo;
  float* ws;  // decode_attn_ws_bytes()
  int* err;   // device error word, may be null
};
// Workspace of a call, from the sizes alone.
size_t decode_attn_ws_bytes(int n_items, int max_q, int max_kv, int n_heads, int n_kv_heads, int head_dim, bool q8);
cudaError_t decode_attn_launch(const DecodeAttnArgs& a, bool bf16, cudaStream_t st);

struct Kv8AppendArgs {
  Kv8 c;
  const void* k;  // new rows [rows, Hkv, D], row strides ldk / ldv
  const void* v;
  long long ldk, ldv;
  const int* new_off;  // [n_seqs + 1]
  const int* lens;     // [n_seqs] tokens, the new ones included
  int n_seqs, rows, max_new;
  int* err;
};
cudaError_t kv8_append_launch(const Kv8AppendArgs& a, bool bf16, cudaStream_t st);
cudaError_t kv8_reorder_launch(const Kv8& c, const int* parent, const int* lens, int B, int K, int* err,
                               cudaStream_t st);

struct BeamSelectArgs {
  const void* logits;  // [B*K, V], row stride ld elements
  long long ld;
  const float* cum;         // [B, K]
  const uint8_t* finished;  // [B, K] or null
  int B, K, V, eos;
  float* score;  // [B, K]; may be cum
  int* parent;
  int* token;
  uint8_t* finished_out;  // may be finished; null: not wanted
};
// dtype 0 f16, 1 bf16, 2 f32
cudaError_t beam_select_launch(const BeamSelectArgs& a, int dtype, cudaStream_t st);
constexpr int kMaxBeams = 32;

struct BeamReorderArgs {
  uint8_t* state;  // [n_outer][B * K] rows
  const int* parent;
  int B, K, n_outer;
  long long outer_stride, row_stride, row_bytes;
  const int* lens;  // [B] or null: live bytes = min(row_bytes, lens[b] * unit_bytes)
  long long unit_bytes;
  int* err;
};
cudaError_t beam_reorder_launch(const BeamReorderArgs& a, cudaStream_t st);

}  // namespace pkc
