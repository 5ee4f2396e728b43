// Host interface of the 4-bit paged KV cache kernels (kv4_cache.cu, kv4_decode.cu, kv4_prefill.cu).
//
// Cache: [blocks][kv heads][block_size / 16] units; a unit holds 16 tokens of one head in
// 18 * head_dim bytes (kv4.cuh describes its inside). head_dim is 64, 128 or 256.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace hk {

struct Kv4PlanArgs {
  const int* seq_rows;  // [S] block-table row of each request
  const int* cached;    // [S] tokens in the cache before the step
  const int* fresh;     // [S] tokens the step appends
  int S;
  int* tables;          // [table_rows, max_blocks]
  int table_rows, max_blocks, block_size;
  const int* free_blocks;  // [n_free] taken in order for new blocks, or null: the tables are complete
  int n_free;
  int *positions, *row_seq, *row_ctx, *slots;  // [cap] outputs
  int cap;
  int* taken;   // [1] blocks taken, or null
  int* status;  // device error word, or null
};

struct Kv4AppendArgs {
  const float* qkv;  // [R, (nh + 2 nkv) * hd], row stride qkv_stride
  int64_t qkv_stride;
  const float *bias, *q_norm, *k_norm;
  float eps;
  const int* positions;
  const int* slots;         // [R] token slots, or null: block_tables / row_seq
  const int* block_tables;  // [table_rows, max_blocks]
  const int* row_seq;
  int max_blocks, table_rows;
  const float* rope;  // [rope_rows, rot_dim / 2, 2]
  int rope_rows, rot_dim, rope_style;
  uint16_t* q_out;  // bf16 [R, nh, hd], row stride q_stride
  int64_t q_stride;
  uint8_t* cache;
  int64_t cache_blocks;
  int R, nh, nkv, hd, block_size;
};

struct Kv4GatherArgs {
  const uint8_t* cache;
  int64_t cache_blocks;
  const int* slots;  // [N]; a slot outside the cache gives zeros
  int N, nkv, hd, block_size;
  uint16_t *k, *v;   // bf16 [N, nkv, hd], either may be null
};

struct Kv4AttnArgs {
  const uint16_t* q;  // bf16 [R, nh, hd], row stride q_stride (elements)
  int64_t q_stride;
  const uint8_t* cache;
  int64_t cache_blocks;
  const int* block_tables;
  int max_blocks, table_rows;
  const int *row_seq, *row_ctx;
  float scale;
  int R, nh, nkv, hd, block_size;
  const float* sinks;   // [nh] extra logit per head, or null (NaN: the head is NaN; +infinity: it is zero)
  uint16_t* out_bf16;   // [R, nh * hd] with row stride out_stride, or null
  float* out;           // fp32, same shape and stride rule (outf_stride), or null
  int64_t out_stride, outf_stride;
  int* status;
  uint32_t wait_polls;  // polls after which a wait gives up (HK_ERR_MBAR_TIMEOUT; the outputs are then undefined)
};
constexpr uint32_t kKv4WaitPolls = 1u << 22;  // a second or so; a wait takes microseconds

// Scratch of the attention launches of one stream. counters are zero between launches.
struct Kv4Workspace {
  float* part;    // kKv4PartFloats
  int* counters;  // kKv4Counters
  int sms;
};
constexpr int kKv4Counters = 2048;  // decode: three per CTA
// Floats per SM. Decode: one CTA, with two partials of its own and one of each of its 15 warps (11 at head_dim 256), of
// an item's heads (at most kKv4ItemHeads: more per kv head make two items) x (head_dim + 4). Prefill with split keys: at
// most one part of 256 rows x (128 + 4).
constexpr int kKv4ItemHeads = 8;
constexpr int kKv4PartFloatsPerSm = 256 * 132;
constexpr int64_t kKv4PartFloats(int sms) { return (int64_t)sms * kKv4PartFloatsPerSm; }

void kv4_plan_launch(const Kv4PlanArgs& a, cudaStream_t s, bool pdl);
void kv4_append_launch(const Kv4AppendArgs& a, cudaStream_t s, bool pdl);
void kv4_gather_launch(const Kv4GatherArgs& a, cudaStream_t s, bool pdl);
void kv4_attention_decode_launch(const Kv4AttnArgs& a, const Kv4Workspace& ws, cudaStream_t s, bool pdl);
void kv4_attention_prefill_launch(const Kv4AttnArgs& a, const Kv4Workspace& ws, cudaStream_t s, bool pdl);

}  // namespace hk
