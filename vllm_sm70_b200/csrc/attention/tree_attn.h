// Host API of tree attention (tree_attn.cu).
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace b200 {

struct TreeAttnArgs {
  const void* q;        // [T, Hq, D] bf16, token stride q_stride_t elements (multiple of 8)
  const void* k_cache;  // [num_blocks, Hkv, block_size, D] bf16
  const void* v_cache;
  void* out;            // [T, Hq, D] bf16, token stride o_stride_t elements (multiple of 8)
  const int* block_table;     // [num_seqs, max_blocks]
  const int* seq_lens;        // [num_seqs], tree nodes included
  const int* cu_q;            // [num_seqs + 1]
  const uint32_t* tree_mask;  // [T, mask_words]
  const float* sinks;         // [Hq] or nullptr
  float* workspace;           // tree_attention_workspace_bytes, 16-byte aligned
  int num_seqs, Hq, Hkv, head_dim, block_size, max_blocks, num_blocks;
  int mask_words, window;
  int64_t num_tokens, q_stride_t, o_stride_t, kv_block_stride;
  float scale;
};

size_t tree_attention_workspace_bytes(int head_dim, int num_sm);
void tree_attention_launch(const TreeAttnArgs& a, cudaStream_t stream);

}  // namespace b200
