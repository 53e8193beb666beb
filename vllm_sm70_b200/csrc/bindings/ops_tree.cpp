// torch.ops._b200_C: tree attention over the paged cache.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>
#include <torch/torch.h>

#include <cmath>

#include "attention/tree_attn.h"

namespace b200 {
namespace {

int sm_count(int dev) {
  int n = 0;
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n > 0 ? n : 148;
}

int64_t tree_attention_workspace(int64_t head_dim, int64_t device) {
  return (int64_t)tree_attention_workspace_bytes((int)head_dim, sm_count((int)device));
}

bool aligned16(const at::Tensor& t) {
  return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
}

void tree_attention(at::Tensor& out, const at::Tensor& q, const at::Tensor& k_cache,
                    const at::Tensor& v_cache, const at::Tensor& block_table,
                    const at::Tensor& seq_lens, const at::Tensor& cu_q,
                    const at::Tensor& tree_mask, double scale, int64_t window,
                    const c10::optional<at::Tensor>& sinks,
                    const c10::optional<at::Tensor>& workspace) {
  const char* what = "tree_attention";
  TORCH_CHECK(q.is_cuda() && q.dim() == 3 && out.dim() == 3, what, ": q / out [T, Hq, D] on CUDA");
  for (const at::Tensor* t : {(const at::Tensor*)&out, &k_cache, &v_cache, &block_table, &seq_lens,
                              &cu_q, &tree_mask})
    TORCH_CHECK(t->device() == q.device(), what, ": every tensor must be on q's device");
  for (const at::Tensor* t : {(const at::Tensor*)&out, &q, &k_cache, &v_cache})
    TORCH_CHECK(t->scalar_type() == at::kBFloat16, what, ": q, out and the caches must be bf16");
  TORCH_CHECK(out.sizes() == q.sizes(), what, ": out must have q's shape");
  const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2);
  TORCH_CHECK(D == 64 || D == 128 || D == 256, what, ": head_dim must be 64, 128 or 256, got ", D);
  for (const at::Tensor* t : {(const at::Tensor*)&out, &q})
    TORCH_CHECK(t->stride(2) == 1 && (Hq == 1 || t->stride(1) == D) && t->stride(0) % 8 == 0 &&
                    (t->numel() == 0 || aligned16(*t)),
                what, ": q / out need dense [Hq, D] rows on 16-byte boundaries");
  TORCH_CHECK(k_cache.dim() == 4 && v_cache.sizes() == k_cache.sizes(), what,
              ": caches must be [blocks, Hkv, block_size, D] of the same shape");
  const int64_t Hkv = k_cache.size(1), BS = k_cache.size(2);
  TORCH_CHECK(k_cache.size(0) >= 1 && Hkv >= 1 && Hq % Hkv == 0 && k_cache.size(3) == D, what,
              ": cache heads / head_dim do not fit q");
  TORCH_CHECK(BS >= 8 && (BS & (BS - 1)) == 0, what, ": block_size must be a power of two >= 8");
  for (const at::Tensor* c : {&k_cache, &v_cache})
    TORCH_CHECK(c->stride(3) == 1 && c->stride(2) == D && c->stride(1) == BS * D &&
                    c->stride(0) % 8 == 0 && c->stride(0) >= Hkv * BS * D && aligned16(*c),
                what, ": cache blocks must be dense [Hkv, block_size, D] on 16-byte boundaries");
  TORCH_CHECK(k_cache.stride(0) == v_cache.stride(0), what, ": K/V block strides differ");
  for (const at::Tensor* t : {&block_table, &seq_lens, &cu_q, &tree_mask})
    TORCH_CHECK(t->scalar_type() == at::kInt && t->is_contiguous(), what,
                ": block_table, seq_lens, cu_q and tree_mask must be contiguous int32");
  const int64_t B = seq_lens.numel();
  TORCH_CHECK(seq_lens.dim() == 1 && cu_q.dim() == 1 && cu_q.numel() == B + 1, what,
              ": seq_lens [B] and cu_q [B + 1]");
  TORCH_CHECK(block_table.dim() == 2 && block_table.size(0) == B && (B == 0 || block_table.size(1) >= 1),
              what, ": block_table [B, max_blocks]");
  TORCH_CHECK(tree_mask.dim() == 2 && tree_mask.size(0) == T && tree_mask.size(1) >= 1, what,
              ": tree_mask [T, words]");
  TORCH_CHECK(std::isfinite(scale) && scale > 0, what, ": scale must be positive, got ", scale);
  TORCH_CHECK(window == 0 || window >= 32 * tree_mask.size(1), what,
              ": a sliding window must be 0 (none) or hold the whole tree (32 x mask words = ",
              32 * tree_mask.size(1), "), got ", window);
  if (sinks)
    TORCH_CHECK(sinks->device() == q.device() && sinks->scalar_type() == at::kFloat &&
                    sinks->is_contiguous() && sinks->numel() == Hq,
                what, ": sinks must be fp32 [Hq]");
  if (T == 0 || B == 0) return;
  c10::cuda::CUDAGuard g(q.device());
  const int64_t need = tree_attention_workspace(D, q.get_device());
  at::Tensor ws;
  if (workspace) {
    ws = *workspace;
    TORCH_CHECK(ws.device() == q.device() && ws.is_contiguous() && aligned16(ws) &&
                    (int64_t)ws.nbytes() >= need,
                what, ": workspace must be contiguous and hold ", need, " bytes");
  } else {
    ws = at::empty({need}, q.options().dtype(at::kByte));
  }
  TreeAttnArgs a{};
  a.q = q.data_ptr();
  a.k_cache = k_cache.data_ptr();
  a.v_cache = v_cache.data_ptr();
  a.out = out.data_ptr();
  a.block_table = block_table.data_ptr<int>();
  a.seq_lens = seq_lens.data_ptr<int>();
  a.cu_q = cu_q.data_ptr<int>();
  a.tree_mask = reinterpret_cast<const uint32_t*>(tree_mask.data_ptr<int>());
  a.sinks = sinks ? sinks->data_ptr<float>() : nullptr;
  a.workspace = reinterpret_cast<float*>(ws.data_ptr());
  a.num_seqs = (int)B;
  a.Hq = (int)Hq;
  a.Hkv = (int)Hkv;
  a.head_dim = (int)D;
  a.block_size = (int)BS;
  a.max_blocks = (int)block_table.size(1);
  a.num_blocks = (int)k_cache.size(0);
  a.mask_words = (int)tree_mask.size(1);
  a.window = (int)std::min<int64_t>(window, 1 << 30);
  a.num_tokens = T;
  a.q_stride_t = q.stride(0);
  a.o_stride_t = out.stride(0);
  a.kv_block_stride = k_cache.stride(0);
  a.scale = (float)scale;
  tree_attention_launch(a, at::cuda::getCurrentCUDAStream().stream());
}

}  // namespace
}  // namespace b200

TORCH_LIBRARY_FRAGMENT(_b200_C, m) {
  m.def("tree_attention(Tensor(a!) out, Tensor q, Tensor k_cache, Tensor v_cache, "
        "Tensor block_table, Tensor seq_lens, Tensor cu_q, Tensor tree_mask, float scale, "
        "int window=0, Tensor? sinks=None, Tensor(b!)? workspace=None) -> ()");
  m.def("tree_attention_workspace(int head_dim, int device) -> int",
        &b200::tree_attention_workspace);
}

TORCH_LIBRARY_IMPL(_b200_C, CUDA, m) { m.impl("tree_attention", &b200::tree_attention); }
