// Attention of trees of drafted tokens over a paged KV cache.
//
// Node j of sequence s sits in the cache at position prior + j, prior = context_lens[s] - L.  It attends to the
// positions below prior and to those prior + i whose bit i its mask has set:
//   out = sum_t p_t V_t,  p = softmax(scale q.K_t) over those t;  zeros where there are none.
#include <math.h>

#include <algorithm>

#include "tree.hpp"

namespace rg {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct TreeArgs {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  const int32_t* table;
  const int32_t* context_lens;
  const int32_t* cu;
  const int32_t* mask;
  float scale_log2;
  int32_t num_heads, num_kv_heads, head_dim, block_size, max_blocks, num_seqs, num_nodes, max_nodes, mask_words;
  int64_t kv_stride;
};

// Any shape: a wave per (sequence, node, q-head), lane l has dims 4 l .. 4 l + 3, the keys one after the other with
// the running maximum m and sum l of their weights.
template <typename T>
__global__ __launch_bounds__(64) void tree_generic_kernel(TreeArgs a) {
  using E = elem<T>;
  using S = typename E::storage;
  const int s = blockIdx.z, h = blockIdx.y, lane = threadIdx.x;
  const Tree t = tree_of(a.cu, s, a.num_nodes, a.max_nodes);
  const int ctx = max(0, min(a.context_lens[s], a.max_blocks * a.block_size)), prior = max(ctx - t.len, 0);
  const int kvh = h / (a.num_heads / a.num_kv_heads);
  const int d0 = lane * 4;
  const bool act = d0 < a.head_dim;
  const int32_t* row = a.table + (int64_t)s * a.max_blocks;
  const S* kc = static_cast<const S*>(a.k);
  const S* vc = static_cast<const S*>(a.v);
  for (int j = blockIdx.x; j < t.nodes; j += gridDim.x) {
    const int64_t at = ((int64_t)(t.first + j) * a.num_heads + h) * a.head_dim;
    const int32_t* bits = a.mask + (int64_t)(t.first + j) * a.mask_words;
    float qv[4] = {0.f, 0.f, 0.f, 0.f}, o[4] = {0.f, 0.f, 0.f, 0.f};
    if (act) {
#pragma unroll
      for (int u = 0; u < 4; ++u) qv[u] = E::load(static_cast<const S*>(a.q) + at, d0 + u);
    }
    float m = -INFINITY, l = 0.f;
    for (int p = 0; p < ctx; ++p) {
      const int i = p - prior;
      if (i >= 0 && (i >= t.nodes || !(bits[i >> 5] >> (i & 31) & 1))) continue;
      const int64_t base = row[p / a.block_size] * a.kv_stride +
                           ((int64_t)kvh * a.block_size + p % a.block_size) * a.head_dim;
      float kv[4] = {0.f, 0.f, 0.f, 0.f}, vv[4] = {0.f, 0.f, 0.f, 0.f};
      if (act) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          kv[u] = E::load(kc, base + d0 + u);
          vv[u] = E::load(vc, base + d0 + u);
        }
      }
      const float x = wave_sum(qv[0] * kv[0] + qv[1] * kv[1] + qv[2] * kv[2] + qv[3] * kv[3]) * a.scale_log2;
      const float m_new = fmaxf(m, x);
      const float alpha = m == m_new ? 1.f : exp2f(m - m_new);
      const float w = x == -INFINITY ? 0.f : exp2f(x - m_new);
      l = l * alpha + w;
#pragma unroll
      for (int u = 0; u < 4; ++u) o[u] = o[u] * alpha + w * vv[u];
      m = m_new;
    }
    const float inv = l != 0.f ? 1.f / l : 1.f;
    if (act) {
#pragma unroll
      for (int u = 0; u < 4; ++u) E::store(static_cast<S*>(a.out) + at, d0 + u, o[u] * inv);
    }
  }
}

}  // namespace

int probe_tree_attention_kernels() {
  hipFuncAttributes at;
  if (hipFuncGetAttributes(&at, reinterpret_cast<const void*>(tree_generic_kernel<bf16_t>)) != hipSuccess) {
    return fail(RG_ERR_HIP, "failed to load the tree attention kernels: %s", hipGetErrorString(hipGetLastError()));
  }
  return RG_OK;
}

}  // namespace rg

using namespace rg;

extern "C" size_t rg_paged_attention_tree_workspace_bytes(int32_t num_seqs, int32_t max_nodes, int32_t num_heads,
                                                          int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                                                          int32_t max_blocks_per_seq) {
  return 0;
}

extern "C" int rg_paged_attention_tree(const void* query, const void* key_cache, const void* value_cache,
                                       const int32_t* block_table, const int32_t* context_lens,
                                       const int32_t* cu_nodes, const int32_t* tree_mask, void* output, float scale,
                                       int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                                       int32_t max_blocks_per_seq, int32_t num_seqs, int32_t num_nodes,
                                       int32_t max_nodes, int32_t mask_words, int32_t dtype, int64_t kv_block_stride,
                                       void* workspace, size_t workspace_bytes, void* stream) {
  const char* op = "paged_attention_tree";
  if (dtype_bytes(dtype) == 0) return fail(RG_ERR_NOT_SUPPORTED, "%s: unknown dtype %d", op, dtype);
  if (head_dim % 4 != 0 || head_dim > RG_MAX_HEAD_DIM || head_dim <= 0) {
    return fail(RG_ERR_NOT_SUPPORTED, "%s: head_dim must be a multiple of 4 and <= %d, got %d", op, RG_MAX_HEAD_DIM,
                head_dim);
  }
  if (num_seqs < 0 || num_nodes < 0 || num_heads <= 0 || num_kv_heads <= 0 || block_size <= 0 || max_blocks_per_seq < 0) {
    return fail(RG_ERR_INVALID_ARGUMENT,
                "%s: need num_seqs, num_nodes and max_blocks_per_seq >= 0 and positive heads / block_size", op);
  }
  if (num_heads % num_kv_heads != 0) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: num_heads %d is not a multiple of num_kv_heads %d", op, num_heads,
                num_kv_heads);
  }
  int st = check_tree_nodes(op, max_nodes);
  if (st != RG_OK) return st;
  if (mask_words < ceil_div(max_nodes, 32)) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: mask_words %d for trees of %d nodes", op, mask_words, max_nodes);
  }
  const int64_t block = (int64_t)num_kv_heads * block_size * head_dim;
  if (kv_block_stride != 0 && kv_block_stride < block) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: kv_block_stride %lld smaller than a block", op, (long long)kv_block_stride);
  }
  if ((int64_t)max_blocks_per_seq * block_size > INT32_MAX - 65536 || num_seqs > 65535 || num_heads > 65535) {
    return fail(RG_ERR_NOT_SUPPORTED, "%s: a block table of %lld tokens, %d sequences, %d heads", op,
                (long long)max_blocks_per_seq * block_size, num_seqs, num_heads);
  }
  if (num_seqs == 0 || num_nodes == 0 || max_nodes == 0) return ok();
  if (!query || !key_cache || !value_cache || !block_table || !context_lens || !cu_nodes || !tree_mask || !output) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: null pointer argument", op);
  }
  const TreeArgs a{query, key_cache, value_cache, output, block_table, context_lens, cu_nodes, tree_mask,
                   scale * kLog2e, num_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq, num_seqs,
                   num_nodes, max_nodes, mask_words, kv_block_stride ? kv_block_stride : block};
  const dim3 grid((unsigned)max_nodes, (unsigned)num_heads, (unsigned)num_seqs);
  return dispatch_dtype(dtype, [&](auto tag) {
    hipLaunchKernelGGL(tree_generic_kernel<decltype(tag)>, grid, dim3(64), 0, as_stream(stream), a);
    return check_launch(op);
  });
}
