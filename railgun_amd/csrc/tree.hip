// A step over drafted tokens, but for its attention (tree_attention.hip): the layout of the trees, which of their
// nodes the model agrees with, and the move of those nodes' cached tokens.
//
// Sequence s owns nodes [cu_nodes[s], cu_nodes[s + 1]) of the packed arrays; node j of it lies in the cache at
// position prior + j, prior = context_lens[s] - L.  A parent is an index in the sequence's own tree below the node's
// own; anything else is no parent.
#include <algorithm>

#include "tree.hpp"

namespace rg {
namespace {

// ------------------------------------------------------------------ layout --

// Ancestors by doubling: with up[j] the node 2^k steps above j (-1: none) and seen[j] the bits of those in between,
//   seen[j] |= seen[up[j]],  depth[j] += depth[up[j]],  up[j] = up[up[j]],
// so a chain of n nodes takes log2 n rounds.  seen is updated in place: what a node reads early are ancestors too.
// A workgroup has kLayoutWords of a tree's mask words, so that 1,024 nodes' fit in LDS; the positions and slots are
// written by the first of a tree's.  Latency: the parents, lengths and table are read in three dependent steps, then a
// barrier a round.  One tree of 64 nodes 3.4 us, 256 of 33 to 256 6.2 us (1.7 MB).
constexpr int kLayoutThreads = 256;
constexpr int kLayoutWords = 8;

struct LayoutArgs {
  const int32_t* parents;
  const int32_t* cu;
  const int32_t* context_lens;
  const int32_t* table;
  const int32_t* text;  // NULL: the root's position is prior
  int32_t* mask;
  int32_t* positions;
  int32_t* slots;
  int32_t num_nodes, max_nodes, mask_words, block_size, max_blocks;
};

__global__ __launch_bounds__(kLayoutThreads) void tree_layout_kernel(LayoutArgs a) {
  __shared__ uint4 seen[kMaxTreeNodes * kLayoutWords / 4];
  __shared__ int16_t up[2][kMaxTreeNodes], depth[2][kMaxTreeNodes];
  static_assert(kLayoutWords == 8, "two 16-byte pieces to a node");
  const int s = blockIdx.x, w0 = blockIdx.y * kLayoutWords, tid = threadIdx.x;
  const Tree t = tree_of(a.cu, s, a.num_nodes, a.max_nodes);
  const int words = min(kLayoutWords, a.mask_words - w0);
  const int ctx = max(0, min(a.context_lens[s], a.max_blocks * a.block_size)), prior = max(ctx - t.len, 0);
  const int root = a.text ? a.text[s] : prior;
  for (int j = tid; j < t.nodes; j += kLayoutThreads) {
    const int p = a.parents[t.first + j];
    if (blockIdx.y == 0) {
      const int at = prior + j;
      int slot = -1;
      if (at < ctx) {
        slot = a.table[(int64_t)s * a.max_blocks + at / a.block_size] * a.block_size + at % a.block_size;
      }
      a.slots[t.first + j] = slot;
    }
    up[0][j] = (int16_t)(p >= 0 && p < j ? p : -1);
    depth[0][j] = (int16_t)(p >= 0 && p < j);
    const uint32_t bit = 1u << (j & 31);
    const int w = (j >> 5) - w0;
    seen[2 * j] = make_uint4(w == 0 ? bit : 0u, w == 1 ? bit : 0u, w == 2 ? bit : 0u, w == 3 ? bit : 0u);
    seen[2 * j + 1] = make_uint4(w == 4 ? bit : 0u, w == 5 ? bit : 0u, w == 6 ? bit : 0u, w == 7 ? bit : 0u);
  }
  __syncthreads();
  int cur = 0;
  while (true) {
    int more = 0;
    for (int j = tid; j < t.nodes; j += kLayoutThreads) {
      const int p = up[cur][j];
      int q = -1, d = depth[cur][j];
      if (p >= 0) {
        uint4 x = seen[2 * j], y = seen[2 * j + 1];
        const uint4 u = seen[2 * p], v = seen[2 * p + 1];
        q = up[cur][p];
        d += depth[cur][p];
        x = make_uint4(x.x | u.x, x.y | u.y, x.z | u.z, x.w | u.w);
        y = make_uint4(y.x | v.x, y.y | v.y, y.z | v.z, y.w | v.w);
        seen[2 * j] = x;
        seen[2 * j + 1] = y;
      }
      depth[cur ^ 1][j] = (int16_t)d;
      up[cur ^ 1][j] = (int16_t)q;
      more |= q >= 0;
    }
    cur ^= 1;
    if (!__syncthreads_or(more)) break;
  }
  const uint32_t* bits = reinterpret_cast<const uint32_t*>(seen);
  for (int j = tid; j < t.nodes; j += kLayoutThreads) {
    int32_t* to = a.mask + (int64_t)(t.first + j) * a.mask_words + w0;
    for (int w = 0; w < words; ++w) to[w] = (int32_t)bits[j * kLayoutWords + w];
    if (blockIdx.y == 0) a.positions[t.first + j] = root + depth[cur][j];
  }
}

// ------------------------------------------------------------ verification --

// A logit and its index as one number that is larger for a larger logit, and for a lower index of equal ones.
// -0 equals +0; a NaN is never compared, so it ranks as -inf.
__device__ __forceinline__ uint64_t rank_of(float v, uint32_t index) {
  const uint32_t u = __float_as_uint(v + 0.f);  // -0 + 0 = +0
  return (uint64_t)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (uint32_t)~index;
}
// The index in it (nothing above -inf: the first).
__device__ __forceinline__ int32_t token_of(uint64_t key) { return key ? (int32_t)~(uint32_t)key : 0; }
__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t other = __shfl_xor((unsigned long long)v, o, kWave);
    v = other > v ? other : v;
  }
  return v;
}

constexpr int kArgmaxThreads = 256;
constexpr int kArgmaxAhead = 4;  // 16-byte pieces of a thread in flight

template <typename T> struct Piece {
  static constexpr int N = 16 / elem<T>::bytes;
  float v[N];
  __device__ __forceinline__ explicit Piece(uint4 u) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (N == 4) v[i] = __uint_as_float(w[i]);
      else {
        v[2 * i] = elem<T>::to_f32((uint16_t)(w[i] & 0xffffu));
        v[2 * i + 1] = elem<T>::to_f32((uint16_t)(w[i] >> 16));
      }
    }
  }
  __device__ __forceinline__ float largest() const {  // (fmaxf passes over NaN)
    float m = v[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = fmaxf(m, v[i]);
    return m;
  }
};

// Workgroup (row, split): the best of one piece of a row of logits.  The row's 16-byte pieces are dealt to the
// splits; what lies before the first and behind the last goes to the first and the last split.  A thread keeps the
// largest value and the piece it was in (of equal ones the first, it goes through them in order) and looks for the
// place in that at the end.  Bound by HBM: 1,469 rows of 128,256 in bf16 58 us, 6.4 TB/s (a row to a workgroup); 64
// rows 5.2 us, 16 pieces to a row.
template <typename T>
__global__ __launch_bounds__(kArgmaxThreads) void argmax_kernel(const typename elem<T>::storage* __restrict__ logits,
                                                                int64_t row_stride, int32_t vocab, int32_t splits,
                                                                const int32_t* __restrict__ cu, int32_t num_seqs,
                                                                uint64_t* __restrict__ best) {
  using E = elem<T>;
  constexpr int N = Piece<T>::N;
  const int tid = threadIdx.x, split = blockIdx.y;
  const int row = blockIdx.x;
  if (row >= cu[num_seqs]) return;
  const typename E::storage* x = logits + (int64_t)row * row_stride;
  const int head = min(vocab, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15u)) % 16) / E::bytes);
  const int pieces = (vocab - head) / N;
  const uint4* body = reinterpret_cast<const uint4*>(x + head);
  const int p0 = (int)((int64_t)pieces * split / splits), p1 = (int)((int64_t)pieces * (split + 1) / splits);
  float top = -INFINITY;
  int at = -1;
  uint4 held = make_uint4(0u, 0u, 0u, 0u);
  for (int p = p0 + tid; p < p1; p += kArgmaxThreads * kArgmaxAhead) {
    uint4 u[kArgmaxAhead];
#pragma unroll
    for (int i = 0; i < kArgmaxAhead; ++i) {
      const int q = p + i * kArgmaxThreads;
      u[i] = stream_load16(body + (q < p1 ? q : p));
    }
#pragma unroll
    for (int i = 0; i < kArgmaxAhead; ++i) {
      const float m = Piece<T>(u[i]).largest();
      const bool better = m > top && p + i * kArgmaxThreads < p1;
      top = better ? m : top;
      at = better ? p + i * kArgmaxThreads : at;
      held = make_uint4(better ? u[i].x : held.x, better ? u[i].y : held.y, better ? u[i].z : held.z,
                        better ? u[i].w : held.w);
    }
  }
  uint64_t key = 0;
  if (at >= 0) {
    const Piece<T> piece(held);
    int e = 0;
#pragma unroll
    for (int i = N - 1; i >= 0; --i) e = piece.v[i] == top ? i : e;
    key = rank_of(top, (uint32_t)(head + at * N + e));
  }
  auto single = [&](int i) {
    const float v = E::to_f32(x[i]);
    if (v > -INFINITY) key = max(key, rank_of(v, (uint32_t)i));
  };
  if (split == 0 && tid < head) single(tid);
  if (split == splits - 1 && head + pieces * N + tid < vocab) single(head + pieces * N + tid);
  key = wave_max64(key);
  __shared__ uint64_t wave_best[kArgmaxThreads / kWave];
  if (tid % kWave == 0) wave_best[tid / kWave] = key;
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int i = 1; i < kArgmaxThreads / kWave; ++i) key = max(key, wave_best[i]);
    best[(int64_t)row * splits + split] = key;
  }
}

struct AcceptArgs {
  const uint64_t* best;  // [num_nodes, splits], or NULL: the targets are given
  int32_t* target;
  const int32_t* draft;
  const int32_t* parents;
  const int32_t* cu;
  int32_t* accepted;
  int32_t* count;
  int32_t* next;
  int32_t num_nodes, max_nodes, max_accepted, splits;
};

// One workgroup per sequence.  child[p] is the lowest node below p that drafted p's target, found by all nodes at
// once; the path from the root is then a walk through LDS, a round trip a token.  With the rows in many splits (few
// sequences, then) the workgroups are large, so that all of a tree's are read at once.  Latency: 2.6 us for a tree
// of 64 nodes and 16 splits, 3.2 for 256 trees whose targets are given.
constexpr int kAcceptThreads = 256, kAcceptMost = 1024;
__global__ __launch_bounds__(kAcceptMost) void accept_tree_kernel(AcceptArgs a) {
  __shared__ int32_t target[kMaxTreeNodes], child[kMaxTreeNodes], path[kMaxTreeNodes];
  __shared__ int32_t length;
  const int s = blockIdx.x, tid = threadIdx.x, threads = blockDim.x;
  const Tree t = tree_of(a.cu, s, a.num_nodes, a.max_nodes);
  // (The first node of a thread is asked for before its target is known.)
  const bool has = tid < t.nodes;
  const int parent0 = has ? a.parents[t.first + tid] : -1, draft0 = has ? a.draft[t.first + tid] : 0;
  if (a.best && a.splits > 1) {
    // 16 lanes to a node.
    const int sub = tid & 15;
    for (int j0 = 0; j0 < t.nodes; j0 += threads / 16) {
      const int j = j0 + (tid >> 4);
      uint64_t key = 0;
      if (j < t.nodes) {
        for (int i = sub; i < a.splits; i += 16) key = max(key, a.best[(int64_t)(t.first + j) * a.splits + i]);
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) {
        const uint64_t other = __shfl_xor((unsigned long long)key, o, kWave);
        key = other > key ? other : key;
      }
      if (sub == 0 && j < t.nodes) target[j] = a.target[t.first + j] = token_of(key);
    }
  } else if (a.best) {
    for (int j = tid; j < t.nodes; j += threads) target[j] = a.target[t.first + j] = token_of(a.best[t.first + j]);
  } else {
    for (int j = tid; j < t.nodes; j += threads) target[j] = a.target[t.first + j];
  }
  for (int j = tid; j < t.nodes; j += threads) child[j] = t.nodes;
  __syncthreads();
  for (int j = tid; j < t.nodes; j += threads) {
    const int p = j == tid ? parent0 : a.parents[t.first + j];
    if (p >= 0 && p < j && (j == tid ? draft0 : a.draft[t.first + j]) == target[p]) atomicMin(&child[p], j);
  }
  __syncthreads();
  if (tid == 0) {
    int n = 0, last = 0;
    for (int j = 0; j < t.nodes && n < a.max_accepted; j = child[j]) path[n++] = last = j;
    length = n;
    a.count[s] = n;
    a.next[s] = t.nodes > 0 ? target[last] : -1;
  }
  __syncthreads();
  for (int i = tid; i < a.max_accepted; i += threads) {
    a.accepted[(int64_t)s * a.max_accepted + i] = i < length ? path[i] : -1;
  }
}

// One split per 16 KB of a row and more while the rows alone do not fill the chip.
int32_t argmax_splits(int32_t num_nodes, int32_t vocab) {
  const int64_t want = ceil_div(4 * (int64_t)device_cu_count(), std::max(num_nodes, 1));
  return (int32_t)std::max<int64_t>(1, std::min<int64_t>({want, ceil_div(vocab, 4096), 64}));
}

// -------------------------------------------------------------- compaction --

struct CompactArgs {
  void* k;
  void* v;
  float* scores;
  const int32_t* table;
  const int32_t* context_lens;
  const int32_t* cu;
  const int32_t* accepted;
  const int32_t* count;
  int32_t* new_lens;
  int64_t layer_stride, kv_stride, score_layer_stride, score_stride;  // kv: in pieces
  int32_t num_nodes, max_accepted, num_kv_heads, block_size, max_blocks;
};

// Workgroup (sequence, layer).  The places of up to kMoveTokens moving tokens are looked up by as many threads; then
// a thread has one piece of a token's rows (K or V, kv-head, place in the row) and takes it from every one of them,
// kMoveAhead at a time: what a token's move overwrites is read by the same thread, before.  (The accepted list rises,
// so a later group's sources lie above what an earlier one wrote.)  Latency: list, table, rows; 64 sequences in 16
// layers, 5.4 MB, 6.7 us, a layer or two of 3 sequences 3.8.
constexpr int kMoveThreads = 256;
constexpr int kMoveTokens = 64;
constexpr int kMoveAhead = 8;
template <typename V>
__global__ __launch_bounds__(kMoveThreads) void compact_tree_kernel(CompactArgs a, int row_pieces) {
  __shared__ int64_t kv_from[kMoveTokens], kv_to[kMoveTokens], score_from[kMoveTokens], score_to[kMoveTokens];
  const int s = blockIdx.x, tid = threadIdx.x;
  const int64_t layer = blockIdx.y;
  const Tree t = tree_of(a.cu, s, a.num_nodes, INT32_MAX);
  const int ctx = max(0, min(a.context_lens[s], a.max_blocks * a.block_size));
  const int prior = max(ctx - t.len, 0);
  const int here = ctx - prior;  // nodes that are in the cache
  const int count = max(0, min(min(a.count[s], a.max_accepted), here));
  if (layer == 0 && tid == 0 && a.new_lens) a.new_lens[s] = prior + count;
  const int32_t* list = a.accepted + (int64_t)s * a.max_accepted;
  const int32_t* row = a.table + (int64_t)s * a.max_blocks;
  const int per_cache = a.num_kv_heads * row_pieces;
  V* const kb = static_cast<V*>(a.k) + layer * a.layer_stride;
  V* const vb = static_cast<V*>(a.v) + layer * a.layer_stride;
  float* const sb = a.scores + layer * a.score_layer_stride;
  for (int i0 = 0; i0 < count; i0 += kMoveTokens) {
    const int n = min(kMoveTokens, count - i0);
    if (tid < n) {
      const int i = i0 + tid, node = list[i];
      int64_t from = -1;
      if (node >= 0 && node < here && node != i) {
        const int src = prior + node, dst = prior + i;
        const int64_t sblk = row[src / a.block_size], dblk = row[dst / a.block_size];
        from = sblk * a.kv_stride + (int64_t)(src % a.block_size) * row_pieces;
        kv_to[tid] = dblk * a.kv_stride + (int64_t)(dst % a.block_size) * row_pieces;
        score_from[tid] = sblk * a.score_stride + src % a.block_size;
        score_to[tid] = dblk * a.score_stride + dst % a.block_size;
      }
      kv_from[tid] = from;
    }
    __syncthreads();
    for (int c = tid; c < 2 * per_cache; c += kMoveThreads) {
      const int in = c < per_cache ? c : c - per_cache;
      const int h = in / row_pieces;
      V* const base = (c < per_cache ? kb : vb) + (int64_t)h * a.block_size * row_pieces + (in - h * row_pieces);
      for (int g = 0; g < n; g += kMoveAhead) {
        V piece[kMoveAhead];
#pragma unroll
        for (int u = 0; u < kMoveAhead; ++u)
          if (g + u < n && kv_from[g + u] >= 0) piece[u] = base[kv_from[g + u]];
#pragma unroll
        for (int u = 0; u < kMoveAhead; ++u)
          if (g + u < n && kv_from[g + u] >= 0) base[kv_to[g + u]] = piece[u];
      }
    }
    if (a.scores) {
      for (int h = tid; h < a.num_kv_heads; h += kMoveThreads) {
        float* const base = sb + h * a.block_size;
        for (int g = 0; g < n; g += kMoveAhead) {
          float x[kMoveAhead];
#pragma unroll
          for (int u = 0; u < kMoveAhead; ++u)
            if (g + u < n && kv_from[g + u] >= 0) x[u] = base[score_from[g + u]];
#pragma unroll
          for (int u = 0; u < kMoveAhead; ++u)
            if (g + u < n && kv_from[g + u] >= 0) base[score_to[g + u]] = x[u];
        }
      }
    }
    __syncthreads();
  }
}

bool overlap(const void* a, size_t an, const void* b, size_t bn) {
  const auto x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + bn && y < x + an;
}

// What the verification's two entries check alike.
int check_accept(const char* op, int32_t num_seqs, int32_t num_nodes, int32_t max_nodes, int32_t max_accepted) {
  if (num_seqs < 0 || num_nodes < 0 || max_accepted < 1) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: need num_seqs and num_nodes >= 0 and max_accepted >= 1, got %d, %d, %d",
                op, num_seqs, num_nodes, max_accepted);
  }
  return check_tree_nodes(op, max_nodes);
}

int run_accept(const char* op, const AcceptArgs& a, int32_t num_seqs, hipStream_t s) {
  hipLaunchKernelGGL(accept_tree_kernel, dim3((unsigned)num_seqs), dim3(a.splits > 1 ? kAcceptMost : kAcceptThreads), 0, s,
                     a);
  return check_launch(op);
}

}  // namespace

int check_tree_nodes(const char* op, int32_t max_nodes) {
  if (max_nodes < 0) return fail(RG_ERR_INVALID_ARGUMENT, "%s: max_nodes %d is negative", op, max_nodes);
  if (max_nodes > kMaxTreeNodes) {
    return fail(RG_ERR_NOT_SUPPORTED, "%s: trees of up to %d nodes, got %d", op, kMaxTreeNodes, max_nodes);
  }
  return RG_OK;
}

int probe_tree_kernels() {
  hipFuncAttributes at;
  if (hipFuncGetAttributes(&at, reinterpret_cast<const void*>(tree_layout_kernel)) != hipSuccess ||
      hipFuncGetAttributes(&at, reinterpret_cast<const void*>(argmax_kernel<bf16_t>)) != hipSuccess ||
      hipFuncGetAttributes(&at, reinterpret_cast<const void*>(accept_tree_kernel)) != hipSuccess ||
      hipFuncGetAttributes(&at, reinterpret_cast<const void*>(compact_tree_kernel<rg_u32x4_t>)) != hipSuccess) {
    return fail(RG_ERR_HIP, "failed to load the tree kernels: %s", hipGetErrorString(hipGetLastError()));
  }
  return RG_OK;
}

}  // namespace rg

using namespace rg;

extern "C" int rg_tree_layout(const int32_t* parents, const int32_t* cu_nodes, const int32_t* context_lens,
                              const int32_t* block_table, const int32_t* text_positions, int32_t* tree_mask,
                              int32_t* positions, int32_t* slot_mapping, int32_t block_size,
                              int32_t max_blocks_per_seq, int32_t num_seqs, int32_t num_nodes, int32_t max_nodes,
                              int32_t mask_words, void* stream) {
  const char* op = "tree_layout";
  int st = check_tree_nodes(op, max_nodes);
  if (st != RG_OK) return st;
  if (num_seqs < 0 || num_nodes < 0 || block_size <= 0 || max_blocks_per_seq < 0) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: need num_seqs, num_nodes and max_blocks_per_seq >= 0 and block_size > 0",
                op);
  }
  if (mask_words < ceil_div(max_nodes, 32) || mask_words > kMaxTreeNodes / 32) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: mask_words %d for trees of %d nodes (at most %d)", op, mask_words,
                max_nodes, kMaxTreeNodes / 32);
  }
  if ((int64_t)max_blocks_per_seq * block_size > INT32_MAX) {
    return fail(RG_ERR_NOT_SUPPORTED, "%s: a block table of %lld tokens", op, (long long)max_blocks_per_seq * block_size);
  }
  if (num_seqs == 0 || num_nodes == 0 || max_nodes == 0) return ok();
  if (!parents || !cu_nodes || !context_lens || !block_table || !tree_mask || !positions || !slot_mapping) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: null pointer argument", op);
  }
  const LayoutArgs a{parents,   cu_nodes,  context_lens, block_table, text_positions, tree_mask,         positions,
                     slot_mapping, num_nodes, max_nodes,    mask_words,  block_size,     max_blocks_per_seq};
  hipLaunchKernelGGL(tree_layout_kernel, dim3((unsigned)num_seqs, (unsigned)ceil_div(mask_words, kLayoutWords)),
                     dim3(kLayoutThreads), 0, as_stream(stream), a);
  return check_launch(op);
}

extern "C" size_t rg_verify_tree_workspace_bytes(int32_t num_nodes, int32_t vocab_size) {
  if (num_nodes <= 0 || vocab_size <= 0) return 0;
  return (size_t)num_nodes * argmax_splits(num_nodes, vocab_size) * sizeof(uint64_t);
}

extern "C" int rg_verify_tree(const void* logits, const int32_t* draft_tokens, const int32_t* parents,
                              const int32_t* cu_nodes, int32_t* target_tokens, int32_t* accepted,
                              int32_t* num_accepted, int32_t* next_tokens, int32_t num_seqs, int32_t num_nodes,
                              int32_t max_nodes, int32_t max_accepted, int32_t vocab_size, int32_t dtype,
                              int64_t logits_row_stride, void* workspace, size_t workspace_bytes, void* stream) {
  const char* op = "verify_tree";
  int st = check_accept(op, num_seqs, num_nodes, max_nodes, max_accepted);
  if (st != RG_OK) return st;
  const int eb = dtype_bytes(dtype);
  if (eb == 0) return fail(RG_ERR_NOT_SUPPORTED, "%s: unknown dtype %d", op, dtype);
  if (vocab_size <= 0 || logits_row_stride < vocab_size) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: need a vocabulary and rows of it, got %d and a row stride of %lld", op,
                vocab_size, (long long)logits_row_stride);
  }
  if (num_seqs == 0) return ok();
  if (!cu_nodes || !accepted || !num_accepted || !next_tokens ||
      (num_nodes > 0 && (!logits || !draft_tokens || !parents || !target_tokens))) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: null pointer argument", op);
  }
  if (reinterpret_cast<uintptr_t>(logits) % eb != 0) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: logits are not aligned to their type", op);
  }
  const size_t need = rg_verify_tree_workspace_bytes(num_nodes, vocab_size);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 7u) != 0)) {
    return fail(RG_ERR_WORKSPACE, "%s: workspace of %zu bytes (8-byte aligned), %zu required", op,
                workspace ? workspace_bytes : (size_t)0, need);
  }
  hipStream_t s = as_stream(stream);
  const AcceptArgs a{static_cast<uint64_t*>(workspace), target_tokens, draft_tokens, parents, cu_nodes, accepted,
                     num_accepted, next_tokens, num_nodes, max_nodes, max_accepted, argmax_splits(num_nodes, vocab_size)};
  if (num_nodes > 0) {
    st = dispatch_dtype(dtype, [&](auto tag) {
      using T = decltype(tag);
      hipLaunchKernelGGL(argmax_kernel<T>, dim3((unsigned)num_nodes, (unsigned)a.splits), dim3(kArgmaxThreads), 0, s,
                         static_cast<const typename elem<T>::storage*>(logits), logits_row_stride, vocab_size, a.splits,
                         cu_nodes, num_seqs, static_cast<uint64_t*>(workspace));
      return check_launch(op);
    });
    if (st != RG_OK) return st;
  }
  return run_accept(op, a, num_seqs, s);
}

extern "C" int rg_accept_tree(const int32_t* target_tokens, const int32_t* draft_tokens, const int32_t* parents,
                              const int32_t* cu_nodes, int32_t* accepted, int32_t* num_accepted, int32_t* next_tokens,
                              int32_t num_seqs, int32_t num_nodes, int32_t max_nodes, int32_t max_accepted,
                              void* stream) {
  const char* op = "accept_tree";
  int st = check_accept(op, num_seqs, num_nodes, max_nodes, max_accepted);
  if (st != RG_OK) return st;
  if (num_seqs == 0) return ok();
  if (!cu_nodes || !accepted || !num_accepted || !next_tokens ||
      (num_nodes > 0 && (!target_tokens || !draft_tokens || !parents))) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: null pointer argument", op);
  }
  const AcceptArgs a{nullptr, const_cast<int32_t*>(target_tokens), draft_tokens, parents, cu_nodes, accepted,
                     num_accepted, next_tokens, num_nodes, max_nodes, max_accepted, 0};
  return run_accept(op, a, num_seqs, as_stream(stream));
}

extern "C" int rg_compact_tree(void* key_cache, void* value_cache, float* scores, const int32_t* block_table,
                               const int32_t* context_lens, const int32_t* cu_nodes, const int32_t* accepted,
                               const int32_t* num_accepted, int32_t* new_context_lens, int32_t max_accepted,
                               int32_t num_layers, int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                               int32_t max_blocks_per_seq, int32_t num_seqs, int32_t num_nodes, int32_t dtype,
                               int64_t layer_stride, int64_t kv_block_stride, int64_t score_layer_stride,
                               int64_t score_block_stride, void* stream) {
  const char* op = "compact_tree";
  const int eb = dtype_bytes(dtype);
  if (eb == 0) return fail(RG_ERR_NOT_SUPPORTED, "%s: unknown dtype %d", op, dtype);
  if (head_dim <= 0 || head_dim > RG_MAX_HEAD_DIM) {
    return fail(RG_ERR_NOT_SUPPORTED, "%s: head_dim must be in 1 .. %d, got %d", op, RG_MAX_HEAD_DIM, head_dim);
  }
  if (num_layers < 0 || num_seqs < 0 || num_nodes < 0 || num_kv_heads <= 0 || block_size <= 0 ||
      max_blocks_per_seq < 0 || max_accepted < 1) {
    return fail(RG_ERR_INVALID_ARGUMENT,
                "%s: need layers, sequences, nodes and table width >= 0 and positive heads, block_size and max_accepted",
                op);
  }
  const int64_t block = (int64_t)num_kv_heads * block_size;
  const int64_t kv_stride = kv_block_stride ? kv_block_stride : block * head_dim;
  const int64_t score_stride = score_block_stride ? score_block_stride : block;
  if (kv_stride < block * head_dim || (scores && score_stride < block)) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: kv_block_stride %lld or score_block_stride %lld smaller than a block", op,
                (long long)kv_stride, (long long)score_stride);
  }
  if (num_layers > 1 && (layer_stride <= 0 || (scores && score_layer_stride <= 0))) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: layer strides must be positive with num_layers > 1", op);
  }
  if ((int64_t)max_blocks_per_seq * block_size > INT32_MAX || block * head_dim > INT32_MAX / 2) {
    return fail(RG_ERR_NOT_SUPPORTED, "%s: a block table of %lld tokens, a block of %lld elements", op,
                (long long)max_blocks_per_seq * block_size, (long long)(block * head_dim));
  }
  if (num_layers > 65535) return fail(RG_ERR_NOT_SUPPORTED, "%s: %d layers", op, num_layers);
  if (num_layers == 0 || num_seqs == 0) return ok();
  if (!key_cache || !value_cache || !block_table || !context_lens || !cu_nodes || !accepted || !num_accepted) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: null pointer argument", op);
  }
  // (Every layer's workgroups read the lengths and the table while the new lengths are written.)
  const size_t entries = 4 * (size_t)num_seqs;
  if (new_context_lens != nullptr && (overlap(new_context_lens, entries, context_lens, entries) ||
                                      overlap(new_context_lens, entries, num_accepted, entries) ||
                                      overlap(new_context_lens, entries, accepted, entries * max_accepted) ||
                                      overlap(new_context_lens, entries, cu_nodes, entries + 4) ||
                                      overlap(new_context_lens, entries, block_table, entries * max_blocks_per_seq))) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: new_context_lens overlaps an input", op);
  }
  const int64_t layers_apart = num_layers > 1 ? layer_stride : 0;
  auto whole = [&](int64_t elements) { return elements * eb % 16 == 0; };
  const bool wide = whole(head_dim) && whole(kv_stride) && whole(layers_apart) &&
                    ((reinterpret_cast<uintptr_t>(key_cache) | reinterpret_cast<uintptr_t>(value_cache)) & 15u) == 0;
  const int piece = wide ? 16 : 2;
  const CompactArgs a{key_cache, value_cache, scores, block_table, context_lens, cu_nodes, accepted, num_accepted,
                      new_context_lens, layers_apart * eb / piece, kv_stride * eb / piece,
                      num_layers > 1 ? score_layer_stride : 0, score_stride, num_nodes, max_accepted, num_kv_heads,
                      block_size, max_blocks_per_seq};
  const dim3 grid((unsigned)num_seqs, (unsigned)num_layers);
  const int row_pieces = head_dim * eb / piece;
  if (wide) hipLaunchKernelGGL(compact_tree_kernel<rg_u32x4_t>, grid, dim3(kMoveThreads), 0, as_stream(stream), a, row_pieces);
  else hipLaunchKernelGGL(compact_tree_kernel<uint16_t>, grid, dim3(kMoveThreads), 0, as_stream(stream), a, row_pieces);
  return check_launch(op);
}
