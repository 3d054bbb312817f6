// Eviction from the paged KV cache by accumulated attention weight.
//
// A segment is one (layer, sequence, kv-head) with n cached tokens, each with an fp32 score in
// `scores` (paged like the cache).  Past the budget it keeps
//   K = { t < protected } + { t >= n - recent } + the (budget - protected - recent) others of the
//       highest score, a tie going to the lower position,
// and the kept rows of K and V and the kept scores move, in the order of their positions, to
// positions 0 .. |K| - 1 of the destination table.
//
// evict_select_kernel (one workgroup per segment) finds the threshold: scores become 32-bit keys in
// the order of the values, and three passes over 11, 11 and 10 bits narrow the key T of the last one
// to be kept, each with a histogram in LDS over the candidates that agree with the bits found so
// far.  A kept candidate's place is then known without a list: before position t lie
//   #{key > T before t} + min(#{key == T before t}, ties to keep)
// kept candidates.  It leaves the kept positions in order (the caller's array, or workspace).
// evict_move_kernel copies: what a segment has to move is cut into chunks, a workgroup each.
#include <algorithm>

#include "rg_common.hpp"

namespace rg {
namespace {

struct EvictArgs {
  void* k;
  void* v;
  float* scores;
  const int32_t* table;
  const int32_t* dst_table;
  const int32_t* context_lens;
  int32_t* new_lens;  // may be null
  int32_t* kept;      // [segments, kept_stride]: the kept positions in order, -1 behind them
  int32_t* in_order;  // [segments]: 1 where a chunk's destination may hold rows still to be read
  int64_t layer_stride, kv_stride, score_layer_stride, score_stride;  // elements
  int32_t kept_stride, budget, recent, guarded;
  int32_t num_kv_heads, head_dim, block_size, max_blocks, max_dst_blocks, batch;
};

struct Segment {
  int layer, seq, kvh;
};
__device__ __forceinline__ Segment segment_of(const EvictArgs& a, int64_t i) {
  Segment s;
  s.kvh = (int)(i % a.num_kv_heads);
  i /= a.num_kv_heads;
  s.seq = (int)(i % a.batch);
  s.layer = (int)(i / a.batch);
  return s;
}
// Contexts longer than the block table's row are clamped to it, negative ones to 0.
__device__ __forceinline__ int context_of(const EvictArgs& a, int seq) {
  return max(0, (int)min<int64_t>(a.context_lens[seq], (int64_t)a.max_blocks * a.block_size));
}
// Cell of (segment, block, offset in the block) in `scores`.
__device__ __forceinline__ int64_t score_cell(const EvictArgs& a, const Segment& s, int64_t blk, int off) {
  return s.layer * a.score_layer_stride + blk * a.score_stride + (int64_t)s.kvh * a.block_size + off;
}

// Unsigned keys in the order of the scores: -0 equals +0, a NaN ranks as -inf.
__device__ __forceinline__ uint32_t order_key(float f) {
  uint32_t u = __float_as_uint(f);
  if ((u & 0x7fffffffu) > 0x7f800000u) u = 0xff800000u;
  if (u == 0x80000000u) u = 0u;
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;
constexpr int kSelBins = 2048;
constexpr int kSelHeldMost = 32768;  // keys held in LDS: 128 KB beside the 16.5 KB of the tables
constexpr int kSelGroup = 64;  // strips of kSelThreads candidates whose counts are scanned together

// Inclusive prefix sum over the wave, and the exclusive one over the workgroup's threads
// (part: kSelWaves words of LDS; ends behind a barrier).
__device__ __forceinline__ int wave_scan(int v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int t = __shfl_up(v, o, 64);
    if (lane >= o) v += t;
  }
  return v;
}
__device__ __forceinline__ int block_scan_excl(int v, int lane, int w, int* part) {
  const int incl = wave_scan(v, lane);
  if (lane == 63) part[w] = incl;
  __syncthreads();
  int before = 0;
  for (int i = 0; i < w; ++i) before += part[i];
  return before + incl - v;
}

// HELD: the candidates' keys are held in LDS (dynamic, one word each), so the scores are read once;
// longer tables read them again in each pass.
template <bool HELD>
__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(EvictArgs a) {
  extern __shared__ uint32_t held[];
  __shared__ int hist[kSelBins];
  __shared__ int part[kSelWaves];
  __shared__ int found[2];               // digit, candidates above it
  __shared__ int strip[2][kSelThreads];  // per (strip, wave): candidates above T, candidates at T
  __shared__ int first_hole, alias;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const Segment sg = segment_of(a, blockIdx.x);
  const int n = context_of(a, sg.seq);
  const int m = min(n, a.budget);
  int32_t* kept = a.kept + (int64_t)blockIdx.x * a.kept_stride;
  const int32_t* row = a.table + (int64_t)sg.seq * a.max_blocks;
  if (a.new_lens != nullptr && sg.layer == 0 && sg.kvh == 0 && tid == 0) a.new_lens[sg.seq] = m;
  for (int i = m + tid; i < a.kept_stride; i += kSelThreads) kept[i] = -1;
  if (n <= a.budget) {
    for (int i = tid; i < n; i += kSelThreads) kept[i] = i;
    if (tid == 0) a.in_order[blockIdx.x] = 0;
    return;
  }
  const int p0 = a.guarded;
  const int count = n - a.recent - p0;           // candidates, positions p0 ..
  const int take = a.budget - a.recent - p0;     // of which this many stay: 0 <= take < count
  for (int i = tid; i < p0; i += kSelThreads) kept[i] = i;
  for (int i = tid; i < a.recent; i += kSelThreads) kept[m - a.recent + i] = n - a.recent + i;
  if (tid == 0) {
    first_hole = n;
    alias = 0;
  }

  auto read_key = [&](int c) -> uint32_t {
    const int p = p0 + c;
    return order_key(a.scores[score_cell(a, sg, row[p / a.block_size], p % a.block_size)]);
  };
  // (A thread reads back only keys that it wrote itself.)
  if constexpr (HELD) {
    // (A table entry, then the score it leads to: two round trips, shared by eight candidates.)
    for (int c0 = tid; c0 < count; c0 += 8 * kSelThreads) {
      uint32_t k[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) k[i] = read_key(min(c0 + i * kSelThreads, count - 1));
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (c0 + i * kSelThreads < count) held[c0 + i * kSelThreads] = k[i];
      }
    }
  }
  auto key_at = [&](int c) -> uint32_t {
    if constexpr (HELD) return held[c];
    else return read_key(c);
  };

  // T: the key of the take-th largest candidate; `left` of those at T are kept.
  uint32_t T = 0xffffffffu;  // (above every key: nothing kept)
  int left = 0;
  if (take > 0) {
    T = 0;
    left = take;
    const int shifts[3] = {21, 10, 0};
#pragma unroll
    for (int ps = 0; ps < 3; ++ps) {
      const int sh = shifts[ps];
      const uint32_t bins = ps == 2 ? 1024u : 2048u;
      for (int i = tid; i < kSelBins; i += kSelThreads) hist[i] = 0;
      __syncthreads();
      const int hi = ps == 0 ? 32 : shifts[ps - 1];  // bits from here on are settled
      for (int c = tid; c < count; c += kSelThreads) {
        const uint32_t k = key_at(c);
        if (ps == 0 || (k >> hi) == (T >> hi)) atomicAdd(&hist[(k >> sh) & (bins - 1)], 1);
      }
      __syncthreads();
      // Candidates in bins above, two bins a thread from the top.
      const int b1 = kSelBins - 1 - 2 * tid, b0 = b1 - 1;
      const int h1 = hist[b1], h0 = hist[b0];
      const int above = block_scan_excl(h1 + h0, lane, w, part);
      if (above < left && left <= above + h1) {
        found[0] = b1;
        found[1] = above;
      } else if (above + h1 < left && left <= above + h1 + h0) {
        found[0] = b0;
        found[1] = above + h1;
      }
      __syncthreads();
      T |= (uint32_t)found[0] << sh;
      left -= found[1];
      __syncthreads();
    }
  }

  // The kept candidates in order.  Strip i holds candidates i * kSelThreads ..; the counts of
  // every (strip, wave) of a group go to LDS and are scanned at once.
  int gt_before = 0, eq_before = 0;  // in the groups before
  const int strips = (count + kSelThreads - 1) / kSelThreads;
  int hole = n;
  for (int g0 = 0; g0 < strips; g0 += kSelGroup) {
    const int gs = min(kSelGroup, strips - g0);
    __syncthreads();
    for (int i = 0; i < gs; ++i) {
      const int c = (g0 + i) * kSelThreads + tid;
      const bool in = c < count;
      const uint32_t k = in ? key_at(c) : 0u;
      const int gt = __popcll(__ballot(in && k > T)), eq = __popcll(__ballot(in && k == T));
      if (lane == 0) {
        strip[0][i * kSelWaves + w] = gt;
        strip[1][i * kSelWaves + w] = eq;
      }
    }
    __syncthreads();
    const bool have = tid < gs * kSelWaves;
    const int gt = have ? strip[0][tid] : 0, eq = have ? strip[1][tid] : 0;
    const int gt_ex = block_scan_excl(gt, lane, w, part);
    int gt_all = 0;
    for (int i = 0; i < kSelWaves; ++i) gt_all += part[i];
    __syncthreads();
    const int eq_ex = block_scan_excl(eq, lane, w, part);
    int eq_all = 0;
    for (int i = 0; i < kSelWaves; ++i) eq_all += part[i];
    strip[0][tid] = gt_before + gt_ex;
    strip[1][tid] = eq_before + eq_ex;
    __syncthreads();
    auto below = [&](uint64_t x) {
      return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(x >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)x, 0));
    };
    for (int i = 0; i < gs; ++i) {
      const int c = (g0 + i) * kSelThreads + tid;
      const bool in = c < count;
      const uint32_t k = in ? key_at(c) : 0u;
      const bool is_gt = in && k > T, is_eq = in && k == T;
      const int g = strip[0][i * kSelWaves + w] + below(__ballot(is_gt));
      const int e = strip[1][i * kSelWaves + w] + below(__ballot(is_eq));
      if (is_gt || (is_eq && e < left)) kept[p0 + g + min(e, left)] = p0 + c;
      else if (in) hole = min(hole, p0 + c);
    }
    gt_before += gt_all;
    eq_before += eq_all;
  }
  // Rows from the first hole on move.  Where a block that receives them is also the block they may
  // come from (the same entry of both tables: eviction in place), the chunks go in order.
  atomicMin(&first_hole, hole);
  __syncthreads();
  const int32_t* drow = a.dst_table + (int64_t)sg.seq * a.max_dst_blocks;
  for (int i = first_hole / a.block_size + tid; i < (m + a.block_size - 1) / a.block_size; i += kSelThreads) {
    if (row[i] == drow[i]) alias = 1;
  }
  __syncthreads();
  if (tid == 0) a.in_order[blockIdx.x] = alias;
}

// ----------------------------------------------------------------- move -----

constexpr int kMoveThreads = 256;
constexpr int kMoveUnroll = 8;     // V-sized pieces of K and V a thread holds
constexpr int kMoveMaxTokens = 128;

// Workgroup (chunk, segment): tokens chunk * TOK .. of the segment's kept list, TOK such that its K
// and V rows fill kMoveUnroll pieces a thread, all of them read before the first is written.  A
// segment that is evicted in place is walked by its first workgroup alone: the chunk at hand is
// written once every thread has read its part of it.  That is enough: kept[j] >= j, so rows
// j .. of the destination never hold a row that a later chunk has yet to read.
template <typename V>
__global__ __launch_bounds__(kMoveThreads, 4) void evict_move_kernel(EvictArgs a, int row_vecs, int tok) {
  __shared__ int64_t src_off[2][kMoveMaxTokens], dst_off[2][kMoveMaxTokens];  // in pieces V; -1: not moved
  const int tid = threadIdx.x;
  const Segment sg = segment_of(a, blockIdx.x);
  const int m = min(context_of(a, sg.seq), a.budget);
  const bool in_order = a.in_order[blockIdx.x] != 0;
  if (in_order && blockIdx.y != 0) return;
  const int32_t* kept = a.kept + (int64_t)blockIdx.x * a.kept_stride;
  const int32_t* row = a.table + (int64_t)sg.seq * a.max_blocks;
  const int32_t* drow = a.dst_table + (int64_t)sg.seq * a.max_dst_blocks;
  constexpr int kSize = (int)sizeof(V);
  const int64_t es = (int64_t)row_vecs * kSize / a.head_dim;  // element bytes
  V* const kb = static_cast<V*>(a.k);
  V* const vb = static_cast<V*>(a.v);
  const int64_t layer = sg.layer * a.layer_stride, head = (int64_t)sg.kvh * a.block_size;
  const int per_token = 2 * row_vecs;
  for (int j0 = (int)blockIdx.y * tok, buf = 0; j0 < m; j0 += tok, buf ^= 1) {
    const int nt = min(tok, m - j0);
    float score = 0.f;
    int64_t to_cell = -1;
    if (tid < nt) {
      const int j = j0 + tid, p = kept[j];
      const int64_t sb = row[p / a.block_size], db = drow[j / a.block_size];
      const int so = p % a.block_size, to = j % a.block_size;
      const bool moved = sb != db || so != to;
      src_off[buf][tid] = moved ? (layer + sb * a.kv_stride + (head + so) * a.head_dim) * es / kSize : -1;
      dst_off[buf][tid] = (layer + db * a.kv_stride + (head + to) * a.head_dim) * es / kSize;
      if (moved) {
        score = a.scores[score_cell(a, sg, sb, so)];
        to_cell = score_cell(a, sg, db, to);
      }
    }
    __syncthreads();
    V piece[kMoveUnroll] = {};
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u) {
      const int i = u * kMoveThreads + tid, t = i / per_token, c = i - t * per_token;
      if (t < nt && src_off[buf][t] >= 0) {
        const int64_t at = src_off[buf][t];
        piece[u] = *((c >= row_vecs ? vb - row_vecs : kb) + at + c);
      }
    }
    if (in_order) {
      // Every thread's reads have landed before any thread writes.
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u) {
      const int i = u * kMoveThreads + tid, t = i / per_token, c = i - t * per_token;
      if (t < nt && src_off[buf][t] >= 0) {
        const int64_t at = dst_off[buf][t];
        *((c >= row_vecs ? vb - row_vecs : kb) + at + c) = piece[u];
      }
    }
    if (to_cell >= 0) a.scores[to_cell] = score;
    if (!in_order) break;
  }
}

// Segments of the call, -1 past what one launch numbers.
int64_t segment_count(int32_t num_layers, int32_t batch, int32_t num_kv_heads) {
  const int64_t pairs = (int64_t)num_layers * batch;
  return pairs <= INT32_MAX && pairs * num_kv_heads <= INT32_MAX ? pairs * num_kv_heads : -1;
}
size_t evict_bytes(int64_t segments, int64_t budget, bool own_list) {
  return align_up((size_t)segments * 4, 256) + (own_list ? align_up((size_t)segments * (size_t)budget * 4, 256) : 0);
}

}  // namespace

int probe_evict_kernels() {
  hipFuncAttributes at;
  if (hipFuncGetAttributes(&at, reinterpret_cast<const void*>(evict_select_kernel<true>)) != hipSuccess ||
      hipFuncGetAttributes(&at, reinterpret_cast<const void*>(evict_move_kernel<rg_u32x4_t>)) != hipSuccess) {
    return fail(RG_ERR_HIP, "failed to load the eviction kernels: %s", hipGetErrorString(hipGetLastError()));
  }
  return RG_OK;
}

}  // namespace rg

using namespace rg;

extern "C" size_t rg_evict_cache_workspace_bytes(int32_t num_layers, int32_t batch_size, int32_t num_kv_heads,
                                                 int32_t budget) {
  if (num_layers <= 0 || batch_size <= 0 || num_kv_heads <= 0 || budget <= 0) return 0;
  const int64_t segments = segment_count(num_layers, batch_size, num_kv_heads);
  return segments < 0 ? 0 : evict_bytes(segments, budget, true);
}

extern "C" int rg_evict_cache(void* key_cache, void* value_cache, float* scores, const int32_t* block_table,
                              const int32_t* dst_block_table, const int32_t* context_lens,
                              int32_t* new_context_lens, int32_t* kept_positions, int32_t budget, int32_t recent,
                              int32_t protected_len, int32_t num_layers, int32_t num_kv_heads, int32_t head_dim,
                              int32_t block_size, int32_t max_blocks_per_seq, int32_t max_dst_blocks_per_seq,
                              int32_t batch_size, int32_t dtype, int64_t layer_stride, int64_t kv_block_stride,
                              int64_t score_layer_stride, int64_t score_block_stride, void* workspace,
                              size_t workspace_bytes, void* stream) {
  const char* op = "evict_cache";
  const int eb = dtype_bytes(dtype);
  if (eb == 0) return fail(RG_ERR_NOT_SUPPORTED, "%s: unknown dtype %d", op, dtype);
  if (head_dim <= 0 || head_dim > RG_MAX_HEAD_DIM) {
    return fail(RG_ERR_NOT_SUPPORTED, "%s: head_dim must be in 1 .. %d, got %d", op, RG_MAX_HEAD_DIM, head_dim);
  }
  if (num_layers < 0 || batch_size < 0 || num_kv_heads <= 0 || block_size <= 0 || max_blocks_per_seq < 0 ||
      max_dst_blocks_per_seq < 0) {
    return fail(RG_ERR_INVALID_ARGUMENT,
                "%s: need num_layers, batch and table widths >= 0 and positive heads and block_size", op);
  }
  if (budget < 1 || recent < 0 || protected_len < 0 || (int64_t)recent + protected_len > budget) {
    return fail(RG_ERR_INVALID_ARGUMENT,
                "%s: need budget >= 1 and recent + protected_len <= budget (both >= 0), got %d, %d, %d", op, budget,
                recent, protected_len);
  }
  const int64_t block = (int64_t)num_kv_heads * block_size;
  const int64_t kv_stride = kv_block_stride ? kv_block_stride : block * head_dim;
  const int64_t score_stride = score_block_stride ? score_block_stride : block;
  if (kv_stride < block * head_dim || score_stride < block) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: kv_block_stride %lld or score_block_stride %lld smaller than a block", op,
                (long long)kv_stride, (long long)score_stride);
  }
  if (num_layers > 1 && (layer_stride <= 0 || score_layer_stride <= 0)) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: layer strides must be positive with num_layers > 1", op);
  }
  const int64_t table_tokens = (int64_t)max_blocks_per_seq * block_size;
  if (table_tokens > INT32_MAX) {
    return fail(RG_ERR_NOT_SUPPORTED, "%s: a block table of %lld tokens", op, (long long)table_tokens);
  }
  const int64_t most = std::min<int64_t>(budget, table_tokens);  // tokens a segment keeps at most
  if (dst_block_table != nullptr && (int64_t)max_dst_blocks_per_seq * block_size < most) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: destination rows of %d blocks hold fewer than %lld tokens", op,
                max_dst_blocks_per_seq, (long long)most);
  }
  if (num_layers == 0 || batch_size == 0) return ok();
  if (!key_cache || !value_cache || !scores || !block_table || !context_lens) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: null pointer argument", op);
  }
  const int64_t segments = segment_count(num_layers, batch_size, num_kv_heads);
  if (segments < 0) {
    return fail(RG_ERR_NOT_SUPPORTED, "%s: more than %d (layer, sequence, kv-head) segments", op, INT32_MAX);
  }
  const size_t need = evict_bytes(segments, budget, kept_positions == nullptr);
  if (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 3u) != 0) {
    return fail(RG_ERR_WORKSPACE, "%s: workspace of %zu bytes (4-byte aligned), %zu required", op,
                workspace ? workspace_bytes : (size_t)0, need);
  }
  EvictArgs a{};
  a.k = key_cache;
  a.v = value_cache;
  a.scores = scores;
  a.table = block_table;
  a.dst_table = dst_block_table ? dst_block_table : block_table;
  a.context_lens = context_lens;
  a.new_lens = new_context_lens;
  a.in_order = static_cast<int32_t*>(workspace);
  a.kept = kept_positions ? kept_positions
                          : reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + align_up((size_t)segments * 4, 256));
  a.layer_stride = num_layers > 1 ? layer_stride : 0;
  a.kv_stride = kv_stride;
  a.score_layer_stride = num_layers > 1 ? score_layer_stride : 0;
  a.score_stride = score_stride;
  a.kept_stride = budget;
  a.budget = budget;
  a.recent = recent;
  a.guarded = protected_len;
  a.num_kv_heads = num_kv_heads;
  a.head_dim = head_dim;
  a.block_size = block_size;
  a.max_blocks = max_blocks_per_seq;
  a.max_dst_blocks = dst_block_table ? max_dst_blocks_per_seq : max_blocks_per_seq;
  a.batch = batch_size;
  hipStream_t s = as_stream(stream);
  const dim3 sel((unsigned)segments);
  if (table_tokens <= kSelHeldMost) {
    hipLaunchKernelGGL(evict_select_kernel<true>, sel, dim3(kSelThreads), (size_t)table_tokens * 4, s, a);
  } else {
    hipLaunchKernelGGL(evict_select_kernel<false>, sel, dim3(kSelThreads), 0, s, a);
  }
  int st = check_launch(op);
  if (st != RG_OK || most == 0) return st;
  // Rows move in 16-byte pieces where every row starts on one, else in 2-byte ones.
  auto whole = [&](int64_t elements) { return elements * eb % 16 == 0; };
  const bool wide = whole(head_dim) && whole(kv_stride) && whole(a.layer_stride) &&
                    ((reinterpret_cast<uintptr_t>(key_cache) | reinterpret_cast<uintptr_t>(value_cache)) & 15u) == 0;
  const int row_vecs = head_dim * eb / (wide ? 16 : 2);
  const int tok = std::max(1, std::min(kMoveMaxTokens, kMoveThreads * kMoveUnroll / (2 * row_vecs)));
  const int64_t chunks = ceil_div(most, tok);
  if (chunks > 65535) return fail(RG_ERR_NOT_SUPPORTED, "%s: a budget of %lld tokens", op, (long long)most);
  const dim3 grid((unsigned)segments, (unsigned)chunks);
  if (wide) {
    hipLaunchKernelGGL(evict_move_kernel<rg_u32x4_t>, grid, dim3(kMoveThreads), 0, s, a, row_vecs, tok);
  } else {
    hipLaunchKernelGGL(evict_move_kernel<uint16_t>, grid, dim3(kMoveThreads), 0, s, a, row_vecs, tok);
  }
  return check_launch(op);
}
