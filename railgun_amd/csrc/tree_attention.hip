// Attention of trees of drafted tokens over a paged KV cache.
//
// Node j of sequence s sits in the cache at position prior + j, prior = context_lens[s] - L.  It attends to the
// positions below prior and to those prior + i whose bit i its mask has set:
//   out = sum_t p_t V_t,  p = softmax(scale q.K_t) over those t;  zeros where there are none.
//
// The L G query rows of a sequence that share a kv-head (row r: node r / G, head r % G of the group) stand against the
// same K and V: an attention product on the matrix cores,
//   S^T = K Q^T,  running maximum and sum per row,  O^T += V^T P^T,
// in row tiles of kRows (32 a wave) and key tiles of kTileKeys.  Only the key tiles that reach into the tree are
// masked.  A (sequence, kv-head, row tile) segment is cut into equal pieces, as many as its length asks for so that the
// batch's pieces fill the chip, whatever the lengths: a workgroup each.  The row tiles of the same keys are neighbours,
// on one XCD at one time: the first to read a key tile brings it to the L2 for the others.  A segment of one piece is
// written out at once; of the others the pieces' softmax partials (m, l, unnormalised O) are joined by
// tree_merge_kernel:
//   M = max m_i,  out = sum 2^(m_i - M) O_i / sum 2^(m_i - M) l_i.
//
// Cells that a row does not attend to must not reach it, and 0 NaN is NaN in a matrix product.  In masked tiles V
// rows behind the context are cleared in LDS; where a tree's V holds something that is not finite it is cleared too,
// and added by hand to the rows that attend to it (which it makes that anyway).
#include "decode_stream.hpp"
#include "tree.hpp"

namespace rg {
namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short v4i16_t __attribute__((ext_vector_type(4)));

template <typename T> struct mfma32;
template <> struct mfma32<bf16_t> {
  __device__ static __forceinline__ f32x16_t run(uint4 a, uint4 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
  }
};
template <> struct mfma32<f16_t> {
  __device__ static __forceinline__ f32x16_t run(uint4 a, uint4 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0,
                                                  0, 0);
  }
};
// acc + lo + hi of a packed pair.
template <typename T> __device__ __forceinline__ float pair_sum(uint32_t pair, float acc);
template <> __device__ __forceinline__ float pair_sum<bf16_t>(uint32_t pair, float acc) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, pair), __builtin_bit_cast(bf16x2_t, 0x3F803F80u),
                                         acc, false);
}
template <> __device__ __forceinline__ float pair_sum<f16_t>(uint32_t pair, float acc) {
  return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, pair), __builtin_bit_cast(f16x2_t, 0x3C003C00u), acc,
                                false);
}

constexpr int kTreeWaves = 4;
constexpr int kTreeThreads = 64 * kTreeWaves;
constexpr int kRows = 32 * kTreeWaves;  // rows of a workgroup's tile, 32 a wave
constexpr int kTileKeys = 32;
constexpr float kSlack = 8.f;           // log2 headroom of the lazy maximum: 2^8 a probability at most

// What is subtracted from the scores of a row whose lazy maximum is m (log2 units): in fp16 the probabilities are
// held times 2^7.  Its normal numbers end at 2^-14, which one token's weight beside those of thousands falls below;
// times 2^7 they fill the type up to 2^(8 + 7).  Past 2^20 the fp32 scores' own steps grow towards the one factor of
// two that is left below 2^16; there they are held as they are.
template <typename T>
__device__ __forceinline__ float reference(float m) {
  if constexpr (std::is_same_v<T, f16_t>) return m - (fabsf(m) < 0x1p20f ? 7.f : 0.f);
  else return m;
}

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
  // The product's.
  float* acc;        // [parts, kRows, D] unnormalised
  float* ml;         // [parts, kRows, 2]: m in log2 units, l
  int2* cuts;        // [num_seqs]: the first of its parts, pieces of a segment
  uint32_t q_sign;   // bit 0: q is taken (else zeros, a scale of 0), bits 15 and 31: negated (a negative scale)
  int32_t group, bs_shift;
  int32_t slots, slots_full;  // pieces that a batch is cut into: as many as are at work together if they are long
  int32_t least;       // key tiles of a piece that is worth its partials
  int32_t long_piece;  // of one that is long
  int32_t short_piece; // of one that is too short for two a CU
  int32_t parts_past;  // partials of short pieces are written past the L2
};

// Any shape: a wave per (sequence, node, q-head), lane l has dims 4 l .. 4 l + 3, the keys one after the other with
// the running maximum m and sum l of their weights.  Bound by a key's chain of load, sum over the wave and exponential,
// 0.9 us for one of few waves: it is there to be right, and slower than a decode row per node, the more so the fewer of
// them there are.  Measured (ms; 32 / 8 heads in bf16): 256 dims, one sequence of 4,096 with 64 nodes 3.9 (plain torch
// operations 0.62, rg_paged_attention_v1 with a row per node 0.18), 64 of 512 to 4,096 with 8 to 32 nodes 21.7 (14.9,
// 4.0); 96 dims 3.6 (0.57, 0.82) and 22.8 (7.7, 21.8).
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


// The arguments, where the kernel has them, read when they are asked for: held in registers from the start, they and
// the state of the line are more than a wave has scalar ones.
typedef __attribute__((address_space(4))) TreeArgs Args;
__device__ __forceinline__ const Args& arguments() {
  const Args* p = (const Args*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *p;
}

// --------------------------------------------------------------- the cuts ---

// A sequence as the cuts see it.  Its context ends with the nodes that are asked for: a tree of more of them than
// max_nodes says has neither rows for the others nor keys.
struct Span {
  Tree t;
  int prior, ctx, tiles, row_tiles;
};
__device__ __forceinline__ Span span_of(const Args& a, int s) {
  Span p;
  p.t = tree_of(a.cu, s, a.num_nodes, a.max_nodes);
  const int cached = max(0, min(a.context_lens[s], a.max_blocks * a.block_size));
  p.prior = max(cached - p.t.len, 0);
  p.ctx = min(cached, p.prior + p.t.nodes);
  p.row_tiles = (p.t.nodes * a.group + kRows - 1) / kRows;
  // (A tree whose context is empty has one tile, without keys: its rows are cleared there.)
  p.tiles = max(1, (p.ctx + kTileKeys - 1) / kTileKeys);
  return p;
}
// Inclusive prefix sum over the 64 lanes: within each row of 16 lanes by shifts of 1, 2, 4 and 8, then lane 15 of rows
// 0 and 2 into rows 1 and 3, then lane 31 into rows 2 and 3.  Lanes whose source falls outside the row receive 0.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);  // row_shr:2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);  // row_shr:4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);  // row_shr:8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return v;
}
// Maximum over the 64 lanes of values not below 0, in lane 63.
__device__ __forceinline__ int wave_top(int v) {
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));
  return v;
}

// Pieces that a batch of so many segments is cut into at most: `slots`, or where the segments alone come near that or
// past it, half of it more than they are.  As many at most are parts of a segment: n cuts make 2 n parts.
__host__ __device__ inline int64_t most_pieces(int64_t segments, int64_t slots) {
  return segments <= slots * 3 / 4 ? slots : segments + slots / 2;
}

// Lengths of pieces, by quarters of the longest: where no two workgroups read the same keys, the long ones come first.
constexpr int kLengths = 4;

struct CutScratch {
  uint32_t spans[kTreeThreads];  // tiles, row tiles of up to so many sequences
  int32_t sums[kTreeWaves][64];
  int32_t wave_sum[1 + kLengths][kTreeWaves];
  // The workgroup's: its sequence; of that, the piece, pieces of a segment, the first part.
  int32_t seq, local, pieces, base;
  Span span;
};

// x / d rounded up, 0 < x, d < 2^22, by = 1 / d: the quotient in fp32 is off by less than one either way.
__device__ __forceinline__ int ceil_quotient(int x, int d, float by) {
  int q = (int)((float)x * by);
  q += (int)__umul24(q, d) < x;
  q += (int)__umul24(q, d) < x;
  return q - ((int)__umul24(q - 1, d) >= x);
}

// Key tiles of a piece from which on the chip is filled with them; of shorter ones two go to a CU, whose start and
// partials cost less than a third hides.  Measured (us, two / three a CU; bf16, 32 / 8 heads of 128): 4 sequences of
// 32,768 with 128 nodes, 160 to 250 tiles a piece 291 / 279; 17 of up to 3,900 with up to 37 (fp16, 28 / 4 heads), 4 to 15
// tiles 39 / 45.  fp32 of 64 dims, whose tiles take longer: 16 of 512 to 2,048 with 8 to 16 nodes 48.5 / 44.4.
constexpr int kLongPiece = 24, kLongPieceF32 = 4;
// Shorter than that, two pieces a CU are worse than one of twice the length: half of the partials.  In batches of few
// segments, whose pieces are all about as long (of many, one a CU is too coarse: 17 of up to 3,900 37 / 42).  Measured
// (us, two / one a CU; 32 / 8 heads): head_dim 128, one sequence of 16,384 with 16 nodes 30.5 / 26.0, four of 4,096 with 32
// 40.2 / 33.7, of 6,000 42.9 / 39.2, but one of 16,384 with 64 in pieces of 16 41.3 / 44.5; fp32, one of 2,048 with 16, 64
// dims, 17.9 / 15.5.  At head_dim 64 in 16 bits no length gained for all (12,288 with 64 nodes 26.7 / 31.9).
constexpr int kShortPiece = 13, kShortPieceF32 = 2, kFewSegments = 16;

// Key tiles to a piece: the least length (a.least and more) that makes no more pieces than most_pieces.  Between
// total / pieces and total / (pieces - segments), where every segment's last piece may be short, a lane each tries 64
// lengths; the waves share the sequences.
// `own`: the thread's sequence of the first kTreeThreads.
struct Cut {
  int tiles, pieces;  // a piece's length; how many there are
  bool alone;         // no sequence has more than one row tile
};
__device__ __forceinline__ Cut piece_tiles(const Args& a, CutScratch& sh, const Span& own, int w, int lane) {
  int tiles = 0, segments = 0, longest = 1, widest = 0;  // tiles: of all segments
  for (int s = threadIdx.x; s < a.num_seqs; s += kTreeThreads) {
    const Span p = s < kTreeThreads ? own : span_of(a, s);
    const int n = p.row_tiles * a.num_kv_heads;
    tiles += n * p.tiles;
    segments += n;
    if (n > 0) longest = max(longest, p.tiles);
    widest = max(widest, p.row_tiles);
    if (s < kTreeThreads) sh.spans[s] = (uint32_t)p.row_tiles << 24 | (uint32_t)p.tiles;
  }
  tiles = wave_scan(tiles);
  segments = wave_scan(segments);
  longest = wave_top(longest);
  widest = wave_top(widest);
  if (lane == 63) {
    sh.sums[w][0] = tiles;
    sh.sums[w][1] = segments;
    sh.sums[w][2] = longest;
    sh.sums[w][3] = widest;
  }
  __syncthreads();
  tiles = segments = 0;
#pragma unroll
  for (int i = 0; i < kTreeWaves; ++i) {
    tiles += sh.sums[i][0];
    segments += sh.sums[i][1];
    longest = max(longest, sh.sums[i][2]);
    widest = max(widest, sh.sums[i][3]);
  }
  Cut cut{longest, segments, widest == 1};
  if (segments == 0) return cut;
  const bool few = kFewSegments * segments <= a.slots && tiles < a.short_piece * a.slots;
  const int most = (int)most_pieces(segments, few ? a.slots / 2 : tiles >= a.long_piece * a.slots_full ? a.slots_full : a.slots);
  const int lo = max(a.least, tiles / most), hi = max(lo, min(longest, tiles / (most - segments) + 1));
  if (lo >= longest) return cut;
  const int mine = lo + (hi - lo) * lane / 63;
  const float by = __builtin_amdgcn_rcpf((float)mine);
  int pieces = 0;
  const int near = min(a.num_seqs, kTreeThreads);
#pragma unroll 4
  for (int s = w; s < near; s += kTreeWaves) {
    const uint32_t span = sh.spans[s];
    pieces += (int)__umul24(span >> 24, ceil_quotient((int)(span & 0xffffffu), mine, by));
  }
  for (int s = kTreeThreads + w; s < a.num_seqs; s += kTreeWaves) {
    const Span p = span_of(a, s);
    pieces += p.row_tiles * ceil_quotient(p.tiles, mine, by);
  }
  pieces *= a.num_kv_heads;
  __syncthreads();  // sums are read
  sh.sums[w][lane] = pieces;
  __syncthreads();
  pieces = 0;
#pragma unroll
  for (int i = 0; i < kTreeWaves; ++i) pieces += sh.sums[i][lane];
  const int first = __builtin_ctzll(__ballot(pieces <= most));  // (hi fits)
  cut.tiles = __builtin_amdgcn_readlane(mine, first);
  cut.pieces = __builtin_amdgcn_readlane(pieces, first);
  return cut;
}

// The piece that workgroup `me` has: its sequence, its place among that one's, and the cuts of those.
__device__ __forceinline__ void find_piece(const Args& a, CutScratch& sh, const Span& own, const Cut& cut, int me, int w,
                                           int lane) {
  // (A batch of more sequences has enough pieces for their order not to matter.)
  const bool sorted = cut.alone && a.num_seqs <= kTreeThreads;
  int before = 0, parts_before = 0;
  for (int s0 = 0; s0 < a.num_seqs; s0 += kTreeThreads) {
    const int s = s0 + threadIdx.x;
    int n = 0, cuts = 0, length = 0;
    Span p = own;
    if (s < a.num_seqs) {
      if (s0 > 0) p = span_of(a, s);
      cuts = (p.tiles + cut.tiles - 1) / cut.tiles;
      n = p.row_tiles * a.num_kv_heads * cuts;
      if (sorted) length = min(kLengths - 1, kLengths - kLengths * ((p.tiles + cuts - 1) / cuts) / cut.tiles);
    }
    const int parts = cuts > 1 ? n : 0, parts_upto = wave_scan(parts);
    int upto[kLengths];
#pragma unroll
    for (int i = 0; i < kLengths; ++i) {
      upto[i] = wave_scan(length == i ? n : 0);
      if (lane == 63) sh.wave_sum[i][w] = upto[i];
    }
    if (lane == 63) sh.wave_sum[kLengths][w] = parts_upto;
    __syncthreads();
    int start = before - n, base = parts_before + parts_upto - parts;
#pragma unroll
    for (int k = 0; k < kTreeWaves; ++k) {
      base += k < w ? sh.wave_sum[kLengths][k] : 0;
      parts_before += sh.wave_sum[kLengths][k];
#pragma unroll
      for (int i = 0; i < kLengths; ++i) {
        start += i < length || (i == length && k < w) ? sh.wave_sum[i][k] : 0;
        before += sh.wave_sum[i][k];
      }
    }
#pragma unroll
    for (int i = 0; i < kLengths; ++i) start += i == length ? upto[i] : 0;
    if (start <= me && me - start < n) {
      sh.seq = s;
      sh.local = me - start;
      sh.pieces = cuts;
      sh.base = base;
      sh.span = p;
    }
    __syncthreads();
    if (me < before) break;
  }
}

// --------------------------------------------------------- the product ------

// One key tile in LDS, two sub-blocks of 16 keys.  K: the 16-byte chunk c of key k of sub-block b at
// b * KB / 2 + 256 c + 16 k, so that a 1 KB copy reads one sub-block only and the A operand of one MFMA is
// 256 contiguous bytes per 16 lanes.  V: rows [key][D] with the 16-byte chunks of a row XORed by
// 2 (key & 3), so that the transposing reads of four rows hit different banks.
template <int D>
struct KeyTile {
  static constexpr int KB = kTileKeys * D * 2;
  static constexpr int BYTES = 2 * KB;
  static constexpr int STAGES = 3;
  static constexpr int VCH = D / 8;          // 16-byte chunks of a V row
  static constexpr int SUB_COPIES = D / 32;  // 1 KB copies of a sub-block's K, and of its V
  __device__ static __forceinline__ int vchunk(int key, int c) { return c ^ (2 * (key & 3)); }
};

// What a piece of a segment is: the rows, the key tiles, where the result goes.
struct Piece {
  int seq, kvh, row0, rows;  // the row tile's first row and the rows of the sequence
  int first, prior, ctx;     // first node; positions
  int kt0, kt1;
  int slot;                  // of the partials, -1: the segment is whole
  bool once;                 // no other row tile reads these keys
};

// Tile kt's attended keys for a node, bit k: key k.  All of it lies before the tree (then no row asks), or its bits
// are shifted out of the node's mask.
__device__ __forceinline__ uint32_t tile_mask(const Piece& p, int node, int kt) {
  const Args& a = arguments();
  const int32_t* bits = a.mask + (int64_t)(p.first + node) * a.mask_words;
  const int at = kt * kTileKeys - p.prior;  // tree index of key 0
  uint32_t m;
  if (at < 0) {
    m = at > -32 ? ((uint32_t)bits[0] << -at) | ((1u << -at) - 1u) : ~0u;
  } else {
    const int w = at >> 5, sh = at & 31;
    const uint32_t lo = w < a.mask_words ? (uint32_t)bits[w] : 0u;
    const uint32_t hi = sh != 0 && w + 1 < a.mask_words ? (uint32_t)bits[w + 1] : 0u;
    m = (uint32_t)(((uint64_t)hi << 32 | lo) >> sh);
  }
  const int left = p.ctx - kt * kTileKeys;
  return left >= 32 ? m : left > 0 ? m & ((1u << left) - 1u) : 0u;
}

// Which keys of a tile hold a value that is not finite: a word for every tile that reaches into the tree, one more than
// its nodes fill where it begins inside a tile.
constexpr int kSickWords = kMaxTreeNodes / kTileKeys + 1;
__device__ __forceinline__ int sick_word(const Piece& p, int kt) { return kt - p.prior / kTileKeys; }

// A row's masks of kMaskTiles key tiles from tile `from` on, into LDS; a row's lanes l and l + 32 do half each.  Read
// by their wave alone.
constexpr int kMaskTiles = 4;
__device__ __forceinline__ void fill_masks(const Piece& p, int node, int from, int in, int hh, uint32_t (&masks)[kMaskTiles][kRows]) {
#pragma unroll
  for (int i = 0; i < kMaskTiles / 2; ++i) {
    const int n = hh * (kMaskTiles / 2) + i;
    masks[n][in] = tile_mask(p, node, from + n);
  }
}

// x where the bit is set, else -inf (by the bit spread over a word: sixteen conditions held as lane masks would take
// 32 scalar registers).
__device__ __forceinline__ float if_bit(uint32_t bits, int b, float x) {
  const uint32_t on = (uint32_t)__builtin_amdgcn_sbfe((int)bits, (uint32_t)b, 1u);
  return __uint_as_float((__float_as_uint(x) & on) | (0xff800000u & ~on));
}

// The lane's row, NB blocks of 32 dims from d0 on.
template <typename T, int D, int NB = D / 32>
__device__ __forceinline__ void store_rows(const Piece& p, int row, int hh, const f32x16_t (&o)[NB], float m, float l,
                                           int d0 = 0) {
  const Args& a = arguments();
  using S = typename elem<T>::storage;
  const int in = row - p.row0;
  if (row >= p.rows) return;
  if (p.slot >= 0) {
    const int64_t at = (int64_t)p.slot * kRows + in;
    float* acc = a.acc + at * D + d0 + 4 * hh;
    auto part = [&](int db, int i) { return f32x4_t{o[db][4 * i], o[db][4 * i + 1], o[db][4 * i + 2], o[db][4 * i + 3]}; };
    if (a.parts_past && p.kt1 - p.kt0 < (std::is_same_v<T, f32_t> ? kLongPieceF32 : kLongPiece)) {
      asm volatile("" ::: "memory");  // (or the two kinds of stores are made one, before the branch or behind it)
#pragma unroll
      for (int db = 0; db < NB; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          __builtin_nontemporal_store(part(db, i), reinterpret_cast<f32x4_t*>(acc + 32 * db + 8 * i));
      asm volatile("" ::: "memory");
    } else {
#pragma unroll
      for (int db = 0; db < NB; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<f32x4_t*>(acc + 32 * db + 8 * i) = part(db, i);
    }
    if (hh == 0 && d0 == 0) *reinterpret_cast<float2*>(a.ml + 2 * at) = make_float2(m, l);
    return;
  }
  const int node = row / a.group, g = row - node * a.group;
  S* out = static_cast<S*>(a.out) + ((int64_t)(p.first + node) * a.num_heads + p.kvh * a.group + g) * D + d0;
  const float inv = l != 0.f ? 1.f / l : 1.f;
#pragma unroll
  for (int db = 0; db < NB; ++db)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x0 = o[db][4 * i] * inv, x1 = o[db][4 * i + 1] * inv, x2 = o[db][4 * i + 2] * inv,
                  x3 = o[db][4 * i + 3] * inv;
      S* to = out + 32 * db + 8 * i + 4 * hh;
      if constexpr (std::is_same_v<T, f32_t>) *reinterpret_cast<float4*>(to) = make_float4(x0, x1, x2, x3);
      else *reinterpret_cast<uint2*>(to) = make_uint2(pack2<T>(x0, x1), pack2<T>(x2, x3));
    }
}

// Adds to the lane's row what V holds that is not finite, of the keys `sick` that the row attends to (`mine`).  The
// values come from the cache, 4 dims at a time as the accumulators have them; times any weight they stay what they are.
template <typename T, int D, int NB = D / 32>
__device__ __forceinline__ void add_not_finite(const Piece& p, int kt, uint32_t sick, uint32_t mine, int hh,
                                               f32x16_t (&o)[NB], int d0 = 0) {
  const Args& a = arguments();
  const int32_t* row_table = a.table + (int64_t)p.seq * a.max_blocks;
  using E = elem<T>;
  using S = typename E::storage;
  while (sick != 0) {
    const int key = __builtin_ctz(sick);
    sick &= sick - 1;
    const int at = kt * kTileKeys + key;
    const S* v = static_cast<const S*>(a.v) + (int64_t)row_table[at / a.block_size] * a.kv_stride +
                 ((int64_t)p.kvh * a.block_size + at % a.block_size) * D + d0;
    const bool takes = mine >> key & 1;
#pragma unroll
    for (int db = 0; db < NB; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = E::to_f32(v[32 * db + 8 * i + 4 * hh + e]);
          o[db][4 * i + e] += takes && !(fabsf(x) < INFINITY) ? x : 0.f;
        }
  }
}

// Not finite: all exponent bits set, of either half of a packed pair.
template <typename T> __device__ __forceinline__ bool pair_not_finite(uint32_t w) {
  constexpr uint32_t e = std::is_same_v<T, bf16_t> ? 0x7f80u : 0x7c00u;
  return (w & e) == e || (w >> 16 & e) == e;
}
template <typename T> __device__ __forceinline__ uint32_t pair_cleared(uint32_t w) {
  constexpr uint32_t e = std::is_same_v<T, bf16_t> ? 0x7f80u : 0x7c00u;
  return ((w & e) == e ? 0u : w & 0xffffu) | ((w >> 16 & e) == e ? 0u : w & 0xffff0000u);
}

// N copies of 1 KB to LDS, `step` bytes apart, non-temporal where they are read once.
template <int N>
__device__ __forceinline__ void copy(const char* base, uint32_t step, uint32_t lane_bytes, uint32_t lds_addr, bool once) {
  if (once) {
#pragma unroll
    for (int i = 0; i < N; ++i) lds_dma16_s_nt(base + step * i, lane_bytes, lds_addr + i * 1024);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) lds_dma16_s(base + step * i, lane_bytes, lds_addr + i * 1024);
  }
}

// Lane l of a wave owns query row l % 32 of it; the other half of that row's keys sits in lane l ^ 32.  sick: a word of
// LDS for every tile that reaches into the tree (sick_word).
template <typename T, int D>
__device__ __forceinline__ void product(const Piece& p, char* lds, uint32_t* sick,
                                        uint32_t (&masks)[kMaskTiles][kRows], int w, int lane) {
  using MF = mfma32<T>;
  using TL = KeyTile<D>;
  constexpr int NKC = D / 16, NDB = D / 32, HALF = TL::SUB_COPIES / 2, COPIES = 2 * HALF;
  static_assert(HALF >= 1, "two waves copy a sub-block");
  const Args& a = arguments();
  const int j = lane & 31, hh = lane >> 5;
  const int row = p.row0 + w * 32 + j;
  const bool busy = p.row0 + w * 32 < p.rows;  // (a wave without rows copies and waits with the others)
  const int node = min(row, p.rows - 1) / a.group, g = min(row, p.rows - 1) - node * a.group;

  // This wave copies half of sub-block cb of every tile.  Lane l of the window holds where that of tile wb + l lies in
  // the caches, in bytes; past the end the last sub-block.
  const int cb = w >> 1, cp = w & 1;
  int wb = p.kt0;
  uint32_t win_lo, win_hi;
  auto fill = [&]() {
    const Args& a = arguments();
    const int subs = (p.ctx + kBS - 1) / kBS, sb = min(2 * (wb + lane) + cb, subs - 1);
    const int64_t block = a.table[(int64_t)p.seq * a.max_blocks + (sb >> a.bs_shift)];
    const int64_t at = 2 * (block * a.kv_stride + ((int64_t)(p.kvh << a.bs_shift) + (sb & ((1 << a.bs_shift) - 1))) * (kBS * D));
    win_lo = (uint32_t)at;
    win_hi = (uint32_t)((uint64_t)at >> 32);
  };
  fill();
  uint4 qb[NKC];
  {
    const uint4* qr = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) +
                                                     ((int64_t)(p.first + node) * a.num_heads + p.kvh * a.group + g) * D);
#pragma unroll
    for (int i = 0; i < NKC; ++i) qb[i] = qr[2 * i + hh];
  }
  int masks_from = max(p.kt0, p.prior / kTileKeys);
  if (masks_from < p.kt1) fill_masks(p, node, masks_from, w * 32 + j, hh, masks);
  // K: copy n of the sub-block takes its chunks 4 n .. 4 n + 3, V: 1024 / (2 D) of its rows; from copy to copy a
  // lane's place moves by the same bytes.
  const uint32_t k_off = (uint32_t)(2 * ((lane & 15) * D + 8 * (4 * cp * HALF + (lane >> 4))));
  constexpr int VROWS = 1024 / (2 * D);
  static_assert(VROWS % 4 == 0, "copies of V that swizzle alike");
  const int v_key = cp * HALF * VROWS + lane / TL::VCH;
  const uint32_t v_off = (uint32_t)(2 * (v_key * D + 8 * TL::vchunk(v_key, lane % TL::VCH)));
  const uint32_t lds_at = (uint32_t)(uintptr_t)((RG_LDS char*)lds) + cb * (TL::KB / 2) + cp * HALF * 1024;
  const char* const kc = static_cast<const char*>(a.k);
  const char* const vc = static_cast<const char*>(a.v);
  auto issue = [&](int kt, int st) {
    const int64_t at = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)win_hi, kt - wb) << 32 |
                                 (uint32_t)__builtin_amdgcn_readlane((int)win_lo, kt - wb));
    copy<HALF>(kc + at, 64, k_off, lds_at + st * TL::BYTES, p.once);
    copy<HALF>(vc + at, 1024, v_off, lds_at + st * TL::BYTES + TL::KB, p.once);
  };

  f32x16_t o[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[db][v] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;
  float ref = -INFINITY;    // reference(m_run)
  float m_thr = -INFINITY;  // m_run + kSlack in raw score units, so a tile's test needs no multiply
  const float scale = a.scale_log2;
  const int xor32 = (lane ^ 32) << 2;
  const int k_lane = (j >> 4) * (TL::KB / 2) + hh * 256 + (j & 15) * 16;
  const int grp = lane >> 4, e_row = (lane >> 2) & 3, qq = lane & 3;

  // A operand m = n NDB + db of the PV product (keys 16 n .., 32-dim block db) by the transposing LDS read: in
  // each 16-lane group, lane 4 e + p points at V[key0 + e][d0 + 4 p ..] and lane i receives V[key0 ..][d0 + i].
  auto v_operand = [&](const char* vbase, int m) {
    const int n = m / NDB, db = m % NDB;
    const int d = 32 * db + 16 * (grp & 1) + 4 * qq;
    uint2 part[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int key = 16 * n + 8 * half + 4 * (grp >> 1) + e_row;
      const int off = key * (D * 2) + TL::vchunk(key, d >> 3) * 16 + (d & 7) * 2;
      part[half] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((RG_LDS v4i16_t*)(vbase + off)));
    }
    return make_uint4(part[0].x, part[0].y, part[1].x, part[1].y);
  };
  constexpr int KA = NKC < 4 ? NKC : 4;          // K operands read ahead of their MFMA
  constexpr int VA = 2 * NDB < 3 ? 2 * NDB : 3;  // V operands, the first of them before the softmax
  // S^T of a tile in LDS: c[v] is key 8 (v >> 2) + 4 hh + (v & 3) of it for query j.
  auto scores = [&](const char* tile) __attribute__((always_inline)) -> f32x16_t {
    const char* kbase = tile + k_lane;
    uint4 ka[KA];
#pragma unroll
    for (int i = 0; i < KA; ++i) ka[i] = *reinterpret_cast<const uint4*>(kbase + i * 512);
    f32x16_t c;
#pragma unroll
    for (int v = 0; v < 16; ++v) c[v] = 0.f;
#pragma unroll
    for (int i = 0; i < NKC; ++i) {
      __builtin_amdgcn_sched_barrier(0);
      c = MF::run(ka[i % KA], qb[i], c);
      if (i + KA < NKC) ka[i % KA] = *reinterpret_cast<const uint4*>(kbase + (i + KA) * 512);
    }
    __builtin_amdgcn_sched_barrier(0);
    return c;
  };
  auto finish = [&](f32x16_t c, const char* tile) __attribute__((always_inline)) {
    const char* vbase = tile + TL::KB;
    uint4 va[VA];
#pragma unroll
    for (int m = 0; m < VA; ++m) va[m] = v_operand(vbase, m);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
    // The maximum moves only when a tile exceeds it by more than kSlack, for both halves of a row alike.
    float tmax = c[0];
#pragma unroll
    for (int v = 1; v < 16; ++v) tmax = fmaxf(tmax, c[v]);
    if (__ballot(tmax > m_thr)) {
      const float other = __int_as_float(__builtin_amdgcn_ds_bpermute(xor32, __float_as_int(tmax)));
      const float both = fmaxf(tmax, other) * scale;
      const bool moves = both > m_run + kSlack;
      const float m_new = moves ? both : m_run;
      const float ref_new = reference<T>(m_new);
      const float alpha = moves ? fast_exp2(ref - ref_new) : 1.f;
      m_run = m_new;
      ref = ref_new;
      m_thr = (m_run + kSlack) / scale;
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[db][v] *= alpha;
    }
    // (A row that has seen no key yet: its scores are -inf, and so are its probabilities' logarithms.)
    const float sub = ref == -INFINITY ? 0.f : ref;
    // Probabilities, rounded to the operand type of the PV product; the sum takes the rounded ones, so
    // the normaliser weighs what enters the product.
    uint32_t pk[8];
#pragma unroll
    for (int v = 0; v < 16; v += 2)
      pk[v / 2] = pack2<T>(fast_exp2(fmaf(c[v], scale, -sub)), fast_exp2(fmaf(c[v + 1], scale, -sub)));
    float s0 = pair_sum<T>(pk[0], l_run), s1 = pair_sum<T>(pk[1], 0.f);
#pragma unroll
    for (int i = 2; i < 8; i += 2) {
      s0 = pair_sum<T>(pk[i], s0);
      s1 = pair_sum<T>(pk[i + 1], s1);
    }
    l_run = s0 + s1;
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int m = 0; m < 2 * NDB; ++m) {
      const int n = m / NDB, db = m % NDB;
      __builtin_amdgcn_sched_barrier(0);
      o[db] = MF::run(va[m % VA], make_uint4(pk[4 * n], pk[4 * n + 1], pk[4 * n + 2], pk[4 * n + 3]), o[db]);
      if (m + VA < 2 * NDB) va[m % VA] = v_operand(vbase, m + VA);
    }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
  };
  // Tile kt reaches into the tree: V rows behind the context and what is not finite are cleared, by the workgroup.
  auto clean = [&](int kt, int st) {
    char* vbase = lds + st * TL::BYTES + TL::KB;
    for (int i = threadIdx.x; i < kTileKeys * TL::VCH; i += kTreeThreads) {
      const int key = i / TL::VCH;
      uint4* at = reinterpret_cast<uint4*>(vbase + i * 16);
      uint4 x = *at;
      if (kt * kTileKeys + key >= p.ctx) {
        *at = make_uint4(0u, 0u, 0u, 0u);
      } else if (pair_not_finite<T>(x.x) || pair_not_finite<T>(x.y) || pair_not_finite<T>(x.z) || pair_not_finite<T>(x.w)) {
        *at = make_uint4(pair_cleared<T>(x.x), pair_cleared<T>(x.y), pair_cleared<T>(x.z), pair_cleared<T>(x.w));
        atomicOr(&sick[sick_word(p, kt)], 1u << key);
      }
    }
    wave_lds_sync();  // (the copies in flight stay in flight)
    tile_barrier();
  };

  static_assert(TL::STAGES == 3 && COPIES < 16, "one tile newer than the awaited one; low bits of vmcnt");
  issue(p.kt0, 0);
  if (p.kt0 + 1 < p.kt1) issue(p.kt0 + 1, 1);
  // Q, the masks and the first tiles have landed (the builtin, which the compiler's own counting follows: behind an asm
  // wait it would wait for Q again in every tile, and with it for every copy in flight).
  __builtin_amdgcn_s_waitcnt(0x70 | 0xF00);  // vmcnt(0)
  // scale_log2 > 0 here: the host passes its magnitude (1 for a scale of 0) and what becomes of q.
  {
    const uint32_t flip = a.q_sign & 0x80008000u, on = a.q_sign & 1 ? 0xffffffffu : 0u;
#pragma unroll
    for (int i = 0; i < NKC; ++i)
      qb[i] = make_uint4((qb[i].x ^ flip) & on, (qb[i].y ^ flip) & on, (qb[i].z ^ flip) & on, (qb[i].w ^ flip) & on);
  }
  // Tile kt has landed (a newer one may not have), for every wave; all are done with tile kt - 1, whose stage takes
  // tile kt + STAGES - 1.  Returns whether there is one.
  auto ready = [&](int kt) __attribute__((always_inline)) {
    asm volatile("" ::: "memory");
    if (kt + 1 < p.kt1) __builtin_amdgcn_s_waitcnt(COPIES | 0x70 | 0xF00);
    else __builtin_amdgcn_s_waitcnt(0x70 | 0xF00);
    tile_barrier();
    const int next = kt + TL::STAGES - 1;
    if (next - wb >= 64) {
      wb = next;
      fill();
      __builtin_amdgcn_s_waitcnt(0x70 | 0xF00);
    }
    return next < p.kt1;
  };
  int kt = p.kt0;
  // The tiles that every row attends to, as far as STAGES of them follow each other.
  const int whole = min(p.kt1, p.prior / kTileKeys);
  for (; kt + TL::STAGES <= whole; kt += TL::STAGES) {
#pragma unroll
    for (int st = 0; st < TL::STAGES; ++st) {
      const bool more = ready(kt + st);
      const char* tile = lds + st * TL::BYTES;
      const int next_st = st == 0 ? TL::STAGES - 1 : st - 1;
      if (busy) {
        __builtin_amdgcn_s_setprio(1);
        const f32x16_t c = scores(tile);
        if (more) issue(kt + st + TL::STAGES - 1, next_st);  // while the QK MFMAs run
        finish(c, tile);
      } else if (more) {
        issue(kt + st + TL::STAGES - 1, next_st);
      }
    }
  }
  int st = 0;
#pragma clang loop unroll(disable)
  for (; kt < p.kt1; ++kt) {
    const bool more = ready(kt);
    const bool masked = kt >= whole;
    if (masked) clean(kt, st);
    const char* tile = lds + st * TL::BYTES;
    const int next_st = st == 0 ? TL::STAGES - 1 : st - 1;
    if (busy) {
      __builtin_amdgcn_s_setprio(1);
      f32x16_t c = scores(tile);
      if (more) issue(kt + TL::STAGES - 1, next_st);
      uint32_t mine = 0;
      if (masked) {
        if (kt - masks_from >= kMaskTiles) fill_masks(p, node, masks_from = kt, w * 32 + j, hh, masks);
        mine = masks[kt - masks_from][w * 32 + j];
        const uint32_t shifted = mine >> (4 * hh);
#pragma unroll
        for (int v = 0; v < 16; ++v) c[v] = if_bit(shifted, 8 * (v >> 2) + (v & 3), c[v]);
      }
      finish(c, tile);
      if (masked && sick[sick_word(p, kt)] != 0) add_not_finite<T, D>(p, kt, sick[sick_word(p, kt)], mine, hh, o);
    } else if (more) {
      issue(kt + TL::STAGES - 1, next_st);
    }
    st = st == TL::STAGES - 1 ? 0 : st + 1;
  }
  const float l = l_run + __shfl_xor(l_run, 32, 64);
  if (busy) store_rows<T, D>(p, row, hh, o, ref, l);
}


// The fp32 product, on v_mfma_f32_32x32x2: step m of S^T = K Q^T takes the k-slot of lane half hh from dim
// hh D/2 + m, so a lane reads its K row in 16-byte pieces; step v of O^T += V^T P^T takes the keys
// 8 (v >> 2) + 4 hh + (v & 3), which is where S^T leaves them, so the probabilities stay in fp32 and in their
// registers.  A key tile is twice as long as in 16 bits and its product 16 times, so one tile in flight ahead of the
// one at hand is enough: two stages.
// K in LDS: rows [key][D], the 16-byte chunk c of a row at c ^ (key & 7) (rows of 256 or 512 bytes would put all
// keys of a read on the same banks); V: rows [key][D] as they are (a read takes 32 neighbours of one row).
template <int D>
struct KeyTileF32 {
  static constexpr int KB = kTileKeys * D * 4;
  static constexpr int BYTES = 2 * KB;
  static constexpr int STAGES = 2;
  static constexpr int CH = D / 4;           // 16-byte chunks of a row
  static constexpr int SUB_COPIES = D / 16;  // 1 KB copies of a sub-block's K, and of its V
  // The scores that waves exchange, 16 a lane: in K's place where they fit, else behind the ring.
  static constexpr int SHARED = 64 * kTreeWaves * 16 * 4;
  static constexpr bool SHARED_IN_RING = KB >= SHARED;
  static constexpr int LDS = STAGES * BYTES + (SHARED_IN_RING ? 0 : SHARED);
};

// WAYS = 2, where a piece has at most 64 rows: waves w and w + 2 have the same rows and half of the dims each.  Each
// adds up its dims' part of the scores, the two exchange them through LDS (at head_dim 128 over the K that all are
// done with; a + b is b + a, so both go on with the same scores), and each has its dims of the output.  Otherwise the
// matrix units of two SIMDs stood idle.  Measured (us, 1 / 2 ways; 32 / 8 heads, 16 sequences of 512 to 2,048 with 8 to 16
// nodes): head_dim 128 117 / 82, 64 66.7 / 48.6.  Four ways up to 32 rows measured the same as two.
template <int D, int WAYS>
__device__ __forceinline__ void product_f32(const Piece& p, char* lds, uint32_t* sick,
                                            uint32_t (&masks)[kMaskTiles][kRows], int w, int lane) {
  const Args& a = arguments();
  using TL = KeyTileF32<D>;
  constexpr int NDB = D / 32 / WAYS, HALF = TL::SUB_COPIES / 2, COPIES = 2 * HALF, HD = D / WAYS / 2;
  const float* q = static_cast<const float*>(a.q);
  const float* kc = static_cast<const float*>(a.k);
  const float* vc = static_cast<const float*>(a.v);
  const int32_t* table = a.table + (int64_t)p.seq * a.max_blocks;
  const int j = lane & 31, hh = lane >> 5;
  const int w_row = WAYS == 2 ? w & 1 : w, d0 = WAYS == 2 ? (w >> 1) * (D / 2) : 0;
  const int row = p.row0 + w_row * 32 + j;
  const bool busy = p.row0 + w_row * 32 < p.rows;
  const int node = min(row, p.rows - 1) / a.group, g = min(row, p.rows - 1) - node * a.group;
  const int subs = (p.ctx + kBS - 1) / kBS;
  const int cb = w >> 1, cp = w & 1;
  int wb = p.kt0, win;
  auto fill = [&]() {
    const int sb = min(2 * (wb + lane) + cb, subs - 1);
    win = (table[sb >> a.bs_shift] << a.bs_shift) | (sb & ((1 << a.bs_shift) - 1));
  };
  fill();
  int masks_from = max(p.kt0, p.prior / kTileKeys);
  if (masks_from < p.kt1) fill_masks(p, node, masks_from, w * 32 + j, hh, masks);
  float qf[HD];
  {
    const float4* qr = reinterpret_cast<const float4*>(q + ((int64_t)(p.first + node) * a.num_heads + p.kvh * a.group + g) * D + d0 + hh * HD);
    const float on = a.q_sign == 0 ? 0.f : a.q_sign & 0x8000u ? -1.f : 1.f;
#pragma unroll
    for (int i = 0; i < HD / 4; ++i) {
      const float4 x = qr[i];
      qf[4 * i] = on != 0.f ? x.x * on : 0.f;
      qf[4 * i + 1] = on != 0.f ? x.y * on : 0.f;
      qf[4 * i + 2] = on != 0.f ? x.z * on : 0.f;
      qf[4 * i + 3] = on != 0.f ? x.w * on : 0.f;
    }
  }
  // Copy n of a sub-block's K or V (1 KB): chunk positions 64 n + lane of its rows.
  uint32_t k_off[HALF], v_off[HALF];  // bytes within the sub-block
#pragma unroll
  for (int i = 0; i < HALF; ++i) {
    const int at = (cp * HALF + i) * 64 + lane, key = at / TL::CH, c = at % TL::CH;
    k_off[i] = (uint32_t)(key * D * 4 + 16 * (c ^ (key & 7)));
    v_off[i] = (uint32_t)(at * 16);
  }
  const uint32_t lds_base = (uint32_t)(uintptr_t)((RG_LDS char*)lds);
  const int64_t head = (int64_t)p.kvh * (kBS << a.bs_shift) * D;
  auto issue = [&](int kt, int st) {
    const int e = __builtin_amdgcn_readlane(win, kt - wb);
    const int64_t off = (int64_t)(e >> a.bs_shift) * a.kv_stride + head + (int64_t)(e & ((1 << a.bs_shift) - 1)) * (kBS * D);
    const uint32_t at = lds_base + st * TL::BYTES + cb * (TL::KB / 2) + cp * HALF * 1024;
#pragma unroll
    for (int i = 0; i < HALF; ++i) lds_dma16_s(reinterpret_cast<const char*>(kc + off), k_off[i], at + i * 1024);
#pragma unroll
    for (int i = 0; i < HALF; ++i) lds_dma16_s(reinterpret_cast<const char*>(vc + off), v_off[i], at + TL::KB + i * 1024);
  };
  f32x16_t o[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[db][v] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;
  const int xor32 = (lane ^ 32) << 2;
  auto clean = [&](int kt, int st) {
    char* vbase = lds + st * TL::BYTES + TL::KB;
    for (int i = threadIdx.x; i < kTileKeys * TL::CH; i += kTreeThreads) {
      const int key = i / TL::CH;
      float4* at = reinterpret_cast<float4*>(vbase + i * 16);
      const float4 x = *at;
      auto fine = [](float v) { return fabsf(v) < INFINITY; };
      if (kt * kTileKeys + key >= p.ctx) {
        *at = make_float4(0.f, 0.f, 0.f, 0.f);
      } else if (!(fine(x.x) && fine(x.y) && fine(x.z) && fine(x.w))) {
        *at = make_float4(fine(x.x) ? x.x : 0.f, fine(x.y) ? x.y : 0.f, fine(x.z) ? x.z : 0.f, fine(x.w) ? x.w : 0.f);
        atomicOr(&sick[sick_word(p, kt)], 1u << key);
      }
    }
    wave_lds_sync();  // (the copies in flight stay in flight)
    tile_barrier();
  };
  auto scores = [&](int st) __attribute__((always_inline)) -> f32x16_t {
    const char* krow = lds + st * TL::BYTES + j * (D * 4);
    f32x16_t c;
#pragma unroll
    for (int v = 0; v < 16; ++v) c[v] = 0.f;
#pragma unroll
    for (int i = 0; i < HD / 4; ++i) {
      const float4 k4 = *reinterpret_cast<const float4*>(krow + 16 * ((d0 / 4 + hh * (HD / 4) + i) ^ (j & 7)));
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(k4.x, qf[4 * i], c, 0, 0, 0);
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(k4.y, qf[4 * i + 1], c, 0, 0, 0);
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(k4.z, qf[4 * i + 2], c, 0, 0, 0);
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(k4.w, qf[4 * i + 3], c, 0, 0, 0);
    }
    return c;
  };
  auto finish = [&](f32x16_t c, int kt, int st, bool masked) __attribute__((always_inline)) {
    uint32_t mine = ~0u;
    if (masked) {
      if (kt - masks_from >= kMaskTiles) fill_masks(p, node, masks_from = kt, w * 32 + j, hh, masks);
      mine = masks[kt - masks_from][w * 32 + j];
      const uint32_t shifted = mine >> (4 * hh);
#pragma unroll
      for (int v = 0; v < 16; ++v) c[v] = if_bit(shifted, 8 * (v >> 2) + (v & 3), c[v]);
    }
    float tmax = c[0];
#pragma unroll
    for (int v = 1; v < 16; ++v) tmax = fmaxf(tmax, c[v]);
    tmax = fmaxf(tmax, __int_as_float(__builtin_amdgcn_ds_bpermute(xor32, __float_as_int(tmax)))) * a.scale_log2;
    if (__ballot(tmax > m_run)) {
      const bool moves = tmax > m_run;
      const float alpha = moves ? fast_exp2(m_run - tmax) : 1.f;
      m_run = moves ? tmax : m_run;
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[db][v] *= alpha;
    }
    const float sub = m_run == -INFINITY ? 0.f : m_run;
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      c[v] = fast_exp2(fmaf(c[v], a.scale_log2, -sub));
      l_run += c[v];
    }
    const float* vrow = reinterpret_cast<const float*>(lds + st * TL::BYTES + TL::KB) + 4 * hh * D + d0 + j;
#pragma unroll
    for (int v = 0; v < 16; ++v)
#pragma unroll
      for (int db = 0; db < NDB; ++db)
        o[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(vrow[(8 * (v >> 2) + (v & 3)) * D + 32 * db], c[v], o[db], 0, 0, 0);
    if (masked && sick[sick_word(p, kt)] != 0) add_not_finite<f32_t, D, NDB>(p, kt, sick[sick_word(p, kt)], mine, hh, o, d0);
  };
  // Both halves' scores of a row.
  auto exchange = [&](f32x16_t& c, int st) __attribute__((always_inline)) {
    float4* const all = reinterpret_cast<float4*>(lds + (TL::SHARED_IN_RING ? st * TL::BYTES : TL::STAGES * TL::BYTES));
    if constexpr (TL::SHARED_IN_RING) {
      wave_lds_sync();
      tile_barrier();  // all are done with K
    }
    if (busy) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        all[(w * 4 + i) * 64 + lane] = make_float4(c[4 * i], c[4 * i + 1], c[4 * i + 2], c[4 * i + 3]);
    }
    wave_lds_sync();
    tile_barrier();
    if (busy) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 x = all[((w ^ 2) * 4 + i) * 64 + lane];
        c[4 * i] += x.x;
        c[4 * i + 1] += x.y;
        c[4 * i + 2] += x.z;
        c[4 * i + 3] += x.w;
      }
    }
  };
  __builtin_amdgcn_s_waitcnt(0x70 | 0xF00);  // vmcnt(0): the window and Q
  issue(p.kt0, 0);
  if (p.kt0 + 1 < p.kt1) issue(p.kt0 + 1, 1);
  static_assert(COPIES < 16, "low bits of vmcnt");
#pragma clang loop unroll(disable)
  for (int kt = p.kt0; kt < p.kt1; ++kt) {
    const int st = (kt - p.kt0) & 1;
    asm volatile("" ::: "memory");
    if (kt + 1 < p.kt1) __builtin_amdgcn_s_waitcnt(COPIES | 0x70 | 0xF00);
    else __builtin_amdgcn_s_waitcnt(0x70 | 0xF00);
    wave_lds_sync();
    tile_barrier();  // tile kt has landed for every wave
    const bool masked = (kt + 1) * kTileKeys > p.prior;
    if (masked) clean(kt, st);
    f32x16_t c{};
    if (busy) c = scores(st);
    if constexpr (WAYS == 2) exchange(c, st);
    if (busy) finish(c, kt, st, masked);
    if (kt + 2 < p.kt1) {
      if (kt + 2 - wb >= 64) {
        wb = kt + 2;
        fill();
        __builtin_amdgcn_s_waitcnt(0x70 | 0xF00);
      }
      wave_lds_sync();
      tile_barrier();  // every wave is done with the stage
      issue(kt + 2, st);
    }
  }
  const float l = l_run + __shfl_xor(l_run, 32, 64);
  if (busy) store_rows<f32_t, D, NDB>(p, row, hh, o, m_run, l, d0);
}

template <typename T, int D>
constexpr int ring_bytes() {
  if constexpr (std::is_same_v<T, f32_t>) return KeyTileF32<D>::LDS;
  else return KeyTile<D>::STAGES * KeyTile<D>::BYTES;
}
// Workgroups to a CU: what their registers allow (168 a wave for three) and the rings, 64 KB in fp32 at head_dim 128
// and 48 at 64.
constexpr int pieces_per_cu(int32_t dtype, int D) { return D == 128 ? (dtype == RG_DTYPE_F32 ? 2 : 3) : dtype == RG_DTYPE_F32 ? 3 : 4; }
template <typename T, int D>
constexpr int groups_per_cu() { return pieces_per_cu(std::is_same_v<T, f32_t> ? RG_DTYPE_F32 : RG_DTYPE_BF16, D); }

// A workgroup to a piece.  What bounds it (bf16, 32 / 8 heads of 128; us):
//  - many sequences, short trees: HBM, and ends apart.  64 of 512 to 4,096 tokens with 8 to 32 nodes, 639 MB: 121 to
//    141, 131 with the merge in a row of calls, 4.9 TB/s.  The pieces are of 17 to 40 tiles: their workgroups end 55 to
//    121 in, at 94 on average.
//  - long trees: the waves' LDS reads and the softmax between two products, which other workgroups' waves hide in part.
//    Four sequences of 30,000 to 32,768 with 101 to 128 nodes, 253 GFLOP: 280 with the merge (12) in a row of calls, 900
//    TFLOP/s; one by one under a profiler the first take 276 to 284, later ones up to 409.  Without the copies to LDS it
//    takes 15 % less, without the exponentials 7 %, without either product 20 %, without both products and
//    the exponentials still 53 % of it.  64 rows a wave would read LDS half as often, in 290 registers: one
//    workgroup a CU.  The next tile's scores under this one's softmax and rings of 4 to 8 tiles gained nothing.
//  - one sequence: latency.  4,096 tokens with 64 nodes: 20.4.  By stamps in the workgroups, on average: 0.4 until they
//    start, 2.0 for the lengths and the cut, 0.9 to find the piece, 2.1 until table, masks and Q are there and 0.3 for
//    the first tile, 6.8 for 8 tiles, 4.5 until the partials are written; the last of them ends at 19.0.
// fp32: v_mfma_f32_32x32x2 has a sixteenth of the rate, and what a row tile lacks of rows is computed all the same; 64
// sequences of 512 to 2,048 with 4 to 8 nodes, 64 dims, 108, 1.5 times the bytes' floor.
template <typename T, int D>
__global__ __launch_bounds__(kTreeThreads, (groups_per_cu<T, D>())) void tree_kernel(TreeArgs) {
  __shared__ __attribute__((aligned(16))) char ring[ring_bytes<T, D>()];
  __shared__ uint32_t sick[kSickWords];
  __shared__ uint32_t masks[kMaskTiles][kRows];
  if (threadIdx.x < kSickWords) sick[threadIdx.x] = 0;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Piece p;
  {
    const Args& a = arguments();
    CutScratch& sh = *reinterpret_cast<CutScratch*>(ring);  // (before the first key tile)
    static_assert(sizeof(CutScratch) <= sizeof(ring), "the cuts' scratch lies in the ring");
    Span own{};
    if (threadIdx.x < (unsigned)a.num_seqs) own = span_of(a, threadIdx.x);
    const Cut cut_to = piece_tiles(a, sh, own, w, lane);
    // Workgroups are dealt to the XCDs in turn.  The row tiles of the same keys go to the same one; where there are none,
    // the order of the pieces is that of their dispatch.
    const int per = (cut_to.pieces + 7) / 8, on_xcd = (int)blockIdx.x / 8;
    const int me = cut_to.alone ? (int)blockIdx.x : on_xcd < per ? (int)(blockIdx.x % 8) * per + on_xcd : cut_to.pieces;
    if (me >= cut_to.pieces) return;
    find_piece(a, sh, own, cut_to, me, w, lane);
    const int s = __builtin_amdgcn_readfirstlane(sh.seq);
    const int local = __builtin_amdgcn_readfirstlane(sh.local), n = __builtin_amdgcn_readfirstlane(sh.pieces);
    const int base = __builtin_amdgcn_readfirstlane(sh.base);
    Span sp;
    sp.t.first = __builtin_amdgcn_readfirstlane(sh.span.t.first);
    sp.t.nodes = __builtin_amdgcn_readfirstlane(sh.span.t.nodes);
    sp.prior = __builtin_amdgcn_readfirstlane(sh.span.prior);
    sp.ctx = __builtin_amdgcn_readfirstlane(sh.span.ctx);
    sp.tiles = __builtin_amdgcn_readfirstlane(sh.span.tiles);
    sp.row_tiles = __builtin_amdgcn_readfirstlane(sh.span.row_tiles);
    __syncthreads();  // the scratch is free
    const int rt = local % sp.row_tiles, cut = local / sp.row_tiles % n;
    p.seq = s;
    p.kvh = local / sp.row_tiles / n;
    p.row0 = rt * kRows;
    p.rows = sp.t.nodes * a.group;
    p.first = sp.t.first;
    p.ctx = sp.ctx;
    p.prior = sp.prior;
    const int each = sp.tiles / n, longer = sp.tiles - each * n;  // the first few are a tile longer
    p.kt0 = each * cut + min(cut, longer);
    p.kt1 = each * (cut + 1) + min(cut + 1, longer);
    p.slot = n > 1 ? base + local : -1;
    p.once = sp.row_tiles == 1;
    if (local == 0 && threadIdx.x == 0) a.cuts[s] = make_int2(base, n);
  }
  if (p.ctx == 0) {
    const int row = p.row0 + w * 32 + (lane & 31);
    f32x16_t o[D / 32];
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int v = 0; v < 16; ++v) o[db][v] = 0.f;
    store_rows<T, D>(p, row, lane >> 5, o, -INFINITY, 0.f);
  } else if constexpr (std::is_same_v<T, f32_t>) {
    if (p.rows - p.row0 <= kRows / 2) product_f32<D, 2>(p, ring, sick, masks, w, lane);
    else product_f32<D, 1>(p, ring, sick, masks, w, lane);
  } else {
    product<T, D>(p, ring, sick, masks, w, lane);
  }
}

// The rows of a cut segment: D / 4 lanes have 4 dims each of a row, a wave N times 256 / D rows.  Where a batch is few
// segments in many pieces (kManyParts), the waves of a workgroup have the same rows (SPLIT), each every fourth piece, and
// their results are joined in LDS: a wave alone would wait for 64 pieces eight times.  AHEAD: pieces in flight, 8, or 2
// where few segments are cut at all.  Measured (us; bf16, 32 / 8 heads of 128, 16 nodes): a wave alone / split, one
// sequence of 32,768 14.5 / 7.4, four of 4,096 6.4 / 6.1, one of 2,048 4.0 / 3.9.  Two rows a wave and four pieces ahead / one
// and eight, 17 sequences of up to 3,900 (fp16, 28 / 4 heads) 8.6 / 7.4, four of 32,768 with 128 nodes 12.4 / 11.4; four
// rows and two pieces / two and two, 64 of up to 4,096 9.1 / 8.0.
constexpr int kMergeWaves = 4;
template <int D> constexpr int merge_rows() { return 256 / D; }

// A row's partials so far, 4 dims of it, and the next.
struct Partial {
  float m, l;
  float4 acc;
  __device__ __forceinline__ void join(float2 x, float4 v, bool is) {
    // (A piece without keys for the row has m = -inf and nothing to add; one whose scores are all NaN has m = -inf
    // too.)
    const bool counts = is && !(x.x == -INFINITY && x.y == 0.f);
    const float mn = counts ? fmaxf(m, x.x) : m;
    const float fo = m == mn ? 1.f : exp2f(m - mn), fq = !counts ? 0.f : x.x == mn ? 1.f : exp2f(x.x - mn);
    l = l * fo + (counts ? x.y * fq : 0.f);
    acc.x = acc.x * fo + (counts ? v.x * fq : 0.f);
    acc.y = acc.y * fo + (counts ? v.y * fq : 0.f);
    acc.z = acc.z * fo + (counts ? v.z * fq : 0.f);
    acc.w = acc.w * fo + (counts ? v.w * fq : 0.f);
    m = mn;
  }
};

template <typename T, int D, int N, int AHEAD, bool SPLIT>
__global__ __launch_bounds__(64 * kMergeWaves) void tree_merge_kernel(TreeArgs a) {
  using S = typename elem<T>::storage;
  constexpr int LANES = D / 4, ROWS = merge_rows<D>(), STEP = SPLIT ? kMergeWaves : 1;
  const int s = blockIdx.z, kvh = blockIdx.y, lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row0 = (SPLIT ? (int)blockIdx.x : (int)blockIdx.x * kMergeWaves + w) * (N * ROWS);
  const int2 cuts = a.cuts[s];  // (not used where the sequence has no tree)
  const Span sp = span_of(arguments(), s);
  const int rows = sp.t.nodes * a.group, n = cuts.y;
  if (row0 >= rows || n <= 1) return;
  const int rt = row0 / kRows, d = lane % LANES * 4;
  static_assert(kRows % (N * ROWS) == 0, "a wave's rows lie in one row tile");
  const int64_t first = (int64_t)(cuts.x + kvh * n * sp.row_tiles + rt) * kRows - rt * kRows;
  const int64_t step = (int64_t)sp.row_tiles * kRows;
  int row[N];
  Partial sum[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    row[k] = min(row0 + k * ROWS + lane / LANES, rows - 1);  // (a row tile's rows are written so far)
    sum[k] = Partial{-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
  }
  int i = SPLIT ? w : 0;
  // AHEAD pieces from i on; `left` of them where they are not all there (`all`): then the split form asks for no others,
  // whose rows four waves would read again.
  auto take = [&](auto all, int left) __attribute__((always_inline)) {
    constexpr bool ALL = decltype(all)::value;
    float2 ml[AHEAD][N];
    float4 v[AHEAD][N];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (!ALL && SPLIT && u >= left) break;
      const int64_t at = first + (ALL ? i + u * STEP : min(i + u * STEP, n - 1)) * step;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        ml[u][k] = *reinterpret_cast<const float2*>(a.ml + 2 * (at + row[k]));
        v[u][k] = *reinterpret_cast<const float4*>(a.acc + (at + row[k]) * D + d);
      }
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (!ALL && SPLIT && u >= left) break;
#pragma unroll
      for (int k = 0; k < N; ++k) sum[k].join(ml[u][k], v[u][k], ALL || u < left);
    }
  };
  for (; i + (AHEAD - 1) * STEP < n; i += AHEAD * STEP) take(std::true_type{}, AHEAD);
  if (i < n) take(std::false_type{}, (n - i + STEP - 1) / STEP);
  if constexpr (SPLIT) {
    static_assert(N == 1, "a row to a lane");
    __shared__ float2 ml[kMergeWaves][64];
    __shared__ float4 acc[kMergeWaves][64];
    ml[w][lane] = make_float2(sum[0].m, sum[0].l);
    acc[w][lane] = sum[0].acc;
    __syncthreads();
    if (w != 0) return;
#pragma unroll
    for (int i = 1; i < kMergeWaves; ++i) sum[0].join(ml[i][lane], acc[i][lane], true);
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    if (row0 + k * ROWS + lane / LANES >= rows) continue;
    const int node = row[k] / a.group, g = row[k] - node * a.group;
    S* out = static_cast<S*>(a.out) + ((int64_t)(sp.t.first + node) * a.num_heads + kvh * a.group + g) * D + d;
    const Partial& x = sum[k];
    const float inv = x.l != 0.f ? 1.f / x.l : 1.f;
    const float x0 = x.acc.x * inv, x1 = x.acc.y * inv, x2 = x.acc.z * inv, x3 = x.acc.w * inv;
    if constexpr (std::is_same_v<T, f32_t>) *reinterpret_cast<float4*>(out) = make_float4(x0, x1, x2, x3);
    else *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(x0, x1), pack2<T>(x2, x3));
  }
}

// ---------------------------------------------------------------- the plan --

// Key tiles of a piece that is worth its partials, 16 bits and fp32 (whose tiles take 16 times the time).  In 16 bits 4
// and 16 measured the same or slower.
constexpr int kLeast = 8, kLeastF32 = 1;

// Parts of a segment from which on a batch is few segments in many: if its pieces are short they end all at once, and
// what the L2s then hold of partials has to leave them before the merge starts.  Written past them the wait is shorter;
// where pieces end one after the other it only costs the merge its L2 hits.  Measured (us, through / past; bf16, 32 / 8
// heads of 128): one sequence of 4,096 with 64 nodes 30.3 / 26.6, of 16,384 42.2 / 40.9, in pieces of 32 tiles of 32,768
// 60.4 / 62.9 and of 65,536 97.9 / 102.5; 64 of up to 4,096 (one or two parts) 133.7 / 139.0; 17 of up to 3,900 (fp16, 28 / 4
// heads; three) 38.8 / 42.6.
constexpr int kManyParts = 8;

struct TreePlan {
  int32_t slots, slots_full, groups, tiles;  // tiles: of the longest sequence
  int32_t cut_in;                                // pieces of a segment that the merge is made for
  size_t ml_at, cuts_at, bytes;
};
TreePlan plan_tree(int32_t num_seqs, int32_t max_nodes, int32_t H, int32_t Hkv, int32_t D, int32_t bs, int32_t MB,
                   int32_t dtype) {
  TreePlan p{};
  const int64_t row_tiles = ceil_div((int64_t)max_nodes * (H / Hkv), kRows), segments = num_seqs * row_tiles * Hkv;
  const int64_t tiles = std::max<int64_t>(1, ceil_div((int64_t)MB * bs, kTileKeys));
  p.tiles = (int32_t)std::min<int64_t>(tiles, INT32_MAX);
  p.slots = device_cu_count() * 2;
  p.slots_full = device_cu_count() * pieces_per_cu(dtype, D);
  // (The kernel goes by either.)
  const int64_t pieces = std::max(most_pieces(segments, p.slots), most_pieces(segments, p.slots_full));
  // (What the product does not take runs on the generic kernel.  The cuts count in 32 bits, a sequence's tiles in 22,
  // its row tiles in 8; a grid has fewer than 2^32 threads.)
  if ((D != 64 && D != 128) || block_shift(bs) < 0 || tiles >= 1 << 22 || row_tiles > 255 ||
      (double)segments * tiles > INT32_MAX || pieces > UINT32_MAX / kTreeThreads - 8) {
    return p;
  }
  p.cut_in = (int32_t)std::min<int64_t>(p.slots_full / segments, kManyParts);
  p.groups = (int32_t)(ceil_div(std::min(pieces, segments * tiles), 8) * 8);
  const int64_t parts = std::min<int64_t>(std::max(p.slots, p.slots_full), segments * tiles);
  p.ml_at = align_up((size_t)parts * kRows * D * 4, 256);
  p.cuts_at = p.ml_at + align_up((size_t)parts * kRows * 8, 256);
  p.bytes = p.cuts_at + align_up((size_t)num_seqs * 8, 256);
  return p;
}

template <typename T, int D>
int launch_product(const char* op, const TreeArgs& a, const TreePlan& p, hipStream_t s) {
  hipLaunchKernelGGL((tree_kernel<T, D>), dim3((unsigned)p.groups), dim3(kTreeThreads), 0, s, a);
  const int st = check_launch(op);                  // (the merge goes by what the product leaves in the workspace)
  if (st != RG_OK || p.tiles <= a.least) return st;  // nothing is cut
  auto merge = [&](auto kernel, int rows) {
    const unsigned groups = (unsigned)ceil_div((int64_t)a.max_nodes * a.group, rows * merge_rows<D>());
    hipLaunchKernelGGL(kernel, dim3(groups, (unsigned)a.num_kv_heads, (unsigned)a.num_seqs), dim3(64 * kMergeWaves), 0, s, a);
  };
  if (p.cut_in >= kManyParts) merge(tree_merge_kernel<T, D, 1, 8, true>, 1);
  else if (p.cut_in >= 2) merge(tree_merge_kernel<T, D, 1, 8, false>, kMergeWaves);
  else merge(tree_merge_kernel<T, D, 2, 2, false>, 2 * kMergeWaves);
  return check_launch(op);
}

}  // namespace

int probe_tree_attention_kernels() {
  hipFuncAttributes at;
  if (hipFuncGetAttributes(&at, reinterpret_cast<const void*>(tree_generic_kernel<bf16_t>)) != hipSuccess ||
      hipFuncGetAttributes(&at, reinterpret_cast<const void*>(tree_kernel<bf16_t, 128>)) != hipSuccess ||
      hipFuncGetAttributes(&at, reinterpret_cast<const void*>(tree_merge_kernel<bf16_t, 128, 1, 8, true>)) != hipSuccess) {
    return fail(RG_ERR_HIP, "failed to load the tree attention kernels: %s", hipGetErrorString(hipGetLastError()));
  }
  return RG_OK;
}

}  // namespace rg

using namespace rg;

extern "C" size_t rg_paged_attention_tree_workspace_bytes(int32_t num_seqs, int32_t max_nodes, int32_t num_heads,
                                                          int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                                                          int32_t max_blocks_per_seq) {
  if (num_seqs <= 0 || max_nodes <= 0 || max_nodes > kMaxTreeNodes || num_heads <= 0 || num_kv_heads <= 0 ||
      num_heads % num_kv_heads != 0 || block_size <= 0 || max_blocks_per_seq < 0 ||
      (int64_t)max_blocks_per_seq * block_size > INT32_MAX - 65536 || num_seqs > 65535 || num_heads > 65535) {
    return 0;
  }
  // (A batch of 16 bits is cut into more pieces.)
  return plan_tree(num_seqs, max_nodes, num_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq, RG_DTYPE_BF16)
      .bytes;
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
  const size_t need = rg_paged_attention_tree_workspace_bytes(num_seqs, max_nodes, num_heads, num_kv_heads, head_dim,
                                                              block_size, max_blocks_per_seq);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned16(workspace))) {
    return fail(RG_ERR_WORKSPACE, "%s: workspace of %zu bytes (16-byte aligned), %zu required", op,
                workspace ? workspace_bytes : (size_t)0, need);
  }
  TreeArgs a{};
  a.q = query;
  a.k = key_cache;
  a.v = value_cache;
  a.out = output;
  a.table = block_table;
  a.context_lens = context_lens;
  a.cu = cu_nodes;
  a.mask = tree_mask;
  a.scale_log2 = scale * kLog2e;
  a.num_heads = num_heads;
  a.num_kv_heads = num_kv_heads;
  a.head_dim = head_dim;
  a.block_size = block_size;
  a.max_blocks = max_blocks_per_seq;
  a.num_seqs = num_seqs;
  a.num_nodes = num_nodes;
  a.max_nodes = max_nodes;
  a.mask_words = mask_words;
  a.kv_stride = kv_block_stride ? kv_block_stride : block;
  if (need > 0 && aligned16(query) && aligned16(key_cache) && aligned16(value_cache) && aligned16(output) &&
      a.kv_stride * dtype_bytes(dtype) % 16 == 0) {
    const TreePlan p = plan_tree(num_seqs, max_nodes, num_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq, dtype);
    char* const ws = static_cast<char*>(workspace);
    a.acc = reinterpret_cast<float*>(ws);
    a.ml = reinterpret_cast<float*>(ws + p.ml_at);
    a.cuts = reinterpret_cast<int2*>(ws + p.cuts_at);
    // The product works with a positive scale: a negative one turns q's signs, 0 takes zeros for q.
    a.q_sign = scale == 0.f ? 0u : scale < 0.f ? 0x80008001u : 1u;
    a.scale_log2 = scale != 0.f ? fabsf(a.scale_log2) : 1.f;
    a.group = num_heads / num_kv_heads;
    a.bs_shift = block_shift(block_size);
    a.slots = p.slots;
    a.slots_full = p.slots_full;
    a.least = dtype == RG_DTYPE_F32 ? kLeastF32 : kLeast;
    a.long_piece = dtype == RG_DTYPE_F32 ? kLongPieceF32 : kLongPiece;
    a.short_piece = dtype == RG_DTYPE_F32 ? kShortPieceF32 : head_dim == 128 ? kShortPiece : 0;
    a.parts_past = p.cut_in >= kManyParts;
    return dispatch_dtype(dtype, [&](auto tag) {
      using T = decltype(tag);
      return head_dim == 128 ? launch_product<T, 128>(op, a, p, as_stream(stream))
                             : launch_product<T, 64>(op, a, p, as_stream(stream));
    });
  }
  const dim3 grid((unsigned)max_nodes, (unsigned)num_heads, (unsigned)num_seqs);
  return dispatch_dtype(dtype, [&](auto tag) {
    hipLaunchKernelGGL(tree_generic_kernel<decltype(tag)>, grid, dim3(64), 0, as_stream(stream), a);
    return check_launch(op);
  });
}
