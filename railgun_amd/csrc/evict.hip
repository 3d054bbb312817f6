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
// the order of the values, and three passes over 11, 11 and 10 bits (13, 11 and 8 for tables of more
// than 16,384 tokens) narrow the key T of the last one to be kept, each with a histogram in LDS over
// the candidates that agree with the bits found so far (after the first pass mostly few, which are
// then listed).  A kept candidate's place is then known: before
// position t lie
//   #{key > T before t} + min(#{key == T before t}, ties to keep)
// kept candidates.  The kernel leaves the kept positions in order (the caller's array, or workspace).
// evict_move_kernel copies: what a segment has to move is cut into chunks, a workgroup each.
// evict_segment_kernel does both, for many or small segments.
#include <algorithm>
#include <type_traits>

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
  int32_t block_shift;  // log2(block_size) where four scores from a multiple of four on are one load, else -1
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

constexpr uint32_t kZeroKey = 0x80000000u;  // order_key(0)

// Inclusive prefix sum over the 64 lanes with DPP: within each row of 16 lanes by shifts of 1, 2, 4 and 8, then
// lane 15 of rows 0 and 2 into rows 1 and 3, then lane 31 into rows 2 and 3.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);  // row_shr:2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);  // row_shr:4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);  // row_shr:8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return v;
}
// Sum over the threads before this one; `all`: over the workgroup.  part: NW words of LDS that no thread
// still reads; holds a barrier.
template <int NW>
__device__ __forceinline__ int block_before(int v, int lane, int w, int* part, int& all) {
  const int incl = wave_scan(v);
  if (lane == 63) part[w] = incl;
  __syncthreads();
  const int waves = wave_scan(lane < NW ? part[lane] : 0);
  all = __builtin_amdgcn_readlane(waves, 63);
  const int before = w > 0 ? __builtin_amdgcn_readlane(waves, w - 1) : 0;
  return before + incl - v;
}

// NT threads.  VPT > 0: every candidate's key sits in a register (VPT a thread, in quads of consecutive ones; a
// wave's candidates are one run), and the scores are read once.  VPT 0: longer tables read them in each pass.
//   A chain of memory round trips and barriers, and past some 16,000 candidates a workgroup's issue rate.  Per
// segment (16 layers x 16 sequences x 8 kv-heads of up to 4,096 tokens, all at once / one of 65,000): keys there
// after 3.0 / 7.9 us, T known at 8 / 16.5, positions written at 10 / 22; the launch 21-23 / 24-25 us.
// Returns, to all threads alike, whether the segment's chunks have to move in order.
template <int NT, int VPT>
__device__ __forceinline__ bool select_segment(const EvictArgs a, const Segment sg, int64_t index) {
  constexpr int NW = NT / 64;
  constexpr int NQ = VPT / 4;                    // quads of candidates in a thread's registers
  constexpr int GROUP = VPT > 0 ? NQ : 16;       // strips of 4 NT candidates whose counts are scanned together
  // Bits of the three passes: with many candidates a first pass over more bins meets fewer equal addresses in
  // the LDS atomics of a wave (65,000 candidates: 9 us over 2,048 bins, 3 over 8,192).
  constexpr int FIRST = VPT > 16 ? 13 : 11, BINS = 1 << FIRST;
  constexpr int shifts[4] = {32, 32 - FIRST, 21 - FIRST, 0};
  constexpr int BPT = BINS / NT;  // bins a thread scans
  constexpr int kList = NT == 1024 ? 2048 : 512;
  __shared__ __attribute__((aligned(16))) int hist[BINS];
  __shared__ int part[2][NW];
  __shared__ int found[3];                          // digit, candidates above it, candidates at it
  __shared__ uint32_t list[kList];                  // the candidates of the first pass's digit, where they fit
  __shared__ int listed, first_hole, last_alias;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = context_of(a, sg.seq);
  const int m = min(n, a.budget);
  int32_t* kept = a.kept + index * a.kept_stride;
  const int32_t* row = a.table + (int64_t)sg.seq * a.max_blocks;
  if (a.new_lens != nullptr && sg.layer == 0 && sg.kvh == 0 && tid == 0) a.new_lens[sg.seq] = m;
  if (n <= a.budget) {
    // (Unsigned: the caller's list may be as long as 32 bits count.)
    for (unsigned i = tid; i < (unsigned)a.kept_stride; i += NT) kept[i] = (int)i < n ? (int)i : -1;
    return false;
  }
  const int p0 = a.guarded;
  const int count = n - a.recent - p0;           // candidates, positions p0 ..
  const int take = a.budget - a.recent - p0;     // of which this many stay: 0 <= take < count
  // Four consecutive positions, from base + c on with c a multiple of four, are a lane's: quads that lie in one
  // block where the block size is a power of two, and are then read in one load (`aligned`).  Keys one at a
  // time cost an address each, which bounded this phase: 65,000 candidates 14.7 us, in quads 7.9.
  const int lead = p0 & 3, base = p0 - lead, extent = lead + count;
  const int strips = (extent + 4 * NT - 1) / (4 * NT);
  const bool aligned = a.block_shift >= 0;

  const float* cells = a.scores + sg.layer * a.score_layer_stride + (int64_t)sg.kvh * a.block_size;
  auto entry = [&](int c) { return row[(uint32_t)(base + min(c, extent - 1)) >> a.block_shift]; };
  auto read_aligned = [&](int c, int blk, uint32_t (&k)[4]) {
    const int off = (base + (min(c, extent - 1) & ~3)) & (a.block_size - 1);
    const float4 v = *reinterpret_cast<const float4*>(&cells[blk * a.score_stride + off]);
    k[0] = __float_as_uint(v.x), k[1] = __float_as_uint(v.y);
    k[2] = __float_as_uint(v.z), k[3] = __float_as_uint(v.w);
  };
  auto read_each = [&](int c, uint32_t (&k)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t p = base + min(c + j, extent - 1), b = p / (uint32_t)a.block_size;
      k[j] = __float_as_uint(cells[row[b] * a.score_stride + (p - b * (uint32_t)a.block_size)]);
    }
  };
  auto to_keys = [&](int c, uint32_t (&k)[4]) {  // of scores; of what is no candidate 0
#pragma unroll
    for (int j = 0; j < 4; ++j) k[j] = c + j >= lead && c + j < extent ? order_key(__uint_as_float(k[j])) : 0u;
  };
  uint32_t key[NQ > 0 ? NQ : 1][4] = {};
  if constexpr (VPT > 0) {
    // A table entry, then the scores it leads to: two round trips, shared by U quads.
    constexpr int U = NQ < 8 ? NQ : 8;
#pragma unroll
    for (int i0 = 0; i0 < NQ; i0 += U) {
      if (i0 < strips) {
        if (aligned) {
          int blk[U];
#pragma unroll
          for (int i = 0; i < U; ++i) blk[i] = entry(((w * strips + i0 + i) * 64 + lane) * 4);
#pragma unroll
          for (int i = 0; i < U; ++i) read_aligned(((w * strips + i0 + i) * 64 + lane) * 4, blk[i], key[i0 + i]);
        } else {
#pragma unroll
          for (int i = i0; i < i0 + U; ++i) read_each(((w * strips + i) * 64 + lane) * 4, key[i]);
        }
      }
#pragma unroll
      for (int i = i0; i < i0 + U; ++i) {
        to_keys(i < strips ? ((w * strips + i) * 64 + lane) * 4 : extent, key[i]);
        // (Finished here, not kept as scores and conditions.)
        asm volatile("" : "+v"(key[i][0]), "+v"(key[i][1]), "+v"(key[i][2]), "+v"(key[i][3]));
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  // The last entry that both tables have alike (before the first stores: a load behind them waits for them).
  const int32_t* drow = a.dst_table + (int64_t)sg.seq * a.max_dst_blocks;
  int alias = -1;
  for (int i = tid; i < (m + a.block_size - 1) / a.block_size; i += NT) {
    if (row[i] == drow[i]) alias = i;
  }
  for (int i = m + tid; i < a.kept_stride; i += NT) kept[i] = -1;
  for (int i = tid; i < a.recent; i += NT) kept[m - a.recent + i] = n - a.recent + i;
  for (int i = tid; i < p0; i += NT) kept[i] = i;
  if (tid == 0) {
    listed = 0;
    first_hole = n;
    last_alias = -1;
  }
  // f(c, the four keys of candidates c ..) over the wave's candidates of the gs strips from g0 on, 256 consecutive
  // ones at a time.  The key of what is no candidate is 0, below every score's.
  auto each = [&](int g0, int gs, auto f) __attribute__((always_inline)) {
    if constexpr (VPT > 0) {
      // (Opaque copies: comparisons are made where they are needed, not kept as masks from call to call.)
      asm volatile("" : "+s"(gs));
      int c = (w * gs * 64 + lane) * 4;
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        uint32_t k[4] = {key[i][0], key[i][1], key[i][2], key[i][3]};
        asm volatile("" : "+v"(k[0]), "+v"(k[1]), "+v"(k[2]), "+v"(k[3]), "+v"(c));
        if (i < gs) f(c + i * 256, k);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < gs; ++i) {
        const int c = g0 * NT * 4 + ((w * gs + i) * 64 + lane) * 4;
        uint32_t k[4];
        if (aligned) read_aligned(c, entry(c), k);
        else read_each(c, k);
        to_keys(c, k);
        f(c, k);
      }
    }
  };

  // T: the key of the take-th largest candidate, or below it and above every key that is not kept; `left` of
  // those at T are kept, the lowest positions first.
  uint32_t T = 0xffffffffu;  // (above every key: nothing kept)
  int left = 0;
  bool whole = false;  // every candidate at or above T is kept
  bool few = false;    // `list` holds the candidates that agree with T's first digit
  auto each_group = [&](auto f) __attribute__((always_inline)) {
    for (int g0 = 0; g0 < (VPT > 0 ? 1 : strips); g0 += GROUP) each(g0, min(GROUP, strips - g0), f);
  };
  if (take > 0) {
    T = 0;
    left = take;
#pragma unroll
    for (int ps = 0; ps < 3; ++ps) {
      if (whole) break;
      const int sh = shifts[ps + 1], hi = shifts[ps];  // bits from hi on are settled
      for (int i = 4 * tid; i < BINS; i += 4 * NT) *reinterpret_cast<int4*>(&hist[i]) = make_int4(0, 0, 0, 0);
      __syncthreads();
      int zeros = 0;
      auto count_in = [&](uint32_t k) __attribute__((always_inline)) {
        // Lanes on one address go one after the other, and a score of 0 is the one that many tokens have in
        // common (weights that underflowed): those are counted in a register.
        if (ps == 0) {
          zeros += __popcll(__ballot(k == kZeroKey));
          if (k == kZeroKey) return;
        }
        if (k != 0 && (ps == 0 || (k >> (hi & 31)) == (T >> (hi & 31))))
          atomicAdd(&hist[(k >> sh) & ((1u << (shifts[ps] - sh)) - 1u)], 1);
      };
      if (ps > 0 && few) {
        for (int i = tid; i < listed; i += NT) count_in(list[i]);
      } else {
        each_group([&](int, const uint32_t (&k)[4]) __attribute__((always_inline)) {
#pragma unroll
          for (int j = 0; j < 4; ++j) count_in(k[j]);
        });
      }
      if (ps == 0 && lane == 0 && zeros > 0) atomicAdd(&hist[kZeroKey >> sh], zeros);
      __syncthreads();
      // Candidates in higher bins; BPT bins a thread, from the top.
      int h[BPT], sum = 0;
#pragma unroll
      for (int i = 0; i < BPT; ++i) {
        h[i] = hist[BINS - 1 - tid * BPT - i];
        sum += h[i];
      }
      int all;
      int above = block_before<NW>(sum, lane, w, part[ps & 1], all);
      if (above < left && left <= above + sum) {
#pragma unroll
        for (int i = 0; i < BPT; ++i) {
          if (above < left && left <= above + h[i]) {
            found[0] = BINS - 1 - tid * BPT - i;
            found[1] = above;
            found[2] = h[i];
          }
          above += h[i];
        }
      }
      __syncthreads();
      T |= (uint32_t)found[0] << sh;
      left -= found[1];
      whole = found[2] == left;  // the digit's candidates are all kept: no need to part them further
      if (ps == 0) few = !whole && found[2] <= kList;
      if (ps == 0 && few) {
        // The other passes part those alone (in no order: they are only counted).
        auto in_digit = [&](uint32_t k) { return k - T < (1u << sh); };  // (T > 0: every score's key is)
        int mine = 0;
        each_group([&](int, const uint32_t (&k)[4]) __attribute__((always_inline)) {
#pragma unroll
          for (int j = 0; j < 4; ++j) mine += in_digit(k[j]);
        });
        const int incl = wave_scan(mine);
        int at = 0;
        if (lane == 63 && incl > 0) at = atomicAdd(&listed, incl);
        at = __builtin_amdgcn_readlane(at, 63) + incl - mine;
        each_group([&](int, const uint32_t (&k)[4]) __attribute__((always_inline)) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (in_digit(k[j])) list[at++] = k[j];
          }
        });
      }
    }
  }

  // The kept candidates in order: a wave's run of candidates is counted, and the waves' counts are scanned.  Where
  // all at T stay, which is so unless scores are equal, there are no ties to count.
  int hole = n;
  auto place = [&](auto with_ties) __attribute__((always_inline)) {
    constexpr bool TIES = decltype(with_ties)::value;
    const uint32_t above_T = TIES ? T : T - 1;
    int gt_before = 0, eq_before = 0;  // in the groups before
    for (int g0 = 0; g0 < (VPT > 0 ? 1 : strips); g0 += GROUP) {
      const int gs = min(GROUP, strips - g0);
      if (g0 > 0) __syncthreads();
      int gt = 0, eq = 0;
      each(g0, gs, [&](int, const uint32_t (&k)[4]) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          gt += k[j] > above_T;
          if constexpr (TIES) eq += k[j] == T;
        }
      });
      const int gt_scan = wave_scan(gt), eq_scan = TIES ? wave_scan(eq) : 0;
      if (lane == 63) {
        part[0][w] = gt_scan;
        part[1][w] = eq_scan;
      }
      __syncthreads();
      const int gsum = wave_scan(lane < NW ? part[0][lane] : 0), esum = TIES ? wave_scan(lane < NW ? part[1][lane] : 0) : 0;
      const int gall = __builtin_amdgcn_readlane(gsum, 63), eall = __builtin_amdgcn_readlane(esum, 63);
      int g = gt_before + (w > 0 ? __builtin_amdgcn_readlane(gsum, w - 1) : 0);
      int e = eq_before + (w > 0 ? __builtin_amdgcn_readlane(esum, w - 1) : 0);
      each(g0, gs, [&](int c, const uint32_t (&k)[4]) __attribute__((always_inline)) {
        int mine = 0;  // (both counts in one scan, ties from bit 16 on)
#pragma unroll
        for (int j = 0; j < 4; ++j) mine += (k[j] > above_T) + (TIES && k[j] == T ? 65536 : 0);
        const int incl = wave_scan(mine), all = __builtin_amdgcn_readlane(incl, 63);
        int gl = g + ((incl - mine) & 0xffff), el = e + ((incl - mine) >> 16);
        g += all & 0xffff;
        e += all >> 16;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool is_gt = k[j] > above_T, is_eq = TIES && k[j] == T;
          if (is_gt || (is_eq && el < left)) kept[p0 + gl + (TIES ? min(el, left) : 0)] = base + c + j;
          else if (k[j] != 0) hole = min(hole, base + c + j);
          gl += is_gt;
          el += is_eq;
        }
      });
      gt_before += gall;
      eq_before += eall;
    }
  };
  if (whole) place(std::false_type{});
  else place(std::true_type{});
  // Rows from the first hole on move.  Where a block that receives them is also the block they may come
  // from (the same entry of both tables: eviction in place), the chunks go in order.
  // (One LDS atomic a wave: lanes on one address go one after the other.)
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    hole = min(hole, __shfl_xor(hole, o, 64));
    alias = max(alias, __shfl_xor(alias, o, 64));
  }
  if (lane == 0) {
    atomicMin(&first_hole, hole);
    atomicMax(&last_alias, alias);
  }
  __syncthreads();
  return last_alias >= first_hole / a.block_size;
}

template <int NT, int VPT>
__global__ __launch_bounds__(NT) void evict_select_kernel(EvictArgs a) {
  const bool in_order = select_segment<NT, VPT>(a, segment_of(a, blockIdx.x), blockIdx.x);
  if (threadIdx.x == 0) a.in_order[blockIdx.x] = in_order;
}

// ----------------------------------------------------------------- move -----

constexpr int kMoveMaxTokens = 512;
constexpr int kInPlacePieces = 8;

// Workgroup (segment, chunk), NT threads: tokens chunk * tok .. of the segment's kept list, tok such that their K
// and V rows fill U pieces V a thread, all of them read before the first is written.  A segment that is evicted in
// place is walked by its first workgroup alone: the chunk at hand is written once every thread has read its part
// of it.  That is enough: kept[j] >= j, so rows j .. of the destination never hold a row that a later chunk has
// yet to read.
//   Bound by the copy: every row is read and written once, with non-temporal accesses (no row is met again).
// Four layers x 17 sequences x 4 kv-heads of up to 1,500 kept tokens of 512 bytes (0.33 GB): 56 us with 256 threads
// of 4 pieces, the rate of a 1 GiB copy being 5.2 TB/s (64 us for these bytes); 8 pieces and ordinary accesses were
// 10 % slower.  In place the round trips of a segment's chunks follow each other, so fewer, larger ones win: two
// sequences of 65,000 tokens down to 8,192 (16 segments) took 447 us a call with 256 threads of 8 pieces, 184 with
// 1,024 of 8, 223 of 16.
//   (The arguments come by value: behind a reference the compiler kept the addresses of all pieces at once, 1,700
// registers of them spilled.)
// Chunk j0 of the segment; in order, or with ALL, that and all later ones.
template <typename V, int NT, int U, bool ALL>
__device__ __forceinline__ void move_rows(const EvictArgs a, const Segment sg, int64_t index, int row_vecs, int tok,
                                          int j0, bool in_order) {
  __shared__ int64_t src_off[2][kMoveMaxTokens], dst_off[2][kMoveMaxTokens];  // in pieces V; -1: not moved
  const int tid = threadIdx.x;
  const int m = min(context_of(a, sg.seq), a.budget);
  const int32_t* kept = a.kept + index * a.kept_stride;
  const int32_t* row = a.table + (int64_t)sg.seq * a.max_blocks;
  const int32_t* drow = a.dst_table + (int64_t)sg.seq * a.max_dst_blocks;
  constexpr int kSize = (int)sizeof(V);
  const int64_t es = (int64_t)row_vecs * kSize / a.head_dim;  // element bytes
  V* const kb = static_cast<V*>(a.k);
  V* const vb = static_cast<V*>(a.v);
  const int64_t layer = sg.layer * a.layer_stride, head = (int64_t)sg.kvh * a.block_size;
  const int per_token = 2 * row_vecs;
#pragma unroll 1
  for (int buf = 0; j0 < m; j0 += tok, buf ^= 1) {
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
    V piece[U] = {};
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = u * NT + tid, t = i / per_token, c = i - t * per_token;
      if (t < nt && src_off[buf][t] >= 0) {
        const int64_t at = src_off[buf][t];
        piece[u] = __builtin_nontemporal_load((c >= row_vecs ? vb - row_vecs : kb) + at + c);
      }
    }
    if (in_order) {
      // Every thread's reads have landed before any thread writes.
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = u * NT + tid, t = i / per_token, c = i - t * per_token;
      if (t < nt && src_off[buf][t] >= 0) {
        const int64_t at = dst_off[buf][t];
        __builtin_nontemporal_store(piece[u], (c >= row_vecs ? vb - row_vecs : kb) + at + c);
      }
    }
    if (to_cell >= 0) a.scores[to_cell] = score;
    if (!ALL && !in_order) break;
  }
}

template <typename V, int NT, int U>
__global__ __launch_bounds__(NT) void evict_move_kernel(EvictArgs a, int row_vecs, int tok) {
  const bool in_order = a.in_order[blockIdx.x] != 0;
  // (A grid has no more than 65,535 workgroups in y, and rows in 2-byte pieces make chunks of a single token.)
  const int64_t chunk = (int64_t)blockIdx.z * gridDim.y + blockIdx.y;
  if ((in_order && chunk != 0) || chunk * tok >= a.budget) return;
  move_rows<V, NT, U, false>(a, segment_of(a, blockIdx.x), blockIdx.x, row_vecs, tok, (int)(chunk * tok), in_order);
}

// Both in one launch, a workgroup per segment: where there are segments enough to fill the chip with one each (the
// moves of some then hide the selection of others), or where a segment moves no more than two chunks.  Else the
// chunks that follow each other in a workgroup cost more than the second launch.  Measured (us, two launches / one;
// rows of 128 bytes): 2,048 segments of 1,024 kept tokens 249 / 231 (in place 225 / 209), 1,024 of 2,000 230 / 225, 48
// of 128 with 256-byte rows 13.0 / 10.6, 256 of 256 15.7 / 14.4; 272 of up to 1,500 with 256-byte rows 64 / 92,
// 64 of 512 13.3 / 16.0.
constexpr int kSegThreads = 512, kSegKeys = 8, kSegPieces = 4;
__global__ __launch_bounds__(kSegThreads) void evict_segment_kernel(EvictArgs a, int row_vecs, int tok) {
  const Segment sg = segment_of(a, blockIdx.x);
  const bool in_order = select_segment<kSegThreads, kSegKeys>(a, sg, blockIdx.x);
  __syncthreads();  // the kept positions stand for the workgroup
  move_rows<rg_u32x4_t, kSegThreads, kSegPieces, true>(a, sg, blockIdx.x, row_vecs, tok, 0, in_order);
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
  if (hipFuncGetAttributes(&at, reinterpret_cast<const void*>(evict_select_kernel<256, 16>)) != hipSuccess ||
      hipFuncGetAttributes(&at, reinterpret_cast<const void*>(evict_segment_kernel)) != hipSuccess ||
      hipFuncGetAttributes(&at, reinterpret_cast<const void*>(evict_move_kernel<rg_u32x4_t, 256, 4>)) != hipSuccess) {
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
  if (table_tokens > INT32_MAX - 65536) {  // (positions are counted in 32 bits, up to a group past the last)
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
  const size_t need = evict_bytes(segments, most, kept_positions == nullptr);
  if (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 3u) != 0) {
    return fail(RG_ERR_WORKSPACE, "%s: workspace of %zu bytes (4-byte aligned), %zu required", op,
                workspace ? workspace_bytes : (size_t)0, need);
  }
  // (The lengths are read by every segment while the new ones are written.)
  const auto lens_at = reinterpret_cast<uintptr_t>(context_lens), new_at = reinterpret_cast<uintptr_t>(new_context_lens);
  if (new_context_lens != nullptr && lens_at < new_at + 4 * (uintptr_t)batch_size &&
      new_at < lens_at + 4 * (uintptr_t)batch_size) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: new_context_lens overlaps context_lens", op);
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
  a.kept_stride = kept_positions ? budget : (int32_t)most;
  a.budget = budget;
  a.recent = recent;
  a.guarded = protected_len;
  a.num_kv_heads = num_kv_heads;
  a.head_dim = head_dim;
  a.block_size = block_size;
  a.max_blocks = max_blocks_per_seq;
  a.max_dst_blocks = dst_block_table ? max_dst_blocks_per_seq : max_blocks_per_seq;
  a.batch = batch_size;
  const bool quads = block_size >= 4 && (block_size & (block_size - 1)) == 0 && score_stride % 4 == 0 &&
                     a.score_layer_stride % 4 == 0 && (reinterpret_cast<uintptr_t>(scores) & 15u) == 0;
  a.block_shift = quads ? __builtin_ctz((unsigned)block_size) : -1;
  hipStream_t s = as_stream(stream);
  const dim3 sel((unsigned)segments);
  // Rows move in 16-byte pieces where every row starts on one, else in 2-byte ones.
  auto whole = [&](int64_t elements) { return elements * eb % 16 == 0; };
  const bool wide = whole(head_dim) && whole(kv_stride) && whole(a.layer_stride) &&
                    ((reinterpret_cast<uintptr_t>(key_cache) | reinterpret_cast<uintptr_t>(value_cache)) & 15u) == 0;
  const int row_vecs = head_dim * eb / (wide ? 16 : 2);
  // Tokens of a chunk.  (A thread looks one token up: no more tokens than threads, which rows of a single piece
  // would allow.)
  auto chunk = [&](int threads, int pieces) {
    return std::max(1, std::min({kMoveMaxTokens, threads, threads * pieces / (2 * row_vecs)}));
  };
  if (wide && table_tokens <= kSegThreads * kSegKeys &&
      (segments >= 4 * (int64_t)device_cu_count() || most * 2 * row_vecs <= 2 * kSegThreads * kSegPieces)) {
    hipLaunchKernelGGL(evict_segment_kernel, sel, dim3(kSegThreads), 0, s, a, row_vecs, chunk(kSegThreads, kSegPieces));
    return check_launch(op);
  }
  auto select = [&](auto kernel, int threads) { hipLaunchKernelGGL(kernel, sel, dim3(threads), 0, s, a); };
  if (table_tokens <= 256 * 4) select(evict_select_kernel<256, 4>, 256);
  else if (table_tokens <= 256 * 16) select(evict_select_kernel<256, 16>, 256);
  else if (table_tokens <= 1024 * 16) select(evict_select_kernel<1024, 16>, 1024);
  else if (table_tokens <= 1024 * 64) select(evict_select_kernel<1024, 64>, 1024);
  else select(evict_select_kernel<1024, 0>, 1024);
  int st = check_launch(op);
  if (st != RG_OK || most == 0) return st;
  auto move = [&](auto kernel, int threads, int pieces) {
    const int tok = chunk(threads, pieces);
    const int64_t chunks = dst_block_table == nullptr ? 1 : ceil_div(most, tok);
    const unsigned y = (unsigned)std::min<int64_t>(chunks, 65535), z = (unsigned)ceil_div(chunks, y);
    hipLaunchKernelGGL(kernel, dim3((unsigned)segments, y, z), dim3(threads), 0, s, a, row_vecs, tok);
    return check_launch(op);
  };
  // (In place without a second table no segment has use for more than one workgroup.)
  if (dst_block_table == nullptr) {
    return wide ? move(evict_move_kernel<rg_u32x4_t, 1024, kInPlacePieces>, 1024, kInPlacePieces)
                : move(evict_move_kernel<uint16_t, 1024, kInPlacePieces>, 1024, kInPlacePieces);
  }
  return wide ? move(evict_move_kernel<rg_u32x4_t, 256, 4>, 256, 4) : move(evict_move_kernel<uint16_t, 256, 4>, 256, 4);
}
