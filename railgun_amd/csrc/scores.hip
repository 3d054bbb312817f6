// Decode attention that also gathers, per cached token and kv-head, the softmax weight that the step's
// queries gave it:
//   out[s, h]  = sum_t p[h, t] V_t,  p[h, t] = e^(x[h, t] - M_h) / L_h,  x[h, t] = scale q[s, h] . K_t
//   scores[t] <- (t < scored_lens[s] ? scores[t] : 0) + sum over the kv-head's G query heads of p[h, t].
//
// The weights need the row's maximum and sum, which stand only once every key has been seen, and a second
// pass over K would cost half of the call's bytes again.  So the pass over K and V, the stream-K decode,
// leaves each raw score q . k in the workspace (4 G bytes a token and kv-head beside the 4 D of K and V in
// 16 bits: 6 % at G 4, head_dim 128, written and read once), and scores_finish_kernel merges the workers'
// partials into the output and turns the raw scores into weights with the merged M and L.
//
//   Bound by the stream of K and V, as the plain decode is: 64 sequences of 512 to 4,096 tokens (bf16, 32 / 8 heads
// of 128, 0.58 GB of K and V) 114 us a call, 101 in the stream (the plain decode's whole call 99) and 10 in the
// finish, whose launch and round trips are most of it; 4 of 32,000 tokens 95 (88).
//
// Shapes outside the tiles (another head_dim, block size or ratio of heads) take scores_generic_kernel, one
// wave per (partition of kGenTokens tokens, query head, sequence), before the same finish.
#include "decode_stream.hpp"

namespace rg {
namespace {

constexpr int kGenTokens = 256;
constexpr int kFinThreads = 256;
constexpr int kFinWaves = kFinThreads / 64;
constexpr int kFinTokens = 1024;   // tokens a workgroup turns into weights at a time
constexpr int kMaxGroup = 512;     // query heads to a kv-head
constexpr int kShortMaxScored = 1024;  // tokens of table that the one-launch kernel holds old scores of

struct ScoreArgs {
  void* out;
  float* scores;
  const float* logits;        // [batch, H_kv, tokens, G] raw scores
  const float* part_acc;      // partials as the stream-K workers leave them
  const float* part_ml;
  const int2* seg_desc;       // null: partial p of segment g is g * num_partitions + p
  const int32_t* block_table;
  const int32_t* context_lens;
  const int32_t* scored_lens;  // may be null: every cell holds a score
  float scale_log2;
  int32_t first;
  int32_t num_heads, num_kv_heads, head_dim, block_size, max_blocks, num_partitions;
  int64_t score_stride;
  int32_t merge_groups, merge_heads;  // workgroups of a segment that merge, and query heads to each (1 or 4)
};

template <typename T, int D, int G>
__global__ __launch_bounds__(64) void scores_stream_kernel(StreamArgs a, const typename DecodeTileFor<T, D, G>::S* __restrict__ q,
                                                           const typename DecodeTileFor<T, D, G>::S* __restrict__ kc,
                                                           const typename DecodeTileFor<T, D, G>::S* __restrict__ vc,
                                                           const int32_t* __restrict__ block_table,
                                                           const int32_t* __restrict__ context_lens) {
  stream_worker<T, D, G, false, StreamVariant::kScores>(a, q, kc, vc, block_table, context_lens, nullptr, nullptr,
                                                        blockIdx.x, 0, threadIdx.x);
}

struct GenericArgs {
  const void* q;
  const void* k_cache;
  const void* v_cache;
  const int32_t* block_table;
  const int32_t* context_lens;
  float* logits;
  float* part_acc;
  float* part_ml;
  float scale_log2;
  int32_t first;
  int32_t num_heads, num_kv_heads, head_dim, block_size, max_blocks, num_partitions;
  int64_t kv_stride;
};

template <typename T>
__global__ __launch_bounds__(64) void scores_generic_kernel(GenericArgs a) {
  using E = elem<T>;
  using S = typename E::storage;
  const int p = blockIdx.x, h = blockIdx.y, s = blockIdx.z, lane = threadIdx.x;
  const int64_t tokens = (int64_t)a.max_blocks * a.block_size;
  const int ctx = (int)max<int64_t>(0, min<int64_t>(a.context_lens[s], tokens));
  const int t0 = p * kGenTokens, t1 = min(ctx, t0 + kGenTokens);
  if (t0 >= t1) return;
  const int D = a.head_dim, G = a.num_heads / a.num_kv_heads;
  const int kvh = h / G, g = h - kvh * G;
  const int d0 = lane * 4;
  const bool act = d0 < D;
  const S* qp = static_cast<const S*>(a.q) + ((int64_t)s * a.num_heads + h) * D;
  const S* kc = static_cast<const S*>(a.k_cache);
  const S* vc = static_cast<const S*>(a.v_cache);
  const int32_t* bt = a.block_table + (int64_t)s * a.max_blocks;
  const int64_t seg = (int64_t)s * a.num_kv_heads + kvh;
  float qv[4] = {0.f, 0.f, 0.f, 0.f};
  if (act) {
#pragma unroll
    for (int u = 0; u < 4; ++u) qv[u] = E::load(qp, d0 + u);
  }
  float m = -INFINITY, l = 0.f;
  float o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int t = t0; t < t1; ++t) {
    const int64_t row = bt[t / a.block_size] * a.kv_stride + ((int64_t)kvh * a.block_size + t % a.block_size) * D;
    float kv[4] = {0.f, 0.f, 0.f, 0.f}, vv[4] = {0.f, 0.f, 0.f, 0.f};
    if (act) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        kv[u] = E::load(kc, row + d0 + u);
        vv[u] = E::load(vc, row + d0 + u);
      }
    }
    const float raw = wave_sum(qv[0] * kv[0] + qv[1] * kv[1] + qv[2] * kv[2] + qv[3] * kv[3]);
    if (lane == 0 && t >= a.first) a.logits[(seg * tokens + t) * G + g] = raw;
    const float x = raw * a.scale_log2;
    const float m_new = fmaxf(m, x);
    const float alpha = exp2f(m - m_new), pe = exp2f(x - m_new);
    l = l * alpha + pe;
#pragma unroll
    for (int u = 0; u < 4; ++u) o[u] = o[u] * alpha + pe * vv[u];
    m = m_new;
  }
  const int64_t part = seg * a.num_partitions + p;
  if (act) {
    float* dst = a.part_acc + (part * G + g) * D + d0;
#pragma unroll
    for (int u = 0; u < 4; ++u) dst[u] = o[u];
  }
  if (lane == 0) {
    a.part_ml[(part * G + g) * 2] = m;
    a.part_ml[(part * G + g) * 2 + 1] = l;
  }
}

// Workgroup (x, kv-head, sequence): the first merge_groups merge the partials of merge_heads query heads each
// into their output rows, the others turn raw scores into weights, kFinTokens tokens at a time.  Each works out
// the maxima and sums it needs from the partials' pairs itself (a few loads), so one launch does both.  The call
// is short against memory latency: what does not depend on the pairs (the accumulators of the merge, the raw
// scores, the old ones) is asked for before they are waited for.  GT: G, or 0 for one known at run time.
template <typename T, int GT>
__global__ __launch_bounds__(kFinThreads) void scores_finish_kernel(ScoreArgs a) {
  using E = elem<T>;
  using S = typename E::storage;
  constexpr int GL = GT > 0 ? GT : kMaxGroup;
  constexpr int UNROLL = kFinTokens / kFinThreads;
  __shared__ float top[GL], inv[GL];
  __shared__ float4 sums[kFinThreads];
  const int kvh = blockIdx.y, s = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int G = GT > 0 ? GT : a.num_heads / a.num_kv_heads;
  const int D = a.head_dim;
  const int64_t tokens = (int64_t)a.max_blocks * a.block_size;
  const int64_t seg = (int64_t)s * a.num_kv_heads + kvh;
  const int2 desc = a.seg_desc != nullptr ? a.seg_desc[seg] : make_int2(0, 0);  // (with the length: one round trip)
  const int ctx = (int)max<int64_t>(0, min<int64_t>(a.context_lens[s], tokens));
  const bool merges = (int)blockIdx.x < a.merge_groups;
  S* out = static_cast<S*>(a.out) + ((int64_t)s * a.num_heads + (int64_t)kvh * G) * D;
  if (ctx == 0) {
    if (blockIdx.x == 0)
      for (int i = tid; i < G * D; i += kFinThreads) E::store(out, i, 0.f);
    return;
  }
  const int64_t first = max(a.first, 0) + (int64_t)((int)blockIdx.x - a.merge_groups) * kFinTokens;
  if (!merges && first >= ctx) return;
  const int64_t pbase = a.seg_desc != nullptr ? desc.x + seg : seg * a.num_partitions;
  const int np = a.seg_desc != nullptr ? desc.y : (ctx + kGenTokens - 1) / kGenTokens;
  const float* ml = a.part_ml + pbase * 2 * G;
  auto pair = [&](int q, int h) { return *reinterpret_cast<const float2*>(ml + ((int64_t)q * G + h) * 2); };
  // Maximum and sum of head h over its partials, in every lane of the wave.
  auto stats = [&](int h, float& m, float& l) {
    m = -INFINITY;
    l = 0.f;
    for (int q0 = 0; q0 < np; q0 += 64) {
      const float2 p = q0 + lane < np ? pair(q0 + lane, h) : make_float2(-INFINITY, 0.f);
      const float mn = fmaxf(m, wave_max(p.x));
      l = l * exp2f(m - mn) + wave_sum(p.y * exp2f(p.x - mn));
      m = mn;
    }
  };
  if (merges) {
    // Whole waves to a head; in it four dims a thread, R partials at a time, their sums added in a fixed order.
    const int per = kFinThreads / a.merge_heads, hw = tid / per, t = tid - hw * per;
    const int h = min((int)blockIdx.x * a.merge_heads + hw, G - 1);
    const int C = D / 4, R = per / C, c = t % C, r = t / C;
    const float* acc = a.part_acc + (pbase * G + h) * D + 4 * c;
    constexpr int AHEAD = 2;
    float4 v[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int q = r + i * R;
      v[i] = r < R && q < np ? *reinterpret_cast<const float4*>(acc + (int64_t)q * G * D) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float m, l;
    stats(h, m, l);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float4 x, int q) {
      const float f = exp2f(pair(q, h).x - m);
      o.x += f * x.x;
      o.y += f * x.y;
      o.z += f * x.z;
      o.w += f * x.w;
    };
    if (r < R) {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (r + i * R < np) add(v[i], r + i * R);
#pragma unroll 4
      for (int q = r + AHEAD * R; q < np; q += R) add(*reinterpret_cast<const float4*>(acc + (int64_t)q * G * D), q);
    }
    sums[tid] = o;
    __syncthreads();
    if (t < C && (int)blockIdx.x * a.merge_heads + hw < G) {
      for (int i = 1; i < min(R, np); ++i) {
        const float4 x = sums[tid + i * C];
        o.x += x.x;
        o.y += x.y;
        o.z += x.z;
        o.w += x.w;
      }
      const float f = l != 0.f ? 1.f / l : 1.f;
      S* row = out + (int64_t)h * D + 4 * t;
      E::store(row, 0, o.x * f);
      E::store(row, 1, o.y * f);
      E::store(row, 2, o.z * f);
      E::store(row, 3, o.w * f);
    }
    return;
  }
  const int scored = a.scored_lens != nullptr ? a.scored_lens[s] : INT32_MAX;
  const int32_t* bt = a.block_table + (int64_t)s * a.max_blocks;
  const float* lg = a.logits + seg * tokens * G;
  float* const cells = a.scores + (int64_t)kvh * a.block_size;
  const int64_t step = (int64_t)(gridDim.x - a.merge_groups) * kFinTokens;
  bool known = false;
  for (int64_t c0 = first; c0 < ctx; c0 += step) {
    // The chunk's cells, old scores and raw scores (a token past the end reads the last one's).
    float* cell[UNROLL];
    float old[UNROLL], raw[UNROLL][GT > 0 ? GT : 1];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int t = (int)min<int64_t>(c0 + u * kFinThreads + tid, ctx - 1), b = t / a.block_size;
      cell[u] = cells + bt[b] * a.score_stride + (t - b * a.block_size);
      if constexpr (GT > 0 && GT % 4 == 0) {
#pragma unroll
        for (int h = 0; h < GT; h += 4) {
          const float4 x = *reinterpret_cast<const float4*>(lg + (int64_t)t * GT + h);
          raw[u][h] = x.x;
          raw[u][h + 1] = x.y;
          raw[u][h + 2] = x.z;
          raw[u][h + 3] = x.w;
        }
      } else if constexpr (GT > 0) {
#pragma unroll
        for (int h = 0; h < GT; ++h) raw[u][h] = lg[(int64_t)t * GT + h];
      }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) old[u] = *cell[u];
    if (!known) {
      for (int h = w; h < G; h += kFinWaves) {
        float m, l;
        stats(h, m, l);
        if (lane == 0) {
          top[h] = m;
          inv[h] = l != 0.f ? 1.f / l : 1.f;
        }
      }
      __syncthreads();
      known = true;
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int64_t t = c0 + u * kFinThreads + tid;
      float sum = 0.f;
      if constexpr (GT > 0) {
#pragma unroll
        for (int h = 0; h < GT; ++h) sum += exp2f(raw[u][h] * a.scale_log2 - top[h]) * inv[h];
      } else if (t < ctx) {
        for (int h = 0; h < G; ++h) sum += exp2f(lg[t * G + h] * a.scale_log2 - top[h]) * inv[h];
      }
      if (t < ctx) *cell[u] = t < scored ? old[u] + sum : sum;
    }
  }
}

// Tables of few tokens (short_applies): one workgroup per segment does it all, one launch.  Its waves take the
// 16-token sub-blocks in turn, as the plain decode's kernel for such tables does; the raw scores stay in LDS
// (`raw`, [tokens][G]), and once the waves' partials are merged every thread turns some tokens' into weights.
//   Bound by latency: two sequences of up to 77 tokens in fp32 (32 / 8 heads of 64) 11.5 us a call, with the
// worker and the finish kernel 14.5.
template <typename T, int D, int G>
__global__ __launch_bounds__(kShortThreads) void scores_short_kernel(
    ScoreArgs a, int64_t kv_stride, int bs_shift, const typename DecodeTileFor<T, D, G>::S* __restrict__ q,
    const typename DecodeTileFor<T, D, G>::S* __restrict__ kc, const typename DecodeTileFor<T, D, G>::S* __restrict__ vc) {
  using Tile = DecodeTileFor<T, D, G>;
  using E = elem<T>;
  constexpr int GP = Tile::GP, HG = Tile::HG, NK = Tile::NK, NV = Tile::NV;
  constexpr int AHEAD = std::is_same_v<T, f32_t> && D == 128 ? 1 : 2, NBUF = AHEAD + 1;
  extern __shared__ float raw[];
  __shared__ float p_lds[kShortWaves][2][kBS * GP];
  __shared__ float alpha_lds[kShortWaves][2][GP];
  __shared__ float acc_lds[kShortWaves][G * D];
  __shared__ float ml_lds[kShortWaves][2][GP];
  const int kvh = blockIdx.x, s = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int max_subs = a.max_blocks << bs_shift, sub_mask = (1 << bs_shift) - 1;
  // Sub-block w + kShortWaves lane of the table row, within the row whatever the context is.
  const int sb = w + kShortWaves * lane;
  const int32_t* row = a.block_table + (int64_t)s * a.max_blocks;
  const int entry = sb < max_subs ? row[sb >> bs_shift] : 0;
  const int len = a.context_lens[s];
  const int scored = a.scored_lens != nullptr ? a.scored_lens[s] : INT32_MAX;
  Tile tile;
  tile.init(lane);
  tile.reset();
  tile.load_q(q + ((int64_t)s * a.num_heads + (int64_t)kvh * G) * D);
  const int ctx = max(0, min(len, max_subs * kBS));
  // The old scores of this thread's tokens, behind nothing but the table.
  constexpr int PER = (kShortMaxScored + kShortThreads - 1) / kShortThreads;
  float old[PER];
  float* cell[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int t = a.first + tid + i * kShortThreads;
    cell[i] = nullptr;
    old[i] = 0.f;
    if (t < ctx) {
      const int b = t >> (4 + bs_shift);
      cell[i] = a.scores + row[b] * a.score_stride + (int64_t)kvh * a.block_size + (t - (b << (4 + bs_shift)));
      if (t < scored) old[i] = *cell[i];
    }
  }
  const int nblk = (ctx + kBS - 1) / kBS;
  const int nb = w < nblk ? (nblk - w + kShortWaves - 1) / kShortWaves : 0;  // this wave's sub-blocks
  if (nb > 0) {
    const int64_t head = (int64_t)kvh * (kBS << bs_shift) * D;
    uint4 kbuf[NBUF][NK], vbuf[NBUF][NV];
    auto load_block = [&](int j, uint4 (&kk)[NK], uint4 (&vv)[NV]) __attribute__((always_inline)) {
      const int e = __builtin_amdgcn_readlane(entry, j);
      const int64_t off = (int64_t)e * kv_stride + head + (int64_t)((w + kShortWaves * j) & sub_mask) * (kBS * D);
      tile.template load_part<1, 0>(kc + off, vc + off, kk, vv);
    };
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) load_block(min(u, nb - 1), kbuf[u], vbuf[u]);
    for (int j0 = 0; j0 < nb; j0 += NBUF) {
#pragma unroll
      for (int u = 0; u < NBUF; ++u) {
        const int j = j0 + u;
        if (j < nb) {
          load_block(min(j + AHEAD, nb - 1), kbuf[(u + AHEAD) % NBUF], vbuf[(u + AHEAD) % NBUF]);
          const int tok0 = (w + kShortWaves * j) * kBS;
          tile.step(kbuf[u], vbuf[u], tok0, ctx, a.scale_log2, p_lds[w][j & 1], alpha_lds[w][j & 1],
                    [&](const f32x4_t (&c)[1]) __attribute__((always_inline)) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (4 * tile.seg + r < G) raw[(tok0 + tile.col) * G + 4 * tile.seg + r] = c[0][r];
          });
        }
      }
    }
  }
  float lsum[4];
  tile.reduce(lsum);
  if (tile.vrow == 0) {
#pragma unroll
    for (int h = 0; h < G; ++h) {
      float4* dst = reinterpret_cast<float4*>(&acc_lds[w][h * D + tile.vd0]);
#pragma unroll
      for (int q4 = 0; q4 < Tile::ACC / 4; ++q4)
        dst[q4] = make_float4(tile.acc[h][4 * q4], tile.acc[h][4 * q4 + 1], tile.acc[h][4 * q4 + 2],
                              tile.acc[h][4 * q4 + 3]);
    }
  }
  if (tile.seg < HG && tile.col == 0) {
    *reinterpret_cast<float4*>(&ml_lds[w][0][4 * tile.seg]) =
        make_float4(tile.m_run[0], tile.m_run[1], tile.m_run[2], tile.m_run[3]);
    *reinterpret_cast<float4*>(&ml_lds[w][1][4 * tile.seg]) = make_float4(lsum[0], lsum[1], lsum[2], lsum[3]);
  }
  __syncthreads();
  // M and 1 / L of head h over the waves.
  auto stats = [&](int h, float& M, float& inv) __attribute__((always_inline)) {
    M = -INFINITY;
#pragma unroll
    for (int ww = 0; ww < kShortWaves; ++ww) M = fmaxf(M, ml_lds[ww][0][h]);
    float L = 0.f;
#pragma unroll
    for (int ww = 0; ww < kShortWaves; ++ww) {
      const float mw = ml_lds[ww][0][h];
      L += (mw == -INFINITY ? 0.f : exp2f(mw - M)) * ml_lds[ww][1][h];
    }
    inv = L != 0.f ? 1.f / L : 1.f;
  };
  for (int i = tid; i < G * D; i += kShortThreads) {
    const int h = i / D;
    float M, inv, o = 0.f;
    stats(h, M, inv);
#pragma unroll
    for (int ww = 0; ww < kShortWaves; ++ww) {
      const float mw = ml_lds[ww][0][h];
      o += (mw == -INFINITY ? 0.f : exp2f(mw - M)) * acc_lds[ww][i];
    }
    E::store(static_cast<typename E::storage*>(a.out), ((int64_t)s * a.num_heads + (int64_t)kvh * G) * D + i, o * inv);
  }
  if (a.first >= ctx) return;
  float M[G], inv[G];
#pragma unroll
  for (int h = 0; h < G; ++h) stats(h, M[h], inv[h]);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int t = a.first + tid + i * kShortThreads;
    if (t < ctx) {
      float sum = 0.f;
#pragma unroll
      for (int h = 0; h < G; ++h) sum += exp2f(raw[t * G + h] * a.scale_log2 - M[h]) * inv[h];
      *cell[i] = old[i] + sum;
    }
  }
}

// The one-launch kernel takes what the plain decode's takes (up to 896 tokens of table at head_dim 64 and 320 at 128
// in 16 bits, 512 and 192 in fp32); fp32 at head_dim 128 with 8 heads to a kv-head fills the registers without the
// scores.
static_assert(short_widest_tokens(64, 2) <= kShortMaxScored && short_widest_tokens(64, 4) <= kShortMaxScored &&
              short_widest_tokens(128, 2) <= kShortMaxScored && short_widest_tokens(128, 4) <= kShortMaxScored);
bool scores_short_applies(const Shape& sh, int32_t dtype) {
  return short_applies(sh, dtype_bytes(dtype)) &&
         !(dtype == RG_DTYPE_F32 && sh.D == 128 && sh.H / sh.Hkv == 8);
}

template <typename T>
void launch_scores_short(const ScoreArgs& f, int64_t kv_stride, int bs_shift, const Shape& sh, const void* q,
                         const void* kc, const void* vc, hipStream_t s) {
  auto go = [&](auto d, auto g) {
    constexpr int D = decltype(d)::value, G = decltype(g)::value;
    using S = typename DecodeTileFor<T, D, G>::S;
    hipLaunchKernelGGL((scores_short_kernel<T, D, G>), dim3(sh.Hkv, sh.B), dim3(kShortThreads),
                       (size_t)sh.MB * sh.bs * G * 4, s, f, kv_stride, bs_shift, static_cast<const S*>(q),
                       static_cast<const S*>(kc), static_cast<const S*>(vc));
  };
  auto by_group = [&](auto d) {
    switch (sh.H / sh.Hkv) {
      case 1: go(d, std::integral_constant<int, 1>{}); break;
      case 2: go(d, std::integral_constant<int, 2>{}); break;
      case 3: go(d, std::integral_constant<int, 3>{}); break;
      case 4: go(d, std::integral_constant<int, 4>{}); break;
      case 5: go(d, std::integral_constant<int, 5>{}); break;
      case 6: go(d, std::integral_constant<int, 6>{}); break;
      case 7: go(d, std::integral_constant<int, 7>{}); break;
      default:  // 8
        if constexpr (!(std::is_same_v<T, f32_t> && decltype(d)::value == 128)) go(d, std::integral_constant<int, 8>{});
        break;
    }
  };
  if (sh.D == 128) by_group(std::integral_constant<int, 128>{});
  else by_group(std::integral_constant<int, 64>{});
}

template <typename T, int D>
void launch_scores_stream(const StreamArgs& sa, int G, const void* q, const void* kc, const void* vc, const int32_t* bt,
                          const int32_t* cl, hipStream_t s) {
  auto go = [&](auto g) {
    constexpr int GC = decltype(g)::value;
    using S = typename DecodeTileFor<T, D, GC>::S;
    hipLaunchKernelGGL((scores_stream_kernel<T, D, GC>), dim3(sa.num_workers), dim3(64), 0, s, sa,
                       static_cast<const S*>(q), static_cast<const S*>(kc), static_cast<const S*>(vc), bt, cl);
  };
  switch (G) {
    case 1: go(std::integral_constant<int, 1>{}); break;
    case 2: go(std::integral_constant<int, 2>{}); break;
    case 4: go(std::integral_constant<int, 4>{}); break;
    case 8: go(std::integral_constant<int, 8>{}); break;
    case 16:
      if constexpr (D <= 128) go(std::integral_constant<int, 16>{});
      break;
    default:
      // G 3, 5, 6, 7 (mfma_group_size admits them at head_dim 64 and 128 only)
      if constexpr (D <= 128) {
        if (G == 3) go(std::integral_constant<int, 3>{});
        else if (G == 5) go(std::integral_constant<int, 5>{});
        else if (G == 6) go(std::integral_constant<int, 6>{});
        else if (G == 7) go(std::integral_constant<int, 7>{});
      }
      break;
  }
}

// A form of its own for every ratio that the tiles take: with G known the raw scores are asked for before the
// pairs are waited for, else behind them.  Measured (the form for any G / its own, us a call; 16 sequences of 500
// to 2,000 tokens, bf16, 8 kv-heads of 128): G 3 25.6 / 24.2, 5 29.3 / 26.4, 6 34.0 / 29.7; 2 kv-heads, G 16
// 28.7 / 27.8; 64 sequences of 500 to 4,000, G 5 125.6 / 120.5; 8 of 64, G 3 21.4 / 19.3; fp32, 8 of 128, G 3
// 38.9 / 36.9.
template <typename T>
void launch_finish(const ScoreArgs& a, int G, dim3 grid, hipStream_t s) {
  auto go = [&](auto g) {
    hipLaunchKernelGGL((scores_finish_kernel<T, decltype(g)::value>), grid, dim3(kFinThreads), 0, s, a);
  };
  switch (G) {
    case 1: go(std::integral_constant<int, 1>{}); break;
    case 2: go(std::integral_constant<int, 2>{}); break;
    case 3: go(std::integral_constant<int, 3>{}); break;
    case 4: go(std::integral_constant<int, 4>{}); break;
    case 5: go(std::integral_constant<int, 5>{}); break;
    case 6: go(std::integral_constant<int, 6>{}); break;
    case 7: go(std::integral_constant<int, 7>{}); break;
    case 8: go(std::integral_constant<int, 8>{}); break;
    case 16: go(std::integral_constant<int, 16>{}); break;
    default: go(std::integral_constant<int, 0>{}); break;
  }
}

int32_t generic_partitions(const Shape& sh) {
  return (int32_t)std::max<int64_t>(1, ceil_div((int64_t)sh.MB * sh.bs, kGenTokens));
}

struct ScoreScratch {
  float* logits;
  void* rest;  // stream-K scratch, or the generic kernel's partials
};

size_t logit_bytes(const Shape& sh) { return align_up((size_t)sh.B * sh.H * sh.MB * sh.bs * 4, 256); }
size_t generic_acc_bytes(const Shape& sh) {
  return align_up((size_t)sh.B * sh.H * generic_partitions(sh) * sh.D * 4, 256);
}
size_t generic_bytes(const Shape& sh) {
  return generic_acc_bytes(sh) + align_up((size_t)sh.B * sh.H * generic_partitions(sh) * 8, 256);
}

// What the entry refuses for its size (the last line: a workspace of more bytes than 64 bits count).
bool too_large(const Shape& sh) {
  const int64_t tokens = (int64_t)sh.MB * sh.bs;
  return tokens > INT32_MAX || sh.B > 65535 || sh.H > 65535 || (int64_t)sh.B * sh.H * tokens > (int64_t)1 << 48;
}

}  // namespace

int probe_scores_kernels() {
  hipFuncAttributes at;
  if (hipFuncGetAttributes(&at, reinterpret_cast<const void*>(scores_stream_kernel<bf16_t, 128, 4>)) != hipSuccess ||
      hipFuncGetAttributes(&at, reinterpret_cast<const void*>(scores_finish_kernel<bf16_t, 4>)) != hipSuccess) {
    return fail(RG_ERR_HIP, "failed to load the scoring decode kernels: %s", hipGetErrorString(hipGetLastError()));
  }
  return RG_OK;
}

}  // namespace rg

using namespace rg;

extern "C" size_t rg_paged_attention_v1_scores_workspace_bytes(int32_t batch_size, int32_t num_heads,
                                                               int32_t num_kv_heads, int32_t head_dim,
                                                               int32_t block_size, int32_t max_blocks_per_seq) {
  if (batch_size <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 || head_dim <= 0 ||
      block_size <= 0 || max_blocks_per_seq <= 0) {
    return 0;
  }
  const Shape sh{num_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq, batch_size};
  if (too_large(sh)) return 0;
  return logit_bytes(sh) + std::max(generic_bytes(sh), stream_bytes(sh, stream_workers(sh), nullptr, nullptr));
}

extern "C" int rg_paged_attention_v1_scores(const void* query, const void* key_cache, const void* value_cache,
                                            const int32_t* block_table, const int32_t* context_lens, void* output,
                                            float* scores, const int32_t* scored_lens, int32_t first_scored,
                                            float scale, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                            int32_t block_size, int32_t max_blocks_per_seq, int32_t batch_size,
                                            int32_t dtype, int64_t kv_block_stride, int64_t score_block_stride,
                                            void* workspace, size_t workspace_bytes, void* stream) {
  const char* op = "paged_attention_v1_scores";
  const Shape sh{num_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq, batch_size};
  int st = check_decode_shape(op, sh, dtype, kv_block_stride);
  if (st != RG_OK) return st;
  const int64_t block = (int64_t)num_kv_heads * block_size;
  const int G = num_heads / num_kv_heads;
  if (G > kMaxGroup) {
    return fail(RG_ERR_NOT_SUPPORTED, "%s: at most %d query heads to a kv-head, got %d", op, kMaxGroup, G);
  }
  if (first_scored < 0) return fail(RG_ERR_INVALID_ARGUMENT, "%s: first_scored %d < 0", op, first_scored);
  if (score_block_stride != 0 && score_block_stride < block) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: score_block_stride %lld smaller than a block", op,
                (long long)score_block_stride);
  }
  const int64_t tokens = (int64_t)max_blocks_per_seq * block_size;
  if (too_large(sh)) {
    return fail(RG_ERR_NOT_SUPPORTED, "%s: a block table of %lld tokens, %d sequences, %d heads", op,
                (long long)tokens, batch_size, num_heads);
  }
  if (batch_size == 0) return ok();
  if (!query || !key_cache || !value_cache || !block_table || !context_lens || !output || !scores) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: null pointer argument", op);
  }
  const int64_t kv_stride = kv_block_stride ? kv_block_stride : block * head_dim;
  // (head_dim 256 with 16 heads to a kv-head fills the registers without the ring of raw scores.)
  const bool tiles = max_blocks_per_seq > 0 && !(head_dim == 256 && G == 16) &&
                     tiles_take(sh, dtype, kv_stride, query, key_cache, value_cache, output);
  const int32_t workers = stream_workers(sh);
  const size_t logits = logit_bytes(sh);
  // (A table of no blocks has no tokens: zeros, from nothing.)
  const size_t need = max_blocks_per_seq == 0 ? 0
                      : logits + (tiles ? stream_bytes(sh, workers, nullptr, nullptr) : generic_bytes(sh));
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned16(workspace))) {
    return fail(RG_ERR_WORKSPACE, "%s: workspace of %zu bytes (16-byte aligned), %zu required", op,
                workspace ? workspace_bytes : (size_t)0, need);
  }
  char* const ws = static_cast<char*>(workspace);
  hipStream_t s = as_stream(stream);
  ScoreArgs f{};
  f.out = output;
  f.scores = scores;
  f.logits = reinterpret_cast<float*>(ws);
  f.block_table = block_table;
  f.context_lens = context_lens;
  f.scored_lens = scored_lens;
  f.scale_log2 = scale * kLog2e;
  f.first = (int32_t)std::min<int64_t>(first_scored, tokens);  // (so that positions counted from it fit 32 bits)
  f.num_heads = num_heads;
  f.num_kv_heads = num_kv_heads;
  f.head_dim = head_dim;
  f.block_size = block_size;
  f.max_blocks = max_blocks_per_seq;
  f.num_partitions = generic_partitions(sh);
  f.score_stride = score_block_stride ? score_block_stride : block;
  if (tiles && scores_short_applies(sh, dtype)) {
    return dispatch_dtype(dtype, [&](auto tag) {
      launch_scores_short<decltype(tag)>(f, kv_stride, block_shift(block_size), sh, query, key_cache, value_cache, s);
      return check_launch(op);
    });
  }
  if (tiles) {
    StreamScratch sc;
    stream_bytes(sh, workers, &sc, ws + logits);
    StreamArgs sa{};
    sa.part_acc = sc.acc;
    sa.part_ml = sc.ml;
    sa.seg_desc = sc.desc;
    sa.scale_log2 = f.scale_log2;
    sa.num_heads = num_heads;
    sa.num_kv_heads = num_kv_heads;
    sa.bs_shift = block_shift(block_size);
    sa.max_blocks = max_blocks_per_seq << sa.bs_shift;
    sa.batch = batch_size;
    sa.num_workers = workers;
    sa.kv_stride = kv_stride;
    sa.table_stride = max_blocks_per_seq;
    sa.logits = reinterpret_cast<float*>(ws);
    f.part_acc = sc.acc;
    f.part_ml = sc.ml;
    f.seg_desc = sc.desc;
    auto go = [&](auto tag) {
      using T = decltype(tag);
      if (head_dim == 256) launch_scores_stream<T, 256>(sa, G, query, key_cache, value_cache, block_table, context_lens, s);
      else if (head_dim == 128) launch_scores_stream<T, 128>(sa, G, query, key_cache, value_cache, block_table, context_lens, s);
      else launch_scores_stream<T, 64>(sa, G, query, key_cache, value_cache, block_table, context_lens, s);
      return check_launch(op);
    };
    st = dispatch_dtype(dtype, go);
    if (st != RG_OK) return st;
  } else {
    float* const acc = reinterpret_cast<float*>(ws + logits);
    float* const ml = reinterpret_cast<float*>(ws + logits + generic_acc_bytes(sh));
    f.part_acc = acc;
    f.part_ml = ml;
    if (max_blocks_per_seq > 0) {
      GenericArgs ga{query, key_cache, value_cache, block_table, context_lens, reinterpret_cast<float*>(ws), acc, ml,
                     f.scale_log2, f.first, num_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq,
                     f.num_partitions, kv_stride};
      st = dispatch_dtype(dtype, [&](auto tag) {
        hipLaunchKernelGGL(scores_generic_kernel<decltype(tag)>, dim3(f.num_partitions, num_heads, batch_size),
                           dim3(64), 0, s, ga);
        return check_launch(op);
      });
      if (st != RG_OK) return st;
    }
  }
  // The output: a workgroup per head where a segment has many partials (a worker of the grid each, so known
  // here up to the contexts), one per four heads where it has few.  The weights: up to one per kFinTokens of the
  // table but no more than some 8192 in all (they step on where the table is longer).
  const int64_t segments = (int64_t)batch_size * num_kv_heads;
  f.merge_heads = (tiles ? workers / segments : f.num_partitions) >= 8 ? 1 : 4;
  f.merge_groups = (int32_t)ceil_div(G, f.merge_heads);
  const int64_t scored = tokens - f.first;
  const int64_t chunks = std::min(ceil_div(scored, kFinTokens), std::max<int64_t>(1, 8192 / segments));
  const dim3 grid((unsigned)(f.merge_groups + chunks), (unsigned)num_kv_heads, (unsigned)batch_size);
  return dispatch_dtype(dtype, [&](auto tag) {
    launch_finish<decltype(tag)>(f, G, grid, s);
    return check_launch(op);
  });
}
