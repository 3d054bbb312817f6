// Paged decode attention (one query token per sequence) for gfx950.
//
// Two partition kernels share one contract.  A workgroup handles one
// (partition p, kv-head, sequence) work item; partition p covers context
// tokens [p*P, min((p+1)*P, ctx)).  Depending on `mode` it writes
//   MODE_FINAL  : the normalised output (the grid has one partition per sequence)
//   MODE_PARTIAL: the unnormalised partial  tmp_out / exp_sums / max_logits
//                 (crates/vllm-cuda/src/kernels/paged_attention_v2_partition.cu:95-106)
//   MODE_AUTO   : MODE_FINAL for sequences that fit one partition, MODE_PARTIAL
//                 otherwise; the merge kernel then skips the single-partition ones.
//
// * decode_mfma_kernel (bf16/f16, head_dim 64/128/256, block_size 16 << j; 16-token
//   sub-blocks of larger blocks): the GQA group's query heads are replicated into the 16 rows
//   of a v_mfma_f32_16x16x32 A operand, each 16-token K sub-block is the B operand, so one K/V
//   block is read from HBM once per kv-head for all of its q-heads.
//   Scores go through an exp2 online softmax whose max is shared by the whole
//   wave (DPP row reductions), P.V runs on the VALU in fp32 with 16-byte V
//   loads, and four waves split the partition's blocks and merge through LDS.
// * decode_generic_kernel: any dtype (fp32 included), head_dim % 4 == 0 up to
//   256, any block size and GQA ratio; one wave per (partition, q-head, seq),
//   each lane owning 4 dims.  Used where the MFMA kernel does not apply.
//
// decode_merge_kernel combines the partials of one (seq, q-head):
//   M = max_p m_p, out = sum_p e^(m_p-M) tmp_p / sum_p e^(m_p-M) l_p
// (crates/vllm-cuda/src/kernels/paged_attention_v2_reduce.cu:50-95).
#include <atomic>
#include <mutex>

#include "decode_stream.hpp"

namespace rg {
namespace {

enum DecodeMode : int32_t { MODE_FINAL = 0, MODE_PARTIAL = 1, MODE_AUTO = 2 };

struct DecodeArgs {
  const void* q;
  const void* k_cache;
  const void* v_cache;
  const int32_t* block_table;
  const int32_t* context_lens;
  void* out;
  float* tmp_out;
  float* exp_sums;
  float* max_logits;
  float scale_log2;  // scale * log2(e)
  int32_t num_heads;
  int32_t num_kv_heads;
  int32_t head_dim;
  int32_t block_size;
  int32_t max_blocks;
  int32_t num_partitions;  // stride of the partial arrays
  int32_t partition_size;  // tokens per partition
  int64_t kv_stride;       // elements between blocks
  int32_t mode;
  // block_size = 16 << bs_shift for the MFMA and stream-K kernels (-1: another size).  They work
  // in 16-token sub-blocks: sub-block b of a sequence is rows 16 (b & mask) .. of the kv-head's
  // slice of physical block table[b >> bs_shift].
  int32_t bs_shift;
};

__device__ __forceinline__ int num_parts_for(int ctx, int P) { return (ctx + P - 1) / P; }

// ------------------------------------------------------------- generic ------

template <typename T>
__global__ __launch_bounds__(64) void decode_generic_kernel(DecodeArgs a) {
  using E = elem<T>;
  using S = typename E::storage;
  const int p = blockIdx.x;
  const int h = blockIdx.y;
  const int s = blockIdx.z;
  const int lane = threadIdx.x;
  // Contexts longer than the block table row are clamped to it, negative ones to 0.
  const int ctx = max(0, min(a.context_lens[s], a.max_blocks * a.block_size));
  const int P = a.partition_size;
  const int np_s = min(num_parts_for(ctx, P), a.num_partitions);
  const int D = a.head_dim;
  const bool final_out = a.mode == MODE_FINAL || (a.mode == MODE_AUTO && np_s <= 1);

  if (p >= np_s) {
    // Empty context: the single-pass kernels leave zeros
    // (paged_attention_v1_plus.cu:38 on a zero-filled output).
    if (ctx == 0 && p == 0 && final_out) {
      S* o = static_cast<S*>(a.out) + ((int64_t)s * a.num_heads + h) * D;
      for (int d = lane; d < D; d += 64) E::store(o, d, 0.f);
    }
    return;
  }
  const int kvh = h / (a.num_heads / a.num_kv_heads);
  const int d0 = lane * 4;
  const bool act = d0 < D;
  const S* qp = static_cast<const S*>(a.q) + ((int64_t)s * a.num_heads + h) * D;
  float qv[4] = {0.f, 0.f, 0.f, 0.f};
  if (act) {
#pragma unroll
    for (int u = 0; u < 4; ++u) qv[u] = E::load(qp, d0 + u);
  }
  const S* kc = static_cast<const S*>(a.k_cache);
  const S* vc = static_cast<const S*>(a.v_cache);
  const int32_t* bt = a.block_table + (int64_t)s * a.max_blocks;

  float m = -INFINITY, l = 0.f;
  float o[4] = {0.f, 0.f, 0.f, 0.f};
  const int t1 = min(ctx, (p + 1) * P);
  for (int t = p * P; t < t1; ++t) {
    const int64_t blk = bt[t / a.block_size];
    const int off = t % a.block_size;
    const int64_t row = blk * a.kv_stride + ((int64_t)kvh * a.block_size + off) * D;
    float kv[4] = {0.f, 0.f, 0.f, 0.f}, vv[4] = {0.f, 0.f, 0.f, 0.f};
    if (act) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        kv[u] = E::load(kc, row + d0 + u);
        vv[u] = E::load(vc, row + d0 + u);
      }
    }
    float dot = qv[0] * kv[0] + qv[1] * kv[1] + qv[2] * kv[2] + qv[3] * kv[3];
    dot = wave_sum(dot);
    const float x = dot * a.scale_log2;
    const float m_new = fmaxf(m, x);
    const float alpha = exp2f(m - m_new);
    const float pe = exp2f(x - m_new);
    l = l * alpha + pe;
#pragma unroll
    for (int u = 0; u < 4; ++u) o[u] = o[u] * alpha + pe * vv[u];
    m = m_new;
  }

  if (final_out) {
    const float inv = l != 0.f ? 1.f / l : 1.f;
    S* op = static_cast<S*>(a.out) + ((int64_t)s * a.num_heads + h) * D;
    if (act) {
#pragma unroll
      for (int u = 0; u < 4; ++u) E::store(op, d0 + u, o[u] * inv);
    }
  } else {
    const int64_t sh = ((int64_t)s * a.num_heads + h) * a.num_partitions + p;
    if (act) {
      float4* tp = reinterpret_cast<float4*>(a.tmp_out + sh * D + d0);
      *tp = make_float4(o[0], o[1], o[2], o[3]);
    }
    if (lane == 0) {
      a.exp_sums[sh] = l;
      a.max_logits[sh] = m * kLn2;
    }
  }
}

// Tuning knobs of the MFMA path (compile-time): waves per workgroup, blocks each wave keeps
// in flight ahead of the one it computes, and an optional occupancy floor.
#ifndef RG_DEC_WAVES
#define RG_DEC_WAVES 4
#endif
#ifndef RG_DEC_PREFETCH
#define RG_DEC_PREFETCH 1
#endif
constexpr int kWaves = RG_DEC_WAVES;
constexpr int kPrefetch = RG_DEC_PREFETCH;
constexpr int kThreads = kWaves * 64;
#if defined(RG_DEC_WAVES_PER_EU) && RG_DEC_WAVES_PER_EU > 0
#define RG_DEC_OCCUPANCY __attribute__((amdgpu_waves_per_eu(RG_DEC_WAVES_PER_EU)))
#else
#define RG_DEC_OCCUPANCY
#endif

// Grid decomposition: workgroup = (partition p, kv-head, sequence), kWaves waves taking the
// partition's blocks round-robin, merged through LDS at the end.
template <typename T, int D, int G>
__global__ __launch_bounds__(kThreads) RG_DEC_OCCUPANCY void decode_mfma_kernel(
    DecodeArgs a, const uint16_t* __restrict__ q_ptr, const uint16_t* __restrict__ kc,
    const uint16_t* __restrict__ vc, const int32_t* __restrict__ block_table,
    const int32_t* __restrict__ context_lens) {
  using Tile = DecodeTile<T, D, G>;
  using S = uint16_t;
  constexpr int GP = Tile::GP;
  constexpr int HG = Tile::HG;
  constexpr int NK = Tile::NK;
  constexpr int NV = Tile::NV;
  constexpr int NBUF = kPrefetch + 1;

  __shared__ float p_lds[kWaves][2][kBS * GP];
  __shared__ float alpha_lds[kWaves][2][GP];
  __shared__ float acc_lds[kWaves][G * D];
  __shared__ float ml_lds[kWaves][2][GP];

  const int p = blockIdx.x;
  const int kvh = blockIdx.y;
  const int s = blockIdx.z;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);

  const int ctx = max(0, min(context_lens[s], a.max_blocks * a.block_size));
  const int P = a.partition_size;
  const int np_s = min(num_parts_for(ctx, P), a.num_partitions);
  const bool final_out = a.mode == MODE_FINAL || (a.mode == MODE_AUTO && np_s <= 1);
  const int H = a.num_heads;

  if (p >= np_s) {
    if (ctx == 0 && p == 0 && final_out) {
      S* o = static_cast<S*>(a.out) + ((int64_t)s * H + (int64_t)kvh * G) * D;
      for (int i = tid; i < G * D; i += kThreads) o[i] = 0;
    }
    return;
  }

  // 16-token sub-blocks of this partition; wave w takes sub-blocks b0+w, b0+w+kWaves, ...
  const int nblk_ctx = (ctx + kBS - 1) / kBS;
  const int b0 = p * (P / kBS);
  const int b1 = min(nblk_ctx, b0 + P / kBS);
  const int nb = b0 + w < b1 ? (b1 - (b0 + w) + kWaves - 1) / kWaves : 0;

  Tile tile;
  tile.init(lane);
  tile.load_q(q_ptr + ((int64_t)s * H + (int64_t)kvh * G) * D);
  tile.reset();
  const int32_t* bt = block_table + (int64_t)s * a.max_blocks;
  const int64_t head_off = (int64_t)kvh * a.block_size * D;
  const int sh = a.bs_shift, sub_mask = (1 << sh) - 1;
  // Block j of this wave, or (j >= nb) one line of its last block per load instruction.
  auto load_block = [&](int j, uint4 (&kk)[NK], uint4 (&vv)[NV]) {
    const int lb = b0 + w + min(j, nb - 1) * kWaves;
    const int64_t off = (int64_t)bt[lb >> sh] * a.kv_stride + head_off + (int64_t)(lb & sub_mask) * (kBS * D);
    tile.load_or_line(kc + off, vc + off, j < nb, kk, vv);
  };

  // Software pipeline: kPrefetch blocks in flight ahead of the one being computed.  Every
  // step issues the same load instructions, so the waits stay exact counts instead of full
  // drains; past the end they read one line of the wave's last block each (a re-read of the
  // whole block was 1 in 8 of a P = 512 partition's requests).
  uint4 kbuf[NBUF][NK], vbuf[NBUF][NV];
  if (nb > 0) {
#pragma unroll
    for (int u = 0; u < kPrefetch; ++u) load_block(u, kbuf[u], vbuf[u]);
  }
  for (int j0 = 0; j0 < nb; j0 += NBUF) {
#pragma unroll
    for (int u = 0; u < NBUF; ++u) {
      const int j = j0 + u;
      if (j < nb) {
        load_block(j + kPrefetch, kbuf[(u + kPrefetch) % NBUF], vbuf[(u + kPrefetch) % NBUF]);
        tile.step(kbuf[u], vbuf[u], (b0 + w + j * kWaves) * kBS, ctx, a.scale_log2, p_lds[w][j & 1],
                  alpha_lds[w][j & 1]);
      }
    }
  }

  float lsum[4];
  tile.reduce(lsum);
  if (tile.vrow == 0) {
#pragma unroll
    for (int h = 0; h < G; ++h) {
      float4* dst = reinterpret_cast<float4*>(&acc_lds[w][h * D + tile.vd0]);
      dst[0] = make_float4(tile.acc[h][0], tile.acc[h][1], tile.acc[h][2], tile.acc[h][3]);
      dst[1] = make_float4(tile.acc[h][4], tile.acc[h][5], tile.acc[h][6], tile.acc[h][7]);
    }
  }
  if (tile.seg < HG && tile.col == 0) {
    *reinterpret_cast<float4*>(&ml_lds[w][0][4 * tile.seg]) =
        make_float4(tile.m_run[0], tile.m_run[1], tile.m_run[2], tile.m_run[3]);
    *reinterpret_cast<float4*>(&ml_lds[w][1][4 * tile.seg]) = make_float4(lsum[0], lsum[1], lsum[2], lsum[3]);
  }
  __syncthreads();

  // Merge the waves and write out two consecutive dims per thread.
  for (int idx = tid; idx < G * D / 2; idx += kThreads) {
    const int h = idx / (D / 2);
    const int d = (idx % (D / 2)) * 2;
    float M = -INFINITY;
#pragma unroll
    for (int ww = 0; ww < kWaves; ++ww) M = fmaxf(M, ml_lds[ww][0][h]);
    float L = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
    for (int ww = 0; ww < kWaves; ++ww) {
      const float mw = ml_lds[ww][0][h];
      const float f = mw == -INFINITY ? 0.f : exp2f(mw - M);
      L += f * ml_lds[ww][1][h];
      o0 += f * acc_lds[ww][h * D + d];
      o1 += f * acc_lds[ww][h * D + d + 1];
    }
    const int hq = kvh * G + h;
    if (final_out) {
      const float inv = L != 0.f ? 1.f / L : 1.f;
      S* op = static_cast<S*>(a.out) + ((int64_t)s * H + hq) * D + d;
      const uint32_t packed = (uint32_t)elem<T>::from_f32(o0 * inv) |
                              ((uint32_t)elem<T>::from_f32(o1 * inv) << 16);
      *reinterpret_cast<uint32_t*>(op) = packed;
    } else {
      const int64_t sh = ((int64_t)s * H + hq) * a.num_partitions + p;
      *reinterpret_cast<float2*>(a.tmp_out + sh * D + d) = make_float2(o0, o1);
      if (d == 0) {
        a.exp_sums[sh] = L;
        a.max_logits[sh] = M * kLn2;
      }
    }
  }
}

template <typename T, int D, int G, bool ROPE = false>
__global__ __launch_bounds__(64) RG_SK_OCCUPANCY void decode_stream_kernel(
    StreamArgs a, const typename DecodeTileFor<T, D, G>::S* __restrict__ q_ptr,
    const typename DecodeTileFor<T, D, G>::S* __restrict__ kc, const typename DecodeTileFor<T, D, G>::S* __restrict__ vc,
    const int32_t* __restrict__ block_table, const int32_t* __restrict__ context_lens,
    const int32_t* __restrict__ positions, const int32_t* __restrict__ slot_mapping) {
  stream_worker<T, D, G, ROPE>(a, q_ptr, kc, vc, block_table, context_lens, positions, slot_mapping, blockIdx.x, 0,
                               threadIdx.x);
}

// One workgroup per segment (sequence, kv-head), one wave per head of the group: merges the
// partials of the segment's workers (the range its first worker recorded in seg_desc) and
// writes the G output rows.  Lane l of wave h holds dims [l*D/64, (l+1)*D/64) of head h, so each
// partial's [G, D] accumulator is read as one contiguous row by the whole workgroup; every
// lane folds the partials in order with an online rescale (loads of consecutive partials
// are independent, so they are issued ahead of the folds).
template <typename T, int D, int G>
__global__ __launch_bounds__(64 * G) void decode_stream_merge_kernel(StreamArgs a,
                                                                    const int32_t* __restrict__ context_lens) {
  using S = typename elem<T>::storage;
  constexpr int PER = D / 64;  // dims per lane
  static_assert(PER == 1 || PER == 2 || PER == 4, "head_dim 64, 128 or 256");
  const int kvh = blockIdx.x;
  const int s = blockIdx.y;
  const int h = threadIdx.x >> 6;
  const int lane = threadIdx.x & 63;
  const int hkv = a.num_kv_heads;
  S* out = static_cast<S*>(a.out) + ((int64_t)s * a.num_heads + (int64_t)kvh * G + h) * D + lane * PER;
  // The segment's workers, as the first of them recorded (their partials: first + g .. ); the
  // descriptor is loaded together with the context length (one memory round trip, not two)
  // and used only when the segment has units (a segment without any keeps a stale entry).
  const int2 dsc = a.seg_desc[(int64_t)s * hkv + kvh];
  const int ctx = context_lens[s];
  asm volatile("" ::"s"(dsc.x), "s"(dsc.y), "s"(ctx));  // both loads issued before either is waited for
  if (min(ctx, a.max_blocks * kBS) <= 0) {  // no blocks (seq_blocks == 0)
#pragma unroll
    for (int e = 0; e < PER; ++e) out[e] = 0;
    return;
  }
  const int64_t pbase = (int64_t)dsc.x + (int64_t)s * hkv + kvh;  // partial index of the first worker
  const int np = dsc.y;

  float m = -INFINITY, l = 0.f;
  float acc[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) acc[e] = 0.f;
#pragma unroll 4
  for (int q = 0; q < np; ++q) {
    const int64_t pi = pbase + q;
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + pi * (2 * G) + 2 * h);
    const float* pa = a.part_acc + pi * (G * D) + h * D + lane * PER;
    float v[PER];
    if constexpr (PER == 4) {
      const float4 t = *reinterpret_cast<const float4*>(pa);
      v[0] = t.x;
      v[1] = t.y;
      v[2] = t.z;
      v[3] = t.w;
    } else if constexpr (PER == 2) {
      const float2 t = *reinterpret_cast<const float2*>(pa);
      v[0] = t.x;
      v[1] = t.y;
    } else {
      v[0] = pa[0];
    }
    const float mn = fmaxf(m, ml.x);
    const float fo = exp2f(m - mn);  // 0 for the first partial (m = -inf)
    const float fq = exp2f(ml.x - mn);
    l = l * fo + ml.y * fq;
#pragma unroll
    for (int e = 0; e < PER; ++e) acc[e] = acc[e] * fo + v[e] * fq;
    m = mn;
  }
  const float inv = l != 0.f ? 1.f / l : 1.f;
  if constexpr (PER == 2 && !std::is_same_v<T, f32_t>) {
    const uint32_t packed = (uint32_t)elem<T>::from_f32(acc[0] * inv) | ((uint32_t)elem<T>::from_f32(acc[1] * inv) << 16);
    *reinterpret_cast<uint32_t*>(out) = packed;
  } else {
#pragma unroll
    for (int e = 0; e < PER; ++e) out[e] = elem<T>::from_f32(acc[e] * inv);
  }
}

// ---------------------------------------------------------------- short -----
//
// Tables of few tokens (short_applies): one workgroup per segment (sequence, kv-head), kShortWaves
// waves taking its 16-token sub-blocks in turn, their partials merged in LDS and the output written:
// one launch, and the workspace, whose size is asked for by shape alone, is left alone.  Such a call is bound by latency and launches, not by bytes: the
// stream-K worker first finds its range by a scan over the context lengths, then its block-table
// window, then its K/V rows, and the merge kernel follows.  Here the table entries (lane l of wave w
// holds sub-block w + kShortWaves l), the context length and q are loaded at once, then the K/V
// rows.  ROPE as in decode_stream_kernel: every wave rotates its q rows, the wave holding the last
// sub-block writes and patches the new token's rows.
// Measured (kernel trace, 4 sequences): 32 / 8 heads of 128 in bf16 at 100 tokens 7.8 us against 9.5 +
// 3.4 of the two kernels and the gap between them; fp32 heads of 64 at 400 tokens 10.4 against 8.8 +
// 3.4.  Its slope is P.V on the VALU, ~1,100 cycles a sub-block and
// wave; 16 tokens a wave more cost 1.1 us.
template <typename T, int D, int G, bool ROPE>
__global__ __launch_bounds__(kShortThreads) void decode_short_kernel(
    StreamArgs a, const typename DecodeTileFor<T, D, G>::S* __restrict__ q_ptr,
    const typename DecodeTileFor<T, D, G>::S* __restrict__ kc, const typename DecodeTileFor<T, D, G>::S* __restrict__ vc,
    const int32_t* __restrict__ block_table, const int32_t* __restrict__ context_lens,
    const int32_t* __restrict__ positions, const int32_t* __restrict__ slot_mapping) {
  using Tile = DecodeTileFor<T, D, G>;
  using S = typename Tile::S;
  static_assert(!ROPE || !std::is_same_v<T, f32_t>, "the fused RoPE runs on the 16-bit tiles");
  constexpr int GP = Tile::GP, HG = Tile::HG, NK = Tile::NK, NV = Tile::NV;
  // Sub-blocks in flight ahead of the one computed (fp32 at head_dim 128: 64 registers each).
  constexpr int AHEAD = std::is_same_v<T, f32_t> && D == 128 ? 1 : 2, NBUF = AHEAD + 1;
  __shared__ float p_lds[kShortWaves][2][kBS * GP];
  __shared__ float alpha_lds[kShortWaves][2][GP];
  __shared__ float acc_lds[kShortWaves][G * D];
  __shared__ float ml_lds[kShortWaves][2][GP];

  const int kvh = blockIdx.x, s = blockIdx.y;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int H = a.num_heads, hkv = a.num_kv_heads;
  const int sh = a.bs_shift, sub_mask = (1 << sh) - 1;

  // Sub-block w + kShortWaves lane of the table row, within the row whatever the context is.
  const int sb = w + kShortWaves * lane;
  const int32_t* row = block_table + (int64_t)s * a.table_stride;
  const int entry = sb < a.max_blocks ? row[sb >> sh] : 0;
  const int ctx_raw = context_lens[s];
  const S* qg = q_ptr + ((int64_t)s * H + (int64_t)kvh * G) * D;
  Tile tile;
  tile.init(lane);
  tile.reset();

  constexpr int QP = G * D <= 128 ? 1 : G * D <= 256 ? 2 : G * D <= 512 ? 4 : 8;
  constexpr int KP = D / 2 >= 64 ? D / 128 : 1;
  __shared__ __attribute__((aligned(16))) uint16_t rope_lds[ROPE ? kShortWaves : 1][ROPE ? G * D + D : 1];
  uint16_t* const rq_lds = rope_lds[ROPE ? w : 0];
  uint16_t* const rk_lds = rq_lds + G * D;
  const int rq_p0 = lane * QP, rk_p0 = lane * KP;
  RopeRun<T, QP> rq;
  RopeRun<T, KP> rk;
  uint4 vnew = make_uint4(0, 0, 0, 0);
  int slot = -1;
  if constexpr (ROPE) {
    slot = slot_mapping[s];
    const int pos = positions[s];  // (of a sequence without a context it is not used)
    const float* cs = a.cos_sin + (int64_t)(ctx_raw > 0 ? pos : 0) * D;
    if (rq_p0 < G * D / 2) rq.load(qg + (rq_p0 / (D / 2)) * D, cs, rq_p0 % (D / 2), D / 2);
    const int64_t nrow = ((int64_t)s * hkv + kvh) * D;
    if (rk_p0 < D / 2) rk.load(static_cast<const S*>(a.k_new) + nrow, cs, rk_p0, D / 2);
    vnew = *reinterpret_cast<const uint4*>(static_cast<const S*>(a.v_new) + nrow + tile.vd0);
  } else {
    tile.load_q(qg);
  }

  const int ctx = max(0, min(ctx_raw, a.max_blocks * kBS));
  const int nblk = (ctx + kBS - 1) / kBS;
  const int nb = w < nblk ? (nblk - w + kShortWaves - 1) / kShortWaves : 0;  // this wave's sub-blocks
  if (nb > 0) {
    const int64_t head = (int64_t)kvh * (kBS << sh) * D;
    uint4 kbuf[NBUF][NK], vbuf[NBUF][NV];
    auto load_block = [&](int j, uint4 (&kk)[NK], uint4 (&vv)[NV]) __attribute__((always_inline)) {
      const int e = __builtin_amdgcn_readlane(entry, j);
      const int64_t off = (int64_t)e * a.kv_stride + head + (int64_t)((w + kShortWaves * j) & sub_mask) * (kBS * D);
      tile.template load_part<1, 0>(kc + off, vc + off, kk, vv);
    };
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) load_block(min(u, nb - 1), kbuf[u], vbuf[u]);
    int patch_j = -1;  // the sub-block of this wave that takes the new token's rows
    if constexpr (ROPE) {
      if (rq_p0 < G * D / 2) rq.rotate_to(rq_lds + (rq_p0 / (D / 2)) * D, rq_p0 % (D / 2), D / 2);
      const int p = ctx_raw - 1, pb = p >> 4;  // the new token's position and sub-block
      if (slot >= 0 && p >= 0 && p < a.max_blocks * kBS && pb % kShortWaves == w) {
        const int e = __builtin_amdgcn_readlane(entry, pb / kShortWaves);
        if (((e << sh) | (pb & sub_mask)) * kBS + (p & (kBS - 1)) == slot) {
          patch_j = pb / kShortWaves;
          if (rk_p0 < D / 2) rk.rotate_to(rk_lds, rk_p0, D / 2);
        }
      }
      wave_lds_sync();
      const uint4* qrow = reinterpret_cast<const uint4*>(rq_lds + (tile.col % G) * D + 8 * tile.seg);
#pragma unroll
      for (int i = 0; i < NK; ++i) tile.qa[i] = qrow[4 * i];
    }
    // Every step issues a sub-block's loads (the last one again past the end), so that the
    // compiler's waits are exact counts.
    for (int j0 = 0; j0 < nb; j0 += NBUF) {
#pragma unroll
      for (int u = 0; u < NBUF; ++u) {
        const int j = j0 + u;
        if (j < nb) {
          load_block(min(j + AHEAD, nb - 1), kbuf[(u + AHEAD) % NBUF], vbuf[(u + AHEAD) % NBUF]);
          if constexpr (ROPE) {
            if (j == patch_j) {
              uint4 knew[NK];
              const uint4* krow = reinterpret_cast<const uint4*>(rk_lds + 8 * tile.seg);
#pragma unroll
              for (int i = 0; i < NK; ++i) knew[i] = krow[4 * i];
              tile.template patch<1>(kbuf[u], vbuf[u], 0, slot & (kBS - 1), knew, vnew);
              const int bsz = kBS << sh;
              const int64_t nrow = (int64_t)(slot >> (4 + sh)) * a.kv_stride +
                                   ((int64_t)kvh * bsz + (slot & (bsz - 1))) * D;
              S* kdst = const_cast<S*>(kc) + nrow;
              S* vdst = const_cast<S*>(vc) + nrow;
              if (tile.col == 0) {
#pragma unroll
                for (int i = 0; i < NK; ++i) *reinterpret_cast<uint4*>(kdst + 32 * i + 8 * tile.seg) = knew[i];
              }
              if (tile.vrow == 0) *reinterpret_cast<uint4*>(vdst + tile.vd0) = vnew;
            }
          }
          tile.step(kbuf[u], vbuf[u], (w + kShortWaves * j) * kBS, ctx, a.scale_log2, p_lds[w][j & 1],
                    alpha_lds[w][j & 1]);
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

  // Merge the waves and write out two consecutive dims per thread (zeros without a context).
  for (int idx = threadIdx.x; idx < G * D / 2; idx += kShortThreads) {
    const int h = idx / (D / 2);
    const int d = (idx % (D / 2)) * 2;
    float M = -INFINITY;
#pragma unroll
    for (int ww = 0; ww < kShortWaves; ++ww) M = fmaxf(M, ml_lds[ww][0][h]);
    float L = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
    for (int ww = 0; ww < kShortWaves; ++ww) {
      const float mw = ml_lds[ww][0][h];
      const float f = mw == -INFINITY ? 0.f : exp2f(mw - M);
      const float2 o = *reinterpret_cast<const float2*>(&acc_lds[ww][h * D + d]);
      L += f * ml_lds[ww][1][h];
      o0 += f * o.x;
      o1 += f * o.y;
    }
    const float inv = L != 0.f ? 1.f / L : 1.f;
    auto* op = static_cast<typename elem<T>::storage*>(a.out) + ((int64_t)s * H + (int64_t)kvh * G + h) * D + d;
    if constexpr (std::is_same_v<T, f32_t>) {
      op[0] = o0 * inv;
      op[1] = o1 * inv;
    } else {
      *reinterpret_cast<uint32_t*>(op) =
          (uint32_t)elem<T>::from_f32(o0 * inv) | ((uint32_t)elem<T>::from_f32(o1 * inv) << 16);
    }
  }
}

// ---------------------------------------------------------------- merge -----

struct MergeArgs {
  void* out;
  const float* exp_sums;
  const float* max_logits;
  const float* tmp_out;
  const int32_t* context_lens;
  int32_t num_heads;
  int32_t head_dim;
  int32_t num_partitions;
  int32_t partition_size;
  int32_t skip_single;  // 1: sequences with one partition were written by the partition kernel
};

// One workgroup of 256 threads per (seq, q-head).  The partition weights e^(m_p - M) go to LDS
// once per partition; thread t accumulates the float4 column chunk c = t % C of the rows
// p = g, g + R, ... of tmp_out (C = D / 4 chunks per row, g = t / C, R = 256 / C row groups),
// so R rows are read at a time, and the R partial sums are added in group order through LDS
// (a fixed order: the result does not depend on timing).
constexpr int kMergeThreads = 256;
template <typename T>
__global__ __launch_bounds__(kMergeThreads) void decode_merge_kernel(MergeArgs a) {
  using E = elem<T>;
  using S = typename E::storage;
  constexpr int kChunk = kMergeThreads;  // partitions whose weights sit in LDS at a time
  constexpr int kWaves = kMergeThreads / 64;
  __shared__ float w_lds[kChunk];
  __shared__ float red[2 * kWaves];
  __shared__ float4 part[kMergeThreads];
  const int h = blockIdx.x;
  const int s = blockIdx.y;
  const int tid = threadIdx.x;
  const int wv = tid >> 6;
  const int D = a.head_dim;
  const int ctx = max(0, a.context_lens[s]);
  const int np_s = min(num_parts_for(ctx, a.partition_size), a.num_partitions);
  if (a.skip_single && np_s <= 1) return;
  S* op = static_cast<S*>(a.out) + ((int64_t)s * a.num_heads + h) * D;
  if (np_s == 0) {
    for (int d = tid; d < D; d += kMergeThreads) E::store(op, d, 0.f);
    return;
  }
  const int64_t sh = ((int64_t)s * a.num_heads + h) * a.num_partitions;
  const float* ml = a.max_logits + sh;
  const float* es = a.exp_sums + sh;
  float M = -INFINITY;
  for (int q = tid; q < np_s; q += kMergeThreads) M = fmaxf(M, ml[q]);
  M = wave_max(M);
  if ((tid & 63) == 0) red[wv] = M;
  __syncthreads();
  M = red[0];
#pragma unroll
  for (int j = 1; j < kWaves; ++j) M = fmaxf(M, red[j]);
  float L = 0.f;
  for (int q = tid; q < np_s; q += kMergeThreads) L += expf(ml[q] - M) * es[q];
  L = wave_sum(L);
  if ((tid & 63) == 0) red[kWaves + wv] = L;
  __syncthreads();
  L = red[kWaves];
#pragma unroll
  for (int j = 1; j < kWaves; ++j) L += red[kWaves + j];
  const float inv = L != 0.f ? 1.f / L : 1.f;
  const float* tp = a.tmp_out + sh * D;
  const int C = D / 4;                    // head_dim % 4 == 0 and <= 1024 (checked on the host)
  const int R = kMergeThreads / C;
  const int c = tid % C, g = tid / C;
  const bool active = g < R;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int q0 = 0; q0 < np_s; q0 += kChunk) {
    const int n = min(kChunk, np_s - q0);
    __syncthreads();  // the previous chunk's weights are no longer read
    if (tid < n) w_lds[tid] = expf(ml[q0 + tid] - M);
    __syncthreads();
    if (active) {
#pragma unroll 4
      for (int q = g; q < n; q += R) {
        const float r = w_lds[q];
        const float4 v = *reinterpret_cast<const float4*>(tp + (int64_t)(q0 + q) * D + 4 * c);
        acc.x += r * v.x;
        acc.y += r * v.y;
        acc.z += r * v.z;
        acc.w += r * v.w;
      }
    }
  }
  if (active) part[g * C + c] = acc;
  __syncthreads();
  if (tid < C) {
    float4 t = part[tid];
    for (int j = 1; j < R; ++j) {
      const float4 u = part[j * C + tid];
      t.x += u.x;
      t.y += u.y;
      t.z += u.z;
      t.w += u.w;
    }
    E::store(op, 4 * tid + 0, t.x * inv);
    E::store(op, 4 * tid + 1, t.y * inv);
    E::store(op, 4 * tid + 2, t.z * inv);
    E::store(op, 4 * tid + 3, t.w * inv);
  }
}

// ------------------------------------------------------------ host side -----

// Tokens per partition the v1 entries use when given a workspace.
#ifndef RG_V1_PARTITION
#define RG_V1_PARTITION 256
#endif
constexpr int kV1PartitionTokens = RG_V1_PARTITION;

template <typename T, int D, int G>
void launch_mfma(const DecodeArgs& a, dim3 grid, hipStream_t s) {
  hipLaunchKernelGGL((decode_mfma_kernel<T, D, G>), grid, dim3(kThreads), 0, s, a,
                     static_cast<const uint16_t*>(a.q), static_cast<const uint16_t*>(a.k_cache),
                     static_cast<const uint16_t*>(a.v_cache), a.block_table, a.context_lens);
}

template <typename T, int D>
bool launch_mfma_g(const DecodeArgs& a, int G, dim3 grid, hipStream_t s) {
  switch (G) {
    case 1: launch_mfma<T, D, 1>(a, grid, s); return true;
    case 2: launch_mfma<T, D, 2>(a, grid, s); return true;
    case 4: launch_mfma<T, D, 4>(a, grid, s); return true;
    case 8: launch_mfma<T, D, 8>(a, grid, s); return true;
    case 3:
    case 5:
    case 6:
    case 7:
      if constexpr (D <= 128) {
        if (G == 3) launch_mfma<T, D, 3>(a, grid, s);
        else if (G == 5) launch_mfma<T, D, 5>(a, grid, s);
        else if (G == 6) launch_mfma<T, D, 6>(a, grid, s);
        else launch_mfma<T, D, 7>(a, grid, s);
        return true;
      }
      return false;
    case 16:
      if constexpr (D < 256) {
        launch_mfma<T, D, 16>(a, grid, s);
        return true;
      }
      return false;
    default: return false;
  }
}

bool mfma_applies(const DecodeArgs& a, int32_t dtype) {
  const int G = a.num_heads / a.num_kv_heads;
  const int eb = dtype_bytes(dtype);
  return (dtype == RG_DTYPE_BF16 || dtype == RG_DTYPE_F16) && a.bs_shift >= 0 &&
         (a.head_dim == 64 || a.head_dim == 128 || a.head_dim == 256) &&
         mfma_group_size(G, a.head_dim) && a.partition_size % kBS == 0 &&
         aligned16(a.q) && aligned16(a.k_cache) && aligned16(a.v_cache) &&
         (a.kv_stride * eb) % 16 == 0 &&
         (a.out == nullptr || (reinterpret_cast<uintptr_t>(a.out) & 3u) == 0);
}

// The grid kernel: the MFMA shapes but head_dim 256 with 16 q-heads per kv-head (whose
// accumulators and two K/V blocks in flight exceed the registers of a wave).
bool grid_mfma_applies(const DecodeArgs& a, int32_t dtype) {
  return mfma_applies(a, dtype) && !(a.head_dim == 256 && a.num_heads / a.num_kv_heads == 16);
}

// The stream-K decode: the MFMA shapes in bf16 / f16, and the same shapes in fp32 (head_dim 64,
// 128 or 256; at 256 a worker holds a block's K and V rows, 128 VGPRs, next to the q row's 64: it
// runs with AGPRs as extra registers, one wave per SIMD as always).
bool stream_applies(const DecodeArgs& a, int32_t dtype) {
  if (dtype != RG_DTYPE_F32) return mfma_applies(a, dtype);
  const int G = a.num_heads / a.num_kv_heads;
  return a.bs_shift >= 0 && (a.head_dim == 64 || a.head_dim == 128 || a.head_dim == 256) &&
         mfma_group_size(G, a.head_dim) && aligned16(a.q) && aligned16(a.k_cache) &&
         aligned16(a.v_cache) && (a.kv_stride * 4) % 16 == 0 && (a.out == nullptr || (reinterpret_cast<uintptr_t>(a.out) & 3u) == 0);
}

// Launches the partition kernel over grid (grid_parts, heads, batch).
int run_partition(const char* op, const DecodeArgs& a, int32_t dtype, int32_t batch,
                  int32_t grid_parts, hipStream_t s) {
  if (batch == 0 || grid_parts == 0) return ok();
  if (grid_mfma_applies(a, dtype)) {
    const int G = a.num_heads / a.num_kv_heads;
    const dim3 grid(grid_parts, a.num_kv_heads, batch);
    if (dtype == RG_DTYPE_BF16) {
      if (a.head_dim == 256) launch_mfma_g<bf16_t, 256>(a, G, grid, s);
      else if (a.head_dim == 128) launch_mfma_g<bf16_t, 128>(a, G, grid, s);
      else launch_mfma_g<bf16_t, 64>(a, G, grid, s);
    } else {
      if (a.head_dim == 256) launch_mfma_g<f16_t, 256>(a, G, grid, s);
      else if (a.head_dim == 128) launch_mfma_g<f16_t, 128>(a, G, grid, s);
      else launch_mfma_g<f16_t, 64>(a, G, grid, s);
    }
    return check_launch(op);
  }
  const dim3 grid(grid_parts, a.num_heads, batch);
  return dispatch_dtype(dtype, [&](auto tag) {
    hipLaunchKernelGGL(decode_generic_kernel<decltype(tag)>, grid, dim3(64), 0, s, a);
    return check_launch(op);
  });
}

int run_merge(const char* op, const MergeArgs& m, int32_t dtype, int32_t batch, hipStream_t s) {
  if (batch == 0) return ok();
  const dim3 grid(m.num_heads, batch);
  return dispatch_dtype(dtype, [&](auto tag) {
    hipLaunchKernelGGL(decode_merge_kernel<decltype(tag)>, grid, dim3(kMergeThreads), 0, s, m);
    return check_launch(op);
  });
}

DecodeArgs make_args(const void* q, const void* kc, const void* vc, const int32_t* bt,
                     const int32_t* cl, void* out, float scale, const Shape& sh,
                     int64_t kv_stride, int32_t P, int32_t NP, int32_t mode) {
  DecodeArgs a;
  a.q = q;
  a.k_cache = kc;
  a.v_cache = vc;
  a.block_table = bt;
  a.context_lens = cl;
  a.out = out;
  a.tmp_out = nullptr;
  a.exp_sums = nullptr;
  a.max_logits = nullptr;
  a.scale_log2 = scale * kLog2e;
  a.num_heads = sh.H;
  a.num_kv_heads = sh.Hkv;
  a.head_dim = sh.D;
  a.block_size = sh.bs;
  a.max_blocks = sh.MB;
  a.num_partitions = NP;
  a.partition_size = P;
  a.kv_stride = kv_stride ? kv_stride : (int64_t)sh.Hkv * sh.bs * sh.D;
  a.mode = mode;
  a.bs_shift = -1;
  for (int j = 0; j <= 4; ++j)
    if (sh.bs == (kBS << j)) a.bs_shift = j;
  return a;
}

struct V2Scratch {
  float* tmp_out;
  float* exp_sums;
  float* max_logits;
};

size_t v2_bytes(int64_t B, int64_t H, int64_t NP, int64_t D, V2Scratch* carve, void* base) {
  const size_t n_stat = (size_t)(B * H * NP);
  const size_t tmp = align_up(n_stat * (size_t)D * 4, 256);
  const size_t stat = align_up(n_stat * 4, 256);
  if (carve) {
    char* p = static_cast<char*>(base);
    carve->tmp_out = reinterpret_cast<float*>(p);
    carve->exp_sums = reinterpret_cast<float*>(p + tmp);
    carve->max_logits = reinterpret_cast<float*>(p + tmp + stat);
  }
  return tmp + 2 * stat;
}

int32_t v1_num_partitions(const Shape& sh) {
  const int64_t max_ctx = (int64_t)sh.MB * sh.bs;
  return (int32_t)ceil_div(max_ctx, kV1PartitionTokens);
}

// ---- stream-K path ----

template <typename T, int D, int G, bool ROPE = false>
void launch_stream(const StreamArgs& sa, const DecodeArgs& a, hipStream_t s) {
  using S = typename DecodeTileFor<T, D, G>::S;
  if constexpr (D <= 128 && G <= 8) {
    if (sa.one_launch) {
      hipLaunchKernelGGL((decode_short_kernel<T, D, G, ROPE>), dim3(sa.num_kv_heads, sa.batch), dim3(kShortThreads), 0,
                         s, sa, static_cast<const S*>(a.q), static_cast<const S*>(a.k_cache),
                         static_cast<const S*>(a.v_cache), a.block_table, a.context_lens, sa.positions,
                         sa.slot_mapping);
      return;
    }
  }
  hipLaunchKernelGGL((decode_stream_kernel<T, D, G, ROPE>), dim3(sa.num_workers), dim3(64), 0, s, sa,
                     static_cast<const S*>(a.q), static_cast<const S*>(a.k_cache),
                     static_cast<const S*>(a.v_cache), a.block_table, a.context_lens, sa.positions,
                     sa.slot_mapping);
  hipLaunchKernelGGL((decode_stream_merge_kernel<T, D, G>), dim3(sa.num_kv_heads, sa.batch), dim3(64 * G), 0, s,
                     sa, a.context_lens);
}

template <typename T, int D>
void launch_stream_g(const StreamArgs& sa, const DecodeArgs& a, int G, hipStream_t s) {
  switch (G) {
    case 1: launch_stream<T, D, 1>(sa, a, s); break;
    case 2: launch_stream<T, D, 2>(sa, a, s); break;
    case 4: launch_stream<T, D, 4>(sa, a, s); break;
    case 8: launch_stream<T, D, 8>(sa, a, s); break;
    case 16: launch_stream<T, D, 16>(sa, a, s); break;
    default:
      // G = 3, 5, 6, 7 (stream_applies admits them at head_dim 64 and 128 only)
      if constexpr (D <= 128) {
        if (G == 3) launch_stream<T, D, 3>(sa, a, s);
        else if (G == 5) launch_stream<T, D, 5>(sa, a, s);
        else if (G == 6) launch_stream<T, D, 6>(sa, a, s);
        else if (G == 7) launch_stream<T, D, 7>(sa, a, s);
      }
      break;
  }
}

// The step's new tokens for the fused RoPE form: rows [batch, H_kv, D] of k and v, token s
// being sequence s's.
struct RopeIn {
  const void* k;
  const void* v;
  const float* cos_sin;
  const int32_t* positions;
  const int32_t* slot_mapping;
};

// The fused RoPE form runs at bf16 / f16, head_dim 64 and 128 and G 1 to 8.
bool rope_stream_applies(const DecodeArgs& a, int32_t dtype, const RopeIn& r) {
  const int G = a.num_heads / a.num_kv_heads;
  return (dtype == RG_DTYPE_BF16 || dtype == RG_DTYPE_F16) && stream_applies(a, dtype) &&
         (a.head_dim == 64 || a.head_dim == 128) && G >= 1 && G <= 8 && aligned16(r.k) && aligned16(r.v) &&
         aligned16(r.cos_sin);
}

template <typename T, int D>
void launch_stream_rope_g(const StreamArgs& sa, const DecodeArgs& a, int G, hipStream_t s) {
  switch (G) {
    case 1: launch_stream<T, D, 1, true>(sa, a, s); break;
    case 2: launch_stream<T, D, 2, true>(sa, a, s); break;
    case 3: launch_stream<T, D, 3, true>(sa, a, s); break;
    case 4: launch_stream<T, D, 4, true>(sa, a, s); break;
    case 5: launch_stream<T, D, 5, true>(sa, a, s); break;
    case 6: launch_stream<T, D, 6, true>(sa, a, s); break;
    case 7: launch_stream<T, D, 7, true>(sa, a, s); break;
    default: launch_stream<T, D, 8, true>(sa, a, s); break;  // G = 8 (rope_stream_applies)
  }
}

// Runs the stream-K decode if it applies and the workspace holds its scratch; returns
// RG_ERR_WORKSPACE (without recording an error) when the workspace is too small.  With rope,
// the fused RoPE form (rope_stream_applies holds).
int run_stream(const char* op, const DecodeArgs& a, int32_t dtype, const Shape& sh, void* ws, size_t ws_bytes,
               hipStream_t s, const RopeIn* rope = nullptr) {
  const int32_t workers = stream_workers(sh);
  StreamScratch sc;
  if (ws_bytes < stream_bytes(sh, workers, &sc, ws)) return RG_ERR_WORKSPACE;
  StreamArgs sa{};
  sa.out = a.out;
  sa.part_acc = sc.acc;
  sa.part_ml = sc.ml;
  sa.seg_desc = sc.desc;
  sa.scale_log2 = a.scale_log2;
  sa.num_heads = sh.H;
  sa.num_kv_heads = sh.Hkv;
  sa.max_blocks = sh.MB << a.bs_shift;
  sa.batch = sh.B;
  sa.num_workers = workers;
  sa.kv_stride = a.kv_stride;
  sa.table_stride = sh.MB;
  sa.bs_shift = a.bs_shift;
  sa.one_launch = short_applies(sh, dtype_bytes(dtype)) ? 1 : 0;
  const int G = sh.H / sh.Hkv;
  if (rope != nullptr) {
    sa.k_new = rope->k;
    sa.v_new = rope->v;
    sa.cos_sin = rope->cos_sin;
    sa.positions = rope->positions;
    sa.slot_mapping = rope->slot_mapping;
    if (dtype == RG_DTYPE_BF16) {
      if (sh.D == 128) launch_stream_rope_g<bf16_t, 128>(sa, a, G, s);
      else launch_stream_rope_g<bf16_t, 64>(sa, a, G, s);
    } else {
      if (sh.D == 128) launch_stream_rope_g<f16_t, 128>(sa, a, G, s);
      else launch_stream_rope_g<f16_t, 64>(sa, a, G, s);
    }
    return check_launch(op);
  }
  if (dtype == RG_DTYPE_BF16) {
    if (sh.D == 256) launch_stream_g<bf16_t, 256>(sa, a, G, s);
    else if (sh.D == 128) launch_stream_g<bf16_t, 128>(sa, a, G, s);
    else launch_stream_g<bf16_t, 64>(sa, a, G, s);
  } else if (dtype == RG_DTYPE_F16) {
    if (sh.D == 256) launch_stream_g<f16_t, 256>(sa, a, G, s);
    else if (sh.D == 128) launch_stream_g<f16_t, 128>(sa, a, G, s);
    else launch_stream_g<f16_t, 64>(sa, a, G, s);
  } else {
    if (sh.D == 256) launch_stream_g<f32_t, 256>(sa, a, G, s);
    else if (sh.D == 128) launch_stream_g<f32_t, 128>(sa, a, G, s);
    else launch_stream_g<f32_t, 64>(sa, a, G, s);
  }
  return check_launch(op);
}

// Body shared by the v1 and v1_plus entries.
int paged_v1(const char* op, const void* q, const void* kc, const void* vc, const int32_t* bt,
             const int32_t* cl, void* out, float scale, const Shape& sh, int32_t dtype,
             int64_t kv_stride, void* ws, size_t ws_bytes, void* stream) {
  int st = check_decode_shape(op, sh, dtype, kv_stride);
  if (st != RG_OK) return st;
  if (sh.B == 0) return ok();
  if (!q || !kc || !vc || !bt || !cl || !out) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: null pointer argument", op);
  }
  hipStream_t s = as_stream(stream);
  if (ws != nullptr) {
    DecodeArgs a = make_args(q, kc, vc, bt, cl, out, scale, sh, kv_stride, kBS, 1, MODE_AUTO);
    if (stream_applies(a, dtype) && sh.MB > 0) {
      st = run_stream(op, a, dtype, sh, ws, ws_bytes, s);
      if (st != RG_ERR_WORKSPACE) return st;
      return fail(RG_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu required", op, ws_bytes,
                  stream_bytes(sh, stream_workers(sh), nullptr, nullptr));
    }
  }
  const int32_t np = v1_num_partitions(sh);
  if (ws != nullptr && np > 1) {
    V2Scratch sc;
    const size_t need = v2_bytes(sh.B, sh.H, np, sh.D, &sc, ws);
    if (ws_bytes < need) {
      return fail(RG_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu required", op, ws_bytes, need);
    }
    DecodeArgs a = make_args(q, kc, vc, bt, cl, out, scale, sh, kv_stride, kV1PartitionTokens, np,
                             MODE_AUTO);
    a.tmp_out = sc.tmp_out;
    a.exp_sums = sc.exp_sums;
    a.max_logits = sc.max_logits;
    st = run_partition(op, a, dtype, sh.B, np, s);
    if (st != RG_OK) return st;
    MergeArgs m{out, sc.exp_sums, sc.max_logits, sc.tmp_out, cl, sh.H, sh.D, np,
                kV1PartitionTokens, 1};
    return run_merge(op, m, dtype, sh.B, s);
  }
  // One partition spans the whole block table.
  const int32_t P = (int32_t)std::max<int64_t>(16, ceil_div((int64_t)sh.MB * sh.bs, 16) * 16);
  DecodeArgs a = make_args(q, kc, vc, bt, cl, out, scale, sh, kv_stride, P, 1, MODE_FINAL);
  return run_partition(op, a, dtype, sh.B, 1, s);
}

// ---- entry without allocation ----
//
// rg_paged_attention_v1_no_alloc keeps the stream-K partials in `scratch` below, one copy per
// device, instead of a caller's workspace.  Host code never passes `scratch` itself to a
// kernel (on the host that name is a stand-in, not a device address): the address of each
// device's copy comes from hipGetSymbolAddress, taken once per device with that device
// current, and is kept in g_scratch_addr.

constexpr int kMaxDevices = 64;
std::atomic<void*> g_scratch_addr[kMaxDevices];
std::mutex g_scratch_mu;

}  // namespace

static __device__ __align__(256) unsigned char scratch[RG_NO_ALLOC_SCRATCH_BYTES];

namespace {

// Address of the current device's copy of `scratch`; looked up on the first call per device.
int no_alloc_scratch(const char* op, void** addr) {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return fail(RG_ERR_HIP, "%s: no current device: %s", op, hipGetErrorString(e));
  if (dev < 0 || dev >= kMaxDevices) {
    return fail(RG_ERR_NOT_SUPPORTED, "%s: device ordinal %d beyond the %d devices supported", op, dev, kMaxDevices);
  }
  void* p = g_scratch_addr[dev].load(std::memory_order_acquire);
  if (p == nullptr) {
    std::lock_guard<std::mutex> lock(g_scratch_mu);
    p = g_scratch_addr[dev].load(std::memory_order_relaxed);
    if (p == nullptr) {
      e = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));
      if (e != hipSuccess || p == nullptr) {
        return fail(RG_ERR_HIP, "%s: cannot locate the static scratch on device %d: %s", op, dev,
                    hipGetErrorString(e));
      }
      g_scratch_addr[dev].store(p, std::memory_order_release);
    }
  }
  *addr = p;
  return RG_OK;
}

}  // namespace

// Called by rg_init with the device being initialised current.
int setup_no_alloc_scratch() {
  void* p = nullptr;
  return no_alloc_scratch("rg_init", &p);
}

int probe_decode_kernels() {
  hipFuncAttributes at;
  if (hipFuncGetAttributes(&at, reinterpret_cast<const void*>(decode_mfma_kernel<bf16_t, 128, 4>)) !=
          hipSuccess ||
      hipFuncGetAttributes(&at, reinterpret_cast<const void*>(decode_generic_kernel<f32_t>)) !=
          hipSuccess) {
    return fail(RG_ERR_HIP, "failed to load the decode kernels: %s",
                hipGetErrorString(hipGetLastError()));
  }
  return RG_OK;
}

}  // namespace rg

using namespace rg;

extern "C" size_t rg_paged_attention_v1_workspace_bytes(int32_t batch_size, int32_t num_heads,
                                                        int32_t num_kv_heads, int32_t head_dim,
                                                        int32_t block_size, int32_t max_blocks_per_seq) {
  if (batch_size <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 ||
      head_dim <= 0 || block_size <= 0 || max_blocks_per_seq <= 0) {
    return 0;
  }
  const Shape sh{num_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq, batch_size};
  const int32_t np = v1_num_partitions(sh);
  const size_t grid = np > 1 ? v2_bytes(batch_size, num_heads, np, head_dim, nullptr, nullptr) : 0;
  return std::max(grid, stream_bytes(sh, stream_workers(sh), nullptr, nullptr));
}

extern "C" int rg_paged_attention_v1(const void* query, const void* key_cache,
                                     const void* value_cache, const int32_t* block_table,
                                     const int32_t* context_lens, void* output, float scale,
                                     int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                     int32_t block_size, int32_t max_blocks_per_seq,
                                     int32_t batch_size, int32_t dtype, int64_t kv_block_stride,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  const Shape sh{num_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq, batch_size};
  return paged_v1("paged_attention_v1", query, key_cache, value_cache, block_table, context_lens,
                  output, scale, sh, dtype, kv_block_stride, workspace, workspace_bytes, stream);
}

extern "C" int rg_rope_reshape_and_cache_paged_attention_v1(
    const void* query, const void* key, const void* value, void* key_cache, void* value_cache,
    const float* cos_sin, const int32_t* positions, const int32_t* slot_mapping, const int32_t* block_table,
    const int32_t* context_lens, void* output, float scale, int32_t num_heads, int32_t num_kv_heads,
    int32_t head_dim, int32_t block_size, int32_t max_blocks_per_seq, int32_t batch_size, int32_t dtype,
    int64_t kv_block_stride, void* workspace, size_t workspace_bytes, void* stream) {
  const char* op = "rope_reshape_and_cache_paged_attention_v1";
  const Shape sh{num_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq, batch_size};
  int st = check_decode_shape(op, sh, dtype, kv_block_stride);
  if (st != RG_OK) return st;
  if (sh.B == 0) return ok();
  if (!query || !key || !value || !key_cache || !value_cache || !cos_sin || !positions || !slot_mapping ||
      !block_table || !context_lens || !output) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: null pointer argument", op);
  }
  if (workspace == nullptr) return fail(RG_ERR_INVALID_ARGUMENT, "%s: needs a workspace", op);
  const DecodeArgs a = make_args(query, key_cache, value_cache, block_table, context_lens, output, scale, sh,
                                 kv_block_stride, kBS, 1, MODE_AUTO);
  const RopeIn rope{key, value, cos_sin, positions, slot_mapping};
  if (sh.MB <= 0 || !rope_stream_applies(a, dtype, rope)) {
    return fail(RG_ERR_NOT_SUPPORTED,
                "%s: runs at bf16 / f16, head_dim 64 or 128, num_heads / num_kv_heads 1 to 8, "
                "block_size 16 * 2^j and 16-byte aligned rows (rg_rope_reshape_and_cache followed by "
                "rg_paged_attention_v1 covers the rest)", op);
  }
  st = run_stream(op, a, dtype, sh, workspace, workspace_bytes, as_stream(stream), &rope);
  if (st != RG_ERR_WORKSPACE) return st;
  return fail(RG_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu required", op, workspace_bytes,
              stream_bytes(sh, stream_workers(sh), nullptr, nullptr));
}

extern "C" int rg_paged_attention_v1_plus(const void* query, const void* key_cache,
                                          const void* value_cache, const int32_t* block_table,
                                          const int32_t* context_lens, void* output,
                                          const float* rotation_metadata, float scale,
                                          int32_t num_heads, int32_t num_kv_heads,
                                          int32_t head_dim, int32_t block_size,
                                          int32_t max_blocks_per_seq, int32_t batch_size,
                                          int32_t dtype, int64_t kv_block_stride, void* workspace,
                                          size_t workspace_bytes, void* stream) {
  (void)rotation_metadata;  // identity rotation
  const Shape sh{num_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq, batch_size};
  return paged_v1("paged_attention_v1_plus", query, key_cache, value_cache, block_table,
                  context_lens, output, scale, sh, dtype, kv_block_stride, workspace,
                  workspace_bytes, stream);
}

extern "C" size_t rg_v2_workspace_bytes(int32_t batch_size, int32_t num_heads,
                                        int32_t num_partitions, int32_t head_dim) {
  if (batch_size <= 0 || num_heads <= 0 || num_partitions <= 0 || head_dim <= 0) return 0;
  return v2_bytes(batch_size, num_heads, num_partitions, head_dim, nullptr, nullptr);
}

extern "C" int rg_paged_attention_v2_partition(
    const void* query, const void* key_cache, const void* value_cache, const int32_t* block_table,
    const int32_t* context_lens, float* tmp_out, float* exp_sums, float* max_logits,
    const float* rotation_metadata, float scale, int32_t num_heads, int32_t num_kv_heads,
    int32_t head_dim, int32_t block_size, int32_t max_blocks_per_seq, int32_t num_partitions,
    int32_t batch_size, int32_t partition_size, int32_t dtype, int64_t kv_block_stride,
    void* stream) {
  (void)rotation_metadata;
  const char* op = "paged_attention_v2_partition";
  const Shape sh{num_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq, batch_size};
  int st = check_decode_shape(op, sh, dtype, kv_block_stride);
  if (st != RG_OK) return st;
  if (partition_size <= 0 || partition_size % block_size != 0) {
    return fail(RG_ERR_INVALID_ARGUMENT,
                "%s: partition_size %d must be a positive multiple of block_size %d", op,
                partition_size, block_size);
  }
  if (num_partitions < 0) return fail(RG_ERR_INVALID_ARGUMENT, "%s: num_partitions < 0", op);
  if (batch_size == 0 || num_partitions == 0) return ok();
  if (!query || !key_cache || !value_cache || !block_table || !context_lens || !tmp_out ||
      !exp_sums || !max_logits) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: null pointer argument", op);
  }
  DecodeArgs a = make_args(query, key_cache, value_cache, block_table, context_lens, nullptr,
                           scale, sh, kv_block_stride, partition_size, num_partitions,
                           MODE_PARTIAL);
  a.tmp_out = tmp_out;
  a.exp_sums = exp_sums;
  a.max_logits = max_logits;
  return run_partition(op, a, dtype, batch_size, num_partitions, as_stream(stream));
}

extern "C" int rg_paged_attention_v2_reduce(void* output, const float* exp_sums,
                                            const float* max_logits, const float* tmp_out,
                                            const int32_t* context_lens,
                                            const float* rotation_metadata, int32_t num_heads,
                                            int32_t head_dim, int32_t num_partitions,
                                            int32_t batch_size, int32_t partition_size,
                                            int32_t dtype, void* stream) {
  (void)rotation_metadata;
  const char* op = "paged_attention_v2_reduce";
  if (dtype_bytes(dtype) == 0) return fail(RG_ERR_NOT_SUPPORTED, "%s: unknown dtype %d", op, dtype);
  if (head_dim > 1024) {
    // MAX_HEAD_DIM_V2_REDUCE (crates/vllm-cuda/src/kernels/mod.rs:477-482)
    return fail(RG_ERR_INVALID_ARGUMENT,
                "head_dim %d exceeds maximum block size 1024 for reduction kernel", head_dim);
  }
  if (head_dim <= 0 || head_dim % 4 != 0) {
    return fail(RG_ERR_NOT_SUPPORTED, "%s: head_dim must be a positive multiple of 4, got %d", op,
                head_dim);
  }
  if (num_heads <= 0 || batch_size < 0 || num_partitions < 0 || partition_size <= 0) {
    return fail(RG_ERR_INVALID_ARGUMENT,
                "%s: need num_heads > 0, batch >= 0, num_partitions >= 0, partition_size > 0",
                op);
  }
  if (batch_size == 0) return ok();
  if (!output || !context_lens || (num_partitions > 0 && (!exp_sums || !max_logits || !tmp_out))) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: null pointer argument", op);
  }
  MergeArgs m{output, exp_sums, max_logits, tmp_out, context_lens, num_heads, head_dim,
              num_partitions, partition_size, 0};
  return run_merge(op, m, dtype, batch_size, as_stream(stream));
}

extern "C" int rg_paged_attention_v2(const void* query, const void* key_cache,
                                     const void* value_cache, const int32_t* block_table,
                                     const int32_t* context_lens, void* output, float scale,
                                     int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                     int32_t block_size, int32_t max_blocks_per_seq,
                                     int32_t batch_size, int32_t max_context_len,
                                     int32_t partition_size, int32_t dtype,
                                     int64_t kv_block_stride, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  const char* op = "paged_attention_v2";
  const Shape sh{num_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq, batch_size};
  int st = check_decode_shape(op, sh, dtype, kv_block_stride);
  if (st != RG_OK) return st;
  if (partition_size <= 0 || partition_size % block_size != 0) {
    return fail(RG_ERR_INVALID_ARGUMENT,
                "%s: partition_size %d must be a positive multiple of block_size %d", op,
                partition_size, block_size);
  }
  if (max_context_len < 0) return fail(RG_ERR_INVALID_ARGUMENT, "%s: max_context_len < 0", op);
  if (batch_size == 0) return ok();
  if (!query || !key_cache || !value_cache || !block_table || !context_lens || !output) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: null pointer argument", op);
  }
  hipStream_t s = as_stream(stream);
  if (workspace != nullptr) {
    // The stream-K decode computes the same merge of split-K partials with balanced splits;
    // it runs whenever it applies and the workspace holds its scratch.
    DecodeArgs a = make_args(query, key_cache, value_cache, block_table, context_lens, output, scale, sh,
                             kv_block_stride, partition_size, 1, MODE_AUTO);
    if (stream_applies(a, dtype) && max_blocks_per_seq > 0) {
      st = run_stream(op, a, dtype, sh, workspace, workspace_bytes, s);
      if (st != RG_ERR_WORKSPACE) return st;
    }
  }
  const int32_t np = (int32_t)std::max<int64_t>(1, ceil_div(max_context_len, partition_size));
  V2Scratch sc;
  const size_t need = v2_bytes(batch_size, num_heads, np, head_dim, &sc, workspace);
  if (workspace == nullptr || workspace_bytes < need) {
    return fail(RG_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu required", op,
                workspace ? workspace_bytes : (size_t)0, need);
  }
  DecodeArgs a = make_args(query, key_cache, value_cache, block_table, context_lens, output, scale,
                           sh, kv_block_stride, partition_size, np, MODE_AUTO);
  a.tmp_out = sc.tmp_out;
  a.exp_sums = sc.exp_sums;
  a.max_logits = sc.max_logits;
  st = run_partition(op, a, dtype, batch_size, np, s);
  if (st != RG_OK) return st;
  MergeArgs m{output, sc.exp_sums, sc.max_logits, sc.tmp_out, context_lens, num_heads, head_dim,
              np, partition_size, 1};
  return run_merge(op, m, dtype, batch_size, s);
}

extern "C" int rg_paged_attention_v1_no_alloc(const void* query, const void* key_cache,
                                              const void* value_cache, const int32_t* block_table,
                                              const int32_t* context_lens, void* output, float scale,
                                              int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                              int32_t block_size, int32_t max_blocks_per_seq,
                                              int32_t batch_size, int32_t dtype, int64_t kv_block_stride,
                                              void* stream) {
  const char* op = "paged_attention_v1_no_alloc";
  const Shape sh{num_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq, batch_size};
  int st = check_decode_shape(op, sh, dtype, kv_block_stride);
  if (st != RG_OK) return st;
  if (sh.B == 0) return ok();
  if (!query || !key_cache || !value_cache || !block_table || !context_lens || !output) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: null pointer argument", op);
  }
  const DecodeArgs a = make_args(query, key_cache, value_cache, block_table, context_lens, output, scale, sh,
                                 kv_block_stride, kBS, 1, MODE_AUTO);
  if (stream_applies(a, dtype) && sh.MB > 0) {
    // The stream-K kernels of rg_paged_attention_v1 with the static scratch as their workspace.
    // Nothing in it needs clearing: every partial and segment descriptor the merge reads is
    // written earlier in the same call.
    const size_t need = stream_bytes(sh, stream_workers(sh), nullptr, nullptr);
    if (need > (size_t)RG_NO_ALLOC_SCRATCH_BYTES) {
      return fail(RG_ERR_WORKSPACE,
                  "%s: this shape needs %zu bytes of split-K scratch, the static scratch holds %zu "
                  "(call rg_paged_attention_v1 with a workspace instead)",
                  op, need, (size_t)RG_NO_ALLOC_SCRATCH_BYTES);
    }
    void* ws = nullptr;
    st = no_alloc_scratch(op, &ws);
    if (st != RG_OK) return st;
    return run_stream(op, a, dtype, sh, ws, RG_NO_ALLOC_SCRATCH_BYTES, as_stream(stream));
  }
  // The other paths of rg_paged_attention_v1 without a workspace use no scratch at all.
  return paged_v1(op, query, key_cache, value_cache, block_table, context_lens, output, scale, sh, dtype,
                  kv_block_stride, nullptr, 0, stream);
}
