// Decode attention of a batch whose sequences begin with the same cached blocks.
//
// With P prefix tokens in shared blocks, the B rows of the batch ask G query heads each of a kv-head's prefix:
// B G rows against the same K and V.  Read per sequence, as the plain decode does, the prefix costs B times
// its bytes; here it is read once per kPreRows rows, as an attention product on the matrix cores:
//   S^T = K Q^T,  running maximum and sum per row,  O^T += V^T P^T.
// The tokens behind the prefix differ per sequence and stay with the stream-K decode worker.  Softmax
// partials (m, l, unnormalised O) of both join in shared_merge_kernel:
//   M = max m_i,  out = sum 2^(m_i - M) O_i / sum 2^(m_i - M) l_i.
//
// One launch computes both: the product is bound by the matrix cores and LDS, the suffixes by HBM, and
// workgroups of either kind sit on every CU, so the shorter of the two hides under the longer (but for the forms
// of more than 256 registers, groups_per_cu: there the product's follow the workers').  A sequence
// whose context ends inside the prefix is not a row of the product (which then needs no mask per row); the
// stream-K worker takes all of its tokens.
//   Measured (bf16, 32 / 8 heads of 128): 256 sequences over 16,384 shared tokens alone 88-92 us a call
// (0.75-0.78 PFLOP/s), with 64 to 1,024 tokens each behind them 158-164 (658 MB; in long runs at the power limit
// up to 188); 16 over 2,048 with up to 700 behind them 17.3, of which the merge takes 4.4.
#include "decode_stream.hpp"

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

constexpr int kPreWaves = 4;
constexpr int kPreThreads = 64 * kPreWaves;
constexpr int kPreRows = 32 * kPreWaves;  // rows of a workgroup, 32 a wave
constexpr int kTileKeys = 32;
constexpr int kStages = 3;                // key tiles in the LDS ring
constexpr float kSlack = 8.f;             // log2 headroom of the lazy maximum: 2^8 a probability at most
// What is subtracted from the scores of a row whose lazy maximum is m (log2 units): in fp16 2^7 times the
// probabilities are held.  Its normal numbers end at 2^-14: one token's weight beside those of thousands that are
// 2^-25 of it each would be all that is left.  Times 2^7 they fill the type up to 2^(8 + 7), and the half step of
// the subnormals, 2^-25, is 2^-32 of the largest weight.  Past 2^20 the fp32 scores' own steps grow towards the one
// factor of two that is left below 2^16; there they are held as they are.
template <typename T>
__device__ __forceinline__ float reference(float m) {
  if constexpr (std::is_same_v<T, f16_t>) return m - (fabsf(m) < 0x1p20f ? 7.f : 0.f);
  else return m;
}

struct PrefixArgs {
  float* acc;  // [H_kv, splits, rows, D] unnormalised
  float* ml;   // [H_kv, splits, rows, 2]: m in log2 units, l
  float scale_log2;  // > 0
  uint32_t q_sign;   // bit 0: q is taken (else zeros, a scale of 0), bits 15 and 31: negated (a negative scale)
  int32_t group, num_heads, num_kv_heads, rows;  // rows = batch * group
  int32_t prefix, subs;                          // prefix tokens, and its 16-token sub-blocks
  int32_t tiles, split_tiles, splits;
  int32_t bs_shift;
  int32_t stream_groups;                         // workgroups of stream-K workers, the first of the grid
  int64_t kv_stride;
};

// One key tile in LDS, two sub-blocks of 16 keys.  K: the 16-byte chunk c of key k of sub-block b at
// b * KB / 2 + 256 c + 16 k, so that a 1 KB copy reads one sub-block only and the A operand of one MFMA is
// 256 contiguous bytes per 16 lanes.  V: rows [key][D] with the 16-byte chunks of a row XORed by
// 2 (key & 3), so that the transposing reads of four rows hit different banks.
template <int D>
struct KeyTile {
  static constexpr int KB = kTileKeys * D * 2;
  static constexpr int BYTES = 2 * KB;
  static constexpr int VCH = D / 8;        // 16-byte chunks of a V row
  static constexpr int SUB_COPIES = D / 32;  // 1 KB copies of a sub-block's K, and of its V
  __device__ static __forceinline__ int vchunk(int key, int c) { return c ^ (2 * (key & 3)); }
};

// The prefix product of workgroup u: kPreRows rows of one kv-head against the key tiles of one split.
// Lane l of a wave owns query row l % 32 of it; the other half of that row's keys sits in lane l ^ 32.
template <typename T, int D>
__device__ __forceinline__ void prefix_product(const PrefixArgs& a, const uint16_t* __restrict__ q,
                                               const uint16_t* __restrict__ kc, const uint16_t* __restrict__ vc,
                                               const int32_t* __restrict__ table, char* lds, int u, int w, int lane) {
  using MF = mfma32<T>;
  using TL = KeyTile<D>;
  constexpr int NKC = D / 16, NDB = D / 32, HALF = TL::SUB_COPIES / 2, COPIES = 2 * HALF;
  static_assert(HALF >= 1, "two waves copy a sub-block");
  const int pairs = a.num_kv_heads * a.splits;
  const int rt = u / pairs, pair = u % pairs;
  const int kvh = pair % a.num_kv_heads, split = pair / a.num_kv_heads;
  const int kt0 = split * a.split_tiles, kt1 = min(a.tiles, kt0 + a.split_tiles);
  const int j = lane & 31, hh = lane >> 5;
  const int wrow = rt * kPreRows + w * 32;  // the wave's first row
  const bool busy = wrow < a.rows;          // (a wave without rows copies and waits with the others)
  const int row = wrow + j;
  const int b = min(row, a.rows - 1) / a.group, g = min(row, a.rows - 1) - b * a.group;

  // This wave copies half of sub-block cb of every tile.  Lane l of the window holds the entry of tile
  // wb + l: (physical block << bs_shift) | sub-block within it; past the end the last sub-block's.
  const int cb = w >> 1, cp = w & 1;
  int wb = kt0, win;
  auto fill = [&]() {
    const int sb = min(2 * (wb + lane) + cb, a.subs - 1);
    win = (table[sb >> a.bs_shift] << a.bs_shift) | (sb & ((1 << a.bs_shift) - 1));
  };
  fill();
  uint4 qb[NKC];
  {
    const uint4* qr = reinterpret_cast<const uint4*>(q + ((int64_t)b * a.num_heads + (int64_t)kvh * a.group + g) * D);
#pragma unroll
    for (int i = 0; i < NKC; ++i) qb[i] = qr[2 * i + hh];
    // scale_log2 > 0 here: the host passes its magnitude (1 for a scale of 0) and what becomes of q.
    const uint32_t flip = a.q_sign & 0x80008000u, on = a.q_sign & 1 ? 0xffffffffu : 0u;
#pragma unroll
    for (int i = 0; i < NKC; ++i)
      qb[i] = make_uint4((qb[i].x ^ flip) & on, (qb[i].y ^ flip) & on, (qb[i].z ^ flip) & on, (qb[i].w ^ flip) & on);
  }
  // Rows whose context lacks part of the prefix are left to the stream-K workers: they compute along
  // (finite or not, no other lane's row sees it) and write nothing that the merge reads.
  int32_t lane_off[COPIES];
  uint32_t ins_lds[COPIES];
#pragma unroll
  for (int ld = 0; ld < COPIES; ++ld) {
    if (ld < HALF) {
      const int n = cp * HALF + ld;
      lane_off[ld] = (lane & 15) * D + 8 * (4 * n + (lane >> 4));
      ins_lds[ld] = cb * (TL::KB / 2) + n * 1024;
    } else {
      const int vi = cb * TL::SUB_COPIES + cp * HALF + ld - HALF;  // of the tile's V
      const int key = vi * (1024 / (D * 2)) + lane / TL::VCH;
      lane_off[ld] = (key & 15) * D + 8 * TL::vchunk(key, lane % TL::VCH);
      ins_lds[ld] = TL::KB + vi * 1024;
    }
  }
  const uint32_t lds_base = (uint32_t)(uintptr_t)((RG_LDS char*)lds);
  const int64_t head = (int64_t)kvh * (kBS << a.bs_shift) * D;
  auto issue = [&](int kt, int st) {
    const int e = __builtin_amdgcn_readlane(win, kt - wb);
    const int64_t off = (int64_t)(e >> a.bs_shift) * a.kv_stride + head + (int64_t)(e & ((1 << a.bs_shift) - 1)) * (kBS * D);
    const char* kb = reinterpret_cast<const char*>(kc + off);
    const char* vb = reinterpret_cast<const char*>(vc + off);
    const uint32_t sbase = lds_base + st * TL::BYTES;
#pragma unroll
    for (int ld = 0; ld < COPIES; ++ld) {
      lds_dma16_s(ld < HALF ? kb : vb, (uint32_t)lane_off[ld] * 2u, sbase + ins_lds[ld]);
    }
  };

  f32x16_t o[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[db][v] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;
  float ref = -INFINITY;    // reference(m_run)
  float m_thr = -INFINITY;  // m_run + kSlack in raw score units, so a tile's test needs no multiply
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
  // Tile kt from ring stage ST.  S^T: c[v] is key 8 (v >> 2) + 4 hh + (v & 3) of the tile for query j.
  auto scores = [&](int kt, auto stc) __attribute__((always_inline)) -> f32x16_t {
    const char* kbase = lds + decltype(stc)::value * TL::BYTES + k_lane;
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
  auto finish = [&](int kt, f32x16_t c, auto stc) __attribute__((always_inline)) {
    const char* vbase = lds + decltype(stc)::value * TL::BYTES + TL::KB;
    uint4 va[VA];
#pragma unroll
    for (int m = 0; m < VA; ++m) va[m] = v_operand(vbase, m);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
    if (2 * kt + 1 >= a.subs) {  // an odd number of sub-blocks: the last tile's second half repeats one
#pragma unroll
      for (int v = 8; v < 16; ++v) c[v] = -INFINITY;
    }
    // The maximum moves only when a tile exceeds it by more than kSlack, for both halves of a row alike.
    float tmax = c[0];
#pragma unroll
    for (int v = 1; v < 16; ++v) tmax = fmaxf(tmax, c[v]);
    if (__ballot(tmax > m_thr)) {
      const float other = __int_as_float(__builtin_amdgcn_ds_bpermute(xor32, __float_as_int(tmax)));
      const float both = fmaxf(tmax, other) * a.scale_log2;
      const float m_new = both > m_run + kSlack ? both : m_run;
      const float ref_new = reference<T>(m_new);
      const float alpha = fast_exp2(ref - ref_new);
      m_run = m_new;
      ref = ref_new;
      m_thr = (m_run + kSlack) / a.scale_log2;
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[db][v] *= alpha;
    }
    // Probabilities, rounded to the operand type of the PV product; the sum takes the rounded ones, so
    // the normaliser weighs what enters the product.
    uint32_t pk[8];
#pragma unroll
    for (int v = 0; v < 16; v += 2)
      pk[v / 2] = pack2<T>(fast_exp2(fmaf(c[v], a.scale_log2, -ref)), fast_exp2(fmaf(c[v + 1], a.scale_log2, -ref)));
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

  // The window and Q have landed (the builtin, which the compiler's own counting follows: behind an asm
  // wait it would wait for Q again in every tile, and with it for every copy in flight).
  __builtin_amdgcn_s_waitcnt(0x70 | 0xF00);  // vmcnt(0)
#pragma unroll
  for (int p = 0; p < kStages - 1; ++p)
    if (kt0 + p < kt1) issue(kt0 + p, p);
  // Tile kt has landed (a newer one may not have), for every wave; all are done with tile kt - 1, whose
  // stage takes tile kt + kStages - 1.
  auto step = [&](int kt, auto stc) __attribute__((always_inline)) {
    constexpr int st = decltype(stc)::value;
    static_assert(kStages == 3 && COPIES < 16, "one tile newer than the awaited one; low bits of vmcnt");
    asm volatile("" ::: "memory");
    if (kt + 1 < kt1) __builtin_amdgcn_s_waitcnt(COPIES | 0x70 | 0xF00);
    else __builtin_amdgcn_s_waitcnt(0x70 | 0xF00);
    tile_barrier();
    const int next = kt + kStages - 1;
    if (next - wb >= 64) {
      wb = next;
      fill();
      __builtin_amdgcn_s_waitcnt(0x70 | 0xF00);
    }
    if (!busy) {
      if (next < kt1) issue(next, st == 0 ? kStages - 1 : st - 1);
      return;
    }
    __builtin_amdgcn_s_setprio(1);
    const f32x16_t c = scores(kt, stc);
    if (next < kt1) issue(next, st == 0 ? kStages - 1 : st - 1);  // while the QK MFMAs run
    finish(kt, c, stc);
  };
  for (int kt = kt0; kt < kt1; kt += kStages) {
    step(kt, std::integral_constant<int, 0>{});
    if (kt + 1 < kt1) step(kt + 1, std::integral_constant<int, 1>{});
    if (kt + 2 < kt1) step(kt + 2, std::integral_constant<int, 2>{});
  }
  if (row < a.rows) {
    const float l = l_run + __shfl_xor(l_run, 32, 64);
    const int64_t at = ((int64_t)kvh * a.splits + split) * a.rows + row;
    float* acc = a.acc + at * D;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int p = 0; p < 4; ++p)
        *reinterpret_cast<float4*>(acc + 32 * db + 8 * p + 4 * hh) =
            make_float4(o[db][4 * p], o[db][4 * p + 1], o[db][4 * p + 2], o[db][4 * p + 3]);
    if (hh == 0) {
      a.ml[2 * at] = ref;
      a.ml[2 * at + 1] = l;
    }
  }
}

// The fp32 product, on v_mfma_f32_32x32x2: step m of S^T = K Q^T takes the k-slot of lane half hh from dim
// hh D/2 + m, so a lane reads its K row in 16-byte pieces; step v of O^T += V^T P^T takes the keys
// 8 (v >> 2) + 4 hh + (v & 3), which is where S^T leaves them, so the probabilities stay in fp32 and in their
// registers.  A key tile is twice as long as in 16 bits and its product 16 times (128 MFMAs of 64 cycles at
// head_dim 128), so one tile in flight ahead of the one at hand is enough: two stages.
// K in LDS: rows [key][D], the 16-byte chunk c of a row at c ^ (key & 7) (rows of 256 or 512 bytes would put all
// keys of a read on the same banks); V: rows [key][D] as they are (a read takes 32 neighbours of one row).
template <int D>
struct KeyTileF32 {
  static constexpr int KB = kTileKeys * D * 4;
  static constexpr int BYTES = 2 * KB;
  static constexpr int STAGES = 2;
  static constexpr int CH = D / 4;            // 16-byte chunks of a row
  static constexpr int SUB_COPIES = D / 16;   // 1 KB copies of a sub-block's K, and of its V
};

template <int D>
__device__ __forceinline__ void prefix_product_f32(const PrefixArgs& a, const float* __restrict__ q,
                                                   const float* __restrict__ kc, const float* __restrict__ vc,
                                                   const int32_t* __restrict__ table, char* lds, int u, int w,
                                                   int lane) {
  using TL = KeyTileF32<D>;
  constexpr int NDB = D / 32, HALF = TL::SUB_COPIES / 2, COPIES = 2 * HALF, HD = D / 2;
  const int pairs = a.num_kv_heads * a.splits;
  const int rt = u / pairs, pair = u % pairs;
  const int kvh = pair % a.num_kv_heads, split = pair / a.num_kv_heads;
  const int kt0 = split * a.split_tiles, kt1 = min(a.tiles, kt0 + a.split_tiles);
  const int j = lane & 31, hh = lane >> 5;
  const int wrow = rt * kPreRows + w * 32;
  const bool busy = wrow < a.rows;
  const int row = wrow + j;
  const int b = min(row, a.rows - 1) / a.group, g = min(row, a.rows - 1) - b * a.group;
  const int cb = w >> 1, cp = w & 1;
  int wb = kt0, win;
  auto fill = [&]() {
    const int sb = min(2 * (wb + lane) + cb, a.subs - 1);
    win = (table[sb >> a.bs_shift] << a.bs_shift) | (sb & ((1 << a.bs_shift) - 1));
  };
  fill();
  float qf[HD];
  {
    const float4* qr = reinterpret_cast<const float4*>(q + ((int64_t)b * a.num_heads + (int64_t)kvh * a.group + g) * D + hh * HD);
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
  const int64_t head = (int64_t)kvh * (kBS << a.bs_shift) * D;
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
  auto compute = [&](int kt, int st) __attribute__((always_inline)) {
    const char* krow = lds + st * TL::BYTES + j * (D * 4);
    f32x16_t c;
#pragma unroll
    for (int v = 0; v < 16; ++v) c[v] = 0.f;
#pragma unroll
    for (int i = 0; i < HD / 4; ++i) {
      const float4 k4 = *reinterpret_cast<const float4*>(krow + 16 * ((hh * (HD / 4) + i) ^ (j & 7)));
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(k4.x, qf[4 * i], c, 0, 0, 0);
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(k4.y, qf[4 * i + 1], c, 0, 0, 0);
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(k4.z, qf[4 * i + 2], c, 0, 0, 0);
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(k4.w, qf[4 * i + 3], c, 0, 0, 0);
    }
    if (2 * kt + 1 >= a.subs) {  // the last tile's second half repeats a sub-block
#pragma unroll
      for (int v = 8; v < 16; ++v) c[v] = -INFINITY;
    }
    float tmax = c[0];
#pragma unroll
    for (int v = 1; v < 16; ++v) tmax = fmaxf(tmax, c[v]);
    tmax = fmaxf(tmax, __int_as_float(__builtin_amdgcn_ds_bpermute(xor32, __float_as_int(tmax)))) * a.scale_log2;
    if (__ballot(tmax > m_run)) {
      const float m_new = fmaxf(m_run, tmax);
      const float alpha = fast_exp2(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[db][v] *= alpha;
    }
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      c[v] = fast_exp2(fmaf(c[v], a.scale_log2, -m_run));
      l_run += c[v];
    }
    const float* vrow = reinterpret_cast<const float*>(lds + st * TL::BYTES + TL::KB) + 4 * hh * D + j;
#pragma unroll
    for (int v = 0; v < 16; ++v)
#pragma unroll
      for (int db = 0; db < NDB; ++db)
        o[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(vrow[(8 * (v >> 2) + (v & 3)) * D + 32 * db], c[v], o[db], 0, 0, 0);
  };
  __builtin_amdgcn_s_waitcnt(0x70 | 0xF00);  // vmcnt(0): the window and Q
  issue(kt0, 0);
  if (kt0 + 1 < kt1) issue(kt0 + 1, 1);
  static_assert(COPIES < 16, "low bits of vmcnt");
  for (int kt = kt0; kt < kt1; ++kt) {
    const int st = (kt - kt0) & 1;
    asm volatile("" ::: "memory");
    if (kt + 1 < kt1) __builtin_amdgcn_s_waitcnt(COPIES | 0x70 | 0xF00);
    else __builtin_amdgcn_s_waitcnt(0x70 | 0xF00);
    tile_barrier();  // tile kt has landed for every wave
    if (busy) compute(kt, st);
    if (kt + 2 < kt1) {
      if (kt + 2 - wb >= 64) {
        wb = kt + 2;
        fill();
        __builtin_amdgcn_s_waitcnt(0x70 | 0xF00);
      }
      tile_barrier();  // every wave is done with the stage
      issue(kt + 2, st);
    }
  }
  if (row < a.rows) {
    const float l = l_run + __shfl_xor(l_run, 32, 64);
    const int64_t at = ((int64_t)kvh * a.splits + split) * a.rows + row;
    float* acc = a.acc + at * D;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int p = 0; p < 4; ++p)
        *reinterpret_cast<float4*>(acc + 32 * db + 8 * p + 4 * hh) =
            make_float4(o[db][4 * p], o[db][4 * p + 1], o[db][4 * p + 2], o[db][4 * p + 3]);
    if (hh == 0) {
      a.ml[2 * at] = m_run;
      a.ml[2 * at + 1] = l;
    }
  }
}

// LDS of the product's ring.
template <typename T, int D>
constexpr int ring_bytes() {
  if constexpr (std::is_same_v<T, f32_t>) return KeyTileF32<D>::STAGES * KeyTileF32<D>::BYTES;
  else return kStages * KeyTile<D>::BYTES;
}

// Workgroups to a CU that the compiler is held to: two, 256 registers a wave, where it fits them without scratch
// memory, which it does not try by itself.  Of the forms that come to more than 256 (or close to it) those are fp32
// at head_dim 128 with up to 4 heads to a kv-head: 252, 254, 264 and 268 by themselves for 1 to 4, at most 256 held.
// Held to that, fp32 with more heads (280 to 330), 16 bits at head_dim 64 with 5, 6, 7 and 16 (264 to 281) and at
// 128 with 16 (280) would spill: those run one workgroup a CU.
//   Measured (fp32, 8 kv-heads of 128, 64 sequences over 2,048 / 8,192 tokens with up to 200 / 1,500 behind them;
// left alone -> held, us): G 1 26 -> 26 / 82 -> 82, 2 32 -> 32 / 93 -> 94, 3 44 -> 38 / 140 -> 113, 4 47 -> 40 /
// 144 -> 118.
template <typename T, int D, int G>
constexpr int groups_per_cu() { return std::is_same_v<T, f32_t> && D == 128 && G <= 4 ? 2 : 1; }

template <typename T, int D, int G>
__global__ __launch_bounds__(kPreThreads, (groups_per_cu<T, D, G>())) void shared_prefix_kernel(
    StreamArgs sa, PrefixArgs pa, const typename DecodeTileFor<T, D, G>::S* __restrict__ q,
    const typename DecodeTileFor<T, D, G>::S* __restrict__ kc, const typename DecodeTileFor<T, D, G>::S* __restrict__ vc,
    const int32_t* __restrict__ block_table, const int32_t* __restrict__ context_lens) {
  __shared__ __attribute__((aligned(16))) char ring[ring_bytes<T, D>()];
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if ((int)blockIdx.x < pa.stream_groups) {
    const int k = (int)blockIdx.x * kPreWaves + w;
    if (k < sa.num_workers) {
      stream_worker<T, D, G, false, StreamVariant::kSuffix, kPreWaves>(sa, q, kc, vc, block_table, context_lens, nullptr,
                                                                       nullptr, k, w, lane);
    }
    return;
  }
  // The prefix's blocks come from the first row that holds all of it: what the rows of a padded batch have in
  // their tables is not looked at.
  int holder = -1;
  for (int s0 = 0; s0 < sa.batch && holder < 0; s0 += 64) {
    const uint64_t mask = __ballot(s0 + lane < sa.batch && context_lens[min(s0 + lane, sa.batch - 1)] >= pa.prefix);
    if (mask != 0) holder = s0 + __builtin_ctzll(mask);
  }
  if (holder < 0) return;
  const int32_t* table = block_table + (int64_t)holder * sa.table_stride;
  const int u = (int)blockIdx.x - pa.stream_groups;
  if constexpr (std::is_same_v<T, f32_t>) prefix_product_f32<D>(pa, q, kc, vc, table, ring, u, w, lane);
  else prefix_product<T, D>(pa, q, kc, vc, table, ring, u, w, lane);
}

// One workgroup per (kv-head, sequence), R waves per query head: lane l of wave r folds dims [l PER, (l + 1) PER) of
// every R-th of the prefix's splits (if the sequence has the whole prefix) and of the stream-K workers' partials,
// in that order; the R results join through LDS.  A chain of memory round trips and little else, so the first of
// the prefix's partials are asked for together with the length and the segment's descriptor: they are there for
// every row, if only as numbers that do not count.
//   Two waves a head: 16 rows over 16,384 shared tokens (32 splits) 22.8 -> 20.9 us a call, 4 over 8,192 18.9 ->
// 17.3; with four splits or fewer one is as fast.
template <typename T, int D, int G, int R>
__global__ __launch_bounds__(64 * G * R) void shared_merge_kernel(StreamArgs sa, PrefixArgs pa,
                                                                  const int32_t* __restrict__ context_lens) {
  using S = typename elem<T>::storage;
  constexpr int PER = D / 64;
  constexpr int AHEAD = 4;
  const int kvh = blockIdx.x, s = blockIdx.y, lane = threadIdx.x & 63;
  const int h = (threadIdx.x >> 6) % G, r = (threadIdx.x >> 6) / G;
  const int64_t seg = (int64_t)s * sa.num_kv_heads + kvh;
  const int2 dsc = sa.seg_desc[seg];  // (stale, and not used, where the segment has no tokens of its own)
  const int len = context_lens[s];
  struct Part {
    float2 ml;
    float v[PER];
  };
  auto load = [&](const float* ml, const float* acc) __attribute__((always_inline)) {
    Part p;
    p.ml = *reinterpret_cast<const float2*>(ml);
#pragma unroll
    for (int e = 0; e < PER; ++e) p.v[e] = acc[lane * PER + e];
    return p;
  };
  const int64_t r0 = (int64_t)kvh * pa.splits * pa.rows + s * G + h;
  auto split = [&](int p) __attribute__((always_inline)) {
    const int64_t at = r0 + (int64_t)min(p, pa.splits - 1) * pa.rows;
    return load(pa.ml + 2 * at, pa.acc + at * D);
  };
  float m = -INFINITY, l = 0.f;
  float acc[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) acc[e] = 0.f;
  auto fold = [&](const Part& p, bool counts) __attribute__((always_inline)) {
    const float x = counts ? p.ml.x : -INFINITY;
    const float mn = fmaxf(m, x);
    const float fo = m == -INFINITY ? 0.f : exp2f(m - mn), fq = counts ? exp2f(x - mn) : 0.f;
    l = l * fo + (counts ? p.ml.y : 0.f) * fq;
#pragma unroll
    for (int e = 0; e < PER; ++e) acc[e] = acc[e] * fo + (counts ? p.v[e] : 0.f) * fq;
    m = counts ? mn : m;
  };
  Part first[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) first[i] = split(r + i * R);
  const int ctx = max(0, min(len, sa.max_blocks * kBS));
  const bool has = ctx >= sa.prefix;
  const int np = past_prefix(ctx, sa.prefix) > 0 ? dsc.y : 0;
  const int64_t p0 = dsc.x + seg;
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) fold(first[i], has && r + i * R < pa.splits);
  if (has) {
#pragma unroll 4
    for (int p = r + AHEAD * R; p < pa.splits; p += R) fold(split(p), true);
  }
#pragma unroll 4
  for (int p = r; p < np; p += R) {
    fold(load(sa.part_ml + (p0 + p) * (2 * G) + 2 * h, sa.part_acc + (p0 + p) * (G * D) + h * D), true);
  }
  if constexpr (R > 1) {
    __shared__ float2 ml_lds[R][G];
    __shared__ float acc_lds[R][G][D];
    if (r > 0) {
      if (lane == 0) ml_lds[r][h] = make_float2(m, l);
#pragma unroll
      for (int e = 0; e < PER; ++e) acc_lds[r][h][lane * PER + e] = acc[e];
    }
    __syncthreads();
    if (r > 0) return;
#pragma unroll
    for (int i = 1; i < R; ++i) {
      Part p;
      p.ml = ml_lds[i][h];
#pragma unroll
      for (int e = 0; e < PER; ++e) p.v[e] = acc_lds[i][h][lane * PER + e];
      fold(p, p.ml.x != -INFINITY);
    }
  }
  S* out = static_cast<S*>(sa.out) + ((int64_t)s * sa.num_heads + (int64_t)kvh * G + h) * D + lane * PER;
  const float inv = l != 0.f ? 1.f / l : 1.f;
#pragma unroll
  for (int e = 0; e < PER; ++e) out[e] = elem<T>::from_f32(acc[e] * inv);
}

template <typename T, int D>
void launch_shared(const StreamArgs& sa, const PrefixArgs& pa, int G, int groups, const void* q, const void* kc,
                   const void* vc, const int32_t* bt, const int32_t* cl, hipStream_t s) {
  auto go = [&](auto g) {
    constexpr int GC = decltype(g)::value;
    using S = typename DecodeTileFor<T, D, GC>::S;
    hipLaunchKernelGGL((shared_prefix_kernel<T, D, GC>), dim3(groups), dim3(kPreThreads), 0, s, sa, pa,
                       static_cast<const S*>(q), static_cast<const S*>(kc), static_cast<const S*>(vc), bt, cl);
    // (Two waves to a head where there are more than four splits, and room in the workgroup.)
    constexpr int R = GC <= 8 ? 2 : 1;
    if (pa.splits > 4) {
      hipLaunchKernelGGL((shared_merge_kernel<T, D, GC, R>), dim3(sa.num_kv_heads, sa.batch), dim3(64 * GC * R), 0, s,
                         sa, pa, cl);
    } else {
      hipLaunchKernelGGL((shared_merge_kernel<T, D, GC, 1>), dim3(sa.num_kv_heads, sa.batch), dim3(64 * GC), 0, s, sa,
                         pa, cl);
    }
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
    default: go(std::integral_constant<int, 16>{}); break;  // shared_applies
  }
}

// What the entry refuses, and what the plan's 32-bit counts would not hold.
bool too_large(const Shape& sh) {
  return (int64_t)sh.MB * sh.bs > INT32_MAX || sh.B > 65535 || (int64_t)sh.B * (sh.H / sh.Hkv) > INT32_MAX;
}

struct SharedPlan {
  int32_t rows, row_tiles, tiles, split_tiles, splits, workers, stream_groups;
};
SharedPlan plan_shared(const Shape& sh, int32_t shared_blocks, bool f32) {
  SharedPlan p;
  const int64_t prefix = (int64_t)shared_blocks * sh.bs;
  p.rows = sh.B * (sh.H / sh.Hkv);
  p.row_tiles = (int32_t)ceil_div(p.rows, kPreRows);
  p.tiles = (int32_t)ceil_div(prefix, kTileKeys);
  // One workgroup of the product per CU beside the one of stream-K workers that its CU also holds.  Two where
  // that leaves splits of many row tiles (few of them, then, for the merge to read) and the table leaves the
  // sequences so little behind the prefix that the product (at 0.7 PFLOP/s) outlasts the workers (at 5 TB/s).
  // Splits of fewer than 8 key tiles (2 in fp32, whose tiles take 16 times the time) are not made: each writes
  // 4 D bytes a row for the merge to read.
  //   Measured (bf16, 32 / 8 heads of 128, us): 256 rows' 16,384 tokens with one token behind them 117 with one,
  // 109 with two, with 64 to 1,024 tokens behind them 159 and 177; 16 rows of 16,384 22.3 and 29.0; 16 rows of 2,048
  // with up to 700 behind them 17.4 with 8 tiles to a split, 18.2 with 4, 20.3 with 2, 22.0 with 16.  fp32, 64 rows of
  // 2,048: 39.8 with 2 tiles, 85 with 16.
  const double product = 4.0 * sh.B * sh.H * sh.D * (double)prefix / (f32 ? 0.1e15 : 0.7e15);
  const double stream = (f32 ? 8.0 : 4.0) * sh.B * sh.Hkv * sh.D * ((double)sh.MB * sh.bs - (double)prefix) / 5e12;
  const int64_t one = std::max<int64_t>(1, device_cu_count() / ((int64_t)sh.Hkv * p.row_tiles));
  const int64_t want = std::min(product > stream && one <= 8 ? 2 * one : one, ceil_div(p.tiles, f32 ? 2 : 8));
  p.split_tiles = (int32_t)ceil_div(p.tiles, std::min<int64_t>(want, p.tiles));
  p.splits = (int32_t)ceil_div(p.tiles, p.split_tiles);
  p.workers = stream_workers(sh);
  p.stream_groups = (int32_t)ceil_div(p.workers, kPreWaves);
  return p;
}
// Whether the shared product takes the call (else every sequence reads the prefix for itself).
bool shared_applies(const Shape& sh, int32_t dtype, int64_t kv_stride, const void* q, const void* kc, const void* vc,
                    const void* out) {
  return sh.D <= 128 && sh.B > 1 && tiles_take(sh, dtype, kv_stride, q, kc, vc, out);
}

// Whether the product saves more than it adds.  It saves all but one reading of the prefix, at the 8 TB/s at which
// the plain decode reads blocks that its sequences share; it adds the product's time over the CUs (a key tile of
// kPreRows rows, full or not: 0.45 us in 16 bits, 3.4 in fp32 at head_dim 128) and the merge's splits and its
// launch where the plain decode of a short table is one kernel (4 us).
//   Measured (32 / 8 heads, 1 to 200 tokens behind the prefix; shared and plain, us): bf16, head_dim 128, 4
// sequences: 512 tokens 15.0 / 13.3, 8,192 18.6 / 30.0; 32: 128 tokens 15.9 / 14.5, 512 16.9 / 20.3, 8,192
// 22.3 / 143; head_dim 64, 32: 512 tokens 18.3 / 11.5, 2,048 18.7 / 29.4.  fp32, head_dim 128, 2: 8,192 tokens
// 48.1 / 35.1; 8: 47.3 / 75.2, 512 tokens 20.4 / 17.5; 64: 512 tokens 29.4 / 48.0.
bool shared_pays(const Shape& sh, int32_t dtype, const SharedPlan& p) {
  const double saved = 2.0 * (sh.B - 1) * p.tiles * kTileKeys * sh.Hkv * sh.D * dtype_bytes(dtype) / 8e12;
  const double product = (double)p.tiles * sh.Hkv * p.row_tiles * sh.D * (dtype == RG_DTYPE_F32 ? 27e-9 : 3.5e-9) /
                         device_cu_count();
  return saved > product + 4e-6;
}

size_t prefix_bytes(const Shape& sh, const SharedPlan& p, size_t* ml_at) {
  const size_t n = (size_t)sh.Hkv * p.splits * p.rows;
  const size_t acc = align_up(n * sh.D * 4, 256);
  if (ml_at) *ml_at = acc;
  return acc + align_up(n * 8, 256);
}

}  // namespace

int probe_shared_prefix_kernels() {
  hipFuncAttributes at;
  if (hipFuncGetAttributes(&at, reinterpret_cast<const void*>(shared_prefix_kernel<bf16_t, 128, 4>)) != hipSuccess ||
      hipFuncGetAttributes(&at, reinterpret_cast<const void*>(shared_merge_kernel<bf16_t, 128, 4, 1>)) != hipSuccess) {
    return fail(RG_ERR_HIP, "failed to load the shared-prefix kernels: %s", hipGetErrorString(hipGetLastError()));
  }
  return RG_OK;
}

}  // namespace rg

using namespace rg;

extern "C" size_t rg_paged_attention_shared_prefix_workspace_bytes(int32_t batch_size, int32_t num_heads,
                                                                   int32_t num_kv_heads, int32_t head_dim,
                                                                   int32_t block_size, int32_t max_blocks_per_seq,
                                                                   int32_t shared_blocks) {
  if (batch_size <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 || head_dim <= 0 ||
      block_size <= 0 || max_blocks_per_seq <= 0 || shared_blocks < 0 || shared_blocks > max_blocks_per_seq) {
    return 0;
  }
  const Shape sh{num_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq, batch_size};
  if (too_large(sh)) return 0;
  size_t n = rg_paged_attention_v1_workspace_bytes(batch_size, num_heads, num_kv_heads, head_dim, block_size,
                                                   max_blocks_per_seq);
  if (shared_blocks > 0) {
    for (const bool f32 : {false, true}) {
      const SharedPlan p = plan_shared(sh, shared_blocks, f32);
      n = std::max(n, prefix_bytes(sh, p, nullptr) + stream_bytes(sh, p.workers, nullptr, nullptr));
    }
  }
  return n;
}

extern "C" int rg_paged_attention_shared_prefix_pays(int32_t batch_size, int32_t num_heads, int32_t num_kv_heads,
                                                     int32_t head_dim, int32_t block_size, int32_t max_blocks_per_seq,
                                                     int32_t shared_blocks, int32_t dtype) {
  if (batch_size <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 || head_dim <= 0 ||
      block_size <= 0 || shared_blocks <= 0 || shared_blocks > max_blocks_per_seq || dtype_bytes(dtype) == 0) {
    return 0;
  }
  const Shape sh{num_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq, batch_size};
  return !too_large(sh) && shared_applies(sh, dtype, 16, nullptr, nullptr, nullptr, nullptr) &&
                 shared_pays(sh, dtype, plan_shared(sh, shared_blocks, dtype == RG_DTYPE_F32))
             ? 1
             : 0;
}

extern "C" int rg_paged_attention_shared_prefix(const void* query, const void* key_cache, const void* value_cache,
                                                const int32_t* block_table, const int32_t* context_lens, void* output,
                                                float scale, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                                int32_t block_size, int32_t max_blocks_per_seq, int32_t batch_size,
                                                int32_t shared_blocks, int32_t dtype, int64_t kv_block_stride,
                                                void* workspace, size_t workspace_bytes, void* stream) {
  const char* op = "paged_attention_shared_prefix";
  const Shape sh{num_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq, batch_size};
  int st = check_decode_shape(op, sh, dtype, kv_block_stride);
  if (st != RG_OK) return st;
  if (shared_blocks < 0 || shared_blocks > max_blocks_per_seq) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: shared_blocks %d outside 0 .. max_blocks_per_seq %d", op, shared_blocks,
                max_blocks_per_seq);
  }
  if (too_large(sh)) {
    return fail(RG_ERR_NOT_SUPPORTED, "%s: a block table of %lld tokens, %d sequences", op,
                (long long)max_blocks_per_seq * block_size, batch_size);
  }
  if (batch_size == 0) return ok();
  if (!query || !key_cache || !value_cache || !block_table || !context_lens || !output) {
    return fail(RG_ERR_INVALID_ARGUMENT, "%s: null pointer argument", op);
  }
  const size_t need = rg_paged_attention_shared_prefix_workspace_bytes(batch_size, num_heads, num_kv_heads, head_dim,
                                                                       block_size, max_blocks_per_seq, shared_blocks);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned16(workspace))) {
    return fail(RG_ERR_WORKSPACE, "%s: workspace of %zu bytes (16-byte aligned), %zu required", op,
                workspace ? workspace_bytes : (size_t)0, need);
  }
  const int64_t kv_stride = kv_block_stride ? kv_block_stride : (int64_t)num_kv_heads * block_size * head_dim;
  if (shared_blocks == 0 || !shared_applies(sh, dtype, kv_stride, query, key_cache, value_cache, output)) {
    return rg_paged_attention_v1(query, key_cache, value_cache, block_table, context_lens, output, scale, num_heads,
                                 num_kv_heads, head_dim, block_size, max_blocks_per_seq, batch_size, dtype,
                                 kv_block_stride, workspace, workspace_bytes, stream);
  }
  const SharedPlan p = plan_shared(sh, shared_blocks, dtype == RG_DTYPE_F32);
  char* const ws = static_cast<char*>(workspace);
  size_t ml_at;
  const size_t pre = prefix_bytes(sh, p, &ml_at);
  StreamScratch sc;
  stream_bytes(sh, p.workers, &sc, ws + pre);
  StreamArgs sa{};
  sa.out = output;
  sa.part_acc = sc.acc;
  sa.part_ml = sc.ml;
  sa.seg_desc = sc.desc;
  sa.scale_log2 = scale * kLog2e;
  sa.num_heads = num_heads;
  sa.num_kv_heads = num_kv_heads;
  sa.bs_shift = block_shift(block_size);
  sa.max_blocks = max_blocks_per_seq << sa.bs_shift;
  sa.batch = batch_size;
  sa.num_workers = p.workers;
  sa.kv_stride = kv_stride;
  sa.table_stride = max_blocks_per_seq;
  sa.prefix = shared_blocks * block_size;
  PrefixArgs pa{};
  pa.acc = reinterpret_cast<float*>(ws);
  pa.ml = reinterpret_cast<float*>(ws + ml_at);
  // The product works with a positive scale: a negative one turns q's signs, 0 takes zeros for q.
  pa.scale_log2 = scale != 0.f ? fabsf(sa.scale_log2) : 1.f;
  pa.q_sign = scale == 0.f ? 0u : scale < 0.f ? 0x80008001u : 1u;
  pa.group = num_heads / num_kv_heads;
  pa.num_heads = num_heads;
  pa.num_kv_heads = num_kv_heads;
  pa.rows = p.rows;
  pa.prefix = sa.prefix;
  pa.subs = sa.prefix / kBS;
  pa.tiles = p.tiles;
  pa.split_tiles = p.split_tiles;
  pa.splits = p.splits;
  pa.bs_shift = sa.bs_shift;
  pa.stream_groups = p.stream_groups;
  pa.kv_stride = kv_stride;
  const int64_t groups = p.stream_groups + (int64_t)num_kv_heads * p.splits * p.row_tiles;
  if (groups > INT32_MAX) return fail(RG_ERR_NOT_SUPPORTED, "%s: %lld workgroups", op, (long long)groups);
  hipStream_t s = as_stream(stream);
  auto go = [&](auto tag) {
    using T = decltype(tag);
    if (head_dim == 128) launch_shared<T, 128>(sa, pa, pa.group, (int)groups, query, key_cache, value_cache, block_table, context_lens, s);
    else launch_shared<T, 64>(sa, pa, pa.group, (int)groups, query, key_cache, value_cache, block_table, context_lens, s);
    return check_launch(op);
  };
  return dispatch_dtype(dtype, go);
}
