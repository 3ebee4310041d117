// Attention of packed query rows (a decode step's, drafts, chunks of prompts) over the
// paged KV cache held in 4 bits (q4_cache.h), for gfx950.
//
// A value is d (c - 8): c the code, d the scale of its block of 32 channels.  Codes are
// multiplied as they are, as the numbers 16 + c (exact: two instructions a pair, with no
// conversion), and what that adds is taken off again:
//   s_t = sum_b dk[t][b] (sum_{c in b} q_c (16 + code) - 24 sum_{c in b} q_c)
//   o_c = sum_t p'[t][b] (16 + code[t][c]) - 24 sum_t p'[t][b],  p' = fp16(p_t dv[t][b])
// with v_mfma_f32_16x16x32, of bf16 numbers and then of fp16 ones, whose 32 channels are one
// block b of K: -24 sum q is its initial accumulator, and dk multiplies its result.  V's
// scale goes into the weights, which are rounded to fp16 once, an eighth of the outputs' own
// rounding (as bf16 numbers, as much as it; 2 to 7% less time but for the longest); sum p'
// is a product with ones.  So no value of the cache is rounded.  Scores, the running maximum,
// sums and outputs are fp32.  (Calls of many rows, is_prompt below, go to the kernels of
// prompt_attention.hip instead, which widen a tile once for all of its rows.)
//
// Products are transposed, S^T = K Q^T and O^T = V^T P^T: a row (a token's q head; "row =
// token * group + head in the group") is a column, lane 16 g + n holds row n's scores of
// tokens 16 t + 4 g + i (t < 2, i < 4) of a tile of 32, and these registers are the
// second product's operand as they stand, V's tokens being read in that order: lane j of
// 16 addresses token 16 (j / 4 % 2) + 4 g + j % 4, and the lower or the upper half of a
// block's 32 channels by j / 8, of a transposing LDS read of half-bytes
// (ds_read_b64_tr_b4: lane n gets channel n of the 16 lanes' tokens and halves).
//
// A workgroup is four waves that take the tiles of its part of the tokens in turn, each with
// its own softmax and its own two tiles in LDS, filled by direct loads a tile
// ahead: nothing is waited for but a wave's own loads, until the four states are joined.
//
// Bound by memory where there are many tokens; by instructions that are not in the
// instruction cache yet where there are few (about 30 cycles each, in every launch): the
// code of a tile and of what is done once is kept short for that.
//
// 32 / 8 heads of 128, us: 48 sequences behind 2000 to 32000 tokens 130 to 150 (635 MB, 4.9 to
// 4.2 TB/s; the same loads without the arithmetic 135, a copy's rate 124), 16 behind 300 to
// 8000 19.4 (2.3 TB/s), 8 of 5 tokens behind them 21, 1 behind 512 9.7.
#include <math.h>

#include <algorithm>

#include "q4_cache.h"
#include "row_items.h"
#include "smx_common.h"
#include "smx_launch.h"

namespace smx {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(1))) const void global_void;
typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) u32x2 lds_u32x2;
typedef __attribute__((address_space(3))) uint32_t lds_u32;
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
typedef __attribute__((address_space(4))) int32_t constant_i32;

// Log2 units: the largest weight times V's largest scale is between 2^TOP and 2^(TOP + LAG) by
// the reference.  (fp16 holds up to 65504, and 11 significant bits of 2^-14 or more: weights
// times scales down to 2^-25 of the largest; all are off by 2^-36 of it at most.)
constexpr float LAG = 4.f, TOP = 11.f;
constexpr float NO_REF = -3e38f;  // before the first token: below the scores of any use
constexpr int KT = 32;            // tokens of a tile
constexpr int WAVES = 4;
constexpr int ROUND = KT * WAVES;
constexpr int BEGIN = 2;          // rounds that the beginning of a tile takes the time of

struct Q4Args {
  const uint16_t* q;
  const uint8_t* codes;
  const uint16_t* scales;
  const int32_t* table;        // [num_seqs, max_blocks]
  const int32_t* query_start;  // [num_seqs + 1], or null: row r is sequence r's one token
  const int32_t* seq_lens;     // [num_seqs]
  uint16_t* out;
  float* part_o;    // [rows, splits, HD], where splits > 1
  float* part_lse;  // [rows, splits], log2 units
  int32_t* counts;  // [rows] parts in use
  int64_t q_stride;
  int num_tokens, num_seqs, max_blocks, num_blocks, bs_log2, n_q, n_kv, group;
  int splits, target;
  float scale_log2;
  float group_inv, target_inv, splits_inv;  // 1 / group, 1 / target, 1 / (splits - 2)
};

// Bytes of a tile in LDS: K's codes, V's codes, K's scales, V's scales.
template <int HD>
struct Tile {
  static constexpr int NB = HD / 32;
  static constexpr int CODES = KT * HD / 2, SCALES = KT * NB * 2;
  static constexpr int BYTES = 2 * (CODES + SCALES);
};

// Eight codes (the half-bytes of w) as numbers 16 + code, pairs of half-bytes j and j + 4:
// bits 3..6 of a bf16, or 6..9 of an fp16, with exponent 4 are whole units.  The masks and the
// exponents come in registers, of which the compiler does not know the value: as literals
// they would make two instructions of v_and_or_b32 (three a pair of codes, not two).
struct CodeBits {
  uint32_t mask = 0x00780078u, one = 0x41804180u;
  uint32_t mask16 = 0x03c003c0u, one16 = 0x4c004c00u;
  float zero = 0.f;  // likewise, for products that are one instruction with a sum only
  __device__ __forceinline__ CodeBits() {
    __asm__("" : "+s"(mask));
    __asm__("" : "+v"(one));
    __asm__("" : "+s"(mask16));
    __asm__("" : "+v"(one16));
    __asm__("" : "+s"(zero));
  }
  __device__ __forceinline__ bf16x8 bf16(uint32_t w) const {
    return __builtin_bit_cast(bf16x8, u32x4{((w << 3) & mask) | one, ((w >> 1) & mask) | one,
                                            ((w >> 5) & mask) | one, ((w >> 9) & mask) | one});
  }
  __device__ __forceinline__ f16x8 f16(uint32_t w) const {
    return __builtin_bit_cast(f16x8, u32x4{((w << 6) & mask16) | one16, ((w << 2) & mask16) | one16,
                                           ((w >> 2) & mask16) | one16, ((w >> 6) & mask16) | one16});
  }
};

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ float half_of(uint32_t w, int i) {
  return (float)__builtin_bit_cast(f16x2, w)[i];
}

// One piece of a workgroup's work: 16 rows from row0 on, tokens [from, to), of a tile of
// rows that `parts` workgroups share, `slot` of them before this one.
struct Q4Item {
  const int32_t* table;
  int token0, row0, rows, from, to, slot, ahead, parts;
};

// a / c for 0 <= a < 2^24 and inv = 1 / c to a few units of the last place.
__device__ __forceinline__ int small_div(int a, int c, float inv) {
  int q = (int)((float)a * inv);
  const int r = a - q * c;
  return q + (r >= c) - (r < 0);
}

template <int HD>
__device__ __forceinline__ void q4_attend(const Q4Args& A, const Q4Item& it, int kvh,
                                          uint8_t* smem) {
  using T = Tile<HD>;
  constexpr int NB = T::NB, DT = HD / 16, RB = HD / 2;  // blocks, tiles of dims, bytes a row
  constexpr int CHUNKS = RB / 16;                       // 16-byte chunks a row
  constexpr int LOADS = KT * CHUNKS / 64;               // direct loads of a K (V) tile
  constexpr int SPAN = 64 / CHUNKS;                     // tokens of one
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int bs = 1 << A.bs_log2;

  // ---- this lane's row (fewer than 2^24 of a sequence: the host sees to it)
  const int row = it.row0 + n, row_tok = small_div(row, A.group, A.group_inv);
  const bool valid = n < it.rows;
  const int64_t tok = it.token0 + row_tok;
  const int head = kvh * A.group + row - row_tok * A.group;
  u32x4 qx[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    qx[b] = u32x4{0u, 0u, 0u, 0u};
    if (valid)
      qx[b] = *reinterpret_cast<const u32x4*>(A.q + tok * A.q_stride + head * HD + 32 * b + 8 * g);
  }
  const int lim = valid ? min(max(it.ahead + row_tok + 1, 0), it.to) : it.to;
  const int lim_min = __builtin_amdgcn_readfirstlane(-wave_max_i32(-lim));

  // ---- direct loads of a tile.  LDS is filled in the lanes' order, 16 bytes each; which
  // 16 bytes those are is the lane's choice: chunk c of token t is put in place
  // c ^ swizzle(t) of its row, so that the lanes of one LDS read are on different banks.
  // A table entry outside the cache is read as page 0 (its tokens' scores become NaN),
  // and tokens past the end are the rest of their page.
  const int ntiles = (it.to - it.from + KT - 1) / KT;
  const constant_i32* const table = (const constant_i32*)it.table;
  const int table_end = max(it.to - 1, 0);
  const int64_t plane = (int64_t)A.num_blocks * A.n_kv << A.bs_log2;  // rows of K
  const int ltok = lane / CHUNKS, lchunk = lane % CHUNKS;
  auto k_swz = [](int t) { return HD == 128 ? (t >> 2) & 3 : (t >> 3) & 1; };
  auto v_swz = [](int t) { return HD == 128 ? (t >> 1 & 2) + (t >> 4 & 1) : t >> 4 & 1; };
  auto look_up = [&](int tile) {
    return table[min(it.from + tile * KT, table_end) >> A.bs_log2];
  };
  auto known = [&](int page) { return (unsigned)page < (unsigned)A.num_blocks; };
  auto stage = [&](lds_u8* __restrict__ dst, int tile, int page) {
    const int t0 = it.from + tile * KT;
    const int64_t row = (((int64_t)(known(page) ? page : 0) * A.n_kv + kvh) << A.bs_log2) +
                        (t0 & (bs - 1));
    {
      // the scales of two tokens (four of 64 channels) a lane, K's and then V's
      constexpr int PER = 16 / (2 * NB), HALF = KT / PER;
      if (lane < 2 * HALF) {
        const int64_t at = row + lane % HALF * PER + (lane < HALF ? 0 : plane);
        __builtin_amdgcn_global_load_lds((global_void*)(A.scales + at * NB),
                                         (lds_void*)(dst + 2 * T::CODES), 16, 0, 0);
      }
    }
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int t = i * SPAN + ltok;
        const int src = t * RB + 16 * (lchunk ^ (v ? v_swz(t) : k_swz(t)));
        __builtin_amdgcn_global_load_lds((global_void*)(A.codes + (row + (v ? plane : 0)) * RB + src),
                                         (lds_void*)(dst + v * T::CODES + i * 1024), 16, 0, 0);
      }
  };

  // ---- the row's state: the exponents' reference (log2 units: TOP below the running maximum
  // and V's largest scale together, or up to LAG less than that), the sum of 2^(score - ref) over this lane's tokens, the output's
  // products with 16 + code and, block by block, the sums of their weights (in every register
  // the same; of its own for each block, so that one that is NaN stays among its dims).
  float ref = NO_REF, l = 0.f;
  f32x4 o[DT], w_sum[NB];
#pragma unroll
  for (int d = 0; d < DT; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int b = 0; b < NB; ++b) w_sum[b] = f32x4{0.f, 0.f, 0.f, 0.f};
  bf16x8 qf[NB];
  const uint32_t one2 = 0x3c003c00u;
  const f16x8 ones = __builtin_bit_cast(f16x8, u32x4{one2, one2, one2, one2});
  f32x4 c0[NB];
  const CodeBits codes;
  const int k_addr = HD == 128 ? n * RB + 16 * (g ^ k_swz(n))
                               : n * RB + 16 * ((g >> 1) ^ k_swz(n)) + 8 * (g & 1);
  const int vt = 16 * (n >> 2 & 1) + 4 * g + (n & 3);
  const int v_addr = T::CODES + vt * RB + 8 * (n >> 3), v_place = v_swz(vt);
  const int s_addr = 2 * T::CODES + 4 * g * 2 * NB;  // scales of tokens 4 g ..

  // Scales of V are below the fp16 number of the bits v_limit, a power of two 2^e, and so
  // weights times them below 2^(score - ref + e): scores up to ref + room leave ref where it is.
  constexpr int PAIRS = T::SCALES / 4;
  uint16_t v_limit = 0x400;
  float room = TOP + LAG + 14.f;

  auto compute = [&](auto plain, const lds_u8* __restrict__ buf, int base, bool bad) {
    // scales of tokens 16 t + 4 g + i, block b: fp16 i * NB + b
    auto scales_of = [&](int v, int t, uint32_t (&w)[2 * NB]) {
#pragma unroll
      for (int j = 0; j < NB / 2; ++j) {
        const u32x4 x = *(const lds_u32x4*)(buf + s_addr + v * T::SCALES + 16 * t * 2 * NB + 16 * j);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[4 * j + i] = x[i];
      }
    };
    float p[2][4];  // scores, then weights
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      uint32_t dk[2 * NB], kw[NB];
      scales_of(0, t, dk);
      if constexpr (HD == 128) {
        const u32x4 x = *(const lds_u32x4*)(buf + t * 16 * RB + k_addr);
#pragma unroll
        for (int b = 0; b < 4; ++b) kw[b] = x[b];
      } else {
        const u32x2 x = *(const lds_u32x2*)(buf + t * 16 * RB + k_addr);
        kw[0] = x[0];
        kw[1] = x[1];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) p[t][i] = 0.f;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const f32x4 s = mfma(codes.bf16(kw[b]), qf[b], c0[b]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          p[t][i] = fmaf(half_of(dk[(i * NB + b) / 2], (i * NB + b) & 1), s[i], p[t][i]);
      }
    }
    const int left = lim - base - 4 * g;  // tokens 16 t + i below it are seen
    if constexpr (!plain) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = bad ? __builtin_nanf("") : p[t][i];
          p[t][i] = 16 * t + i < left ? x : -INFINITY;
        }
    }
    // Two of V's scales a lane, those of the tile once: whether one is past the largest so far
    // (an unseen token's, an infinity and a NaN do not count).
    uint32_t sizes = *(const lds_u32*)(buf + 2 * T::CODES + T::SCALES + 4 * (lane % PAIRS));
    sizes &= 0x7fff7fffu;
    if constexpr (!plain) sizes = lane % PAIRS * 2 / NB < it.to - base ? sizes : 0u;
    const u16x2 past = __builtin_bit_cast(u16x2, sizes) - u16x2{v_limit, v_limit};
    const bool larger = __builtin_elementwise_min(past[0], past[1]) < (uint16_t)(0x7c00 - v_limit);
    float mx = p[0][0];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, p[t][i]);
    mx = xor_max<32>(xor_max<16>(mx)) * A.scale_log2;
    if (__builtin_amdgcn_ballot_w64(mx > ref + room || larger)) {
      const int lo = sizes & 0xffff, hi = sizes >> 16;
      const int most = wave_max_i32(max(lo < 0x7c00 ? lo : 0, hi < 0x7c00 ? hi : 0));
      v_limit = (uint16_t)__builtin_amdgcn_readfirstlane(max((int)v_limit, (most & 0x7c00) + 0x400));
      const float above = (float)(v_limit >> 10) - 15.f;
      room = TOP + LAG - above;
      const float next = fmaxf(ref, mx + above - TOP);
      const float alpha = __builtin_amdgcn_exp2f(ref - next);
      ref = next;
      l *= alpha;
#pragma unroll
      for (int b = 0; b < NB; ++b) w_sum[b] *= alpha;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= alpha;
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        p[t][i] = __builtin_amdgcn_exp2f(fmaf(p[t][i], A.scale_log2, -ref));
    l += ((p[0][0] + p[0][1]) + (p[0][2] + p[0][3])) + ((p[1][0] + p[1][1]) + (p[1][2] + p[1][3]));
    // O^T += V^T P'^T, block by block
    uint32_t dv[2][2 * NB];
    scales_of(1, 0, dv[0]);
    scales_of(1, 1, dv[1]);
    if constexpr (!plain) {  // (an unseen token's scale may be anything)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i)
          dv[t][i] = 16 * t + i * 2 / NB < left ? dv[t][i] : 0u;
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      u32x4 x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = i * NB + b;
        // (one instruction with the conversion, where a product alone would be two)
        x[i] = cvt_pk_f16(fmaf(p[0][i], half_of(dv[0][e / 2], e & 1), codes.zero),
                          fmaf(p[1][i], half_of(dv[1][e / 2], e & 1), codes.zero));
      }
      const f16x8 w = __builtin_bit_cast(f16x8, x);
      w_sum[b] = mfma(ones, w, w_sum[b]);
      const i32x2 v = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
          (lds_i32x2*)(buf + v_addr + 16 * (b ^ v_place)));
      o[2 * b] = mfma(codes.f16((uint32_t)v[0]), w, o[2 * b]);
      o[2 * b + 1] = mfma(codes.f16((uint32_t)v[1]), w, o[2 * b + 1]);
    }
  };

  // ---- this wave's tiles
  lds_u8* const lds = (lds_u8*)smem + wave * 2 * T::BYTES;
  int tile = wave, page = look_up(tile), next_page = look_up(tile + WAVES);
  if (tile < ntiles) stage(lds, tile, page);
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    qf[b] = __builtin_bit_cast(bf16x8, qx[b]);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum = dot2_bf16(qx[b][i], 0x3f803f80u, sum);
    sum = -24.f * xor_sum<32>(xor_sum<16>(sum));
    c0[b] = f32x4{sum, sum, sum, sum};
  }
  auto round = [&](lds_u8* __restrict__ next, const lds_u8* __restrict__ cur) {
    __builtin_amdgcn_s_waitcnt(0x0f70);  // this tile's loads have arrived
    __asm__ volatile("" ::: "memory");
    const bool bad = !known(page);
    if (tile + WAVES < ntiles) stage(next, tile + WAVES, next_page);
    page = next_page;
    next_page = look_up(tile + 2 * WAVES);
    const int base = it.from + tile * KT;
    if (!bad && base + KT <= lim_min)
      compute(std::true_type{}, cur, base, false);
    else
      compute(std::false_type{}, cur, base, bad);
  };
  for (int at = 0; tile < ntiles; tile += WAVES, at ^= 1)
    round(lds + (at ^ 1) * T::BYTES, lds + at * T::BYTES);

  // ---- what 16 + code added, then the waves' states: each leaves its own in the place of
  // its tiles, and joins the four of a quarter of the dims
  l = xor_sum<32>(xor_sum<16>(l));
  constexpr int QT = DT / WAVES;            // tiles of dims a wave joins
  constexpr int STATE = 2 * T::BYTES / 4;  // floats between two waves' states
  static_assert(STATE >= 16 * HD + 32, "a state fits in the place of the tiles");
  float* const jo = reinterpret_cast<float*>(smem);
  float* const mine = jo + wave * STATE;
#pragma unroll
  for (int d = 0; d < DT; ++d)
    *reinterpret_cast<f32x4*>(mine + (d * 64 + lane) * 4) = o[d] + -24.f * w_sum[d / 2][0];
  if (g == 0) {
    mine[16 * HD + n] = ref;
    mine[16 * HD + 16 + n] = l;
  }
  __syncthreads();
  float refs[WAVES];
  ref = NO_REF;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    refs[w] = jo[w * STATE + 16 * HD + n];
    ref = fmaxf(ref, refs[w]);
  }
  l = 0.f;
#pragma unroll
  for (int d = 0; d < QT; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const float a = __builtin_amdgcn_exp2f(refs[w] - ref);
    l = fmaf(jo[w * STATE + 16 * HD + 16 + n], a, l);
#pragma unroll
    for (int d = 0; d < QT; ++d)
      o[d] += a * *reinterpret_cast<const f32x4*>(jo + w * STATE +
                                                  ((wave * QT + d) * 64 + lane) * 4);
  }
  if (!valid) return;
  // l == 0 only where the row sees no token: its output is 0, its weight none
  const float inv = l == 0.f ? 0.f : 1.f / l;
  // (the row again, from its number: not kept in registers through the tiles)
  int row_again = it.row0 + n;
  __asm__ volatile("" : "+v"(row_again));
  const int again_tok = small_div(row_again, A.group, A.group_inv);
  const int64_t orow = (int64_t)(it.token0 + again_tok) * A.n_q + kvh * A.group + row_again -
                       again_tok * A.group;
  const int dim = wave * QT * 16 + 4 * g;
  if (it.parts == 1) {
#pragma unroll
    for (int d = 0; d < QT; ++d)
      st_agent(reinterpret_cast<u32x2*>(A.out + orow * HD + dim + 16 * d),
               u32x2{cvt_pk_bf16(o[d][0] * inv, o[d][1] * inv),
                     cvt_pk_bf16(o[d][2] * inv, o[d][3] * inv)});
  } else if (l != 0.f) {  // the merge reads no partial whose weight is none
    float* const dst = A.part_o + (orow * A.splits + it.slot) * HD + dim;
#pragma unroll
    for (int d = 0; d < QT; ++d)
      st_agent_b128(dst + 16 * d, __builtin_bit_cast(u32x4, o[d] * inv));
  }
  if (wave == 0 && g == 0 && A.splits > 1) {
    if (it.slot == 0) st_agent(A.counts + orow, it.parts == 1 ? 0 : it.parts);
    if (it.parts > 1)
      st_agent(A.part_lse + orow * A.splits + it.slot, l == 0.f ? -INFINITY : ref + log2f(l));
  }
}

// Sequence r's queries are the tokens [query_start[r], query_start[r + 1]), the last n of
// its L tokens; its work is its tiles of 16 rows times the rounds (ROUND tokens) of L.  The
// work of all sequences, end to end, is cut into parts of `chunk` rounds, one a workgroup.
// Equal parts, whatever the lengths, can be the end of a tile and the beginning of the next,
// each with its partial; every beginning costs about 4 us (the chain of length, table entry
// and first tile, and the join), as much as BEGIN rounds.  So every tile begins a new part
// where parts no longer than that allow it.  Grid: kv heads, parts.
template <int HD>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(HD == 64 ? 4 : 2)))
void q4_attention_kernel(Q4Args A) {
  constexpr int M = 16;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[WAVES * 2 * Tile<HD>::BYTES];
  const int kvh = blockIdx.x, lane = threadIdx.x & 63;
  const int cap = A.max_blocks << A.bs_log2;
  int q0, nq, len, tiles, rounds;  // of sequence b + lane
  auto load = [&](int b) {
    const int r = b + lane;
    q0 = nq = len = tiles = rounds = 0;
    if (r < A.num_seqs) {
      len = min(max(A.seq_lens[r], 0), cap);
      q0 = r;
      nq = 1;
      if (A.query_start) {
        q0 = min(max(A.query_start[r], 0), A.num_tokens);
        nq = max(min(A.query_start[r + 1], A.num_tokens) - q0, 0);
      }
      tiles = (nq * A.group + M - 1) / M;
      rounds = tiles ? max((len + ROUND - 1) / ROUND, 1) : 0;
    }
  };
  load(0);
  float all = (float)tiles * (float)rounds;
  int top = wave_max_i32(rounds);
  for (int b = 64; b < A.num_seqs; b += 64) {
    load(b);
    all += (float)tiles * (float)rounds;
    top = max(top, wave_max_i32(rounds));
  }
  if (A.num_seqs > 64) load(0);
  all = wave_sum(all);
  // (the host has bounded the sum for offsets in order; there is no work in others)
  if (all > 0x1p28f) return;
  // `chunk` need not be exact (workgroups take a second part where there is one), but a
  // tile of `top` rounds must lie in at most (top - 2) / chunk + 2 <= splits parts
  int chunk = (int)(all * A.target_inv + 0.999f);
  if (A.splits > 2) chunk = max(chunk, (int)((float)top * A.splits_inv) + 1);
  chunk = max(chunk, A.splits == 1 ? top : 1);
  const int equal = chunk;
  float inv = __builtin_amdgcn_rcpf((float)chunk);
  // (so much work that a part's length is nothing beside it: the sums below stay in int32,
  // and so do a part's tokens, where parts end past the tokens of a tile)
  bool apart = A.num_seqs <= 64 && all < 0x1p22f;
  auto padded = [&](int r) {
    if (!apart) return r;
    const int q = small_div(r, chunk, inv);
    return q * chunk < r ? (q + 1) * chunk : r;
  };
  while (apart) {
    const float sum = wave_sum((float)(tiles * padded(rounds)));
    if (sum <= (float)(chunk * A.target) || chunk >= top) break;
    // the tiles' ends make too many: somewhat longer parts
    chunk = min(max(chunk + 1, (int)(sum * A.target_inv + 0.999f)), top);
    apart = chunk <= equal + BEGIN;
    if (!apart) chunk = equal;
    inv = __builtin_amdgcn_rcpf((float)chunk);
  }
  chunk = __builtin_amdgcn_readfirstlane(chunk);
  // Part after part (one, unless there are more than workgroups), piece after piece.
  // What is known of the sequences is loaded again for each: it would be in registers
  // through the tiles.
  int part = blockIdx.y, at = part * chunk, b = 0, base = 0;
  for (;;) {
    const int work = tiles * padded(rounds);
    const int incl = wave_scan_i32(work), here = __builtin_amdgcn_readlane(incl, 63);
    if (at >= base + here) {  // in a later 64 sequences
      base += here;
      b += 64;
      if (b >= A.num_seqs) break;
      load(b);
      continue;
    }
    const int i = __ffsll((unsigned long long)__ballot(base + incl > at)) - 1;
    const int r = padded(__builtin_amdgcn_readlane(rounds, i));
    int tile_at = base + __builtin_amdgcn_readlane(incl, i) - __builtin_amdgcn_readlane(work, i);
    int tile = 0;
    if (at - tile_at >= r) {
      tile = (at - tile_at) / r;
      tile_at += tile * r;
    }
    const int begin = part * chunk, end = begin + chunk;
    const int from = at - tile_at, to = min(r, end - tile_at);
    Q4Item it;
    it.table = A.table + (int64_t)(b + i) * A.max_blocks;
    it.token0 = __builtin_amdgcn_readlane(q0, i);
    const int n = __builtin_amdgcn_readlane(nq, i), L = __builtin_amdgcn_readlane(len, i);
    it.row0 = tile * M;
    it.rows = min(M, n * A.group - it.row0);
    it.ahead = L - n;  // the position of the first query token
    const int range = min(max(it.ahead + (it.row0 + it.rows - 1) / A.group + 1, 0), L);
    it.from = min(from * ROUND, range);
    it.to = min(to * ROUND, range);
    // the parts of this tile that end at or before `begin`, and from `end` on
    it.slot = from > 0 ? small_div(begin - tile_at + chunk - 1, chunk, inv) : 0;
    it.parts = it.slot + 1 +
               (tile_at + r > end ? small_div(tile_at + r - end + chunk - 1, chunk, inv) : 0);
    q4_attend<HD>(A, it, kvh, smem);
    at += to - from;
    if (at >= end) {
      part += A.target;
      at = part * chunk;
    }
    if (A.num_seqs <= 64 && at >= here) break;
    load(b);
    __syncthreads();  // the states are read out
  }
  stores_done();
}

// How a call is cut, from its sizes (lengths are on the device).  512 workgroups fill the
// chip once (two a compute unit, by their registers).  Twice as many parts, 48 sequences
// behind 2000 to 32000 152 us for 155, but 16 behind 300 to 8000 22 for 19.  Heads of 64
// leave registers for four, which few rows a sequence are cut for from 16 rounds (of the
// tables' capacity) a part of 512 on: us with 512 / 768 / 1024 parts, 32 / 8 heads, 48
// sequences behind 2000 to 32000 92 / 90 / 85, 128 behind 500 to 4000 50 / 44 / 41, 32 behind 500
// to 8000 24.3 / 21.2 / 20.6, 8 behind 32000 42 / 40 / 40, 64 behind 300 to 2000 (21 rounds) 20 /
// 19 / 17, 24 behind 1000 to 20000, 16 / 4 18.8 / 18.0 / 19.1, but 2 behind 32000 (12) 15.7 and
// 16.9 with 1024.
constexpr int FILL = 512, MAX_PARTS = 64;

int tune(const char* name, int v) {
  const char* e = tuning_env(name);
  return e ? atoi(e) : v;
}

struct Q4Choice {
  int splits, target;
};

// Tiles of 16 rows, the most there can be.
int64_t q4_tiles(int64_t num_tokens, int64_t num_seqs, int group) {
  return (num_tokens * group + 15) / 16 + num_seqs - 1;
}

// Whether a call's rows are prompts': more than two tiles of a sequence on average, and
// more work altogether than tiles of 16 rows, which widen every code and scale again,
// are done with first (the tables' capacity stands for the lengths, and a tile's
// beginning counts as three rounds).  us by tiles / by the prompt kernels, and the work, 32
// / 8 heads of 128: 100 tokens 6.0 / 10.3 (0.8k), 8 x 20 behind 1000 24 / 31 (3.5k), 300
// tokens 12.5 / 14.7 (3.6k), 40 behind 8000 26 / 29 (5.3k), 16 x 60 21 / 14 (7.7k), 8 x 60
// behind 1000 38 / 33 (12k), 60 behind 15000 53 / 43 (15k); heads of 64: 1000 tokens, 14 / 2
// heads 19 / 24 (9.6k), 8 x 100 behind 500, 16 / 4 15.8 / 17.6 (6.4k), 500 behind 4000, 14 / 2
// 44 / 34 (17k).
bool is_prompt(int64_t num_tokens, int64_t num_seqs, int64_t cap, int group, int n_kv, int hd) {
  if (num_tokens * group <= 32 * num_seqs) return false;
  const int64_t work = q4_tiles(num_tokens, num_seqs, group) * ((cap + ROUND - 1) / ROUND + 3) * n_kv;
  return work > tune("SMX_Q4_WORK", hd == 64 ? 9600 : 5500);
}

Q4Choice choose_q4(int64_t num_tokens, int64_t num_seqs, int64_t cap, int group, int n_kv, int hd) {
  Q4Choice c{};
  const int64_t rounds = (cap + ROUND - 1) / ROUND;  // the most of a tile
  const bool few = num_tokens * group <= 32 * num_seqs;
  const int64_t work = q4_tiles(num_tokens, num_seqs, group) * rounds * n_kv;
  const int fill = hd == 64 && few && work > 16 * FILL ? 2 * FILL : FILL;
  c.target = std::max(1, fill / n_kv);
  // uneven lengths: the longest may take four times the parts of even ones
  const int64_t even = (c.target + num_seqs - 1) / num_seqs;
  c.splits = (int)std::clamp<int64_t>(4 * even + 2, 3, MAX_PARTS);
  // Tiles of few rounds are not cut (up to 64 sequences, each can begin a part of its own): the
  // merge takes longer than they do.  us cut / whole, 32 / 8 heads of 128: 200 tokens (3 rounds
  // of capacity) 8.0 / 6.5, 100 queries 7.7 / 5.9, 16 sequences of 100 to 500 (5) 9.4 / 8.5, 48
  // 13.9 / 12.0, 512 tokens (6) 9.2 / 9.25, but 700 (7) 9.3 / 10.3.
  const bool whole = rounds == 1 || (num_seqs <= 64 && rounds <= 6);
  c.splits = whole ? 1 : (int)std::min<int64_t>(c.splits, rounds + 1);
  return c;
}

int64_t q4_workspace(int64_t rows, int64_t splits, int hd) {
  return splits == 1 ? 0 : rows * (splits * (hd + 1) + 1) * 4;
}

}  // namespace
}  // namespace smx

#include "smx_abi_util.h"

extern "C" int64_t smx_q4_attention_workspace(int32_t num_tokens, int32_t num_seqs,
                                              int32_t max_blocks, int32_t block_size, int32_t n_q,
                                              int32_t n_kv, int32_t head_dim) {
  if (num_tokens < 1 || num_seqs < 1 || max_blocks < 1 || block_size < 1 || n_kv < 1 ||
      n_q < n_kv || n_q % n_kv || head_dim < 1)
    return -1;
  if (smx::is_prompt(num_tokens, num_seqs, (int64_t)max_blocks * block_size, n_q / n_kv,
                     n_kv, head_dim)) {
    smx::Q4Prompt p{};
    p.num_tokens = num_tokens;
    p.num_seqs = num_seqs;
    p.max_blocks = max_blocks;
    while ((1 << p.bs_log2) < block_size) ++p.bs_log2;
    p.n_q = n_q;
    p.n_kv = n_kv;
    p.head_dim = head_dim;
    return smx::q4_prompt_workspace(p);
  }
  const smx::Q4Choice c = smx::choose_q4(num_tokens, num_seqs, (int64_t)max_blocks * block_size,
                                         n_q / n_kv, n_kv, head_dim);
  return smx::q4_workspace((int64_t)num_tokens * n_q, c.splits, head_dim);
}

extern "C" int smx_q4_attention(void* stream, const void* q, int64_t q_stride, const void* codes,
                                const void* scales, const int32_t* block_table,
                                const int32_t* query_start_loc, const int32_t* seq_lens,
                                void* workspace, int64_t workspace_bytes, void* out,
                                int32_t num_tokens, int32_t num_seqs, int32_t max_blocks,
                                int32_t num_blocks, int32_t block_size, int32_t n_q, int32_t n_kv,
                                int32_t head_dim, float scale) {
  SMX_REQUIRE(q && codes && scales && block_table && seq_lens && out, "null pointer argument");
  SMX_REQUIRE(head_dim == 64 || head_dim == 128, "head_dim must be 64 or 128");
  SMX_REQUIRE(n_kv >= 1 && n_kv <= 65535 && n_q >= n_kv && n_q % n_kv == 0,
              "n_q must be a multiple of n_kv");
  SMX_REQUIRE(num_blocks >= 1, "num_blocks must be >= 1");
  SMX_REQUIRE(block_size >= 32 && block_size <= 4096 && (block_size & (block_size - 1)) == 0,
              "block_size must be a power of two in [32, 4096]");
  SMX_REQUIRE(max_blocks >= 1 && (int64_t)max_blocks * block_size <= INT32_MAX - 4096,
              "max_blocks * block_size (a sequence's capacity) must fit in int32");
  SMX_REQUIRE(num_seqs >= 1 && num_seqs <= 65535, "num_seqs must be in [1, 65535]");
  SMX_REQUIRE(num_tokens >= 1 && (int64_t)num_tokens * n_q < (1ll << 30),
              "num_tokens * n_q must be in [1, 2^30)");
  SMX_REQUIRE(query_start_loc || num_tokens == num_seqs,
              "without query_start_loc there must be a row for each sequence");
  SMX_REQUIRE(scale > 0.f && isfinite(scale), "scale must be positive and finite");
  SMX_REQUIRE((uintptr_t)q % 16 == 0 && (uintptr_t)codes % 16 == 0 &&
                  (uintptr_t)scales % 16 == 0 && (uintptr_t)out % 16 == 0,
              "q, codes, scales and out must be 16-byte aligned");
  SMX_REQUIRE(((uintptr_t)block_table | (uintptr_t)seq_lens | (uintptr_t)query_start_loc) % 4 == 0,
              "int arrays must be 4-byte aligned");
  SMX_REQUIRE(q_stride >= (int64_t)n_q * head_dim && q_stride % 8 == 0,
              "q_stride must be a multiple of 8 and hold n_q heads");
  int bs_log2 = 0;
  while ((1 << bs_log2) < block_size) ++bs_log2;
  const float scale_log2 = scale * 1.44269504088896340736f;
  if (smx::is_prompt(num_tokens, num_seqs, (int64_t)max_blocks * block_size, n_q / n_kv,
                     n_kv, head_dim)) {
    const smx::Q4Prompt p{(const uint16_t*)q, (const uint8_t*)codes, (const uint16_t*)scales,
                          block_table, query_start_loc, seq_lens, workspace, out, q_stride,
                          num_tokens, num_seqs, max_blocks, num_blocks, bs_log2, n_q, n_kv,
                          head_dim, scale_log2};
    const int64_t need = smx::q4_prompt_workspace(p);
    SMX_REQUIRE(need >= 0, "too many row tiles for one launch");
    SMX_REQUIRE(need == 0 || (workspace && (uintptr_t)workspace % 16 == 0 &&
                              workspace_bytes >= need),
                "workspace must be 16-byte aligned and hold smx_q4_attention_workspace bytes");
    return smx::q4_prompt((hipStream_t)stream, p);
  }
  const smx::Q4Choice c = smx::choose_q4(num_tokens, num_seqs, (int64_t)max_blocks * block_size,
                                         n_q / n_kv, n_kv, head_dim);
  SMX_REQUIRE(smx::q4_tiles(num_tokens, num_seqs, n_q / n_kv) *
                      (((int64_t)max_blocks * block_size + smx::ROUND - 1) / smx::ROUND) <
                  (1ll << 28),
              "row tiles times the sequences' capacity / 128 must be below 2^28");
  const int64_t rows = (int64_t)num_tokens * n_q;
  SMX_REQUIRE(c.splits == 1 || (workspace && (uintptr_t)workspace % 16 == 0 &&
                                workspace_bytes >= smx::q4_workspace(rows, c.splits, head_dim)),
              "workspace must be 16-byte aligned and hold smx_q4_attention_workspace bytes");
  smx::Q4Args a{};
  a.q = (const uint16_t*)q;
  a.codes = (const uint8_t*)codes;
  a.scales = (const uint16_t*)scales;
  a.table = block_table;
  a.query_start = query_start_loc;
  a.seq_lens = seq_lens;
  a.out = (uint16_t*)out;
  a.part_o = (float*)workspace;
  a.part_lse = a.part_o + rows * c.splits * head_dim;
  a.counts = (int32_t*)(a.part_lse + rows * c.splits);
  a.q_stride = q_stride;
  a.num_tokens = num_tokens;
  a.num_seqs = num_seqs;
  a.max_blocks = max_blocks;
  a.num_blocks = num_blocks;
  a.bs_log2 = bs_log2;
  a.n_q = n_q;
  a.n_kv = n_kv;
  a.group = n_q / n_kv;
  a.splits = c.splits;
  a.target = c.target;
  a.scale_log2 = scale_log2;
  a.group_inv = 1.f / a.group;
  a.target_inv = 1.f / c.target;
  a.splits_inv = c.splits > 2 ? 1.f / (c.splits - 2) : 0.f;
  const dim3 grid(n_kv, c.target);
  const auto kernel = head_dim == 128 ? smx::q4_attention_kernel<128>
                                      : smx::q4_attention_kernel<64>;
  SMX_LAUNCH(kernel, grid, dim3(64 * smx::WAVES), 0, (hipStream_t)stream, a);
  const int rc = (int)hipGetLastError();
  if (rc || c.splits == 1) return rc;
  return smx::merge_rows((hipStream_t)stream, head_dim, a.part_o, a.part_lse, a.counts, out,
                         query_start_loc, num_seqs, num_tokens, n_q, c.splits);
}
