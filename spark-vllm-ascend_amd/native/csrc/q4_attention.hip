// Attention of packed query rows (a decode step's, drafts, chunks of prompts) over the
// paged KV cache held in 4 bits (q4_cache.h), for gfx950.
//
// A value is d (c - 8): c the code, d the scale of its block of 32 channels.  Codes are
// multiplied as they are, as the bf16 numbers 16 + c (exact: two instructions a pair,
// with no conversion), and what that adds is taken off again:
//   s_t = sum_b dk[t][b] (sum_{c in b} q_c (16 + code) - 24 sum_{c in b} q_c)
//   o_c = sum_t p'[t][b] (16 + code[t][c]) - 24 sum_t p'[t][b],  p' = bf16(p_t dv[t][b])
// with v_mfma_f32_16x16x32_bf16, whose 32 channels are one block b of K: -24 sum q is its
// initial accumulator, and dk multiplies its result.  V's scale goes into the weights,
// which are rounded to bf16 once, as they are over a bf16 cache; sum p' is a product
// with ones.  So no value of the cache is rounded.  Scores, the running maximum, sums
// and outputs are fp32.
//
// Products are transposed, S^T = K Q^T and O^T = V^T P^T: a row (a token's q head; "row =
// token * group + head in the group") is a column, lane 16 g + n holds row n's scores of
// tokens 16 t + 4 g + i (i < 4) of a tile's sixteens t, and these registers are the
// second product's operand as they stand, V's tokens being read in that order: lane j
// of 16 addresses token 16 (j / 4) + 4 g + j % 4 of a transposing LDS read of half-bytes
// (ds_read_b64_tr_b4: lane n gets channel n of the 16 lanes' tokens).
//
// A workgroup is four waves that take the tiles (64 tokens) of its part of the tokens in
// turn, each with its own softmax and its own buffers in LDS, filled by direct loads:
// nothing is waited for but a wave's own loads, until the four states are joined.
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
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(1))) const void global_void;
typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) u32x2 lds_u32x2;
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
typedef __attribute__((address_space(4))) int32_t constant_i32;

constexpr float LAG = 8.f;        // log2 units
constexpr float NO_REF = -3e38f;  // before the first token: below the scores of any use
constexpr int KT = 64;            // tokens of a tile
constexpr int WAVES = 4;
constexpr int ROUND = KT * WAVES;

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
  int splits, target, least;
  float scale_log2;
};

// Bytes of a wave's buffer: K's codes, V's codes, and their scales.
template <int HD>
struct Tile {
  static constexpr int NB = HD / 32;
  static constexpr int K = KT * HD / 2, V = K, S = KT * NB * 2;
  static constexpr int BYTES = K + V + 1024;
};

// Eight codes (the half-bytes of w) as bf16 numbers 16 + code, pairs of half-bytes j and
// j + 4: bits 3..6 of a bf16 with exponent 4 are whole units.
__device__ __forceinline__ bf16x8 codes_bf16(uint32_t w) {
  constexpr uint32_t M = 0x00780078u, E = 0x41804180u;
  return __builtin_bit_cast(bf16x8, u32x4{((w << 3) & M) | E, ((w >> 1) & M) | E,
                                          ((w >> 5) & M) | E, ((w >> 9) & M) | E});
}

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ float half_of(uint32_t w, int i) {
  return (float)__builtin_bit_cast(f16x2, w)[i];
}

// What one workgroup computes: rows of 16 RT from row0 on, tokens [from, to).
struct Q4Item {
  const int32_t* table;
  int token0, row0, rows, from, to, slot, ahead, parts;
};

template <int HD, int RT>
__device__ __forceinline__ void q4_attend(const Q4Args& A, const Q4Item& it, int kvh,
                                          uint8_t* smem) {
  using T = Tile<HD>;
  constexpr int NB = T::NB, DT = HD / 16, RB = HD / 2;  // blocks, tiles of dims, bytes a row
  constexpr int CHUNKS = RB / 16;                       // 16-byte chunks a row
  constexpr int LOADS = KT * CHUNKS / 64;               // direct loads of a K (V) tile
  constexpr int SPAN = 64 / CHUNKS;                     // tokens of one
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int bs = 1 << A.bs_log2;

  // ---- this lane's rows
  int lim[RT], tok[RT], head[RT];
  bool valid[RT];
  bf16x8 qf[RT][NB];
  f32x4 c0[RT][NB];
  int lim_min = it.to;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int row = it.row0 + 16 * r + n;
    valid[r] = 16 * r + n < it.rows;
    tok[r] = it.token0 + row / A.group;
    head[r] = kvh * A.group + row % A.group;
    lim[r] = it.to;
    if (valid[r]) lim[r] = min(max(it.ahead + row / A.group + 1, 0), it.to);
    lim_min = min(lim_min, lim[r]);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      u32x4 x = {0u, 0u, 0u, 0u};
      if (valid[r])
        x = *reinterpret_cast<const u32x4*>(A.q + (int64_t)tok[r] * A.q_stride + head[r] * HD +
                                            32 * b + 8 * g);
      qf[r][b] = __builtin_bit_cast(bf16x8, x);
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += bf16_lo(x[i]) + bf16_hi(x[i]);
      sum = -24.f * xor_sum<32>(xor_sum<16>(sum));
      c0[r][b] = f32x4{sum, sum, sum, sum};
    }
  }
  lim_min = __builtin_amdgcn_readfirstlane(-wave_max_i32(-lim_min));

  // ---- direct loads of a tile.  LDS is filled in the lanes' order, 16 bytes each; which
  // 16 bytes those are is the lane's choice: chunk c of token t is put in place
  // c ^ swizzle(t) of its row, so that the lanes of one LDS read are on different banks.
  // A table entry outside the cache is read as page 0 (its tokens' scores become NaN),
  // and tokens past the end are the rest of their page.
  const int ntiles = it.to > it.from ? (it.to - it.from + KT - 1) / KT : 0;
  const constant_i32* const table = (const constant_i32*)it.table;
  const int table_end = max(it.to - 1, 0);
  const int64_t plane = (int64_t)A.num_blocks * A.n_kv << A.bs_log2;  // rows of K
  const int ltok = lane / CHUNKS, lchunk = lane % CHUNKS;
  // (K: the 16 lanes of a read are 16 tokens' chunks of one g; V: see v_addr)
  const int k_src = HD == 128 ? 16 * (lchunk ^ ((ltok >> 2) & 3)) : 16 * (lchunk ^ ((ltok >> 3) & 1));
  int page[2];
  auto look_up = [&](int tile) {
    const int base = it.from + tile * KT;
    page[0] = table[min(base, table_end) >> A.bs_log2];
    page[1] = table[min(base + 32, table_end) >> A.bs_log2];
  };
  auto row_of = [&](int u, int t) -> int64_t {  // of token t, in page[u]
    const bool known = (unsigned)page[u] < (unsigned)A.num_blocks;
    return (((int64_t)(known ? page[u] : 0) * A.n_kv + kvh) << A.bs_log2) + (t & (bs - 1));
  };
  auto stage = [&](lds_u8* dst, int tile) {
    const int base = it.from + tile * KT;
    int64_t row[2];
    row[0] = row_of(0, base);
    row[1] = row_of(1, base + 32);
    {
      // the scales of two tokens (four of 64 channels) a lane, K's and then V's
      constexpr int PER = 16 / (2 * NB), HALF = KT / PER;
      const int i = lane % HALF, v = lane / HALF;
      if (v < 2) {
        const int t = i * PER;
        const int64_t at = (t < 32 ? row[0] : row[1]) + (t & 31) + (v ? plane : 0);
        __builtin_amdgcn_global_load_lds((global_void*)(A.scales + at * NB),
                                         (lds_void*)(dst + T::K + T::V), 16, 0, 0);
      }
    }
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int t0 = i * SPAN;  // the load's first token
        const int64_t r0 = row[t0 / 32] + (t0 & 31) + (v ? plane : 0);
        const int v_src = HD == 128 ? 16 * (lchunk ^ (i & 3))
                                    : 16 * (lchunk ^ (ltok >> 4 & 1));
        const uint8_t* const src = A.codes + r0 * RB;
        __builtin_amdgcn_global_load_lds((global_void*)(src + (ltok * RB + (v ? v_src : k_src))),
                                         (lds_void*)(dst + v * T::K + i * 1024), 16, 0, 0);
      }
  };
  constexpr int STAGE_LOADS = 1 + 2 * LOADS;
  auto bad_pages = [&]() {
    return ((unsigned)page[0] >= (unsigned)A.num_blocks ? 1 : 0) |
           ((unsigned)page[1] >= (unsigned)A.num_blocks ? 2 : 0);
  };

  // ---- a row's state: the exponents' reference (log2 units: the running maximum, or up
  // to LAG below it), the sum of 2^(score - ref) over this lane's tokens, the output's
  // products with 16 + code and (register b: block b) the sums of their weights.
  float ref[RT], l[RT];
  f32x4 o[RT][DT], w_sum[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    ref[r] = NO_REF;
    l[r] = 0.f;
    w_sum[r] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < DT; ++d) o[r][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // ones in the rows 4 x + b of the weights' product, so that its register b is block b's
  bf16x8 ones[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const uint32_t x = (lane & 3) == b ? 0x3f803f80u : 0u;
    ones[b] = __builtin_bit_cast(bf16x8, u32x4{x, x, x, x});
  }
  const int k_addr = HD == 128 ? n * RB + 16 * (g ^ (n >> 2))
                               : n * RB + 16 * ((g >> 1) ^ (n >> 3)) + 8 * (g & 1);
  // V: lane n of 16 addresses token 16 (n / 4) + 4 g + n % 4
  const int vt = 16 * (n >> 2) + 4 * g + (n & 3);
  const int v_swz = HD == 128 ? n >> 2 : (vt >> 4) & 1;

  auto compute = [&](auto plain, const lds_u8* buf, int tile, int bad) {
    const int base = it.from + tile * KT;
    const lds_u8* const sk = buf + T::K + T::V;
    const lds_u8* const sv = sk + T::S;
    // scales of tokens 16 t + 4 g + i, block b: fp16 i * NB + b of 8 NB bytes
    auto scales_of = [&](const lds_u8* s, int t, uint32_t (&w)[2 * NB]) {
#pragma unroll
      for (int j = 0; j < NB / 2; ++j) {
        const u32x4 x = *(const lds_u32x4*)(s + (16 * t + 4 * g) * 2 * NB + 16 * j);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[4 * j + i] = x[i];
      }
    };
    float p[RT][4][4];  // scores, then weights: [16 tokens][i]
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      uint32_t dk[2 * NB], kw[NB];
      scales_of(sk, t, dk);
      if constexpr (HD == 128) {
        const u32x4 x = *(const lds_u32x4*)(buf + t * 16 * RB + k_addr);
#pragma unroll
        for (int b = 0; b < 4; ++b) kw[b] = x[b];
      } else {
        // (a load's 32 tokens are swizzled by their own bit 3)
        const u32x2 x = *(const lds_u32x2*)(buf + t * 16 * RB + k_addr);
        kw[0] = x[0];
        kw[1] = x[1];
      }
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) p[r][t][i] = 0.f;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const bf16x8 a = codes_bf16(kw[b]);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const f32x4 s = mfma(a, qf[r][b], c0[r][b]);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            p[r][t][i] = fmaf(half_of(dk[(i * NB + b) / 2], (i * NB + b) & 1), s[i], p[r][t][i]);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      if constexpr (!plain) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = bad >> (t / 2) & 1 ? __builtin_nanf("") : p[r][t][i];
            p[r][t][i] = base + 16 * t + 4 * g + i < lim[r] ? x : -INFINITY;
          }
      }
      float mx = p[r][0][0];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, p[r][t][i]);
      mx = xor_max<32>(xor_max<16>(mx)) * A.scale_log2;
      if (__builtin_amdgcn_ballot_w64(mx > ref[r] + LAG)) {
        const float next = fmaxf(ref[r], mx);
        const float alpha = __builtin_amdgcn_exp2f(ref[r] - next);
        ref[r] = next;
        l[r] *= alpha;
        w_sum[r] *= alpha;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[r][d] *= alpha;
      }
      float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[r][t][i] = __builtin_amdgcn_exp2f(fmaf(p[r][t][i], A.scale_log2, -ref[r]));
          part[i] += p[r][t][i];
        }
      l[r] += (part[0] + part[1]) + (part[2] + part[3]);
    }
    // O^T += V^T P'^T, block by block
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      uint32_t dv0[2 * NB], dv1[2 * NB];  // of sixteens 2 m and 2 m + 1
      scales_of(sv, 2 * m, dv0);
      scales_of(sv, 2 * m + 1, dv1);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        bf16x8 w[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          u32x4 x;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int e = i * NB + b;
            float w0 = p[r][2 * m][i] * half_of(dv0[e / 2], e & 1);
            float w1 = p[r][2 * m + 1][i] * half_of(dv1[e / 2], e & 1);
            if constexpr (!plain) {  // (an unseen token's scale may be anything)
              const int t = base + 32 * m + 4 * g + i;
              w0 = t < lim[r] ? w0 : 0.f;
              w1 = t + 16 < lim[r] ? w1 : 0.f;
            }
            x[i] = cvt_pk_bf16(w0, w1);
          }
          w[r] = __builtin_bit_cast(bf16x8, x);
          w_sum[r] = mfma(ones[b], w[r], w_sum[r]);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int d = 2 * b + c;  // 16 dims: chunk d of 8 bytes of every row
          const i32x2 x = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
              (lds_i32x2*)(buf + T::K + vt * RB + 16 * (b ^ v_swz) + 8 * c));
          const bf16x8 a = codes_bf16((uint32_t)x[m]);
#pragma unroll
          for (int r = 0; r < RT; ++r) o[r][d] = mfma(a, w[r], o[r][d]);
        }
      }
    }
  };

  // ---- this wave's tiles: the next one's loads in flight during the current one
  lds_u8* const lds = (lds_u8*)smem + wave * 2 * T::BYTES;
  if (wave < ntiles) {
    look_up(wave);
    stage(lds, wave);
    int bad = bad_pages(), buf = 0;
    look_up(wave + WAVES);
    auto round = [&](lds_u8* __restrict__ next, const lds_u8* __restrict__ cur, int tile) {
      int bad_next = 0;
      if (tile + WAVES < ntiles) {
        stage(next, tile + WAVES);
        bad_next = bad_pages();
        look_up(tile + 2 * WAVES);
        __builtin_amdgcn_s_waitcnt(0x0f70 | (STAGE_LOADS & 15));  // this tile's have arrived
      } else {
        __builtin_amdgcn_s_waitcnt(0x0f70);
      }
      __asm__ volatile("" ::: "memory");
      if (!bad && it.from + tile * KT + KT <= lim_min)
        compute(std::true_type{}, cur, tile, 0);
      else
        compute(std::false_type{}, cur, tile, bad);
      bad = bad_next;
    };
    for (int tile = wave; tile < ntiles; tile += WAVES) {
      round(lds + (buf ^ 1) * T::BYTES, lds + buf * T::BYTES, tile);
      buf ^= 1;
    }
  }

  // ---- what 16 + code added, then the four waves' states
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    l[r] = xor_sum<32>(xor_sum<16>(l[r]));
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[r][d][i] = fmaf(-24.f, w_sum[r][d / 2], o[r][d][i]);
  }
  constexpr int STATE = RT * (16 * HD + 32);  // floats of a wave's
  if (ntiles > 1) {
    float* const jo = reinterpret_cast<float*>(smem);
    __syncthreads();  // the tiles are read out
    if (wave > 0) {
      float* const dst = jo + (wave - 1) * STATE;
#pragma unroll
      for (int r = 0; r < RT; ++r) {
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) dst[((r * DT + d) * 4 + i) * 64 + lane] = o[r][d][i];
        if (g == 0) {
          dst[RT * 16 * HD + r * 32 + n] = ref[r];
          dst[RT * 16 * HD + r * 32 + 16 + n] = l[r];
        }
      }
    }
    __syncthreads();
  }
  if (wave > 0) return;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    if (ntiles > 1) {
      const float* const jo = reinterpret_cast<const float*>(smem);
#pragma unroll
      for (int w = 1; w < WAVES; ++w) {
        const float* const src = jo + (w - 1) * STATE;
        const float ro = src[RT * 16 * HD + r * 32 + n], lo = src[RT * 16 * HD + r * 32 + 16 + n];
        const float next = fmaxf(ref[r], ro);
        const float a = __builtin_amdgcn_exp2f(ref[r] - next);
        const float b = __builtin_amdgcn_exp2f(ro - next);
        ref[r] = next;
        l[r] = l[r] * a + lo * b;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            o[r][d][i] = o[r][d][i] * a + src[((r * DT + d) * 4 + i) * 64 + lane] * b;
      }
    }
    if (!valid[r]) continue;
    const int64_t orow = (int64_t)tok[r] * A.n_q + head[r];
    // l == 0 only where the row sees no token: its output is 0, its weight none
    const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];
    if (it.slot == 0 && A.splits > 1 && g == 0)
      st_agent(A.counts + orow, it.parts == 1 ? 0 : it.parts);
    if (it.parts == 1) {
      uint16_t* const dst = A.out + orow * HD;
#pragma unroll
      for (int d = 0; d < DT; ++d)
        st_agent(reinterpret_cast<u32x2*>(dst + 16 * d + 4 * g),
                 u32x2{cvt_pk_bf16(o[r][d][0] * inv, o[r][d][1] * inv),
                       cvt_pk_bf16(o[r][d][2] * inv, o[r][d][3] * inv)});
    } else {
      const int64_t prow = orow * A.splits + it.slot;
      if (g == 0) st_agent(A.part_lse + prow, l[r] == 0.f ? -INFINITY : ref[r] + log2f(l[r]));
      if (l[r] != 0.f) {  // the merge reads no partial whose weight is none
        float* const dst = A.part_o + prow * HD;
#pragma unroll
        for (int d = 0; d < DT; ++d)
          st_agent_b128(dst + 16 * d + 4 * g,
                        u32x4{__float_as_uint(o[r][d][0] * inv), __float_as_uint(o[r][d][1] * inv),
                              __float_as_uint(o[r][d][2] * inv),
                              __float_as_uint(o[r][d][3] * inv)});
      }
    }
  }
}

// Sequence r's queries are the tokens [query_start[r], query_start[r + 1]), the last n of
// its L tokens.  Grid: kv heads, items.
template <int HD, int RT>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(2)))
void q4_attention_kernel(Q4Args A) {
  constexpr int M = 16 * RT;
  constexpr int BUF = WAVES * 2 * Tile<HD>::BYTES, JOIN = (WAVES - 1) * RT * (16 * HD + 32) * 4;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[BUF > JOIN ? BUF : JOIN];
  const int kvh = blockIdx.x;
  const int cap = A.max_blocks << A.bs_log2;
  auto queries = [&](int r, int& s0) {
    if (!A.query_start) {
      s0 = r;
      return 1;
    }
    s0 = min(max(A.query_start[r], 0), A.num_tokens);
    return max(min(A.query_start[r + 1], A.num_tokens) - s0, 0);
  };
  auto length = [&](int r) { return min(max(A.seq_lens[r], 0), cap); };
  int my_q0 = 0, my_nq = 0, my_len = 0;  // of sequence `lane` where there are up to 64
  auto seg_of = [&](int r, int& tiles, int& rounds) {
    my_nq = queries(r, my_q0);
    my_len = length(r);
    tiles = (int)(((int64_t)my_nq * A.group + M - 1) / M);
    rounds = tiles ? (int)(((int64_t)my_len + ROUND - 1) / ROUND) : 0;
  };
  Place place;
  if (!find_item<ROUND>(seg_of, A.num_seqs, blockIdx.y, A.target, A.splits, A.least, -INFINITY,
                        false, place))
    return;
  const int seq = place.seg;
  int q0, nq, L;
  if (A.num_seqs <= 64) {  // (a second look in memory is a round trip)
    q0 = __builtin_amdgcn_readlane(my_q0, seq);
    nq = __builtin_amdgcn_readlane(my_nq, seq);
    L = __builtin_amdgcn_readlane(my_len, seq);
  } else {
    nq = queries(seq, q0);
    L = length(seq);
  }
  const int tiles = (int)(((int64_t)nq * A.group + M - 1) / M);
  const int split = place.x / tiles;
  Q4Item it;
  it.table = A.table + (int64_t)seq * A.max_blocks;
  it.token0 = q0;
  it.row0 = (place.x - split * tiles) * M;
  it.rows = min(M, nq * A.group - it.row0);
  it.ahead = L - nq;  // the position of the first query token
  const int range = max(it.ahead + (it.row0 + it.rows - 1) / A.group + 1, 0);
  it.from = part_end(0, split * place.chunk, range);
  it.to = part_end(it.from, place.chunk, range);
  it.slot = split;
  it.parts = place.parts;
  q4_attend<HD, RT>(A, it, kvh, smem);
  stores_done();
}

// How a call is cut, from its sizes (lengths are on the device).
constexpr int FILL = 512, MAX_PARTS = 64;

struct Q4Choice {
  int rt, splits, tiles, target;
};

// Whether a call's rows are prompts': more than a tile of a sequence on average.
bool is_prompt(int64_t num_tokens, int64_t num_seqs, int group) {
  const char* e = tuning_env("SMX_Q4_ROWS");
  return num_tokens * group > (e ? atoi(e) : 32) * num_seqs;
}

Q4Choice choose_q4(int64_t num_tokens, int64_t num_seqs, int64_t cap, int group, int n_kv) {
  Q4Choice c{};
  const int64_t rows = (num_tokens * group + num_seqs - 1) / num_seqs;  // of a sequence
  c.rt = rows > 16 ? 2 : 1;
  const int m = 16 * c.rt;
  c.tiles = (int)((num_tokens * group + m - 1) / m + num_seqs - 1);
  c.target = std::max(1, FILL / n_kv);
  const int64_t groups = (rows + m - 1) / m * num_seqs * n_kv;
  const int64_t even = (FILL + groups - 1) / groups;
  c.splits = (int)std::clamp<int64_t>(num_seqs == 1 ? even : 4 * even, 1,
                                      std::min<int64_t>(MAX_PARTS, std::max<int64_t>(1, cap / ROUND)));
  if (groups >= 2 * FILL) c.splits = 1;
  return c;
}

int64_t q4_items(const Q4Choice& c) {
  return std::min<int64_t>((int64_t)c.tiles * c.splits, (int64_t)c.target + c.tiles + 1);
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
  if (smx::is_prompt(num_tokens, num_seqs, n_q / n_kv)) {
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
                                         n_q / n_kv, n_kv);
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
  if (smx::is_prompt(num_tokens, num_seqs, n_q / n_kv)) {
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
                                         n_q / n_kv, n_kv);
  SMX_REQUIRE(smx::q4_items(c) <= 65535, "too many row tiles for one launch");
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
  a.least = 1;
  a.scale_log2 = scale_log2;
  const dim3 grid(n_kv, (unsigned)smx::q4_items(c));
  const auto kernel = head_dim == 128
      ? (c.rt == 1 ? smx::q4_attention_kernel<128, 1> : smx::q4_attention_kernel<128, 2>)
      : (c.rt == 1 ? smx::q4_attention_kernel<64, 1> : smx::q4_attention_kernel<64, 2>);
  SMX_LAUNCH(kernel, grid, dim3(64 * smx::WAVES), 0, (hipStream_t)stream, a);
  const int rc = (int)hipGetLastError();
  if (rc || c.splits == 1) return rc;
  return smx::merge_rows((hipStream_t)stream, head_dim, a.part_o, a.part_lse, a.counts, out,
                         query_start_loc, num_seqs, num_tokens, n_q, c.splits);
}
