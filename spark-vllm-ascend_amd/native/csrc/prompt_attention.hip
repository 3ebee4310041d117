// Attention of several query rows per sequence over the paged bf16 KV cache,
// for gfx950: packed causal prompts (whole prompts, chunks behind a context,
// drafted tokens) and decode batches whose sequences share a prefix.
//
// A query row is one (token, q head); the rows of one kv head read the same K
// and V, so a workgroup takes 32 WM of them ("row = token * group + head in
// the group") against one range of tokens.  With p = softmax of the scores a
// row sees (token t is seen iff from <= t < the row's limit),
//   S^T = K Q^T     v_mfma_f32_32x32x16_bf16, A = 32 tokens of K, B = 32 rows
//   O^T = V^T P^T   the same instruction, A = 32 dims of V, B = P of 16 tokens
// one online softmax a row: running maximum m and sum l in fp32, P rounded to
// bf16 for the second product (the sum keeps the unrounded values, as split-KV
// decode does).  Transposed products keep a row's scores in one lane pair: lane
// 32 h + n holds row n's scores of tokens 8 a + 4 h + b (a, b < 4) of every 32,
// so the maximum and the sum are in-lane but for one lane swap, and the B
// operand of the second product is those registers as they stand, with V's
// token order permuted to match: its A operand is two transposing LDS reads
// (ds_read_b64_tr_b16) of 4 tokens each.
#include <limits.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "smx_common.h"
#include "smx_launch.h"

namespace smx {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(1))) const void global_void;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) uint16_t lds_u16;
typedef __attribute__((address_space(4))) int32_t constant_i32;

// (lo, hi) as one v_cvt_pk_bf16_f32
__device__ __forceinline__ uint32_t cvt_pk_bf16(float lo, float hi) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), bf16x2));
}

// A dword of two bf16 values with those that are infinite or NaN replaced by 0.
__device__ __forceinline__ uint32_t finite_bf16x2(uint32_t w) {
  if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
  if ((w & 0x7f800000u) == 0x7f800000u) w &= 0x0000ffffu;
  return w;
}

constexpr float LAG = 8.f;        // log2 units
constexpr float NO_REF = -3e38f;  // before the first token: below the scores of any use

struct RowsArgs {
  const uint16_t* q;
  const uint16_t* kc;
  const uint16_t* vc;
  const int32_t* table;         // [num_seqs, max_blocks]
  const int32_t* query_start;   // [num_seqs + 1] (prompts)
  const int32_t* prefix_table;  // [prefix_blocks] (shared prefix)
  const int32_t* prefix_len;    // [1]
  const int32_t* seq_lens;      // [num_seqs]
  uint16_t* out;
  float* part_o;    // [rows, slots, HD], where slots > 1
  float* part_lse;  // [rows, slots], log2 units
  int32_t* counts;  // [rows] slots in use, of the prefix's and then [rows] of the suffix's
  int64_t q_stride;  // elements from a token's q to the next token's
  int num_tokens, num_seqs, max_blocks, prefix_blocks, num_blocks, bs_log2, n_q, n_kv, group;
  int splits;         // most parts of a tile's tokens (prompts), of the prefix (shared prefix)
  int suffix_splits;  // most parts of a sequence's own tokens (shared prefix)
  int tiles;          // row tiles: the most there can be (prompts), of the prefix's rows
  int target;         // workgroups a kv head to aim at
  int least;          // rounds of a part at least (prompts)
  int zigzag;         // period of the order of the tiles (prompts)
  float gain;         // of find_item (prompts)
  float scale_log2;
};

// What one workgroup computes: `rows` rows from row0 on (row -> token row / group
// from token0 on, head kvh * group + row % group) over the tokens [from, to) of
// the pages in `table`.  query_at: the position of token token0, or NO_QUERY
// where every row is a sequence's one decode token.
constexpr int NO_QUERY = INT_MIN;
struct Item {
  const int32_t* table;
  int token0, row0, rows, from, to, slot, slots, query_at;
  int32_t* counts;  // where the first part's workgroup writes `parts` for its rows, or null
  int parts;
  bool direct;  // the only part of its rows: the output itself, no partial
};

// HD: head_dim.  WM waves take 32 rows each, WN groups of them take every WN-th
// tile of KT tokens; ST tiles of K and V a group are in LDS, one that is read and
// ST - 1 that are on their way.
template <int HD, int WM, int WN, int KT, int ST>
struct Shape {
  static constexpr int M = 32 * WM, NT = 64 * WM * WN;
  static constexpr int CH = HD / 8;                  // 16-byte chunks of a row
  static constexpr int TILE = KT * CH;               // chunks of a K or V tile
  static constexpr int GROUP = ST * 2 * TILE;        // the buffers of K and V
  static constexpr int JOIN = WN > 1 ? (WN - 1) * WM * (32 * HD + 64) / 4 : 0;
  static constexpr int LDS = WN * GROUP > JOIN ? WN * GROUP : JOIN;
  static constexpr int LOADS = TILE / 64 / WM;       // a wave's loads of a K (V) tile
  static_assert(TILE % (64 * WM) == 0, "whole loads per wave");
};

// Chunk c of row r sits in slot c ^ k_swz(r) (K) or c ^ v_swz(r) (V) of its row, so
// that the lanes of one LDS read are spread over all banks: K is read 16 bytes
// a lane from 32 rows, V 8 bytes a lane, 64 bytes from each of 8 rows.
template <int HD>
__device__ __forceinline__ int k_swz(int r) {
  return HD == 128 ? (r & 15) : ((r >> 1) & 7);
}
template <int HD>
__device__ __forceinline__ int v_swz(int r) {
  return HD == 128 ? 4 * (r & 3) : 4 * ((r >> 1) & 1);
}

// s_waitcnt operand: at most `vm` vector loads outstanding, no LDS operation
constexpr int wait_vm(int vm) { return (vm & 15) | ((vm >> 4) << 14) | (7 << 4); }

// Every wave of the workgroup is here.  (__syncthreads would also wait for all
// vector loads.)
__device__ __forceinline__ void meet() {
  __asm__ volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  __asm__ volatile("" ::: "memory");
}

// The largest of a wave's values, for every lane.
__device__ __forceinline__ int wave_max_i32(int v) {
  auto dpp = [](int x, auto ctrl) {
    return __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, 0xf, 0xf, false);
  };
  v = max(v, dpp(v, std::integral_constant<int, DPP_QUAD_XOR1>{}));
  v = max(v, dpp(v, std::integral_constant<int, DPP_QUAD_XOR2>{}));
  v = max(v, dpp(v, std::integral_constant<int, DPP_ROW_HALF_MIRROR>{}));
  v = max(v, dpp(v, std::integral_constant<int, DPP_ROW_MIRROR>{}));
  const auto a = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
  v = max((int)a[0], (int)a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
  return max((int)b[0], (int)b[1]);
}

// BS: the least block_size, 32 or 64: a tile is looked up and addressed by NP pieces
// of BT tokens that are within a page.
template <int HD, int WM, int WN, int KT, int ST, int BS>
__device__ __forceinline__ void attend(const RowsArgs& A, const Item& it, int kvh, u32x4* smem) {
  using S = Shape<HD, WM, WN, KT, ST>;
  constexpr int KS = HD / 16, DT = HD / 32, NU = KT / 32, CH = S::CH;
  constexpr int BT = KT < BS ? KT : BS, NP = KT / BT;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % WM, wn = wave / WM;
  const int bs = 1 << A.bs_log2;
  const int tok_stride = A.n_kv * HD;
  const int64_t page_stride = (int64_t)tok_stride << A.bs_log2;

  // ---- this lane's row
  const int row = it.row0 + 32 * wm + n;
  const bool valid = 32 * wm + n < it.rows;
  const int tok = it.token0 + row / A.group, head = kvh * A.group + row % A.group;
  // The row sees the tokens below lim: of a prompt up to its own position, of a
  // decode row all of its sequence.  (A row past the tile's end is not stored: it
  // sees everything, so that no tile is masked for it.)
  int lim = it.to;
  if (valid) {
    const int len = it.query_at == NO_QUERY ? A.seq_lens[tok] : it.query_at + row / A.group + 1;
    lim = min(max(len, 0), it.to);
  }
  u32x4 qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    qf[ks] = u32x4{0u, 0u, 0u, 0u};
    if (valid)
      qf[ks] = *reinterpret_cast<const u32x4*>(A.q + (int64_t)tok * A.q_stride + head * HD +
                                               16 * ks + 8 * h);
  }
  const int lim_min = __builtin_amdgcn_readfirstlane(-wave_max_i32(-lim));

  // ---- staging: wave wm of a group loads every WM-th kilobyte of its tile, by
  // buffer loads into LDS whose resource is one piece of BT tokens: tokens past the
  // end, and those of a table entry outside the cache, are past the resource's end
  // and read as 0 without an access.  Pages are looked up a round before they are
  // used, by scalar loads (the table is constant while the kernel runs), which do
  // not queue behind the tiles' loads.  (Whole tiles of 64 by one resource where
  // pages allow it: a third less scalar arithmetic, 8192-token prompt 541 us, 531.)
  const int first = it.from & ~(KT - 1);
  const int ntiles = it.to > it.from ? (it.to - first + KT - 1) / KT : 0;
  const int rounds = (ntiles + WN - 1) / WN;
  lds_u32x4* const lds = (lds_u32x4*)smem + wn * S::GROUP;
  const int lrow = lane / CH, lc = lane % CH;  // the lane's row and chunk of a load
  const int tok_bytes = 2 * tok_stride;
  const constant_i32* const table = (const constant_i32*)it.table;
  // (an empty range may lie past the table's end, with a prefix longer than it)
  const int table_end = it.to > it.from ? it.to - 1 : 0;
  auto look_up = [&](int (&page)[NP], int base) {
#pragma unroll
    for (int u = 0; u < NP; ++u)
      page[u] = table[min(base + BT * u, table_end) >> A.bs_log2];
  };
  auto stage = [&](const uint16_t* cache, lds_u32x4* dst, const int (&page)[NP], int base,
                   auto swz) {
    __amdgpu_buffer_rsrc_t piece[NP];
#pragma unroll
    for (int u = 0; u < NP; ++u) {
      const int t = base + BT * u;
      const bool known = (unsigned)page[u] < (unsigned)A.num_blocks;
      const int rows = known ? min(it.to - t, BT) : 0;
      const uint16_t* const at = cache + (int64_t)(known ? page[u] : 0) * page_stride +
                                 (t & (bs - 1)) * tok_stride + kvh * HD;
      piece[u] = __builtin_amdgcn_make_buffer_rsrc(
          (void*)at, 0, rows > 0 ? (rows - 1) * tok_bytes + 2 * HD : 0, 0x00027000);
    }
#pragma unroll
    for (int i = 0; i < S::LOADS; ++i) {
      const int c0 = (i * WM + wm) * 64;  // first chunk of this load
      const int r0 = c0 / CH;             // its row
      const int off = lrow * tok_bytes + 16 * (lc ^ swz(r0 + lrow));
      const __amdgpu_buffer_rsrc_t src =
          NP > 1 && (i * WM * 64 / CH >= BT || r0 >= BT) ? piece[NP - 1] : piece[0];
      __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (lds_void*)(dst + c0), 16, off,
                                               (r0 & (BT - 1)) * tok_bytes, 0, 0);
    }
  };
  auto stage_k = [&](lds_u32x4* dst, const int (&page)[NP], int base) {
    stage(A.kc, dst, page, base, [](int r) { return k_swz<HD>(r); });
  };
  auto stage_v = [&](lds_u32x4* dst, const int (&page)[NP], int base) {
    stage(A.vc, dst, page, base, [](int r) { return v_swz<HD>(r); });
  };
  auto bad_pages = [&](const int (&page)[NP]) {
    int bad = 0;
#pragma unroll
    for (int u = 0; u < NP; ++u) bad |= (unsigned)page[u] >= (unsigned)A.num_blocks ? 1 << u : 0;
    return bad;
  };

  // The exponents' reference of the row, log2 units: the running maximum, or up to
  // LAG below it (NO_REF before the first token), and the running sum of
  // 2^(score - ref) over this lane's tokens.
  float ref = NO_REF, l = 0.f;
  f32x16 o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
  f32x16 s[NU];       // scores: s[u][4 a + b] is token 32 u + 8 a + 4 h + b of row n
  uint32_t p[NU][8];  // and their 2^(score - ref), bf16 pairs

  auto scores = [&](const lds_u32x4* kt) {
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[u][i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        const u32x4 a = kt[(32 * u + n) * CH + ((2 * ks + h) ^ k_swz<HD>(n))];
        s[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, qf[ks]), s[u],
                                                       0, 0, 0);
      }
  };
  // A plain tile: every row of the wave sees all of it, and its pages are known.  The
  // others have code of their own, so that the accumulators are not moved at every
  // tile where the paths join.
  auto is_plain = [&](int base, int bad) {
    return base >= it.from && base + KT <= lim_min && !bad;
  };
  auto softmax = [&](auto plain, int base, int bad) {
    // the scores of tokens without a page are NaN, and so is every row that sees one
    if constexpr (!plain) {
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int t = base + 32 * u + 8 * (i / 4) + 4 * h + i % 4;
          const float x = bad >> (NP == NU ? u : 0) & 1 ? __builtin_nanf("") : s[u][i];
          s[u][i] = t >= it.from && t < lim ? x : -INFINITY;
        }
    }
    float mx = s[0][0];
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[u][i]);
    mx = xor_max<32>(mx) * A.scale_log2;
    // The reference follows the maximum only once that has grown by LAG: p is then
    // at most 2^LAG, which neither fp32 nor bf16 minds, and most tiles leave o and
    // l as they are.
    if (__builtin_amdgcn_ballot_w64(mx > ref + LAG)) {
      const float next = fmaxf(ref, mx);
      const float alpha = __builtin_amdgcn_exp2f(ref - next);
      ref = next;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= alpha;
    }
    float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[u][2 * i], A.scale_log2, -ref));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(s[u][2 * i + 1], A.scale_log2, -ref));
        part[2 * (i & 1)] += p0;
        part[2 * (i & 1) + 1] += p1;
        p[u][i] = cvt_pk_bf16(p0, p1);
      }
    l += (part[0] + part[1]) + (part[2] + part[3]);
  };
  // O^T += V^T P^T
  const int vr = 4 * h + ((lane & 15) >> 2), vcol = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  auto v_operand = [&](const lds_u16* vt, int kk, int d) -> u32x4 {  // 16 tokens, dims 32 d + n
    u32x2 half[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = 16 * kk + 8 * j + vr;
      const lds_u16* src = vt + (r * CH + ((4 * d + vcol) ^ v_swz<HD>(r))) * 8 + 4 * (lane & 1);
      half[j] = __builtin_bit_cast(u32x2,
                                   __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)src));
    }
    return u32x4{half[0].x, half[0].y, half[1].x, half[1].y};
  };
  auto p_operand = [&](int kk) -> u32x4 {
    return u32x4{p[kk / 2][4 * (kk & 1)], p[kk / 2][4 * (kk & 1) + 1],
                 p[kk / 2][4 * (kk & 1) + 2], p[kk / 2][4 * (kk & 1) + 3]};
  };
  // A masked token must not reach a row by 0 * infinity or 0 * NaN: where a tile
  // that some row sees in part holds such values (0 * V tells), they are left out
  // of the product and added to the rows that see them.
  auto odd_values = [&](const lds_u16* vt) {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.f;
    const u32x4 none = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int kk = 0; kk < 2 * NU; ++kk)
#pragma unroll
      for (int d = 0; d < DT; ++d)
        z = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            __builtin_bit_cast(bf16x8, v_operand(vt, kk, d)), __builtin_bit_cast(bf16x8, none), z,
            0, 0, 0);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) sum += z[i];
    return __builtin_amdgcn_ballot_w64(sum != sum) != 0;
  };
  auto weigh = [&](auto plain, const lds_u32x4* vtile, int base) {
    const lds_u16* const vt = (const lds_u16*)vtile;
    bool odd = false;
    if constexpr (!plain) odd = odd_values(vt);
    if (!odd) {
#pragma unroll
      for (int kk = 0; kk < 2 * NU; ++kk)
#pragma unroll
        for (int d = 0; d < DT; ++d)
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              __builtin_bit_cast(bf16x8, v_operand(vt, kk, d)),
              __builtin_bit_cast(bf16x8, p_operand(kk)), o[d], 0, 0, 0);
    } else {
#pragma unroll
      for (int kk = 0; kk < 2 * NU; ++kk)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          u32x4 a = v_operand(vt, kk, d);
          a = u32x4{finite_bf16x2(a.x), finite_bf16x2(a.y), finite_bf16x2(a.z),
                    finite_bf16x2(a.w)};
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                         __builtin_bit_cast(bf16x8, p_operand(kk)),
                                                         o[d], 0, 0, 0);
        }
      for (int r = 0; r < KT; ++r) {
        const bool seen = base + r >= it.from && base + r < lim;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int dim = 32 * d + 8 * (i / 4) + 4 * h + i % 4;
            const uint32_t v = vt[(r * CH + ((dim / 8) ^ v_swz<HD>(r))) * 8 + dim % 8];
            if (seen && (v & 0x7f80u) == 0x7f80u) o[d][i] += bf16_bits_to_f32(v);
          }
      }
    }
  };

  // One round after another: the loads of the tile ST - 1 rounds ahead into `next`,
  // whose last readers are past the barrier, then the tile in `cur`.  Both are
  // restrict so that the compiler does not wait for the loads into the one before
  // it reads the other; the wait that counts is the one before the barrier.
  int bad[ST];  // of the tiles in LDS, that of this round first
  int page[NP];
#pragma unroll
  for (int i = 0; i < ST; ++i) bad[i] = 0;
  look_up(page, first + wn * KT);
#pragma unroll
  for (int i = 0; i < ST - 1; ++i) {
    const int tile = i * WN + wn, base = first + tile * KT;
    if (tile < ntiles) {
      lds_u32x4* const dst = lds + i * 2 * S::TILE;
      stage_k(dst, page, base);
      stage_v(dst + S::TILE, page, base);
      bad[i] = bad_pages(page);
      look_up(page, base + WN * KT);
    }
  }
  auto round = [&](auto plain, lds_u32x4* __restrict__ next, const lds_u32x4* __restrict__ cur,
                   int tile) {
    const int base = first + tile * KT, ahead = base + (ST - 1) * WN * KT;
    // (a tile past the end is of no rows: a plain round loads nothing there, without
    // the branch that would keep the addresses' arithmetic from the products' shadow)
    if (plain || tile + (ST - 1) * WN < ntiles) {
      stage_k(next, page, ahead);
      stage_v(next + S::TILE, page, ahead);
      bad[ST - 1] = bad_pages(page);
      look_up(page, ahead + WN * KT);
    }
    if ((!plain && tile >= ntiles) || 32 * wm >= it.rows) return;
    scores(cur);
    softmax(plain, base, bad[0]);
    weigh(plain, cur + S::TILE, base);
  };
  int at = 0, rd = 0;  // the buffer of this round's tile
  auto step = [&](auto plain) {
    // this wave's loads of the tile have arrived (those of later ones may be on
    // their way), then every wave's have, and the last round's tile is read out
    if (ST > 2 && (rd + ST - 2) * WN + wn < ntiles)
      __builtin_amdgcn_s_waitcnt(wait_vm((ST - 2) * 2 * S::LOADS));
    else
      __builtin_amdgcn_s_waitcnt(wait_vm(0));
    meet();
    const int before = at == 0 ? ST - 1 : at - 1;
    round(plain, lds + before * 2 * S::TILE, lds + at * 2 * S::TILE, rd * WN + wn);
    at = at == ST - 1 ? 0 : at + 1;
#pragma unroll
    for (int i = 0; i < ST - 1; ++i) bad[i] = bad[i + 1];
    ++rd;
  };
  while (rd < rounds) {
    while (rd * WN + wn < ntiles && is_plain(first + (rd * WN + wn) * KT, bad[0]))
      step(std::true_type{});
    if (rd < rounds) step(std::false_type{});
  }

  // ---- the lane pair's sums, then the WN groups' states (of one tile the first's only)
  l = xor_sum<32>(l);
  if (WN > 1 && ntiles > 1) {
    float* const jo = reinterpret_cast<float*>(smem);
    __builtin_amdgcn_s_waitcnt(wait_vm(0));
    __syncthreads();  // the tiles are read out, nothing is on its way into them
    if (wn > 0) {
      float* const dst = jo + ((wn - 1) * WM + wm) * (32 * HD + 64);
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) dst[(16 * d + i) * 64 + lane] = o[d][i];
      if (h == 0) {
        dst[32 * HD + n] = ref;
        dst[32 * HD + 32 + n] = l;
      }
    }
    __syncthreads();
    if (wn > 0) return;
#pragma unroll
    for (int w = 1; w < WN; ++w) {
      const float* const src = jo + ((w - 1) * WM + wm) * (32 * HD + 64);
      const float ro = src[32 * HD + n], lo = src[32 * HD + 32 + n];
      const float next = fmaxf(ref, ro);
      const float a = __builtin_amdgcn_exp2f(ref - next), b = __builtin_amdgcn_exp2f(ro - next);
      ref = next;
      l = l * a + lo * b;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = o[d][i] * a + src[(16 * d + i) * 64 + lane] * b;
    }
  }
  if (WN > 1 && wn > 0) return;  // (a single tile: the first group's)
  // The row again, from its number: not kept in registers through the rounds.
  int row_again = row;
  __asm__ volatile("" : "+v"(row_again));
  const int64_t orow = (int64_t)(it.token0 + row_again / A.group) * A.n_q + kvh * A.group +
                       row_again % A.group;
  // l == 0 only where the row sees no token: its output is 0, its weight none
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (valid && it.direct) {
    if (h == 0 && it.counts) st_agent(it.counts + orow, 0);  // nothing to merge
    uint16_t* const dst = A.out + orow * HD;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int a = 0; a < 4; ++a)
        st_agent(reinterpret_cast<u32x2*>(dst + 32 * d + 8 * a + 4 * h),
                 u32x2{cvt_pk_bf16(o[d][4 * a] * inv, o[d][4 * a + 1] * inv),
                       cvt_pk_bf16(o[d][4 * a + 2] * inv, o[d][4 * a + 3] * inv)});
  } else if (valid) {
    const int64_t prow = orow * it.slots + it.slot;
    if (h == 0 && it.counts) st_agent(it.counts + orow, it.parts);
    if (h == 0)
      st_agent(A.part_lse + prow, l == 0.f ? -INFINITY : ref + log2f(l));
    if (l != 0.f) {  // the merge reads no partial whose weight is none
      float* const dst = A.part_o + prow * HD;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int a = 0; a < 4; ++a)
          st_agent_b128(dst + 32 * d + 8 * a + 4 * h,
                        u32x4{__float_as_uint(o[d][4 * a] * inv),
                              __float_as_uint(o[d][4 * a + 1] * inv),
                              __float_as_uint(o[d][4 * a + 2] * inv),
                              __float_as_uint(o[d][4 * a + 3] * inv)});
    }
  }
}

// The end of a part that begins at `from`, at most `end`.
__device__ __forceinline__ int part_end(int from, int chunk, int end) {
  return (int)min((int64_t)from + chunk, (int64_t)end);
}

// Where a workgroup stands in a launch's work: segment seg (a sequence, or the
// prefix), item x of its tiles times parts, the segment's parts of `chunk` tokens.
struct Place {
  int seg, x, parts, chunk;
};

// Finds item `item` of segments whose row tiles and rounds (of ROUND tokens) seg_of
// gives, 64 at a time, a lane each.  With max_parts > 1 every segment's tokens
// are cut into parts of one length, the least (of at least `least` rounds) that
// makes about `target` items of all segments and at most max_parts of any, so
// that the workgroups are alike whatever the lengths: every workgroup derives
// it from the lengths.  Nothing is cut where that would not save `gain` rounds of
// the longest item (a round beside another workgroup's takes 1.45 of one alone), or
// where the items read memory at its rate as they are (`memory`: few rows a
// sequence): from 160 of 512 workgroups on, none 1.3 times as long as the average.  us
// whole / cut of sequences of 5 tokens behind 5000, a fourth of them r times the
// average: 16 (128 workgroups) r = 1 97 / 63; 20 (160) 110 / 91, behind 2500
// 38 / 41; 29 (232) 122 / 130, r = 1.15 133 / 130, 1.3 146 / 140, 1.5 160 / 131.
template <int ROUND, typename Seg>
__device__ __forceinline__ bool find_item(Seg seg_of, int num_segs, int item, int target,
                                          int max_parts, int least, float gain, bool memory,
                                          Place& place) {
  const int lane = threadIdx.x & 63;
  int chunk = INT_MAX / ROUND;  // in rounds
  int tiles0 = 0, rounds0 = 0;
  if (lane < num_segs) seg_of(lane, tiles0, rounds0);
  if (max_parts > 1) {
    float work = wave_sum((float)tiles0 * (float)rounds0), all = wave_sum((float)tiles0);
    int top = wave_max_i32(rounds0);
    for (int b = 64; b < num_segs; b += 64) {
      int tiles = 0, rounds = 0;
      if (b + lane < num_segs) seg_of(b + lane, tiles, rounds);
      work += wave_sum((float)tiles * (float)rounds);
      all += wave_sum((float)tiles);
      top = max(top, wave_max_i32(rounds));
    }
    chunk = max(max((int)fminf(ceilf(work / (float)target), 1e9f),
                    (top + max_parts - 1) / max_parts), least);
    const float alone = all / (float)target;
    if ((float)top * (1.f - 1.45f * alone) < gain ||
        (memory && alone > 0.31f && (float)top * all < 1.3f * work))
      chunk = max(chunk, top);
    // every segment rounds up: a little longer parts where that made too many
    for (int i = 0; i < 3 && num_segs <= 64; ++i) {
      const float items = wave_sum((float)tiles0 * (float)max(1, (rounds0 + chunk - 1) / chunk));
      if (items <= (float)target || chunk >= top) break;
      chunk = max(chunk + 1, min((int)fminf((float)chunk * items / (float)target, 1e9f), top));
    }
    chunk = __builtin_amdgcn_readfirstlane(chunk);
  }
  int done = 0;
  for (int b = 0; b < num_segs; b += 64) {
    int tiles = tiles0, rounds = rounds0;
    if (b > 0) {
      tiles = rounds = 0;
      if (b + lane < num_segs) seg_of(b + lane, tiles, rounds);
    }
    const int parts = max(1, (rounds + chunk - 1) / chunk);
    const int items = tiles * parts;
    const int incl = wave_scan_i32(items);
    const int total = __builtin_amdgcn_readlane(incl, 63);
    if (item < done + total) {
      const int i = __ffsll((unsigned long long)__ballot(done + incl > item)) - 1;
      place.seg = b + i;
      place.x = item - done - (__builtin_amdgcn_readlane(incl, i) -
                               __builtin_amdgcn_readlane(items, i));
      place.parts = __builtin_amdgcn_readlane(parts, i);
      place.chunk = chunk * ROUND;
      return true;
    }
    done += total;
  }
  return false;
}

// Shapes.  Rounds of 64 tokens: a workgroup of 64 rows takes 0.85 us alone on its
// compute unit and 1.2 beside another (heads of 64: 0.6 alone), one of 128 rows 1.3
// and 2.07, so 128 rows multiply 1.16 times as fast where the chip is full.  64 KB of
// LDS and at most 256 registers let two be resident.  Two waves a SIMD from two
// workgroups overlap matrix and vector work by themselves; 8 waves a workgroup (256
// rows, or four token groups) were slower on full chips.
//
// Packed prompts.  Bound by matrix and vector work in turn where there are many rows:
// one prompt of 8192 tokens, 32 / 8 heads of 128, 515 to 545 us = 1070 to 1010 TFLOP/s,
// a large library product 1406; of 1.05 million cycles at 1.94 GHz the matrix units
// are busy for 0.53, other vector instructions issue for 0.42.  By the longest
// workgroups where all are resident (2048 tokens 50 us); by memory for a few drafted
// tokens (8 x 5 behind 300 to 8000: 20 us, 4.9 TB/s).  Sequence r's queries are the tokens [query_start[r],
// query_start[r + 1]), the last n of its L tokens: token i of them is at position
// L - n + i and sees the tokens up to itself.  Grid: kv heads, items.
template <int HD, int WM, int WN, int KT, int ST, int BS>
__global__ __launch_bounds__(64 * WM * WN) __attribute__((amdgpu_waves_per_eu(2)))
void prompt_attention_kernel(RowsArgs A) {
  using S = Shape<HD, WM, WN, KT, ST>;
  __shared__ __attribute__((aligned(16))) u32x4 smem[S::LDS];
  constexpr int ROUND = WN * KT;
  const int kvh = blockIdx.x;
  const int cap = A.max_blocks << A.bs_log2;
  auto queries = [&](int r, int& s0) {
    s0 = min(max(A.query_start[r], 0), A.num_tokens);
    return max(min(A.query_start[r + 1], A.num_tokens) - s0, 0);
  };
  auto length = [&](int r) { return min(max(A.seq_lens[r], 0), cap); };
  int my_q0 = 0, my_nq = 0, my_len = 0;  // of sequence `lane` where there are up to 64
  auto seg_of = [&](int r, int& tiles, int& rounds) {
    my_nq = queries(r, my_q0);
    my_len = length(r);
    tiles = (int)(((int64_t)my_nq * A.group + S::M - 1) / S::M);
    rounds = tiles ? (int)(((int64_t)my_len + ROUND - 1) / ROUND) : 0;
  };
  // Whole tiles: the last (longest) first, every other run of `zigzag` of them in
  // turned order, so that a compute unit that starts with a long tile of one run
  // gets a short one of the next (one prompt of 2048 tokens 50.8 us without, 48.5,
  // 4096 149 and 146; from more than two fillings on not: 8192 515, 522).
  int item = blockIdx.y;
  if (A.splits == 1) {
    const int run = item / A.zigzag, i = item % A.zigzag;
    const int here = min(A.zigzag, A.tiles - run * A.zigzag);
    item = A.tiles - 1 - (run * A.zigzag + (run & 1 ? here - 1 - i : i));
  }
  Place place;
  // (the grid has room for the most items there can be)
  // (a gain below 14 is choose_prompt's for fewer than 64 rows a sequence)
  if (!find_item<ROUND>(seg_of, A.num_seqs, item, A.target, A.splits, A.least,
                        A.gain, A.gain < 14.f, place))
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
  const int tiles = (int)(((int64_t)nq * A.group + S::M - 1) / S::M);
  const int split = place.x / tiles;
  Item it;
  it.table = A.table + (int64_t)seq * A.max_blocks;
  it.token0 = q0;
  it.row0 = (place.x - split * tiles) * S::M;
  it.rows = min(S::M, nq * A.group - it.row0);
  const int ahead = L - nq;  // the position of the first query token
  const int last = (it.row0 + it.rows - 1) / A.group;
  const int range = max(ahead + last + 1, 0);
  it.from = part_end(0, split * place.chunk, range);
  it.to = part_end(it.from, place.chunk, range);
  it.slot = split;
  it.slots = A.splits;
  it.query_at = ahead;
  it.counts = split == 0 && A.splits > 1 ? A.counts : nullptr;
  it.parts = place.parts;
  it.direct = place.parts == 1;
  attend<HD, WM, WN, KT, ST, BS>(A, it, kvh, smem);
  stores_done();
}

// Decode rows (one token a sequence) under a shared prefix: the prefix with the
// rows of all sequences, and each sequence's own tokens [prefix, L).  Grid: kv
// heads, items.  Up to 64 rows the prefix and the sequences are segments of one
// work list in parts of one length.  More (BIG): the prefix's items come first,
// workgroups of 128 rows, one a compute unit, bound by a round's chain alone on its
// unit; the sequences' items, bound by memory, run beside them.  64 sequences of 100
// to 2048 tokens under 32700: 80 us, 440 TFLOP/s and 3.9 TB/s at once, the matrix
// units busy for a fifth of it; 8 under 4096 9.8 us.
template <int HD, bool BIG, int BS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))
void shared_prefix_kernel(RowsArgs A) {
  constexpr int WM = 2, WN = 2, KT = 32, ST = 2;
  using S = Shape<HD, WM, WN, KT, ST>;
  using B = Shape<HD, 4, 1, 64, 2>;  // the prefix's where BIG
  static_assert(B::LDS <= S::LDS, "one LDS array serves both");
  __shared__ __attribute__((aligned(16))) u32x4 smem[S::LDS];
  constexpr int ROUND = WN * KT;
  const int kvh = blockIdx.x;
  const int prefix = min(max(A.prefix_len[0], 0), A.prefix_blocks << A.bs_log2);
  const int cap = A.max_blocks << A.bs_log2;
  const int64_t rows = (int64_t)A.num_seqs * A.n_q;
  Item it;
  it.slots = A.splits + A.suffix_splits;
  it.query_at = NO_QUERY;
  it.direct = false;
  auto prefix_item = [&](int split, int tile, int m, int chunk, int parts) {
    it.table = A.prefix_table;
    it.token0 = 0;
    it.row0 = tile * m;
    it.rows = min(m, A.num_seqs * A.group - it.row0);
    it.from = part_end(0, split * chunk, prefix);
    it.to = part_end(it.from, chunk, prefix);
    it.slot = split;
    it.counts = split > 0 ? nullptr : A.counts;
    it.parts = parts;
  };
  auto prefix_part = [&]() {  // the item of a BIG launch's first tiles * splits
    const int rounds = (prefix + 63) / 64;
    const int chunk = max((rounds + A.splits - 1) / A.splits, 1);
    const int parts = max((rounds + chunk - 1) / chunk, 1);
    const int split = blockIdx.y / A.tiles;
    if (split >= parts) return;
    prefix_item(split, blockIdx.y - split * A.tiles, B::M, chunk * 64, parts);
    attend<HD, 4, 1, 64, 2, BS>(A, it, kvh, smem);
  };
  auto listed_part = [&](int item) {
    const int group_tiles = (A.group + S::M - 1) / S::M;
    // a sequence's tiles are aligned, so that a tile's halves of 32 tokens are within a page
    const int first = prefix & ~(KT - 1);
    auto length = [&](int r) { return min(max(A.seq_lens[r], 0), cap); };
    constexpr int SEG0 = BIG ? 1 : 0;  // segment 0 is the prefix, r + 1 sequence r
    int my_len = 0;  // of segment `lane` where there are up to 64
    auto seg_of = [&](int i, int& tiles, int& rounds) {
      const int s = SEG0 + i;
      tiles = s == 0 ? A.tiles : group_tiles;
      my_len = s == 0 ? prefix : length(s - 1);
      const int span = s == 0 ? prefix : my_len > prefix ? my_len - first : 0;
      rounds = (span + ROUND - 1) / ROUND;
    };
    Place place;
    if (!find_item<ROUND>(seg_of, A.num_seqs + 1 - SEG0, item, A.target, A.suffix_splits, 1,
                          -INFINITY, false, place))
      return;
    const int seg = SEG0 + place.seg;
    const int tiles = seg == 0 ? A.tiles : group_tiles;
    const int split = place.x / tiles, tile = place.x - split * tiles;
    if (seg == 0) {
      prefix_item(split, tile, S::M, place.chunk, place.parts);
    } else {
      const int L = A.num_seqs + 1 - SEG0 <= 64 ? __builtin_amdgcn_readlane(my_len, place.seg)
                                               : length(seg - 1);
      it.table = A.table + (int64_t)(seg - 1) * A.max_blocks;
      it.token0 = seg - 1;
      it.row0 = tile * S::M;
      it.rows = min(S::M, A.group - it.row0);
      const int end = max(L, prefix);
      const int begin = part_end(first, split * place.chunk, end);
      it.from = max(begin, prefix);
      it.to = max(part_end(begin, place.chunk, end), it.from);
      it.slot = A.splits + split;
      it.counts = split > 0 ? nullptr : A.counts + rows;
      it.parts = place.parts;
    }
    attend<HD, WM, WN, KT, ST, 32>(A, it, kvh, smem);
  };
  const int big = BIG ? A.tiles * A.splits : 0;
  if (BIG && (int)blockIdx.y < big)
    prefix_part();
  else
    listed_part((int)blockIdx.y - big);
  stores_done();
}

// out = sum_s 2^(lse_s - max) o_s / sum_s 2^(lse_s - max) over a row's partials: the
// counts[row] first slots and the counts[rows + row] from slot `second` on.  WPR
// waves a row take chunks of MCH partials in turn, lane j of a wave the weight of
// partial j of its chunk, every lane HD / 64 dims; all of a chunk's loads are
// issued before the first is used (64 partials of 256 rows 3.8 us; with one wave a
// row 4.9).  A partial of weight 0 may not have been
// written and is left out.  Rows that are of no sequence, and rows of one part
// (no partials: counts 0), stay as they are.
constexpr int MCH = 16;

template <int HD, int WPR>
__global__ __launch_bounds__(256) void rows_merge_kernel(
    const float* part_o, const float* part_lse, const int32_t* counts, uint16_t* out,
    const int32_t* query_start, int num_seqs, int num_tokens, int n_q, int slots, int second) {
  constexpr int D = HD / 64, ROWS = 4 / WPR;
  __shared__ float top_s[4], sum_s[4], acc_s[4][HD];
  __shared__ int bad_s[4];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), v = wave % WPR;
  const int64_t rows = (int64_t)num_tokens * n_q;
  const int64_t row = (int64_t)blockIdx.x * ROWS + wave / WPR;
  if (row >= rows) return;
  const int tok = (int)(row / n_q);
  if (query_start && (tok < query_start[0] || tok >= query_start[num_seqs])) return;
  const int c0 = min(max(counts[row], 0), second);
  const int c1 = second < slots ? min(max(counts[rows + row], 0), slots - second) : 0;
  const int cnt = c0 + c1;
  if (cnt == 0) return;  // written by the only part
  auto slot = [&](int i) { return i < c0 ? i : second + i - c0; };
  const float* const lse = part_lse + row * slots;
  const float* const po = part_o + row * slots * HD + D * lane;
  float top = -INFINITY, sum = 0.f, acc[D] = {};
  bool bad = false;
  for (int i0 = v * MCH; i0 < cnt; i0 += WPR * MCH) {
    const int last = min(MCH, cnt - i0) - 1;
    const float x = lse[slot(i0 + min(lane, last))];
    float pv[MCH][D];
#pragma unroll
    for (int j = 0; j < MCH; ++j) {
      const float* const src = po + (int64_t)slot(i0 + min(j, last)) * HD;
#pragma unroll
      for (int d = 0; d < D; ++d) pv[j][d] = src[d];
    }
    __builtin_amdgcn_sched_barrier(0);
    const float mine = lane <= last ? x : -INFINITY;
    bad |= __builtin_amdgcn_ballot_w64(mine != mine) != 0;
    const float next = fmaxf(top, wave_max(mine));
    const float w = mine == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mine - next);
    const float a = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - next);
    sum = sum * a + wave_sum(w);
#pragma unroll
    for (int d = 0; d < D; ++d) acc[d] *= a;
#pragma unroll
    for (int j = 0; j < MCH; ++j) {
      const float wj = __builtin_bit_cast(
          float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), j));
#pragma unroll
      for (int d = 0; d < D; ++d) acc[d] = wj == 0.f ? acc[d] : fmaf(wj, pv[j][d], acc[d]);
    }
    top = next;
  }
  if constexpr (WPR > 1) {
#pragma unroll
    for (int d = 0; d < D; ++d) acc_s[wave][D * lane + d] = acc[d];
    if (lane == 0) {
      top_s[wave] = top;
      sum_s[wave] = sum;
      bad_s[wave] = bad;
    }
    __syncthreads();
    if (v != 0) return;
    const float mine = top;
    for (int w = 1; w < WPR; ++w) top = fmaxf(top, top_s[wave + w]);
    const float a = mine == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mine - top);
    sum *= a;
#pragma unroll
    for (int d = 0; d < D; ++d) acc[d] *= a;
    for (int w = 1; w < WPR; ++w) {
      const float t = top_s[wave + w];
      const float b = t == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(t - top);
      sum = fmaf(b, sum_s[wave + w], sum);
      bad |= bad_s[wave + w] != 0;
#pragma unroll
      for (int d = 0; d < D; ++d) acc[d] = fmaf(b, acc_s[wave + w][D * lane + d], acc[d]);
    }
  }
  const float inv = sum > 0.f ? 1.f / sum : 0.f;
  uint16_t* const dst = out + row * HD + D * lane;
  float r[D];
#pragma unroll
  for (int d = 0; d < D; ++d) r[d] = bad ? __builtin_nanf("") : acc[d] * inv;
  if constexpr (D == 2)
    st_agent(reinterpret_cast<uint32_t*>(dst), cvt_pk_bf16(r[0], r[1]));
  else
    st_agent(dst, f32_to_bf16(r[0]));
  stores_done();
}

int log2_of(int v) {
  int b = 0;
  while ((1 << b) < v) ++b;
  return b;
}

template <int HD>
int launch_merge(hipStream_t stream, const RowsArgs& a, int slots, int second, bool prompts) {
  const int64_t rows = (int64_t)a.num_tokens * a.n_q;
  const int32_t* const start = prompts ? a.query_start : nullptr;
  if (slots > MCH)
    SMX_LAUNCH((rows_merge_kernel<HD, 4>), dim3((unsigned)rows), dim3(256), 0, stream, a.part_o,
               a.part_lse, a.counts, a.out, start, a.num_seqs, a.num_tokens, a.n_q, slots, second);
  else
    SMX_LAUNCH((rows_merge_kernel<HD, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream,
               a.part_o, a.part_lse, a.counts, a.out, start, a.num_seqs, a.num_tokens, a.n_q,
               slots, second);
  return (int)hipGetLastError();
}

int tune(const char* name, int v) {
  const char* e = tuning_env(name);
  return e ? atoi(e) : v;
}

// How a call is cut, from its sizes (lengths are on the device).  512 workgroups of
// 64 KB of LDS and 256 threads fill the chip once.
constexpr int FILL = 512, MAX_PARTS = 64;

struct Choice {
  int m;  // rows of a workgroup: 64 (two waves share them, two groups the tokens) or 128
  int splits, suffix_splits, tiles, target;
  float gain;
};

// 128 rows a workgroup multiply faster (a K tile read from L2 serves twice the
// rows), 64 fill the chip sooner and halve the longest workgroup.  us at 32 / 8
// heads of 128, rows of 64 / of 128: a prompt of 1000 tokens 22 / 27, 1500 35 / 38,
// 2048 54 / 50, 3000 103 / 85; behind a context, where all ranges are about as long,
// 128 from one filling on (1000 behind 3000, 40 / 8 heads 114 / 100, 32 / 8 74 / 83).
// Sequences of 65 to 128 rows are one tile of 128, so that fewer workgroups share a
// compute unit: 28 tokens of 12 sequences (192 workgroups of 64) 7.2 / 8.6, 16 (256) 7.6 /
// 8.7, 20 (320) 9.4 / 9.1, 40 (640) 14.9 / 13.5; behind 600 12 15.9 / 20.0, 16 17.2 /
// 20.7, 20 21.3 / 21.2, 40 34.5 / 32.5.
//
// Cutting tiles' tokens into parts costs partials and a second launch, about 11 us
// (14 rounds of 64 tokens), 5 where a tile has few rows, and two workgroups a
// compute unit take 1.45 of a round alone: it pays for long ranges of few
// workgroups.  us whole / cut: 300 tokens behind 16000 201 / 116 (rows of 64), 64
// behind 1000 20 / 14, 1000 behind 3000, 8 / 1 heads 55 / 36, but 16 / 16 heads
// 56.6 / 56.9 and 512 behind 2000 38 / 41.  (The tables' capacity stands for the
// lengths here, find_item asks again with them.)  Sequences of few rows read memory
// at its rate from 160 workgroups on: 23 of up to 11 tokens behind 2821 51 / 59; only
// uneven ones are cut then (find_item), and those of a small capacity not even asked:
// 20 of 5 behind 2500 38 / 41, a fourth of them 1.3 times that 47 / 41, 29 such 57 / 63
// and 65 / 63.  Lengths below the longest take fewer parts, so the longest may take 2
// or 4 times the parts of even ones: 1, 2, 4 times 8 of 5 behind 300 to 8000
// 32.0, 29.6, 29.8; 60 each behind 500, 12000, 900, 700 47.1, 33.6, 32.2; 200 each
// behind 500, 12000, 900 91.8, 75.7, 79.6.  Cut for long
// contexts 128 rows are better: 509 behind 16000 170 / 153, 500 behind 4000 60 / 60.
// Parts are of at least 256 tokens: 300 behind 1500 31.5 at 512, 32.2 at 256, one
// token behind 900 14.6 at 512, 12.3 at 256.
Choice choose_prompt(int64_t num_tokens, int64_t num_seqs, int64_t cap, int group, int n_kv) {
  Choice c{};
  const int64_t rows = (num_tokens * group + num_seqs - 1) / num_seqs;  // of a sequence
  auto groups = [&](int m) { return (rows + m - 1) / m * num_seqs * n_kv; };  // of even lengths
  const bool behind = cap > 2 * ((num_tokens + num_seqs - 1) / num_seqs);
  c.m = groups(64) > (behind ? FILL : 800) || (rows > 64 && rows <= 128 && groups(64) >= 256)
            ? 128 : 64;
  c.gain = 6.f + 8.f * std::min<int64_t>(rows, 64) / 64;
  const bool few = (float)(cap / 64) * (1.f - 1.45f * groups(64) / FILL) >= c.gain &&
                   !(rows <= 64 && cap < 4096 && groups(64) >= 160);
  if (few && rows > 1024 && cap >= 8192) c.m = 128;
  c.m = tune("SMX_PA_M", c.m) < 128 ? 64 : 128;
  c.tiles = (int)((num_tokens * group + c.m - 1) / c.m + num_seqs - 1);
  c.target = std::max(1, FILL / n_kv);
  if (few) {
    const int64_t even = (FILL + groups(c.m) - 1) / groups(c.m);
    const int64_t most = num_seqs == 1 ? even : num_tokens * group <= 1024 ? 4 * even : 2 * even;
    c.splits = (int)std::min<int64_t>({most, MAX_PARTS, cap / 256});
  }
  c.splits = std::clamp(tune("SMX_PA_SPLITS", c.splits), 1, MAX_PARTS);
  return c;
}

// Rows of 128 for the prefix (its own workgroups, one a compute unit) where that is
// much work; else one list of 64-row workgroups for the prefix and the sequences.
// us, list / own: 64 sequences (256 rows) under 2000 tokens 25.6 / 30.2, 8000 32.8 /
// 32.1, 32700 134 / 90; 24 (96 rows) under 4000 16.9 / 19.3, 16000 28.6 / 25.2.
// Beside the prefix's own workgroups a long sequence may take 4 times the parts of
// even ones: 1, 2, 4 times 64 of 100 to 2048 under 32700 93, 88, 88, 48 of 1 to 6000
// under 16000 60, 52, 48, one of 7000 among 31 of 100 46, 36, 33, 40 of 1 to 600 52, 53, 54.
Choice choose_prefix(int64_t num_seqs, int64_t prefix_cap, int64_t cap, int group, int n_kv) {
  Choice c{};
  const int64_t rows = num_seqs * group;
  c.m = tune("SMX_SP_M", rows > 64 && rows * prefix_cap >= 1500000 ? 128 : 64) < 128 ? 64 : 128;
  c.tiles = (int)((rows + c.m - 1) / c.m);
  const int64_t prefix_parts = std::max<int64_t>(1, prefix_cap / 64);
  const int64_t suffix_parts = std::max<int64_t>(1, cap / 64);
  if (c.m == 64) {
    c.target = std::max(1, FILL / n_kv);
    c.suffix_splits = (int)std::min<int64_t>(
        {MAX_PARTS, c.target, std::max(prefix_parts, suffix_parts)});
    c.splits = c.suffix_splits;
  } else {
    c.splits = (int)std::max<int64_t>(
        1, std::min<int64_t>({FILL / 2 / n_kv / c.tiles, MAX_PARTS, prefix_parts}));
    c.target = std::max(1, 2 * FILL / n_kv);
    const int64_t even = (c.target + num_seqs - 1) / num_seqs;
    c.suffix_splits = (int)std::min<int64_t>({4 * even, MAX_PARTS, suffix_parts});
  }
  return c;
}

int64_t partial_bytes(int64_t rows, int64_t slots, int hd) {
  if (slots == 1) return 0;
  return rows * (slots * (hd + 1) + 2) * 4;
}

void set_workspace(RowsArgs& a, void* workspace, int64_t rows, int slots, int hd) {
  a.part_o = (float*)workspace;
  a.part_lse = a.part_o + rows * slots * hd;
  a.counts = (int32_t*)(a.part_lse + rows * slots);
}

// Tiles times parts: at most the target (whose parts' length comes from a sum in
// fp32, so perhaps one more) and one more part of every tile.
int64_t items_bound(int64_t tiles, int target, int splits) {
  return std::min<int64_t>(tiles * splits, target + tiles + 1);
}

template <int HD>
int launch_prompt(hipStream_t stream, RowsArgs& a, const Choice& c) {
  a.zigzag = a.num_seqs == 1 && (int64_t)c.tiles * a.n_kv <= 2 * FILL ? std::max(1, 256 / a.n_kv)
                                                                      : 1 << 30;
  a.target = c.target;
  a.least = 256 / 64;
  a.gain = c.gain;
  const dim3 grid(a.n_kv, (unsigned)items_bound(c.tiles, c.target, c.splits));
  if (c.m == 64)
    SMX_LAUNCH((prompt_attention_kernel<HD, 2, 2, 32, 2, 32>), grid, dim3(256), 0, stream, a);
  else if (a.bs_log2 > 5)
    SMX_LAUNCH((prompt_attention_kernel<HD, 4, 1, 64, 2, 64>), grid, dim3(256), 0, stream, a);
  else
    SMX_LAUNCH((prompt_attention_kernel<HD, 4, 1, 64, 2, 32>), grid, dim3(256), 0, stream, a);
  const int rc = (int)hipGetLastError();
  return rc || c.splits == 1 ? rc : launch_merge<HD>(stream, a, c.splits, c.splits, true);
}

// Workgroups a kv head of the shared-prefix launch.
int64_t prefix_items(int64_t num_seqs, int64_t group, const Choice& c) {
  const int64_t own = num_seqs * ((group + 63) / 64);
  return c.m == 64 ? items_bound(c.tiles + own, c.target, c.splits)
                   : (int64_t)c.tiles * c.splits + items_bound(own, c.target, c.suffix_splits);
}

template <int HD>
int launch_prefix(hipStream_t stream, RowsArgs& a, const Choice& c) {
  a.target = c.target;
  const dim3 grid(a.n_kv, (unsigned)prefix_items(a.num_seqs, a.group, c));
  if (c.m == 64)
    SMX_LAUNCH((shared_prefix_kernel<HD, false, 32>), grid, dim3(256), 0, stream, a);
  else if (a.bs_log2 > 5)
    SMX_LAUNCH((shared_prefix_kernel<HD, true, 64>), grid, dim3(256), 0, stream, a);
  else
    SMX_LAUNCH((shared_prefix_kernel<HD, true, 32>), grid, dim3(256), 0, stream, a);
  const int rc = (int)hipGetLastError();
  return rc ? rc : launch_merge<HD>(stream, a, c.splits + c.suffix_splits, c.splits, false);
}

}  // namespace
}  // namespace smx

#include "smx_abi_util.h"

#define SMX_ROWS_SIZES(num_tokens)                                                               \
  SMX_REQUIRE(head_dim == 64 || head_dim == 128, "head_dim must be 64 or 128");                  \
  SMX_REQUIRE(n_kv >= 1 && n_kv <= 65535 && n_q >= n_kv && n_q % n_kv == 0,                      \
              "n_q must be a multiple of n_kv");                                                 \
  SMX_REQUIRE(block_size >= 32 && block_size <= 4096 && (block_size & (block_size - 1)) == 0,    \
              "block_size must be a power of two in [32, 4096]");                                \
  SMX_REQUIRE((int64_t)n_kv * head_dim * block_size < (1ll << 30),                               \
              "a page must have fewer than 2^30 elements");                                      \
  SMX_REQUIRE(max_blocks >= 1 && (int64_t)max_blocks * block_size <= INT32_MAX - 4096,           \
              "max_blocks * block_size (a sequence's capacity) must fit in int32");              \
  SMX_REQUIRE(num_seqs >= 1 && num_seqs <= 65535, "num_seqs must be in [1, 65535]");             \
  SMX_REQUIRE(num_tokens >= 1 && (int64_t)(num_tokens) * n_q < (1ll << 30),                      \
              "num_tokens * n_q must be in [1, 2^30)")

#define SMX_ROWS_CHECKS()                                                                        \
  SMX_REQUIRE(q && k_cache && v_cache && block_table && seq_lens && out,                         \
              "null pointer argument");                                                          \
  SMX_REQUIRE(num_blocks >= 1, "num_blocks must be >= 1");                                       \
  SMX_REQUIRE(scale > 0.f && isfinite(scale), "scale must be positive and finite");              \
  SMX_REQUIRE((uintptr_t)q % 16 == 0 && (uintptr_t)k_cache % 16 == 0 &&                          \
                  (uintptr_t)v_cache % 16 == 0 && (uintptr_t)out % 16 == 0,                      \
              "q, k_cache, v_cache and out must be 16-byte aligned");                            \
  SMX_REQUIRE((uintptr_t)block_table % 4 == 0 && (uintptr_t)seq_lens % 4 == 0,                   \
              "int arrays must be 4-byte aligned")

extern "C" int64_t smx_prompt_attention_workspace(int32_t num_tokens, int32_t num_seqs,
                                                  int32_t max_blocks, int32_t block_size,
                                                  int32_t n_q, int32_t n_kv, int32_t head_dim) {
  if (num_tokens < 1 || num_seqs < 1 || max_blocks < 1 || block_size < 1 || n_kv < 1 ||
      n_q < n_kv || n_q % n_kv || head_dim < 1)
    return -1;
  const smx::Choice c = smx::choose_prompt(num_tokens, num_seqs, (int64_t)max_blocks * block_size,
                                           n_q / n_kv, n_kv);
  return smx::partial_bytes((int64_t)num_tokens * n_q, c.splits, head_dim);
}

extern "C" int smx_prompt_attention(void* stream, const void* q, int64_t q_stride,
                                    const void* k_cache, const void* v_cache,
                                    const int32_t* block_table, const int32_t* query_start_loc,
                                    const int32_t* seq_lens, void* workspace,
                                    int64_t workspace_bytes, void* out, int32_t num_tokens,
                                    int32_t num_seqs, int32_t max_blocks, int32_t num_blocks,
                                    int32_t block_size, int32_t n_q, int32_t n_kv,
                                    int32_t head_dim, float scale) {
  SMX_ROWS_CHECKS();
  SMX_ROWS_SIZES(num_tokens);
  SMX_REQUIRE(query_start_loc && (uintptr_t)query_start_loc % 4 == 0,
              "query_start_loc must be non-null and 4-byte aligned");
  SMX_REQUIRE(q_stride >= (int64_t)n_q * head_dim && q_stride % 8 == 0,
              "q_stride must be a multiple of 8 and hold n_q heads");
  const smx::Choice c = smx::choose_prompt(num_tokens, num_seqs, (int64_t)max_blocks * block_size,
                                           n_q / n_kv, n_kv);
  SMX_REQUIRE(smx::items_bound(c.tiles, c.target, c.splits) <= 65535,
              "too many row tiles for one launch");
  const int64_t rows = (int64_t)num_tokens * n_q;
  SMX_REQUIRE(c.splits == 1 || (workspace && (uintptr_t)workspace % 16 == 0 &&
                                workspace_bytes >= smx::partial_bytes(rows, c.splits, head_dim)),
              "workspace must be 16-byte aligned and hold smx_prompt_attention_workspace bytes");
  smx::RowsArgs a{};
  a.q = (const uint16_t*)q;
  a.kc = (const uint16_t*)k_cache;
  a.vc = (const uint16_t*)v_cache;
  a.table = block_table;
  a.query_start = query_start_loc;
  a.seq_lens = seq_lens;
  a.out = (uint16_t*)out;
  smx::set_workspace(a, workspace, rows, c.splits, head_dim);
  a.q_stride = q_stride;
  a.num_tokens = num_tokens;
  a.num_seqs = num_seqs;
  a.max_blocks = max_blocks;
  a.num_blocks = num_blocks;
  a.bs_log2 = smx::log2_of(block_size);
  a.n_q = n_q;
  a.n_kv = n_kv;
  a.group = n_q / n_kv;
  a.splits = c.splits;
  a.tiles = c.tiles;
  a.scale_log2 = scale * 1.44269504088896340736f;
  return head_dim == 128 ? smx::launch_prompt<128>((hipStream_t)stream, a, c)
                         : smx::launch_prompt<64>((hipStream_t)stream, a, c);
}

extern "C" int64_t smx_shared_prefix_attention_workspace(int32_t num_seqs, int32_t prefix_blocks,
                                                         int32_t max_blocks, int32_t block_size,
                                                         int32_t n_q, int32_t n_kv,
                                                         int32_t head_dim) {
  if (num_seqs < 1 || prefix_blocks < 1 || max_blocks < 1 || block_size < 1 || n_kv < 1 ||
      n_q < n_kv || n_q % n_kv || head_dim < 1)
    return -1;
  const smx::Choice c =
      smx::choose_prefix(num_seqs, (int64_t)prefix_blocks * block_size,
                         (int64_t)max_blocks * block_size, n_q / n_kv, n_kv);
  return smx::partial_bytes((int64_t)num_seqs * n_q, c.splits + c.suffix_splits, head_dim);
}

extern "C" int smx_shared_prefix_attention(
    void* stream, const void* q, int64_t q_stride, const void* k_cache, const void* v_cache,
    const int32_t* prefix_table, const int32_t* prefix_len, const int32_t* block_table,
    const int32_t* seq_lens, void* workspace, int64_t workspace_bytes, void* out,
    int32_t num_seqs, int32_t prefix_blocks, int32_t max_blocks, int32_t num_blocks,
    int32_t block_size, int32_t n_q, int32_t n_kv, int32_t head_dim, float scale) {
  SMX_ROWS_CHECKS();
  SMX_ROWS_SIZES(num_seqs);
  SMX_REQUIRE(prefix_table && prefix_len && (uintptr_t)prefix_table % 4 == 0 &&
                  (uintptr_t)prefix_len % 4 == 0,
              "prefix_table and prefix_len must be non-null and 4-byte aligned");
  SMX_REQUIRE(prefix_blocks >= 1 && (int64_t)prefix_blocks * block_size <= INT32_MAX - 4096,
              "prefix_blocks * block_size must fit in int32");
  SMX_REQUIRE(q_stride >= (int64_t)n_q * head_dim && q_stride % 8 == 0,
              "q_stride must be a multiple of 8 and hold n_q heads");
  const smx::Choice c =
      smx::choose_prefix(num_seqs, (int64_t)prefix_blocks * block_size,
                         (int64_t)max_blocks * block_size, n_q / n_kv, n_kv);
  const int64_t rows = (int64_t)num_seqs * n_q;
  const int slots = c.splits + c.suffix_splits;
  SMX_REQUIRE(smx::prefix_items(num_seqs, n_q / n_kv, c) <= 65535,
              "too many row tiles for one launch");
  SMX_REQUIRE(workspace && (uintptr_t)workspace % 16 == 0 &&
                  workspace_bytes >= smx::partial_bytes(rows, slots, head_dim),
              "workspace must be 16-byte aligned and hold "
              "smx_shared_prefix_attention_workspace bytes");
  smx::RowsArgs a{};
  a.q = (const uint16_t*)q;
  a.kc = (const uint16_t*)k_cache;
  a.vc = (const uint16_t*)v_cache;
  a.table = block_table;
  a.prefix_table = prefix_table;
  a.prefix_len = prefix_len;
  a.seq_lens = seq_lens;
  a.out = (uint16_t*)out;
  smx::set_workspace(a, workspace, rows, slots, head_dim);
  a.q_stride = q_stride;
  a.num_tokens = num_seqs;
  a.num_seqs = num_seqs;
  a.max_blocks = max_blocks;
  a.prefix_blocks = prefix_blocks;
  a.num_blocks = num_blocks;
  a.bs_log2 = smx::log2_of(block_size);
  a.n_q = n_q;
  a.n_kv = n_kv;
  a.group = n_q / n_kv;
  a.splits = c.splits;
  a.suffix_splits = c.suffix_splits;
  a.tiles = c.tiles;
  a.scale_log2 = scale * 1.44269504088896340736f;
  return head_dim == 128 ? smx::launch_prefix<128>((hipStream_t)stream, a, c)
                         : smx::launch_prefix<64>((hipStream_t)stream, a, c);
}
