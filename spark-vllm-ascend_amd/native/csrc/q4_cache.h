// The paged KV cache held in 4 bits: its format and layout (gfx950).
//
// Blocks of 32 channels of one head of a token share an fp16 scale d and hold codes c of
// 0..15 for the values d (c - 8), the block format of the Q4_0 weights: m the first
// value of largest magnitude, d = fp16(m / -8) (kept finite), c = floor(x / d + 8.5)
// kept within 0..15; 8 where d is 0.  A block with a NaN has the scale NaN, codes 0.
//
// codes  [2][num_blocks][n_kv][block_size][head_dim / 2] bytes, K first
// scales [2][num_blocks][n_kv][block_size][head_dim / 32] fp16
// One head's page is contiguous, so that a tile of it is read in whole kilobytes.  V's
// codes are in channel order, two a byte, the lower half first.  K's dword
// g * (head_dim / 32) + b holds channels 32 b + 8 g + (0, 2, 4, 6, 1, 3, 5, 7), lowest
// half-byte first: lane group g of a matrix instruction reads its channels of every
// block at once, and (w >> s) & 0x000f000f is a pair of neighbours.
#pragma once

#include "smx_common.h"

namespace smx {

struct Q4Cache {
  uint8_t* codes;
  uint16_t* scales;
  int num_blocks, bs_log2, n_kv;
};

// The row of (plane, slot, head): its codes are the bytes [row * HD / 2, + HD / 2), its
// scales the fp16 values [row * HD / 32, + HD / 32).  slot is in [0, num_blocks * bs).
__device__ __forceinline__ int64_t q4_row(const Q4Cache& c, int plane, int64_t slot, int head) {
  const int64_t page = ((int64_t)plane * c.num_blocks + (slot >> c.bs_log2)) * c.n_kv + head;
  return (page << c.bs_log2) + (slot & ((1 << c.bs_log2) - 1));
}

// Quantises a head's chunk of 8 bf16 channels a lane (16 bytes: lane j of the head's
// HD / 8 neighbours has channels 8 j ..), four lanes a block, and stores it.  Every lane
// of the four must be active; `store` says whether this head is kept.
//
// x / d is taken as x * (1 / d), off by 1e-6 at most.  A code's border is an odd h with
// x / d = h / 2.  With x of 8 and d of 11 significant bits, 2 x - h d is 0 or so large that
// the quotient is 2^-12 or more from the border: 2^-14 added before the floor puts
// those that hit one on its upper side and leaves the others on theirs.
template <int HD>
__device__ __forceinline__ void q4_store_chunk(const Q4Cache& c, int plane, int64_t slot,
                                               int head, int j, u32x4 x, bool store) {
  const int g = j & 3, b = j >> 2;
  // (magnitude, lowest index, sign) as one word
  uint32_t best = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t w = x[i / 2];
    const uint32_t v = i & 1 ? w >> 16 : w & 0xffffu;
    best = max(best, ((v & 0x7fffu) << 6) | (uint32_t)((31 - 8 * g - i) << 1) | (v >> 15));
  }
  best = max(best, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)best, DPP_QUAD_XOR1, 0xf, 0xf,
                                                         false));
  best = max(best, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)best, DPP_QUAD_XOR2, 0xf, 0xf,
                                                         false));
  const uint32_t mag = best >> 6;
  const float m = bf16_bits_to_f32(mag | ((best & 1u) << 15));
  const float limit = 65504.f;
  const float df = fminf(fmaxf(m * -0.125f, -limit), limit);
  const _Float16 d = mag > 0x7f80u ? (_Float16)__builtin_nanf("") : (_Float16)df;
  const float dr = (float)d;
  const float inv = dr == 0.f ? 0.f : 1.0f / dr;
  uint32_t code[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = i & 1 ? bf16_hi(x[i / 2]) : bf16_lo(x[i / 2]);
    // (1 / NaN makes every code of a block with a NaN 0)
    code[i] = (uint32_t)fminf(fmaxf(floorf(fmaf(v, inv, 8.5f + 0x1p-14f)), 0.f), 15.f);
  }
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) w |= code[i] << (plane == 0 ? 4 * (i / 2) + 16 * (i & 1) : 4 * i);
  if (store) {
    const int64_t row = q4_row(c, plane, slot, head);
    const int dword = plane == 0 ? g * (HD / 32) + b : j;
    st_agent(reinterpret_cast<uint32_t*>(c.codes + row * (HD / 2)) + dword, w);
    if (g == 0) st_agent(c.scales + row * (HD / 32) + b, __builtin_bit_cast(uint16_t, d));
  }
}

}  // namespace smx
