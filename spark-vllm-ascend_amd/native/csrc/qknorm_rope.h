// Per-head RMSNorm and neox rotary positions of q and k, 16 lanes a head of 128.
#pragma once

#include <math.h>

#include "smx_common.h"

namespace smx {

// The 8 channels 8 j .. of one head (src, 128 channels): normalised with gam and rotated
// to position pos (kept within the table) where `turn`, as they are elsewhere.  Lane j of
// the 16; lane j ^ 8 holds the other half of each rotation pair.  All lanes of a wave call it.
__device__ __forceinline__ u32x4 qknorm_rope_chunk(const uint16_t* __restrict__ src,
                                                   const uint16_t* __restrict__ gam,
                                                   const uint16_t* __restrict__ cos_sin,
                                                   int64_t pos, bool turn, int j,
                                                   int max_position, float eps) {
  constexpr int HD = 128, HALF = 64;
  const int dim = 8 * (j & 7);
  const u32x4 own = *reinterpret_cast<const u32x4*>(src + 8 * j);
  const u32x4 gv = *reinterpret_cast<const u32x4*>(gam + 8 * j);
  pos = pos < 0 ? 0 : (pos >= max_position ? max_position - 1 : pos);
  const u32x4 cv = *reinterpret_cast<const u32x4*>(cos_sin + pos * HD + dim);
  const u32x4 sv = *reinterpret_cast<const u32x4*>(cos_sin + pos * HD + HALF + dim);
  auto other_half = [](uint32_t v) {  // lane j ^ 8's register
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, DPP_ROW_ROR8, 0xf, 0xf, false);
  };
  u32x4 val = own;
  // (every head of a wave is a V head, or all lanes stay: the row moves need them)
  if (__builtin_amdgcn_ballot_w64(turn) != 0) {
    const bool lo = j < 8;
    float sq[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t p = other_half(own[i]);
      const uint32_t aw = lo ? own[i] : p, bw = lo ? p : own[i];
      sq[2 * i] = bf16_lo(aw) * bf16_lo(aw) + bf16_lo(bw) * bf16_lo(bw);
      sq[2 * i + 1] = bf16_hi(aw) * bf16_hi(aw) + bf16_hi(bw) * bf16_hi(bw);
    }
    const float ss = sum8(((sq[0] + sq[1]) + (sq[2] + sq[3])) + ((sq[4] + sq[5]) + (sq[6] + sq[7])));
    const float inv = 1.0f / sqrtf(ss / (float)HD + eps);
    const uint32_t flip = lo ? 0x80008000u : 0u;  // u = a c - b s, v = b c + a s
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // the rounded norm of this half, and the other half's from lane j ^ 8
      const uint32_t nw = pack_bf16x2(bf16_lo(own[i]) * inv * bf16_lo(gv[i]),
                                      bf16_hi(own[i]) * inv * bf16_hi(gv[i]));
      const uint32_t ow = other_half(nw), sw = sv[i] ^ flip;
      r[i] = pack_bf16x2(fmaf(bf16_lo(nw), bf16_lo(cv[i]), bf16_lo(ow) * bf16_lo(sw)),
                         fmaf(bf16_hi(nw), bf16_hi(cv[i]), bf16_hi(ow) * bf16_hi(sw)));
    }
    if (turn) val = u32x4{r[0], r[1], r[2], r[3]};
  }
  return val;
}

}  // namespace smx
