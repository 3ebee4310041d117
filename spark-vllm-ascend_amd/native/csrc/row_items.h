// What the attentions over packed rows share (prompt_attention.hip,
// q4_attention.hip): how a launch's work is cut from lengths on the device, and
// the merge of its partials.
#pragma once

#include <limits.h>

#include <type_traits>

#include "smx_common.h"
#include "smx_launch.h"

namespace smx {

// Enqueues the merge of a row attention's partials (prompt_attention.hip): row r's
// out = the softmax mean of its counts[r] first of `slots` slots; rows of count 0 and
// rows of no sequence (query_start, null: none) stay as they are.
int merge_rows(hipStream_t stream, int head_dim, const float* part_o, const float* part_lse,
               const int32_t* counts, void* out, const int32_t* query_start, int num_seqs,
               int num_tokens, int n_q, int slots);

// Packed rows of many tokens a sequence over a cache held in 4 bits, by
// prompt_attention.hip's kernels.
struct Q4Prompt {
  const uint16_t* q;
  const uint8_t* codes;
  const uint16_t* scales;
  const int32_t* table;
  const int32_t* query_start;
  const int32_t* seq_lens;
  void* workspace;  // q4_prompt_workspace bytes
  void* out;
  int64_t q_stride;
  int num_tokens, num_seqs, max_blocks, num_blocks, bs_log2, n_q, n_kv, head_dim;
  float scale_log2;
};
int64_t q4_prompt_workspace(const Q4Prompt& p);  // -1: more row tiles than a launch holds
int q4_prompt(hipStream_t stream, const Q4Prompt& p);

namespace {

// (lo, hi) as one v_cvt_pk_bf16_f32
__device__ __forceinline__ uint32_t cvt_pk_bf16(float lo, float hi) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), bf16x2));
}

// (lo, hi) as one v_cvt_pk_f16_f32
__device__ __forceinline__ uint32_t cvt_pk_f16(float lo, float hi) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), f16x2));
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

}  // namespace
}  // namespace smx
