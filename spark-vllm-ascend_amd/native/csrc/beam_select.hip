// Beam search's selection over beams and vocabulary, for gfx950: of a sequence's beams b
// with scores c_b and logits x_b the `width` best continuations
//   score(b, v) = c_b + x_b[v] - log sum_u exp(x_b[u])
// in order, ties to the lowest b * vocab + v.
//
// One pass over the logits.  A beam's best are its largest logits, so a workgroup keeps
// the `width` largest of its part of a row and the part's maximum and sum of exponentials
// (beam_parts_kernel); a workgroup a sequence then takes the best of the parts'
// (beam_merge_kernel).  Beams are compared by their sums, so these are of exponentials in
// 64 bits, each good to 8e-13 of itself, relative to a part's maximum: a score is good to
// 3e-12, and rows that differ by a constant have the same sums.  (The transcendental unit's
// exponentials with a correction for most of a peaked row's sum were 1.4 times as fast, but
// their error of some 1e-8 is a function of the value: in a row of few distinct logits it
// does not average out.)
//
// Bound by vector instructions where there are many rows: 512 rows of 151936 bf16 values,
// a tenth of them done, 16 best of 8 beams: 75 us, the parts 67 (2.1 TB/s; about 25
// instructions a value, 18 of them in 64 bits), the merge 7.4.  4 rows 10.8 us: two launches
// of short latencies one after another.
//
// A NaN logit counts as -inf, a token that is never chosen; of several logits of +inf each
// has an equal share.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "smx_common.h"
#include "smx_launch.h"

namespace smx {
namespace {

typedef u32x4 u32x4_a2 __attribute__((aligned(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));

constexpr int MAX_WIDTH = 64, MAX_BEAMS = 64;
constexpr int CAP = 128;     // candidates of a wave
constexpr int CHUNKS = 128;  // loads of a wave that hold candidates
constexpr int NT = 256, WAVES = NT / 64;
// Of 16 bytes, a lane: a part is 16 KB of a row.  us with 2 / 4 / 8 of them, rows of 151936
// bf16 values: 1 row 9.5 / 10.0 / 11.4, 16 rows 11.4 / 11.7 / 12.0, 128 rows 33 / 27 / 26,
// 512 rows (a tenth done) 94 / 75 / 75; 64 rows of 32000 10.7 / 10.9 / 12.3, 512 rows 27 /
// 24 / 24.
constexpr int LOADS = 4;

struct BeamArgs {
  const void* logits;
  const float* scores;   // [rows]
  const uint8_t* done;   // [rows] or null
  double* part_sum;      // [rows, parts]
  float* part_max;       // [rows, parts]
  float* cand_value;     // [seqs, width, beams * parts]: rank first
  int32_t* cand_token;   // likewise, -1: none
  int32_t* parents;      // [seqs, width]
  int64_t* tokens;
  float* out_scores;
  int64_t stride;  // of a row of logits, in elements
  int seqs, beams, width, vocab, parts, pad_id;
};

// exp(a) for |a| <= 700, relative error 8e-13: a = n ln 2 + r with |r| <= ln 2 / 2, a
// polynomial of degree 8 fitted to exp on that interval by least squares reweighted
// towards the largest relative error, and n added to the exponent's bits.
__device__ __forceinline__ double exp_any(double a) {
  const double magic = 0x1.8p52;  // its sum's low bits are the rounded quotient
  const double t = fma(a, 1.4426950408889634, magic);
  const double r = fma(t - magic, -0.6931471805599453, a);
  double p = 0x1.9eda514635a5bp-16;
  p = fma(p, r, 0x1.a1a83103871fap-13);
  p = fma(p, r, 0x1.6c18b3a477d5cp-10);
  p = fma(p, r, 0x1.111082a0498a6p-7);
  p = fma(p, r, 0x1.55555404b7c02p-5);
  p = fma(p, r, 0x1.555555a08d61dp-3);
  p = fma(p, r, 0x1.0000000088227p-1);
  p = fma(p, r, 0x1.ffffffffd55a3p-1);
  p = fma(p, r, 0x1.ffffffffff79dp-1);
  const uint64_t bits = __builtin_bit_cast(uint64_t, p);
  uint32_t hi = (uint32_t)(bits >> 32);
  asm("" : "+v"(hi));  // (so that 32 bits are added in one instruction, not 64 in five)
  hi += (uint32_t)__builtin_bit_cast(uint64_t, t) << 20;
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | (uint32_t)bits);
}

// exp(x - top) for a part's maximum x <= top, either of them infinite (top not -inf, or
// neither counts: their sums are 0).
__device__ __forceinline__ double exp_between(float x, float top) {
  return x == top ? 1.0 : exp_any(fmax((double)x - (double)top, -700.0));
}

// Values in their order as signed integers: the bits of positive ones, minus those of
// negative ones' magnitudes, so that -0 is 0.
__device__ __forceinline__ int order_key(uint32_t u) {
  const int m = (int)u >> 31;
  return (int)((u & 0x7fffffffu) ^ m) - m;
}
__device__ __forceinline__ float order_value(int k) {
  return __uint_as_float(k < 0 ? (uint32_t)-k | 0x80000000u : (uint32_t)k);
}
// Where -0 may be below 0: negative values' bits but the sign's flipped, and back.  (Of
// bf16 values 16 bits, the upper ones of a key.)
__device__ __forceinline__ int quick_key(float f) {
  const int u = (int)__float_as_uint(f);
  return u ^ ((u >> 31) & 0x7fffffff);
}
template <int BITS>
__device__ __forceinline__ float key_value(int k) {
  return __uint_as_float((uint32_t)(k ^ ((k >> 31) & 0x7fffffff)) & (~0u << (32 - BITS)));
}
constexpr int INF_KEY = 0x7f800000;

// The value of lane ^ MASK, once the lanes of each group of MASK hold the same value.
template <int MASK, typename K>
__device__ __forceinline__ K other(K v) {
  auto move = [](uint32_t x) -> uint32_t {
    if constexpr (MASK <= 8) {
      constexpr int CTRL = MASK == 1   ? DPP_QUAD_XOR1
                           : MASK == 2 ? DPP_QUAD_XOR2
                           : MASK == 4 ? DPP_ROW_HALF_MIRROR
                                       : DPP_ROW_MIRROR;
      return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, false);
    } else {
      return (uint32_t)__shfl_xor((int)x, MASK);
    }
  };
  if constexpr (sizeof(K) == 4) {
    return __builtin_bit_cast(K, move(__builtin_bit_cast(uint32_t, v)));
  } else {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(K, (uint64_t)move((uint32_t)u) | (uint64_t)move((uint32_t)(u >> 32)) << 32);
  }
}

// The sum over a wave, in an order that does not depend on the lane.
__device__ __forceinline__ double wave_sum64(double v) {
  v += other<1>(v);
  v += other<2>(v);
  v += other<4>(v);
  v += other<8>(v);
  v += other<16>(v);
  v += other<32>(v);
  return v;
}

// One part (NT * LOADS * V logits) of one row, a wave's share of it in registers: its
// maximum, the values that reach a bound which `width` of the part do (found from maxima
// over a lane of each wave), and its sum of exponentials; the few collected of all waves are ranked
// by counting.
template <typename L>
__global__ __launch_bounds__(NT) void beam_parts_kernel(BeamArgs A) {
  constexpr int V = 16 / sizeof(L);  // logits of a load
  constexpr int PART = NT * LOADS * V;
  __shared__ uint64_t list[WAVES][CAP + 4];
  __shared__ u32x4 tail_s, chunk_s[WAVES][CHUNKS];
  __shared__ int where_s[WAVES][CHUNKS];
  __shared__ int count_s[WAVES], best_s[WAVES][64];
  __shared__ double sum_s[WAVES];
  const int part = blockIdx.x, row = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // a beam that is done, or has no score, offers nothing from its logits
  if (A.done && A.done[row]) return;
  if (!(A.scores[row] > -INFINITY)) return;
  const int first = part * PART, here = min(A.vocab - first, PART);
  const L* const src = reinterpret_cast<const L*>(A.logits) + (int64_t)row * A.stride + first;
  typedef L __attribute__((may_alias)) Value;
  constexpr uint32_t NONE = sizeof(L) == 2 ? 0xff80ff80u : 0xff800000u;  // -inf

  u32x4 x[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int at = (i * NT + tid) * V;
    x[i] = u32x4{NONE, NONE, NONE, NONE};
    if (at + V <= here) x[i] = *reinterpret_cast<const u32x4_a2*>(src + at);
  }
  if (here < PART) {
    // the row's last few logits, by the thread that has their place
    const int chunk = here / V;
    if (tid == chunk % NT) {
      tail_s = u32x4{NONE, NONE, NONE, NONE};
      for (int j = chunk * V; j < here; ++j)
        reinterpret_cast<Value*>(&tail_s)[j - chunk * V] = src[j];
#pragma unroll
      for (int i = 0; i < LOADS; ++i)
        if (i == chunk / NT) x[i] = tail_s;
    }
  }
  // ---- the loads' and the lanes' maxima, as keys
  constexpr int STEP = V == 8 ? 0x10000 : 1;  // between two keys
  constexpr int NO_KEY = (int)0x807fffff & -STEP;  // of -inf
  constexpr int BITS = V == 8 ? 16 : 32;
  typedef typename std::conditional<V == 8, s16x2, int>::type Key;
  Key most[LOADS];  // V == 8: of the even values and of the odd ones
  auto key = [](Key k) -> int {
    if constexpr (V == 8)
      return max((int)k[0], (int)k[1]) << 16;
    else
      return k;
  };
  auto maxima = [&]() {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t u = x[i][j];  // (an element itself is no operand for a bit_cast)
        const Key w = __builtin_bit_cast(Key, u);
        const Key k = w ^ ((w >> (V == 8 ? 15 : 31)) & (Key)(V == 8 ? 0x7fff : 0x7fffffff));
        most[i] = j == 0 ? k : __builtin_elementwise_max(most[i], k);
      }
    }
    Key best = most[0];
#pragma unroll
    for (int i = 1; i < LOADS; ++i) best = __builtin_elementwise_max(best, most[i]);
    return key(best);
  };
  int best = maxima();
  if (__builtin_amdgcn_ballot_w64(best > INF_KEY)) {
    // -inf in the place of a NaN without a sign (one with it is below -inf in this order)
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t w = x[i][j];
        if constexpr (V == 8) {
          if ((w & 0xffffu) - 0x7f81u < 0x7fu) w = (w & 0xffff0000u) | 0xff80u;
          if ((w >> 16) - 0x7f81u < 0x7fu) w = (w & 0xffffu) | 0xff800000u;
        } else {
          if (w - 0x7f800001u < 0x7fffffu) w = NONE;
        }
        x[i][j] = w;
      }
    best = maxima();
  }
  // Of the lanes l of all waves.
  best_s[wave][lane] = best;
  __syncthreads();
  best = best_s[0][lane];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) best = max(best, best_s[w][lane]);
  int top_key = best;
  top_key = max(top_key, other<1>(top_key));
  top_key = max(top_key, other<2>(top_key));
  top_key = max(top_key, other<4>(top_key));
  top_key = max(top_key, other<8>(top_key));
  top_key = max(top_key, other<16>(top_key));
  top_key = max(top_key, other<32>(top_key));

  // ---- the largest
  // The bound: the width-th largest of these 64 maxima, which 1.15 times `width` of a part's
  // values are expected to reach at a width of 16; bit by bit from above, of 16.
  int64_t least_key = NO_KEY + STEP;
  for (int64_t bit = 1ll << 31; bit >= 1 << 16; bit >>= 1)
    if (least_key + bit <= INF_KEY &&
        __popcll(__builtin_amdgcn_ballot_w64(best >= (int)(least_key + bit))) >= A.width)
      least_key += bit;
  // (0 and -0 are the same value, but not the same key: a bound of 0 is -0's)
  const int bound_key = least_key == 0 ? -STEP : (int)least_key;
  const float bound = key_value<BITS>(bound_key);
  const float top = key_value<BITS>(max(top_key, NO_KEY));
  uint64_t* const mine = list[wave];
  int n = 0;
  // (what is computed of a load's values is not kept over this)
  auto opaque = [&](int i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t w = x[i][j];
      asm volatile("" : "+v"(w));
      x[i][j] = w;
    }
  };
  auto value = [&](int i, int j) -> float {
    if constexpr (V == 8)
      return j & 1 ? bf16_hi(x[i][j / 2]) : bf16_lo(x[i][j / 2]);
    else
      return __uint_as_float(x[i][j]);
  };
  // The few lanes' loads that hold a value which reaches it go to LDS, and their values are
  // looked at there, a lane each.
  auto below = [](uint64_t m) {  // its bits below this lane's
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
  };
  int chunks = 0;
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const bool hit = key(most[i]) >= bound_key;
    if (const uint64_t m = __builtin_amdgcn_ballot_w64(hit)) {
      const int at = chunks + below(m);
      if (hit && at < CHUNKS) {
        chunk_s[wave][at] = x[i];
        where_s[wave][at] = i * NT + tid;
      }
      chunks += __popcll(m);
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  typedef typename std::conditional<V == 8, uint16_t, uint32_t>::type __attribute__((may_alias)) Raw;
  const Raw* const chunk = reinterpret_cast<const Raw*>(chunk_s[wave]);
  for (int e = lane; e - lane < min(chunks, CHUNKS) * V; e += 64) {
    const uint32_t w = e < chunks * V ? (uint32_t)chunk[e] << (V == 8 ? 16 : 0) : 0xff800000u;
    const bool in = __uint_as_float(w) >= bound;
    const uint64_t m = __builtin_amdgcn_ballot_w64(in);
    const int at = n + below(m);
    if (in && at < CAP)
      mine[at] = (uint64_t)((uint32_t)order_key(w) ^ 0x80000000u) << 32 |
                 (0xffffffffu - (uint32_t)(where_s[wave][e / V] * V + e % V));
    n += __popcll(m);
  }
  // Puts the values of load i that `in(j)` says into the list, in no particular order: a
  // bit a value, the set ones lane by lane.
  auto collect = [&](int i, auto in) {
    uint32_t bits = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) bits = bits + bits + (in(j) ? 1u : 0u);
    while (const uint64_t m = __builtin_amdgcn_ballot_w64(bits != 0)) {
      const int at = n + below(m);
      if (bits && at < CAP) {
        const int low = __ffs(bits) - 1, j = V - 1 - low;
        uint32_t w;
        if constexpr (V == 8) {
          const uint32_t lo = j & 2 ? x[i][1] : x[i][0], hi = j & 2 ? x[i][3] : x[i][2];
          w = j & 4 ? hi : lo;
          w = j & 1 ? w & 0xffff0000u : w << 16;
        } else {
          const uint32_t lo = j & 1 ? x[i][1] : x[i][0], hi = j & 1 ? x[i][3] : x[i][2];
          w = j & 2 ? hi : lo;
        }
        mine[at] = (uint64_t)((uint32_t)order_key(w) ^ 0x80000000u) << 32 |
                   (0xffffffffu - (uint32_t)((i * NT + tid) * V + j));
      }
      bits &= bits - 1;
      n += __popcll(m);
    }
  };
  if (n > CAP || chunks > CHUNKS) {
    // (sorted or equal logits: the bound is loose)  The width-th largest value, bit by bit
    // from above; then those above it, and as many of its equals as are missing, the
    // lowest places first: load by load, lane by lane.
    auto key_of = [&](int i, int j) { return order_key(__float_as_uint(value(i, j))); };
    auto reach = [&](int b) {
      int c = 0;
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        opaque(i);
#pragma unroll
        for (int j = 0; j < V; ++j)
          c += __popcll(__builtin_amdgcn_ballot_w64(key_of(i, j) >= b));
      }
      return c;
    };
    // (more than `width` reach `bound`, so the value is not below it)
    int64_t least = order_key(__float_as_uint(bound));
#pragma unroll 1
    for (int64_t bit = 1ll << 31; bit >= STEP; bit >>= 1)
      if (least + bit <= INF_KEY && reach((int)(least + bit)) >= A.width) least += bit;
    n = 0;
    int missing = A.width - reach((int)least + STEP);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      int equal = 0;
      opaque(i);
#pragma unroll
      for (int j = 0; j < V; ++j) equal += key_of(i, j) == (int)least;
      const int incl = wave_scan_i32(equal);
      int before = incl - equal;
      collect(i, [&](int j) {
        const int k = key_of(i, j);
        const bool same = k == (int)least;
        const bool in = k > (int)least || (same && before < missing);
        before += same;
        return in;
      });
      missing = max(missing - __builtin_amdgcn_readlane(incl, 63), 0);
    }
  }

  // ---- the sum of exponentials relative to `top` (-inf and NaN with a sign: below -700)
  double sum = 0.0;
  if (top_key < INF_KEY && top_key > NO_KEY) {
    double s[2] = {0.0, 0.0};
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      opaque(i);
#pragma unroll
      for (int j = 0; j < V; ++j)
        s[j & 1] += exp_any(fmax((double)value(i, j) - (double)top, -700.0));
    }
    sum = s[0] + s[1];
  } else if (top_key == INF_KEY) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) sum += value(i, j) == INFINITY;
  }
  sum = wave_sum64(sum);
  if (lane < 4) mine[n + lane] = 0;  // four of them are compared at a time
  if (lane == 0) {
    count_s[wave] = n;
    sum_s[wave] = sum;
  }
  __syncthreads();

  const int seq = row / A.beams, lists = A.beams * A.parts;
  const int64_t out = (int64_t)seq * A.width * lists + (row - seq * A.beams) * A.parts + part;
  int total = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) total += count_s[w];
  for (int i = lane; i < n; i += 64) {
    const uint64_t key = mine[i];
    int rank = 0;
    for (int w = 0; w < WAVES; ++w)
      for (int j = 0; j < count_s[w]; j += 4)
#pragma unroll
        for (int k = 0; k < 4; ++k) rank += list[w][j + k] > key;
    if (rank < A.width) {
      st_agent(A.cand_value + out + (int64_t)rank * lists,
               order_value((int)((uint32_t)(key >> 32) ^ 0x80000000u)));
      st_agent(A.cand_token + out + (int64_t)rank * lists,
               first + (int)(0xffffffffu - (uint32_t)key));
    }
  }
  for (int i = total + tid; i < A.width; i += NT)
    st_agent(A.cand_token + out + (int64_t)i * lists, -1);
  if (tid == 0) {
    double s = 0.0;
    for (int w = 0; w < WAVES; ++w) s += sum_s[w];
    st_agent(A.part_max + (int64_t)row * A.parts + part, top);
    st_agent(reinterpret_cast<uint64_t*>(A.part_sum) + (int64_t)row * A.parts + part,
             __builtin_bit_cast(uint64_t, s));
  }
  stores_done();
}

// In order: the larger score first, then the lower place, beam << 24 | token.
__device__ __forceinline__ bool before(double s, int p, double t, int r) {
  return s > t || (s == t && p < r);
}

// a / c for 0 <= a < 2^24 and inv = 1 / c to a few units of the last place.
__device__ __forceinline__ int small_div(int a, int c, float inv) {
  const int q = (int)((float)a * inv);
  const int r = a - q * c;
  return q + (r >= c) - (r < 0);
}

// One workgroup a sequence.  A beam's parts are joined to its log sum; the candidates that
// reach a bound found as above are collected and ranked.  Where too many do (equal scores,
// or more are wanted than there are lists, beams times parts, whose first the bound is of),
// they are found one after another instead: 49 of 4 x 16 rows of 16000 142 us, 16 of them
// 11.7.  Bound by instructions that are not in the cache yet: one loop does for the bound and
// for the candidates.
constexpr int MERGE_NT = 512, MERGE_WAVES = MERGE_NT / 64;
constexpr int MERGE_CAP = 1024, HELD = 4;

__global__ __launch_bounds__(MERGE_NT) void beam_merge_kernel(BeamArgs A) {
  __shared__ float top_s[MAX_BEAMS];
  __shared__ double log_s[MAX_BEAMS];  // score - the log of the sum relative to the maximum
  __shared__ float own_s[MAX_BEAMS];   // the score of a beam that is done
  __shared__ double cs[MERGE_CAP];
  __shared__ int cp[MERGE_CAP];
  __shared__ double best_s[MERGE_WAVES];
  __shared__ int place_s[MERGE_WAVES];
  __shared__ int count_s;
  const int seq = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lists = A.beams * A.parts;
  const float lists_inv = __builtin_amdgcn_rcpf((float)lists);
  const float parts_inv = __builtin_amdgcn_rcpf((float)A.parts);
  if (tid == 0) count_s = 0;
  // Candidate e of `n`: rank, beam, part.  The first list head of a lane and the first
  // candidates of a thread are on their way before anything else.
  const int n = A.width * lists;
  const int32_t* const token_of = A.cand_token + (int64_t)seq * n;
  const float* const value_of = A.cand_value + (int64_t)seq * n;
  int token[HELD];
  float value[HELD];
#pragma unroll
  for (int i = 0; i < HELD; ++i) {
    const int e = min(i == 0 ? lane : tid + (i - 1) * MERGE_NT, n - 1);
    token[i] = token_of[e];
    value[i] = value_of[e];
  }
  // a beam that offers nothing from its logits has the score -inf
  for (int b = wave; b < A.beams; b += MERGE_WAVES) {
    const int row = seq * A.beams + b;
    const float* const pm = A.part_max + (int64_t)row * A.parts;
    const double* const ps = A.part_sum + (int64_t)row * A.parts;
    const float c = A.scores[row];
    const uint8_t flag = *(A.done ? A.done + row : reinterpret_cast<const uint8_t*>(A.scores));
    const int at = min(lane, A.parts - 1);
    const float m0 = pm[at];
    const double s0 = ps[at];
    float m = m0;
    for (int p = lane + 64; p < A.parts; p += 64) m = fmaxf(m, pm[p]);
    m = wave_max(m);
    double s = 0.0;
    for (int p = lane; p < A.parts; p += 64) {
      const bool held = p == lane;
      s += (held ? s0 : ps[p]) * exp_between(held ? m0 : pm[p], m);
    }
    s = wave_sum64(s);
    // log s: fp32's, and what is missing from s exp(-log s) = 1
    const double y = (double)(__builtin_amdgcn_logf((float)s) * 0x1.62e430p-1f);
    const double d = s * exp_any(-y) - 1.0;
    if (lane == 0) {
      top_s[b] = m;
      const bool done = A.done && flag;
      log_s[b] = done || !(c > -INFINITY) || !(s > 0.0) ? -INFINITY
                                                        : (double)c - (y + (d - 0.5 * d * d));
      own_s[b] = done ? c : -INFINITY;
    }
  }
  __syncthreads();

  auto candidate = [&](int e, int tok, float v, double& s, int& place) {
    const int list = e - small_div(e, lists, lists_inv) * lists;
    const int b = small_div(list, A.parts, parts_inv);
    s = log_s[b];
    if (s == -INFINITY || tok < 0) {
      s = -INFINITY;
      return;
    }
    s += v == top_s[b] ? 0.0 : (double)v - (double)top_s[b];
    place = b << 24 | tok;
  };
  // The bound: the width-th largest of the lanes' best list heads (ranks of 0), lane l of
  // every wave with the lists l, l + 64, .., rounded downwards and found bit by bit (of 16);
  // -inf where there are fewer.  Then all of them.
  float bound = -INFINITY;
  for (int pass = 0; pass < 2; ++pass) {
    double best = -INFINITY;
    const int step = pass ? MERGE_NT : 64, end = pass ? n : lists;
    int i = pass;
#pragma unroll 1
    for (int e = pass ? tid : lane; e < end; e += step, ++i) {
      double s;
      int p, tok;
      float v;
      if (pass ? i < HELD : i == 0) {
        tok = i == 0 ? token[0] : token[1];
        v = i == 0 ? value[0] : value[1];
#pragma unroll
        for (int h = 2; h < HELD; ++h) {
          tok = i == h ? token[h] : tok;
          v = i == h ? value[h] : v;
        }
      } else {
        tok = token_of[e];
        v = value_of[e];
      }
      candidate(e, tok, v, s, p);
      best = fmax(best, s);
      if (pass && s >= (double)bound && s > -INFINITY) {
        const int i = atomicAdd(&count_s, 1);  // (any order: they are ranked)
        if (i < MERGE_CAP) {
          cs[i] = s;
          cp[i] = p;
        }
      }
    }
    if (pass) break;
    int least = quick_key((float)best);
    least -= (double)(float)best > best;
    int64_t key = quick_key(-INFINITY);
#pragma unroll 1
    for (int64_t bit = 1ll << 31; bit >= 1 << 16; bit >>= 1)
      if (key + bit <= INF_KEY &&
          __popcll(__builtin_amdgcn_ballot_w64(least >= (int)(key + bit))) >= A.width)
        key += bit;
    bound = key_value<32>((int)key);
  }
  // a beam that is done: itself
  if (tid < A.beams && own_s[tid] > -INFINITY) {
    const int i = atomicAdd(&count_s, 1);
    if (i < MERGE_CAP) {
      cs[i] = (double)own_s[tid];
      cp[i] = tid << 24 | A.pad_id;
    }
  }
  __syncthreads();
  const int64_t out = (int64_t)seq * A.width;
  auto put = [&](int rank, double s, int p) {
    st_agent(A.parents + out + rank, seq * A.beams + (p >> 24));
    st_agent(reinterpret_cast<uint64_t*>(A.tokens) + out + rank, (uint64_t)(p & 0xffffff));
    st_agent(A.out_scores + out + rank, (float)s);
  };
  int found = count_s;
  if (found <= MERGE_CAP) {
    // eight lanes a candidate
    for (int i0 = 0; i0 < found; i0 += MERGE_NT / 8) {
      const int i = i0 + tid / 8, at = min(i, found - 1);
      const double s = cs[at];
      const int p = cp[at];
      int rank = 0;
#pragma unroll 4
      for (int j = tid & 7; j < found; j += 8)
        rank += (int)(cs[j] > s) | ((int)(cs[j] == s) & (int)(cp[j] < p));
      rank += other<1>(rank);
      rank += other<2>(rank);
      rank += other<4>(rank);
      if ((tid & 7) == 0 && i < found && rank < A.width) put(rank, s, p);
    }
  } else {
    double last_s = INFINITY;
    int last_p = -1;
    for (found = 0; found < A.width; ++found) {
      double bs = -INFINITY;
      int bp = INT_MAX;
      for (int e = tid; e < n + A.beams; e += MERGE_NT) {
        double s = -INFINITY;
        int p = 0;
        if (e < n)
          candidate(e, token_of[e], value_of[e], s, p);
        else if (e - n < A.beams)
          s = (double)own_s[e - n], p = (e - n) << 24 | A.pad_id;
        if (s > -INFINITY && before(last_s, last_p, s, p) && before(s, p, bs, bp)) {
          bs = s;
          bp = p;
        }
      }
#pragma unroll
      for (int mask = 1; mask < 64; mask <<= 1) {
        const double s = __shfl_xor(bs, mask);
        const int p = __shfl_xor(bp, mask);
        if (before(s, p, bs, bp)) {
          bs = s;
          bp = p;
        }
      }
      __syncthreads();  // the last round's have been read
      if (lane == 0) {
        best_s[wave] = bs;
        place_s[wave] = bp;
      }
      __syncthreads();
      for (int w = 0; w < MERGE_WAVES; ++w)
        if (before(best_s[w], place_s[w], bs, bp)) {
          bs = best_s[w];
          bp = place_s[w];
        }
      if (!(bs > -INFINITY)) break;
      if (tid == 0) put(found, bs, bp);
      last_s = bs;
      last_p = bp;
    }
  }
  for (int i = found + tid; i < A.width; i += MERGE_NT) {
    st_agent(A.parents + out + i, -1);
    st_agent(reinterpret_cast<uint64_t*>(A.tokens) + out + i, (uint64_t)-1);
    st_agent(A.out_scores + out + i, -INFINITY);
  }
  stores_done();
}

// Parts of a row of `vocab` logits of `elem` bytes.
int num_parts(int64_t vocab, int elem) {
  const int64_t size = NT * LOADS * 16 / elem;
  return (int)((vocab + size - 1) / size);
}

}  // namespace
}  // namespace smx

#include "smx_abi_util.h"

extern "C" int64_t smx_beam_select_workspace(int32_t seqs, int32_t beams, int32_t width,
                                             int32_t vocab, int32_t element_size) {
  if (seqs < 1 || beams < 1 || width < 1 || vocab < 1 || (element_size != 2 && element_size != 4))
    return -1;
  const int64_t rows = (int64_t)seqs * beams;
  return rows * smx::num_parts(vocab, element_size) * (8 + 4 + 8 * (int64_t)width);
}

extern "C" int smx_beam_select(void* stream, const void* logits, int64_t stride,
                               int32_t element_size, const float* scores, const uint8_t* done,
                               void* workspace, int64_t workspace_bytes, int32_t* parents,
                               int64_t* tokens, float* out_scores, int32_t seqs, int32_t beams,
                               int32_t width, int32_t vocab, int32_t pad_id) {
  SMX_REQUIRE(logits && scores && workspace && parents && tokens && out_scores,
              "null pointer argument");
  SMX_REQUIRE(element_size == 2 || element_size == 4, "logits must be bf16 or fp32");
  SMX_REQUIRE(beams >= 1 && beams <= smx::MAX_BEAMS, "beams must be in [1, 64]");
  SMX_REQUIRE(width >= 1 && width <= smx::MAX_WIDTH, "width must be in [1, 64]");
  SMX_REQUIRE(vocab >= 1 && vocab <= (1 << 24), "vocab must be in [1, 2^24]");
  SMX_REQUIRE(seqs >= 1 && (int64_t)seqs * beams <= 65535, "seqs * beams must be in [1, 65535]");
  SMX_REQUIRE(stride >= vocab, "a row's stride must hold the vocabulary");
  SMX_REQUIRE(pad_id >= 0 && pad_id < vocab, "pad_id must be a token");
  SMX_REQUIRE((uintptr_t)logits % element_size == 0 && (uintptr_t)workspace % 16 == 0 &&
                  ((uintptr_t)scores | (uintptr_t)parents | (uintptr_t)out_scores) % 4 == 0 &&
                  (uintptr_t)tokens % 8 == 0,
              "misaligned pointer");
  SMX_REQUIRE(out_scores != scores || width == beams,
              "out_scores may be scores only where width is beams");
  SMX_REQUIRE(workspace_bytes >= smx_beam_select_workspace(seqs, beams, width, vocab, element_size),
              "workspace must hold smx_beam_select_workspace bytes");
  const int64_t rows = (int64_t)seqs * beams;
  const int parts = smx::num_parts(vocab, element_size);
  smx::BeamArgs a{};
  a.logits = logits;
  a.scores = scores;
  a.done = done;
  a.part_sum = (double*)workspace;
  a.part_max = (float*)(a.part_sum + rows * parts);
  a.cand_value = a.part_max + rows * parts;
  a.cand_token = (int32_t*)(a.cand_value + rows * parts * width);
  a.parents = parents;
  a.tokens = tokens;
  a.out_scores = out_scores;
  a.stride = stride;
  a.seqs = seqs;
  a.beams = beams;
  a.width = width;
  a.vocab = vocab;
  a.parts = parts;
  a.pad_id = pad_id;
  const auto kernel = element_size == 2 ? smx::beam_parts_kernel<uint16_t>
                                        : smx::beam_parts_kernel<float>;
  SMX_LAUNCH(kernel, dim3(parts, (unsigned)rows), dim3(smx::NT), 0, (hipStream_t)stream, a);
  const int rc = (int)hipGetLastError();
  if (rc) return rc;
  SMX_LAUNCH(smx::beam_merge_kernel, dim3(seqs), dim3(smx::MERGE_NT), 0, (hipStream_t)stream, a);
  return (int)hipGetLastError();
}
