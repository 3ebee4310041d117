// Beam search's selection over beams and vocabulary, for gfx950: of a sequence's beams b
// with scores c_b and logits x_b the `width` best continuations
//   score(b, v) = c_b + x_b[v] - log sum_u exp(x_b[u])
// in order, ties to the lowest b * vocab + v.
//
// One pass over the logits.  A beam's best are its largest logits, so a workgroup keeps
// the `width` largest of its part of a row and the part's maximum and sum of exponentials
// (beam_parts_kernel); a workgroup a sequence then takes the best of the parts'
// (beam_merge_kernel).  Beams are compared by their sums, so these are taken in 64 bits,
// with exponentials good to 4e-11: two beams' candidates whose scores differ by less
// than that might be taken in the wrong order, where fp32 sums would confuse those within
// 1e-6.  64-bit fma runs at the rate of the 32-bit one on this chip.
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
typedef double f64x2 __attribute__((ext_vector_type(2)));

constexpr int MAX_WIDTH = 64, MAX_BEAMS = 64;
constexpr int CAP = 128;  // candidates of a wave
constexpr int NT = 256, WAVES = NT / 64;

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

// exp(a) for a <= 0, relative error 4e-11 (a below -700: something below 1e-304):
// a = n ln 2 + r with |r| <= ln 2 / 2, a polynomial of degree 7 fitted to exp on that
// interval by least squares reweighted towards the largest relative error, and n added to
// the exponent's bits.
__device__ __forceinline__ double exp_le0(double a) {
  a = fmax(a, -700.0);
  const double magic = 0x1.8p52;  // its sum's low bits are the rounded quotient
  const double t = fma(a, 1.4426950408889634, magic);
  const double n = t - magic;
  const double r = fma(n, -0.6931471805599453, a);
  double p = 0x1.9eb71c629715ep-13;
  p = fma(p, r, 0x1.6da4bf9e8e8dfp-10);
  p = fma(p, r, 0x1.1112fa548f5cbp-7);
  p = fma(p, r, 0x1.5554685b28249p-5);
  p = fma(p, r, 0x1.55555343bd2bcp-3);
  p = fma(p, r, 0x1.00000059d83e1p-1);
  p = fma(p, r, 0x1.000000010b76ep+0);
  p = fma(p, r, 0x1.ffffffffabae7p-1);
  const uint64_t bits = __builtin_bit_cast(uint64_t, p);
  const uint32_t low = (uint32_t)__builtin_bit_cast(uint64_t, t);
  return __builtin_bit_cast(double, bits + ((uint64_t)(low << 20) << 32));
}

// Values in their order as unsigned integers (no NaN, no -0 among them).
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t u = __float_as_uint(f);
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
constexpr uint32_t LEAST = 0x00800000u;  // the order key of the least finite value

// A candidate of a part: bf16 values and the place in the part (below 65536) in 32 bits,
// fp32 ones in 64; a larger key is a larger value, or the same at a lower place.
template <typename L>
struct Keys;
template <>
struct Keys<uint16_t> {
  typedef uint32_t Key;
  static constexpr Key NONE = LEAST - 1;
  static __device__ __forceinline__ Key make(float f, uint32_t at) {
    return (order_key(f) & 0xffff0000u) | (0xffffu - at);
  }
  static __device__ __forceinline__ float value(Key k) {
    // (a negative value's low bits are the complement of its key's)
    return order_value(k & 0x80000000u ? k & 0xffff0000u : k | 0xffffu);
  }
  static __device__ __forceinline__ uint32_t place(Key k) { return 0xffffu - (k & 0xffffu); }
};
template <>
struct Keys<float> {
  typedef uint64_t Key;
  static constexpr Key NONE = (uint64_t)LEAST << 32 | 0;
  static __device__ __forceinline__ Key make(float f, uint32_t at) {
    return (uint64_t)order_key(f) << 32 | (0xffffffffu - at);
  }
  static __device__ __forceinline__ float value(Key k) { return order_value((uint32_t)(k >> 32)); }
  static __device__ __forceinline__ uint32_t place(Key k) { return 0xffffffffu - (uint32_t)k; }
};

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

// The least of the maxima of `groups` (a power of two up to 64) equal groups of a wave's
// neighbouring lanes: `groups` values or more are at least that.
template <typename K>
__device__ __forceinline__ K least_of_maxima(K v, int groups) {
  auto step = [&](auto mask) {
    constexpr int MASK = decltype(mask)::value;
    const K o = other<MASK>(v);
    const bool up = groups * MASK < 64;  // still within a group: the maximum
    v = (o > v) == up ? o : v;
  };
  step(std::integral_constant<int, 1>{});
  step(std::integral_constant<int, 2>{});
  step(std::integral_constant<int, 4>{});
  step(std::integral_constant<int, 8>{});
  step(std::integral_constant<int, 16>{});
  step(std::integral_constant<int, 32>{});
  return v;
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

// One part (NT * E logits) of one row.  Each wave reads its share once into registers,
// finds a bound that `width` of its values reach from its lanes' maxima, and collects
// those that reach it; the few collected of all waves are ranked by counting.
template <typename L, int E>
__global__ __launch_bounds__(NT) void beam_parts_kernel(BeamArgs A) {
  typedef Keys<L> Ks;
  typedef typename Ks::Key Key;
  constexpr int V = 16 / sizeof(L);  // logits of a load
  constexpr int LOADS = E / V;
  __shared__ Key list[WAVES * CAP];
  __shared__ int count_s[WAVES];
  __shared__ float max_s[WAVES];
  __shared__ double sum_s[WAVES];
  const int part = blockIdx.x, row = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // a beam that is done, or has no score, offers nothing from its logits
  if (A.done && A.done[row]) return;
  if (!(A.scores[row] > -INFINITY)) return;
  const int first = part * (NT * E), here = min(A.vocab - first, NT * E);
  const L* const src = reinterpret_cast<const L*>(A.logits) + (int64_t)row * A.stride + first;

  float x[E];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int at = (i * NT + tid) * V;
    u32x4 w;
    if (at + V <= here) {
      w = *reinterpret_cast<const u32x4_a2*>(src + at);
    } else {
      if constexpr (V == 8) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t lo = at + 2 * j < here ? (uint32_t)src[at + 2 * j] : 0xff80u;
          const uint32_t hi = at + 2 * j + 1 < here ? (uint32_t)src[at + 2 * j + 1] : 0xff80u;
          w[j] = lo | hi << 16;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          w[j] = at + j < here ? __float_as_uint(src[at + j]) : 0xff800000u;
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float f;
      if constexpr (V == 8)
        f = j & 1 ? bf16_hi(w[j / 2]) : bf16_lo(w[j / 2]);
      else
        f = __uint_as_float(w[j]);
      x[i * V + j] = fmaxf(f, -INFINITY) + 0.f;  // NaN as -inf, -0 as 0
    }
  }
  float top = -INFINITY;
#pragma unroll
  for (int e = 0; e < E; ++e) top = fmaxf(top, x[e]);
  top = wave_max(top);

  // ---- the sum of exponentials
  double sum = 0.0;
  if (top > -INFINITY) {
    double s0 = 0.0, s1 = 0.0;
    const double topd = (double)top;
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      s0 += exp_le0(x[e] == top ? 0.0 : (double)x[e] - topd);
      s1 += exp_le0(x[e + 1] == top ? 0.0 : (double)x[e + 1] - topd);
    }
    sum = wave_sum64(s0 + s1);
  }

  // ---- the largest
  Key key[E], best = 0;
#pragma unroll
  for (int i = 0; i < LOADS; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int e = i * V + j;
      key[e] = Ks::make(x[e], (uint32_t)((i * NT + tid) * V + j));
      best = max(best, key[e]);
    }
  int groups = 1;
  while (groups < A.width) groups <<= 1;
  Key bound = max(least_of_maxima(best, groups), (Key)(Ks::NONE + 1));
  auto reach = [&](Key b) {
    int c = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) c += __popcll(__builtin_amdgcn_ballot_w64(key[e] >= b));
    return c;
  };
  int n = reach(bound);
  if (n > CAP) {
    // (sorted or equal logits: the bound is loose)  The largest bound that `width` keys
    // reach, bit by bit from above; all keys are different, so it ends at `width`.
    Key b = 0;
    for (int bit = 8 * (int)sizeof(Key) - 1; bit >= 0; --bit) {
      const Key c = b | (Key)1 << bit;
      const int m = reach(c);
      if (m < A.width) continue;
      b = c;
      if (m <= CAP) break;
    }
    bound = max(b, (Key)(Ks::NONE + 1));
    n = reach(bound);
  }
  int at = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const bool in = key[e] >= bound;
    const uint64_t m = __builtin_amdgcn_ballot_w64(in);
    if (m) {
      if (in) list[wave * CAP + at + __popcll(m & ((1ull << lane) - 1))] = key[e];
      at += __popcll(m);
    }
  }
  if (lane == 0) {
    count_s[wave] = n;
    max_s[wave] = top;
    sum_s[wave] = sum;
  }
  __syncthreads();

  const int seq = row / A.beams, lists = A.beams * A.parts;
  const int64_t out = (int64_t)seq * A.width * lists + (row - seq * A.beams) * A.parts + part;
  int total = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) total += count_s[w];
  for (int i = tid; i < WAVES * CAP; i += NT) {
    if ((i & (CAP - 1)) >= count_s[i / CAP]) continue;
    const Key mine = list[i];
    int rank = 0;
    for (int w = 0; w < WAVES; ++w)
      for (int j = 0; j < count_s[w]; ++j) rank += list[w * CAP + j] > mine;
    if (rank < A.width) {
      st_agent(A.cand_value + out + (int64_t)rank * lists, Ks::value(mine));
      st_agent(A.cand_token + out + (int64_t)rank * lists, first + (int)Ks::place(mine));
    }
  }
  for (int i = total + tid; i < A.width; i += NT)
    st_agent(A.cand_token + out + (int64_t)i * lists, -1);
  if (tid == 0) {
    float m = max_s[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) m = fmaxf(m, max_s[w]);
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w)
      if (max_s[w] > -INFINITY)
        s += sum_s[w] * exp_le0(max_s[w] == m ? 0.0 : (double)max_s[w] - (double)m);
    st_agent(A.part_max + (int64_t)row * A.parts + part, m);
    st_agent(reinterpret_cast<uint64_t*>(A.part_sum) + (int64_t)row * A.parts + part,
             __builtin_bit_cast(uint64_t, s));
  }
  stores_done();
}

// A continuation in order: the larger score first, then the lower place.
struct Cand {
  double score;
  int64_t place;  // beam * vocab + token
};
__device__ __forceinline__ bool before(double s, int64_t p, double t, int64_t r) {
  return s > t || (s == t && p < r);
}

// One workgroup a sequence.  A beam's parts are joined to its log sum; the candidates that
// reach a bound found as above are collected and ranked.  Where too many do (equal
// scores), they are found one after another instead.
constexpr int MERGE_CAP = 1024;

__global__ __launch_bounds__(NT) void beam_merge_kernel(BeamArgs A) {
  __shared__ float top_s[MAX_BEAMS];
  __shared__ double log_s[MAX_BEAMS];  // the log of the sum relative to the maximum
  __shared__ float score_s[MAX_BEAMS];
  __shared__ double cs[MERGE_CAP];
  __shared__ int64_t cp[MERGE_CAP];
  __shared__ double bound_s[WAVES];
  __shared__ int64_t best_s[WAVES];
  __shared__ int count_s;
  const int seq = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lists = A.beams * A.parts;
  // score_s: NaN marks a beam that offers nothing, log_s NaN one that is done
  for (int b = wave; b < A.beams; b += WAVES) {
    const int row = seq * A.beams + b;
    const float c = A.scores[row];
    const bool dead = !(c > -INFINITY), done = A.done && A.done[row];
    float m = -INFINITY;
    double s = 0.0;
    if (!dead && !done) {
      for (int p = lane; p < A.parts; p += 64) m = fmaxf(m, A.part_max[(int64_t)row * A.parts + p]);
      m = wave_max(m);
      for (int p = lane; p < A.parts; p += 64) {
        const float pm = A.part_max[(int64_t)row * A.parts + p];
        if (pm > -INFINITY)
          s += A.part_sum[(int64_t)row * A.parts + p] *
               exp_le0(pm == m ? 0.0 : (double)pm - (double)m);
      }
      s = wave_sum64(s);
    }
    if (lane == 0) {
      top_s[b] = m;
      log_s[b] = done ? __builtin_nan("") : log(s);
      score_s[b] = dead ? __builtin_nanf("") : c;
    }
  }
  if (tid == 0) count_s = 0;
  __syncthreads();

  // Candidate e of `n`: rank, beam, part; the done beams' own ones come last.
  const int n = A.width * lists, all = n + A.beams;
  auto candidate = [&](int e, double& s, int64_t& place) {
    s = -INFINITY;
    if (e >= n) {
      const int b = e - n;
      if (log_s[b] != log_s[b] && score_s[b] == score_s[b]) {
        s = (double)score_s[b];
        place = (int64_t)b * A.vocab + A.pad_id;
      }
      return;
    }
    const int list = e % lists, b = list / A.parts;
    if (log_s[b] != log_s[b] || score_s[b] != score_s[b]) return;
    const int64_t at = (int64_t)seq * A.width * lists + e;
    const int token = A.cand_token[at];
    if (token < 0) return;
    const float v = A.cand_value[at];
    s = (double)score_s[b] + ((v == top_s[b] ? 0.0 : (double)v - (double)top_s[b]) - log_s[b]);
    place = (int64_t)b * A.vocab + token;
  };
  double best = -INFINITY;
  for (int e = tid; e < all; e += NT) {
    double s;
    int64_t p;
    candidate(e, s, p);
    best = fmax(best, s);
  }
  // (a group of lanes sees every rank of its lists)
  int groups = WAVES;
  while (groups < A.width) groups <<= 1;
  const double bound_w = least_of_maxima(best, groups / WAVES);
  if (lane == 0) bound_s[wave] = bound_w;
  __syncthreads();
  double bound = bound_s[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) bound = fmin(bound, bound_s[w]);
  for (int e = tid; e < all; e += NT) {
    double s;
    int64_t p;
    candidate(e, s, p);
    if (s >= bound && s > -INFINITY) {
      const int i = atomicAdd(&count_s, 1);  // (any order: they are ranked)
      if (i < MERGE_CAP) {
        cs[i] = s;
        cp[i] = p;
      }
    }
  }
  __syncthreads();
  const int64_t out = (int64_t)seq * A.width;
  auto put = [&](int rank, double s, int64_t p) {
    const int b = (int)(p / A.vocab);
    st_agent(A.parents + out + rank, seq * A.beams + b);
    st_agent(reinterpret_cast<uint64_t*>(A.tokens) + out + rank,
             (uint64_t)(p - (int64_t)b * A.vocab));
    st_agent(A.out_scores + out + rank, (float)s);
  };
  int found = count_s;
  if (found <= MERGE_CAP) {
    for (int i = tid; i < found; i += NT) {
      const double s = cs[i];
      const int64_t p = cp[i];
      int rank = 0;
      for (int j = 0; j < found; ++j) rank += before(cs[j], cp[j], s, p);
      if (rank < A.width) put(rank, s, p);
    }
  } else {
    double last_s = INFINITY;
    int64_t last_p = -1;
    for (found = 0; found < A.width; ++found) {
      double bs = -INFINITY;
      int64_t bp = INT64_MAX;
      for (int e = tid; e < all; e += NT) {
        double s;
        int64_t p;
        candidate(e, s, p);
        if (s > -INFINITY && before(last_s, last_p, s, p) && before(s, p, bs, bp)) {
          bs = s;
          bp = p;
        }
      }
#pragma unroll
      for (int mask = 1; mask < 64; mask <<= 1) {
        const double s = __shfl_xor(bs, mask);
        const int64_t p = __shfl_xor(bp, mask);
        if (before(s, p, bs, bp)) {
          bs = s;
          bp = p;
        }
      }
      __syncthreads();  // the last round's have been read
      if (lane == 0) {
        bound_s[wave] = bs;
        best_s[wave] = bp;
      }
      __syncthreads();
      for (int w = 0; w < WAVES; ++w)
        if (before(bound_s[w], best_s[w], bs, bp)) {
          bs = bound_s[w];
          bp = best_s[w];
        }
      if (!(bs > -INFINITY)) break;
      if (tid == 0) put(found, bs, bp);
      last_s = bs;
      last_p = bp;
    }
  }
  for (int i = found + tid; i < A.width; i += NT) {
    st_agent(A.parents + out + i, -1);
    st_agent(reinterpret_cast<uint64_t*>(A.tokens) + out + i, (uint64_t)-1);
    st_agent(A.out_scores + out + i, -INFINITY);
  }
  stores_done();
}

// Logits of a part: many rows take long ones, few rows short ones that fill the chip.
int part_size(int64_t rows, int64_t vocab, int elem) {
  const int large = elem == 2 ? 16384 : 8192, small = large / 4;
  return rows * ((vocab + large - 1) / large) >= 512 ? large : small;
}

}  // namespace
}  // namespace smx

#include "smx_abi_util.h"

extern "C" int64_t smx_beam_select_workspace(int32_t seqs, int32_t beams, int32_t width,
                                             int32_t vocab, int32_t element_size) {
  if (seqs < 1 || beams < 1 || width < 1 || vocab < 1 || (element_size != 2 && element_size != 4))
    return -1;
  const int64_t rows = (int64_t)seqs * beams;
  const int64_t size = smx::part_size(rows, vocab, element_size);
  const int64_t parts = (vocab + size - 1) / size;
  return rows * parts * (8 + 4 + 8 * (int64_t)width);
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
  const int size = smx::part_size(rows, vocab, element_size);
  const int parts = (vocab + size - 1) / size;
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
  const auto kernel = element_size == 2
      ? (size == 16384 ? smx::beam_parts_kernel<uint16_t, 64> : smx::beam_parts_kernel<uint16_t, 16>)
      : (size == 8192 ? smx::beam_parts_kernel<float, 32> : smx::beam_parts_kernel<float, 8>);
  SMX_LAUNCH(kernel, dim3(parts, (unsigned)rows), dim3(smx::NT), 0, (hipStream_t)stream, a);
  const int rc = (int)hipGetLastError();
  if (rc) return rc;
  SMX_LAUNCH(smx::beam_merge_kernel, dim3(seqs), dim3(smx::NT), 0, (hipStream_t)stream, a);
  return (int)hipGetLastError();
}
