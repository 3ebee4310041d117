// Writes to and reads from the paged KV cache held in 4 bits (q4_cache.h), for gfx950:
// a step's keys and values, the same behind q/k RMSNorm and RoPE, and tokens' values.
// Bound by memory: 2 bytes a value in, 4.5 bits out (read: 4.5 bits in, 4 bytes out).  8000
// tokens of 8 heads of 128: written in 10.8 us (3.9 TB/s; 12.0 with one load a lane), read in
// 14.5 (5.2 TB/s; 18.1 with K or V of a lane); 16 tokens 2.8 and 3.2 (2.7).
#include <math.h>

#include "q4_cache.h"
#include "qknorm_rope.h"
#include "smx_launch.h"

namespace smx {
namespace {

// HD / 8 lanes a (token, head) pair, its K and its V: two loads a lane on their way.  Lanes
// past the end work on the last pair (a block's four lanes trade values) and store nothing.
template <int HD>
__global__ __launch_bounds__(256) void q4_write_kernel(const uint16_t* __restrict__ key,
                                                       const uint16_t* __restrict__ value,
                                                       const int64_t* __restrict__ slots,
                                                       Q4Cache c, int64_t pairs, int64_t key_stride,
                                                       int64_t value_stride, int64_t cache_slots) {
  constexpr int LANES = HD / 8, PER = 256 / LANES;
  const int j = threadIdx.x % LANES;
  const int64_t raw = (int64_t)blockIdx.x * PER + threadIdx.x / LANES;
  const int64_t pair = min(raw, pairs - 1);
  const int64_t t = (uint32_t)pair / (uint32_t)c.n_kv;
  const int head = (int)(pair - t * c.n_kv);
  const int64_t slot = slots[t];
  const u32x4 k = *reinterpret_cast<const u32x4*>(key + t * key_stride + head * HD + 8 * j);
  const u32x4 v = *reinterpret_cast<const u32x4*>(value + t * value_stride + head * HD + 8 * j);
  const bool store = raw < pairs && slot >= 0 && slot < cache_slots;
#pragma unroll 1
  for (int plane = 0; plane < 2; ++plane)  // (one time the code: it is not in the cache)
    q4_store_chunk<HD>(c, plane, store ? slot : 0, head, j, plane ? v : k, store);
  stores_done();
}

// 16 lanes a (token, head) pair of 128 channels, as qknorm_rope_kv_vec_kernel.
__global__ __launch_bounds__(256) void q4_qknorm_rope_write_kernel(
    const uint16_t* __restrict__ qkv, const uint16_t* __restrict__ q_gamma,
    const uint16_t* __restrict__ k_gamma, const uint16_t* __restrict__ cos_sin,
    const int64_t* __restrict__ positions, const int64_t* __restrict__ slots,
    uint16_t* __restrict__ q_out, Q4Cache c, uint32_t items, int n_q, int64_t cache_slots,
    int max_position, float eps) {
  const int j = threadIdx.x & 15;
  const uint32_t raw = blockIdx.x * 16u + (threadIdx.x >> 4);
  const uint32_t item = min(raw, items - 1);
  const uint32_t nh = (uint32_t)(n_q + 2 * c.n_kv);
  const uint32_t t = item / nh;
  const int h = (int)(item - t * nh);
  const int64_t slot = slots[t];
  const u32x4 val = qknorm_rope_chunk(qkv + (int64_t)item * 128, h < n_q ? q_gamma : k_gamma,
                                      cos_sin, positions[t], h < n_q + c.n_kv, j, max_position,
                                      eps);
  // (a wave's pairs can be of both kinds: every lane takes part in the codes' search)
  const bool kv = raw < items && h >= n_q && slot >= 0 && slot < cache_slots;
  const int plane = h >= n_q + c.n_kv;
  q4_store_chunk<128>(c, plane, kv ? slot : 0, kv ? h - n_q - plane * c.n_kv : 0, j, val, kv);
  if (raw < items && h < n_q)
    st_agent_b128(q_out + ((int64_t)t * n_q + h) * 128 + 8 * j, val);
  stores_done();
}

// A lane 4 channels of K and of V (a 16-byte store each); 0 for a slot outside the cache.
template <int HD>
__global__ __launch_bounds__(256) void q4_read_kernel(Q4Cache c, const int64_t* __restrict__ slots,
                                                      float* __restrict__ key,
                                                      float* __restrict__ value, int64_t pairs,
                                                      int64_t cache_slots) {
  constexpr int LANES = HD / 4, PER = 256 / LANES;
  const int j = threadIdx.x % LANES;
  const int64_t pair = (int64_t)blockIdx.x * PER + threadIdx.x / LANES;
  if (pair < pairs) {
    const int64_t t = (uint32_t)pair / (uint32_t)c.n_kv;
    const int head = (int)(pair - t * c.n_kv);
    const int64_t slot = slots[t];
    const bool in = slot >= 0 && slot < cache_slots;
    const int b = j / 8, g = (j & 7) / 2, half = j & 1;  // channels 4 j .. of block b
    uint32_t w[2] = {0u, 0u};
    float d[2] = {0.f, 0.f};
#pragma unroll
    for (int plane = 0; plane < 2; ++plane)
      if (in) {
        const int64_t row = q4_row(c, plane, slot, head);
        const int dword = plane == 0 ? g * (HD / 32) + b : j / 2;
        w[plane] = reinterpret_cast<const uint32_t*>(c.codes + row * (HD / 2))[dword];
        d[plane] = f16_bits_to_f32(c.scales[row * (HD / 32) + b]);
      }
#pragma unroll
    for (int plane = 0; plane < 2; ++plane) {
      u32x4 out = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int ch = 4 * half + i;
        const int bit = plane == 0 ? 4 * (ch / 2) + 16 * (ch & 1) : 4 * ch;
        if (in) out[i] = __float_as_uint(d[plane] * (float)((int)((w[plane] >> bit) & 15u) - 8));
      }
      st_agent_b128((plane ? value : key) + pair * HD + 4 * j, out);
    }
  }
  stores_done();
}

}  // namespace
}  // namespace smx

#include "smx_abi_util.h"

#define SMX_Q4_CACHE_CHECKS()                                                                    \
  SMX_REQUIRE(codes && scales && slot_mapping, "null pointer argument");                         \
  SMX_REQUIRE(head_dim == 64 || head_dim == 128, "head_dim must be 64 or 128");                  \
  SMX_REQUIRE(n_kv >= 1 && n_kv <= 65535, "n_kv must be in [1, 65535]");                         \
  SMX_REQUIRE(num_tokens >= 1 && (int64_t)num_tokens * n_kv < (1ll << 26),                       \
              "num_tokens * n_kv must be in [1, 2^26)");                                         \
  SMX_REQUIRE(num_blocks >= 1, "num_blocks must be >= 1");                                       \
  SMX_REQUIRE(block_size >= 32 && block_size <= 4096 && (block_size & (block_size - 1)) == 0,    \
              "block_size must be a power of two in [32, 4096]");                                \
  SMX_REQUIRE((uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 16 == 0,                         \
              "codes and scales must be 16-byte aligned");                                       \
  SMX_REQUIRE((uintptr_t)slot_mapping % 8 == 0, "int64 arrays must be 8-byte aligned")

namespace {
smx::Q4Cache q4_cache(const void* codes, const void* scales, int num_blocks, int block_size,
                      int n_kv) {
  smx::Q4Cache c{(uint8_t*)const_cast<void*>(codes), (uint16_t*)const_cast<void*>(scales),
                 num_blocks, 0, n_kv};
  while ((1 << c.bs_log2) < block_size) ++c.bs_log2;
  return c;
}
}  // namespace

extern "C" int smx_q4_reshape_and_cache(void* stream, const void* key, int64_t key_stride,
                                        const void* value, int64_t value_stride, void* codes,
                                        void* scales, const int64_t* slot_mapping,
                                        int32_t num_tokens, int32_t n_kv, int32_t head_dim,
                                        int32_t num_blocks, int32_t block_size) {
  SMX_REQUIRE(key && value, "null pointer argument");
  SMX_Q4_CACHE_CHECKS();
  SMX_REQUIRE((uintptr_t)key % 16 == 0 && (uintptr_t)value % 16 == 0 && key_stride % 8 == 0 &&
                  value_stride % 8 == 0,
              "key and value tokens must be 16-byte aligned");
  SMX_REQUIRE(key_stride >= (int64_t)n_kv * head_dim && value_stride >= (int64_t)n_kv * head_dim,
              "a token's stride must hold its heads");
  const smx::Q4Cache c = q4_cache(codes, scales, num_blocks, block_size, n_kv);
  const int64_t pairs = (int64_t)num_tokens * n_kv, per = 256 * 8 / head_dim;
  const dim3 grid((unsigned)((pairs + per - 1) / per));
  SMX_LAUNCH((head_dim == 128 ? smx::q4_write_kernel<128> : smx::q4_write_kernel<64>), grid,
             dim3(256), 0, (hipStream_t)stream, (const uint16_t*)key, (const uint16_t*)value,
             slot_mapping, c, pairs, key_stride, value_stride, (int64_t)num_blocks * block_size);
  return (int)hipGetLastError();
}

extern "C" int smx_q4_qknorm_rope_kv_write(void* stream, const void* qkv, const void* q_gamma,
                                           const void* k_gamma, const void* cos_sin,
                                           const int64_t* positions, const int64_t* slot_mapping,
                                           void* q_out, void* codes, void* scales,
                                           int32_t num_tokens, int32_t n_q, int32_t n_kv,
                                           int32_t head_dim, int32_t num_blocks,
                                           int32_t block_size, int32_t max_position, float eps) {
  SMX_REQUIRE(qkv && q_gamma && k_gamma && cos_sin && positions && q_out,
              "null pointer argument");
  SMX_Q4_CACHE_CHECKS();
  SMX_REQUIRE(head_dim == 128, "head_dim must be 128");
  SMX_REQUIRE(num_tokens <= 65535, "num_tokens must be in [1, 65535]");
  SMX_REQUIRE(n_q >= 1 && n_q + 2 * n_kv <= 65535, "bad head counts");
  SMX_REQUIRE(max_position >= 1, "max_position must be >= 1");
  SMX_REQUIRE(eps >= 0.f && isfinite(eps), "eps must be finite and >= 0");
  SMX_REQUIRE((uintptr_t)positions % 8 == 0, "int64 arrays must be 8-byte aligned");
  SMX_REQUIRE(((uintptr_t)qkv | (uintptr_t)q_gamma | (uintptr_t)k_gamma | (uintptr_t)cos_sin |
               (uintptr_t)q_out) % 16 == 0,
              "bf16 tensors must be 16-byte aligned");
  const int64_t items = (int64_t)num_tokens * (n_q + 2 * n_kv);
  SMX_REQUIRE(items < (1ll << 28), "num_tokens * (n_q + 2 n_kv) must be below 2^28");
  const smx::Q4Cache c = q4_cache(codes, scales, num_blocks, block_size, n_kv);
  SMX_LAUNCH(smx::q4_qknorm_rope_write_kernel, dim3((unsigned)((items + 15) / 16)), dim3(256), 0,
             (hipStream_t)stream, (const uint16_t*)qkv, (const uint16_t*)q_gamma,
             (const uint16_t*)k_gamma, (const uint16_t*)cos_sin, positions, slot_mapping,
             (uint16_t*)q_out, c, (uint32_t)items, n_q, (int64_t)num_blocks * block_size,
             max_position, eps);
  return (int)hipGetLastError();
}

extern "C" int smx_q4_kv_read(void* stream, const void* codes, const void* scales,
                              const int64_t* slot_mapping, void* key, void* value,
                              int32_t num_tokens, int32_t n_kv, int32_t head_dim,
                              int32_t num_blocks, int32_t block_size) {
  SMX_REQUIRE(key && value, "null pointer argument");
  SMX_Q4_CACHE_CHECKS();
  SMX_REQUIRE((uintptr_t)key % 16 == 0 && (uintptr_t)value % 16 == 0,
              "key and value must be 16-byte aligned");
  const smx::Q4Cache c = q4_cache(codes, scales, num_blocks, block_size, n_kv);
  const int64_t pairs = (int64_t)num_tokens * n_kv, per = 256 * 4 / head_dim;
  const dim3 grid((unsigned)((pairs + per - 1) / per));
  SMX_LAUNCH((head_dim == 128 ? smx::q4_read_kernel<128> : smx::q4_read_kernel<64>), grid,
             dim3(256), 0, (hipStream_t)stream, c, slot_mapping, (float*)key, (float*)value, pairs,
             (int64_t)num_blocks * block_size);
  return (int)hipGetLastError();
}
