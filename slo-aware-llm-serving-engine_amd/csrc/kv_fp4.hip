// KV write into a 4-bit pool, and the read back of cached tokens (gfx950).
#include "capi_internal.h"
#include "fp4.h"

namespace slo {

// Both kernels: a workgroup takes TOK tokens, a lane 8 channels of K or V, and
// lanes go by channel, token, then K or V and head, so that tokens that lie
// side by side in a page of a 4-bit pool are read and written as one piece.
// All of a lane's loads are issued before the first is used.
struct Unit {
  int token, head, j;
  bool is_v, live;
};

template <int TOK>
__device__ __forceinline__ Unit unit_of(int u, int hkv, int shift, int tokens) {
  Unit x;
  x.j = u & ((1 << shift) - 1);
  u >>= shift;
  x.token = blockIdx.x * TOK + u % TOK;
  u /= TOK;
  x.is_v = u >= hkv;
  x.head = x.is_v ? u - hkv : u;
  x.live = u < 2 * hkv && x.token < tokens;
  return x;
}

// Slot-mapped write into a 4-bit pool (format and scale rule: fp4.h): 16 bytes
// a lane in, the group's largest magnitude over 4 lanes by DPP, 4 code bytes
// out; the first of the 4 lanes writes the scale byte.  Bound by the round trip
// to memory at a decode step's size (24 tokens of 8 heads 2.9 us) and by HBM
// above a few thousand tokens (4,096 tokens, 21 MB, 7.4 us).
template <int TOK, int DEPTH>
__global__ void __launch_bounds__(256)
store_fp4_kernel(const uint16_t* __restrict__ key, int64_t key_stride, const uint16_t* __restrict__ value,
                 int64_t value_stride, const int32_t* __restrict__ slot_mapping, int tokens, int hkv, int shift,
                 uint8_t* __restrict__ k_cache, uint8_t* __restrict__ v_cache, uint8_t* __restrict__ k_scale,
                 uint8_t* __restrict__ v_scale, int64_t num_slots, int block_size, int floor_code) {
  const int units = (2 * hkv * TOK) << shift;
  for (int u0 = 0; u0 < units; u0 += 256 * DEPTH) {
    u32x4 x[DEPTH];
    int slot[DEPTH];
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const Unit t = unit_of<TOK>(u0 + 256 * d + threadIdx.x, hkv, shift, tokens);
      slot[d] = -1;
      x[d] = u32x4{0, 0, 0, 0};
      if (!t.live) continue;
      x[d] = *reinterpret_cast<const u32x4*>((t.is_v ? value + t.token * value_stride : key + t.token * key_stride) +
                                             (((t.head << shift) + t.j) << 3));
      slot[d] = slot_mapping[t.token];
    }
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const Unit t = unit_of<TOK>(u0 + 256 * d + threadIdx.x, hkv, shift, tokens);
      int code;
      const uint32_t w = e2m1_encode8(x[d], floor_code, code);
      if (slot[d] < 0 || slot[d] >= num_slots) continue;
      const int page = slot[d] / block_size, off = slot[d] - page * block_size;
      const int64_t row = ((int64_t)page * hkv + t.head) * block_size + off;
      reinterpret_cast<uint32_t*>(t.is_v ? v_cache : k_cache)[(row << shift) + t.j] = w;
      if ((t.j & 3) == 0) (t.is_v ? v_scale : k_scale)[(row << (shift - 2)) + (t.j >> 2)] = (uint8_t)code;
    }
  }
}

// Cached tokens as bf16 rows.  E4M3FN values are code * scale in fp32, rounded
// once; 4-bit values are exact.  A slot outside the pool gives zeros.
template <int KV, int TOK, int DEPTH>
__global__ void __launch_bounds__(256)
load_kv_kernel(const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache,
               const void* __restrict__ k_scale, const void* __restrict__ v_scale,
               const int32_t* __restrict__ slot_mapping, int tokens, int hkv, int shift, int64_t num_slots, int block_size,
               uint16_t* __restrict__ k_out, uint16_t* __restrict__ v_out) {
  const int units = (2 * hkv * TOK) << shift;
  for (int u0 = 0; u0 < units; u0 += 256 * DEPTH) {
    u32x4 x[DEPTH];
    float scale[DEPTH];
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const Unit t = unit_of<TOK>(u0 + 256 * d + threadIdx.x, hkv, shift, tokens);
      x[d] = u32x4{0, 0, 0, 0};
      scale[d] = 1.0f;
      if (!t.live) continue;
      const int slot = slot_mapping[t.token];
      if (slot < 0 || slot >= num_slots) continue;
      const uint8_t* cache = t.is_v ? v_cache : k_cache;
      const void* scales = t.is_v ? v_scale : k_scale;
      if (KV == KV_FP4_E2M1) {
        const int page = slot / block_size, off = slot - page * block_size;
        const int64_t row = ((int64_t)page * hkv + t.head) * block_size + off;
        x[d][0] = reinterpret_cast<const uint32_t*>(cache)[(row << shift) + t.j];
        scale[d] = e8m0(static_cast<const uint8_t*>(scales)[(row << (shift - 2)) + (t.j >> 2)]);
      } else {
        const int64_t row = (int64_t)slot * hkv + t.head;
        if (KV == KV_BF16) {
          x[d] = reinterpret_cast<const u32x4*>(cache)[(row << shift) + t.j];
        } else {
          const u32x2 w = reinterpret_cast<const u32x2*>(cache)[(row << shift) + t.j];
          x[d][0] = w.x;
          x[d][1] = w.y;
          scale[d] = static_cast<const float*>(scales)[row];
        }
      }
    }
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const Unit t = unit_of<TOK>(u0 + 256 * d + threadIdx.x, hkv, shift, tokens);
      if (!t.live) continue;
      u32x4 o = x[d];
      if (KV == KV_FP4_E2M1) {
        o = e2m1_decode8(x[d][0], scale[d]);
      } else if (KV == KV_FP8_E4M3FN) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const u32x2 b = fp8x4_to_bf16x4(x[d][i]);
#pragma unroll
          for (int h = 0; h < 2; ++h)
            o[2 * i + h] = pack_bf16x2(__uint_as_float(b[h] << 16) * scale[d], __uint_as_float(b[h] & 0xffff0000u) * scale[d]);
        }
      }
      u32x4* to = reinterpret_cast<u32x4*>(t.is_v ? v_out : k_out) + ((((int64_t)t.token * hkv + t.head) << shift) + t.j);
      if constexpr (TOK > 1)
        __builtin_nontemporal_store(o, to);
      else
        *to = o;
    }
  }
}

// Four tokens a workgroup, and four loads a lane in flight, from here on: the
// read back of 262,144 tokens of 8 heads takes 347 us so and 376 us with one
// token a workgroup, that of 4,096 tokens 8.7 and 7.0 us.  What such a read back
// writes is larger than the caches, so it is stored past them: 338 us, and what
// the next kernel finds there is not displaced (a move of 16 rows in the pool
// that was read back before takes 160 us instead of 184).
constexpr int kManyTokens = 16384;

}  // namespace slo

using namespace slo;

static inline bool unaligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; }

extern "C" int slo_store_kvcache_fp4(const void* key, int64_t key_row_stride, const void* value, int64_t value_row_stride,
                                     const int32_t* slot_mapping, int32_t num_tokens, int32_t num_kv_heads,
                                     int32_t head_dim, void* k_cache, void* v_cache, void* k_scale, void* v_scale,
                                     int32_t num_blocks, int32_t block_size, float scale_floor, slo_stream_t stream) {
  if (num_tokens < 0 || num_kv_heads <= 0) return fail(SLO_ERR_INVALID, "store_kvcache_fp4: bad token/head count");
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(SLO_ERR_UNSUPPORTED, "store_kvcache_fp4: head_dim must be 64, 128 or 256");
  uint32_t bits;
  __builtin_memcpy(&bits, &scale_floor, 4);
  const int floor_code = (int)(bits >> 23);  // the sign is bit 8 of this
  if ((bits & 0x7fffffu) || floor_code < 27 || floor_code > kFp4MaxCode)
    return fail(SLO_ERR_INVALID, "store_kvcache_fp4: scale_floor must be a power of two from 2^-100 to 2^125");
  if (num_tokens == 0) return SLO_OK;
  if (!key || !value || !slot_mapping || !k_cache || !v_cache || !k_scale || !v_scale)
    return fail(SLO_ERR_INVALID, "store_kvcache_fp4: null pointer");
  if (num_blocks <= 0 || block_size <= 0) return fail(SLO_ERR_INVALID, "store_kvcache_fp4: no KV pool");
  if ((key_row_stride % 8) || (value_row_stride % 8) || unaligned16(key) || unaligned16(value) || unaligned16(k_cache) ||
      unaligned16(v_cache))
    return fail(SLO_ERR_INVALID, "store_kvcache_fp4: rows must be 16-byte aligned (stride multiple of 8 elements)");
  const int64_t per = 2 * (int64_t)num_kv_heads * (head_dim / 8);
  if (per > 65536) return fail(SLO_ERR_UNSUPPORTED, "store_kvcache_fp4: too many heads");
  const int shift = head_dim == 64 ? 3 : head_dim == 128 ? 4 : 5;
  const bool many = num_tokens >= kManyTokens;
  hipLaunchKernelGGL((many ? store_fp4_kernel<4, 4> : store_fp4_kernel<1, 1>), dim3(many ? (num_tokens + 3) / 4 : num_tokens),
                     dim3(256), 0, static_cast<hipStream_t>(stream), static_cast<const uint16_t*>(key), key_row_stride,
                     static_cast<const uint16_t*>(value), value_row_stride, slot_mapping, num_tokens, num_kv_heads, shift,
                     static_cast<uint8_t*>(k_cache), static_cast<uint8_t*>(v_cache), static_cast<uint8_t*>(k_scale),
                     static_cast<uint8_t*>(v_scale), (int64_t)num_blocks * block_size, block_size, floor_code);
  return check_launch("store_kvcache_fp4");
}

extern "C" int slo_load_kvcache(const void* k_cache, const void* v_cache, const void* k_scale, const void* v_scale,
                                int32_t kv_dtype, int32_t num_blocks, int32_t block_size, const int32_t* slot_mapping,
                                int32_t num_tokens, int32_t num_kv_heads, int32_t head_dim, void* k_out, void* v_out,
                                slo_stream_t stream) {
  if (num_tokens < 0 || num_kv_heads <= 0) return fail(SLO_ERR_INVALID, "load_kvcache: bad token/head count");
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(SLO_ERR_UNSUPPORTED, "load_kvcache: head_dim must be 64, 128 or 256");
  if (kv_dtype < KV_BF16 || kv_dtype > KV_FP4_E2M1) return fail(SLO_ERR_INVALID, "load_kvcache: bad kv_dtype");
  if (num_tokens == 0) return SLO_OK;
  if (!k_cache || !v_cache || !slot_mapping || !k_out || !v_out) return fail(SLO_ERR_INVALID, "load_kvcache: null pointer");
  if (kv_dtype != KV_BF16 && (!k_scale || !v_scale))
    return fail(SLO_ERR_INVALID, "load_kvcache: a quantised pool needs its scales");
  if (num_blocks <= 0 || block_size <= 0) return fail(SLO_ERR_INVALID, "load_kvcache: no KV pool");
  if (unaligned16(k_cache) || unaligned16(v_cache) || unaligned16(k_out) || unaligned16(v_out))
    return fail(SLO_ERR_INVALID, "load_kvcache: pools and outputs must be 16-byte aligned");
  const int64_t per = 2 * (int64_t)num_kv_heads * (head_dim / 8);
  if (per > 65536) return fail(SLO_ERR_UNSUPPORTED, "load_kvcache: too many heads");
  const int shift = head_dim == 64 ? 3 : head_dim == 128 ? 4 : 5;
  const bool many = num_tokens >= kManyTokens;
  auto* kernel = kv_dtype == KV_BF16         ? (many ? load_kv_kernel<KV_BF16, 4, 4> : load_kv_kernel<KV_BF16, 1, 1>)
                 : kv_dtype == KV_FP8_E4M3FN ? (many ? load_kv_kernel<KV_FP8_E4M3FN, 4, 4> : load_kv_kernel<KV_FP8_E4M3FN, 1, 1>)
                                             : (many ? load_kv_kernel<KV_FP4_E2M1, 4, 4> : load_kv_kernel<KV_FP4_E2M1, 1, 1>);
  hipLaunchKernelGGL(kernel, dim3(many ? (num_tokens + 3) / 4 : num_tokens), dim3(256), 0, static_cast<hipStream_t>(stream),
                     static_cast<const uint8_t*>(k_cache), static_cast<const uint8_t*>(v_cache), k_scale, v_scale, slot_mapping,
                     num_tokens, num_kv_heads, shift, (int64_t)num_blocks * block_size, block_size,
                     static_cast<uint16_t*>(k_out), static_cast<uint16_t*>(v_out));
  return check_launch("load_kvcache");
}
