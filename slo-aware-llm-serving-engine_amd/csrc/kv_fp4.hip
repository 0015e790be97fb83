// KV write into a 4-bit pool, and the read back of cached tokens (gfx950).
#include "capi_internal.h"
#include "fp4.h"

namespace slo {

// Slot-mapped write into a 4-bit pool (format and scale rule: fp4.h).  One
// workgroup per token, one lane per 8 channels of K or V: a 16-byte load, the
// group's largest magnitude over 4 lanes by DPP, and 4 code bytes; the first
// of the 4 lanes writes the scale byte.  Bound by the round trip to memory at
// a decode step's size and by HBM above a few thousand tokens.
__global__ void __launch_bounds__(256)
store_fp4_kernel(const uint16_t* __restrict__ key, int64_t key_stride, const uint16_t* __restrict__ value,
                 int64_t value_stride, const int32_t* __restrict__ slot_mapping, int hkv, int head_dim,
                 uint8_t* __restrict__ k_cache, uint8_t* __restrict__ v_cache, uint8_t* __restrict__ k_scale,
                 uint8_t* __restrict__ v_scale, int64_t num_slots, int block_size, int floor_code) {
  const int64_t tok = blockIdx.x;
  const int cph = head_dim >> 3, per = hkv * cph;
  for (int c = threadIdx.x; c < 2 * per; c += blockDim.x) {
    const bool is_v = c >= per;
    const int cc = is_v ? c - per : c;
    const u32x4 x = *reinterpret_cast<const u32x4*>((is_v ? value + tok * value_stride : key + tok * key_stride) + cc * 8);
    const int slot = slot_mapping[tok];
    if (slot < 0 || slot >= num_slots) return;
    const int page = slot / block_size, off = slot - page * block_size;
    const int head = cc / cph, j = cc - head * cph;
    int code;
    const uint32_t w = e2m1_encode8(x, floor_code, code);
    const int64_t row = ((int64_t)page * hkv + head) * block_size + off;
    reinterpret_cast<uint32_t*>((is_v ? v_cache : k_cache) + row * (head_dim >> 1))[j] = w;
    if ((j & 3) == 0) (is_v ? v_scale : k_scale)[row * (head_dim / kFp4Group) + (j >> 2)] = (uint8_t)code;
  }
}

// Cached tokens as bf16 rows: one workgroup per token, one lane per 8
// channels.  E4M3FN values are code * scale in fp32, rounded once; 4-bit
// values are exact.  A slot outside the pool gives zeros.
template <int KV>
__global__ void __launch_bounds__(256)
load_kv_kernel(const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache,
               const void* __restrict__ k_scale, const void* __restrict__ v_scale,
               const int32_t* __restrict__ slot_mapping, int hkv, int head_dim, int64_t num_slots, int block_size,
               uint16_t* __restrict__ k_out, uint16_t* __restrict__ v_out) {
  const int64_t tok = blockIdx.x;
  const int cph = head_dim >> 3, per = hkv * cph;
  const int slot = slot_mapping[tok];
  const bool live = slot >= 0 && slot < num_slots;
  for (int c = threadIdx.x; c < 2 * per; c += blockDim.x) {
    const bool is_v = c >= per;
    const int cc = is_v ? c - per : c;
    const uint8_t* cache = is_v ? v_cache : k_cache;
    const void* scales = is_v ? v_scale : k_scale;
    const int head = cc / cph, j = cc - head * cph;
    u32x4 o = {0, 0, 0, 0};
    if (live) {
      if (KV == KV_BF16) {
        o = reinterpret_cast<const u32x4*>(cache)[(int64_t)slot * per + cc];
      } else if (KV == KV_FP8_E4M3FN) {
        const u32x2 w = reinterpret_cast<const u32x2*>(cache)[(int64_t)slot * per + cc];
        const float scale = static_cast<const float*>(scales)[(int64_t)slot * hkv + head];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const u32x2 b = fp8x4_to_bf16x4(w[i]);
#pragma unroll
          for (int h = 0; h < 2; ++h)
            o[2 * i + h] = pack_bf16x2(__uint_as_float(b[h] << 16) * scale, __uint_as_float(b[h] & 0xffff0000u) * scale);
        }
      } else {
        const int page = slot / block_size, off = slot - page * block_size;
        const int64_t row = ((int64_t)page * hkv + head) * block_size + off;
        const uint32_t w = reinterpret_cast<const uint32_t*>(cache + row * (head_dim >> 1))[j];
        o = e2m1_decode8(w, e8m0(static_cast<const uint8_t*>(scales)[row * (head_dim / kFp4Group) + (j >> 2)]));
      }
    }
    reinterpret_cast<u32x4*>(is_v ? v_out : k_out)[tok * per + cc] = o;
  }
}

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
  hipLaunchKernelGGL(store_fp4_kernel, dim3(num_tokens), dim3(per < 256 ? (unsigned)((per + 63) / 64 * 64) : 256), 0,
                     static_cast<hipStream_t>(stream), static_cast<const uint16_t*>(key), key_row_stride,
                     static_cast<const uint16_t*>(value), value_row_stride, slot_mapping, num_kv_heads, head_dim,
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
  const dim3 grid(num_tokens), block(per < 256 ? (unsigned)((per + 63) / 64 * 64) : 256);
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto* kernel = kv_dtype == KV_BF16         ? load_kv_kernel<KV_BF16>
                 : kv_dtype == KV_FP8_E4M3FN ? load_kv_kernel<KV_FP8_E4M3FN>
                                             : load_kv_kernel<KV_FP4_E2M1>;
  hipLaunchKernelGGL(kernel, grid, block, 0, s, static_cast<const uint8_t*>(k_cache), static_cast<const uint8_t*>(v_cache),
                     k_scale, v_scale, slot_mapping, num_kv_heads, head_dim, (int64_t)num_blocks * block_size, block_size,
                     static_cast<uint16_t*>(k_out), static_cast<uint16_t*>(v_out));
  return check_launch("load_kvcache");
}
