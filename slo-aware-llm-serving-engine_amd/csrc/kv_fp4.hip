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
// to memory at a decode step's size (24 tokens of 8 heads 2.9 us) and still by
// two of them at a prompt's (4,096 tokens, 21 MB, 7.4 us or 2.9 TB/s; 262,144
// tokens, 1.36 GB, 267 us or 5.1 TB/s).
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
template <int KV, int TOK, int DEPTH, bool NT>
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
      if constexpr (NT)
        __builtin_nontemporal_store(o, to);
      else
        *to = o;
    }
  }
}

// Four tokens a workgroup, and four loads a lane in flight, from 16,384 tokens
// on where one token leaves lanes of a workgroup idle or, packed, just fills it;
// with more heads a token's workgroup has loads enough, and bf16's are four
// times a code's.  us with one token / with four, at head_dim 128:
//   store       8 heads: 16,384 tokens 18.2 / 18.4, 65,536 78 / 65, 262,144
//               302 / 267; 1 head 65,536 34 / 24; 16 heads 65,536 137 / 137
//   read back   4 bits, 8 heads: 16,384 17.1 / 17.0, 262,144 408 / 335; 1 head
//               65,536 23 / 14; 16 heads 65,536 165 / 173
//               E4M3FN, 8 heads: 262,144 324 / 291; 16 heads 65,536 142 / 155
//               bf16, 4 heads: 131,072 104 / 95; 8 heads 262,144 355 / 379
// A grid holds less than 2^32 threads, so from 2^24 tokens on there are always
// four.
constexpr int kManyTokens = 16384, kMostSingle = 1 << 24;

static bool four_tokens(int tokens, int64_t lanes, bool bf16) {
  return tokens >= kMostSingle || (tokens >= kManyTokens && lanes <= (bf16 ? 128 : 256));
}

// A read back that writes 256 MiB and more, the size of the last-level cache,
// passes it by: little of it would be found there by what reads it next, and the
// pool would be displaced.  us of a read back and a copy of what it wrote, through the
// cache / past it, 8 heads of 4 bits: 67 MB 37 / 43, 134 MB 82 / 84, 268 MB 195
// / 184, 1,074 MB 745 / 725; E4M3FN 37 / 42, 81 / 87, 184 / 178, 696 / 687.  bf16
// reads as much as it writes and gains nothing: 200 / 204 and 781 / 795.
constexpr int64_t kPastCache = 256ll << 20;

template <int KV>
static auto* load_kernel(bool four, bool past) {
  if constexpr (KV != KV_BF16) {
    if (four && past) return load_kv_kernel<KV, 4, 4, true>;
  }
  return four ? load_kv_kernel<KV, 4, 4, false> : load_kv_kernel<KV, 1, 1, false>;
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
  const int shift = head_dim == 64 ? 3 : head_dim == 128 ? 4 : 5;
  const bool four = four_tokens(num_tokens, per, false);
  hipLaunchKernelGGL((four ? store_fp4_kernel<4, 4> : store_fp4_kernel<1, 1>), dim3(four ? (num_tokens + 3) / 4 : num_tokens),
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
  const bool four = four_tokens(num_tokens, per, kv_dtype == KV_BF16), past = 16 * per * num_tokens >= kPastCache;
  auto* kernel = kv_dtype == KV_BF16         ? load_kernel<KV_BF16>(four, past)
                 : kv_dtype == KV_FP8_E4M3FN ? load_kernel<KV_FP8_E4M3FN>(four, past)
                                             : load_kernel<KV_FP4_E2M1>(four, past);
  hipLaunchKernelGGL(kernel, dim3(four ? (num_tokens + 3) / 4 : num_tokens), dim3(256), 0, static_cast<hipStream_t>(stream),
                     static_cast<const uint8_t*>(k_cache), static_cast<const uint8_t*>(v_cache), k_scale, v_scale, slot_mapping,
                     num_tokens, num_kv_heads, shift, (int64_t)num_blocks * block_size, block_size,
                     static_cast<uint16_t*>(k_out), static_cast<uint16_t*>(v_out));
  return check_launch("load_kvcache");
}
