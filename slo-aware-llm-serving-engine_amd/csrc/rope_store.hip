// Norms of q and k (or none), rotary embedding in any layout, and the
// slot-mapped KV write, in one pass over the fused QKV projection's output
// (gfx950).  For a 4-bit pool q and k only: the store kernel then reads k and V
// again (4,096 tokens, 32 and 8 heads of 128: 23.7 us in both launches, a bf16 pool
// 19.7).
//
// With the first R channels of a head rotated, h the head after the norm
// (h = x rsqrt(mean x^2 + eps) w, or x itself) and a pair's channels (a, b)
// neighbours (2i, 2i + 1) or half of R apart (i, i + R / 2), i < R / 2:
//   y[a] = h[a] cos_i - h[b] sin_i,  y[b] = h[b] cos_i + h[a] sin_i
// and y = h on the other channels, all in fp32 and rounded once to bf16.  (The
// layout of qk_norm_rope.hip, all 128 channels in halves with both norms, keeps
// its own kernel and the rounding points of the model that it serves.)  K goes
// to the pool after the rotation and that rounding, V as given; E4M3FN pools
// use the quantisation of the store kernel.
#include "common.h"
#include "capi_internal.h"

namespace slo {
namespace {

// Threads per workgroup, and heads that a lane group has in flight.  Up to 1,024
// tokens all workgroups of 512 threads are on the GPU at once, and a token's
// heads side by side end soonest; past that, small ones that hold more heads a
// lane keep more loads in flight.  us for 512 x 2 / 128 x 3, 32 and 8 heads of
// 128: 128 tokens 3.5 / 4.8, 768 6.9 / 8.2, 2,000 12.5 / 11.0, 8,192 (221 MB) 60.6
// / 44.8 (4.9 TB/s; 256 x 3 45.3, 128 x 6 43.0 but 11.7 for the 2,000); 16 and 1 heads,
// 8,192 28.0 / 16.6; heads of 64 29.2 / 21.1; E4M3FN, 4,096 (103 MB) 26.1 / 21.0.
constexpr int kFewThreads = 512, kFewHeads = 2, kManyThreads = 128, kManyHeads = 3, kMany = 1024;

struct RopeParams {
  const uint16_t* qkv;
  int64_t qkv_stride;
  const int64_t* positions;
  int tokens, num_heads, num_kv_heads;
  const uint16_t *q_w, *k_w;  // null: no norm
  float eps;
  const float* cos_sin;  // [max_position, rot]: cosines, then sines
  int max_position, rot;
  uint16_t *q_out, *k_out;
  const int32_t* slots;
  int kv_dtype;
  void *k_cache, *v_cache;
  float *k_scale, *v_scale;
  int64_t num_slots;
  float scale_floor;
};

// Sum over GROUP adjacent lanes, the same bits in every lane.
template <int GROUP>
__device__ __forceinline__ float group_sum(float x) {
  x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0xb1, 0xf, 0xf, false));   // quad_perm 1, 0, 3, 2
  x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x4e, 0xf, 0xf, false));   // quad_perm 2, 3, 0, 1
  x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x141, 0xf, 0xf, false));  // row_half_mirror
  if constexpr (GROUP >= 16) x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x140, 0xf, 0xf, false));  // row_mirror
  if constexpr (GROUP >= 32) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  }
  return x;
}

__device__ __forceinline__ void unpack4(const u32x2& w, float* f) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

// One workgroup per token (and turn); D / 8 lanes per head, each with 8
// channels in two pieces of 4: lane j of a head has channels 8j.. and 8j + 4..,
// or, with FAR pairs on a rotated lane (j < R / 8), 4j.. and R / 2 + 4j.., so
// that both channels of a pair are in one lane in either layout.
template <int D, bool FAR, int THREADS, int U>
__global__ void __launch_bounds__(THREADS)
rope_store_kernel(RopeParams p) {
  constexpr int LANES = D / 8, GROUPS = THREADS / LANES;
  const int j = threadIdx.x % LANES, grp = threadIdx.x / LANES;
  const int heads = p.num_heads + 2 * p.num_kv_heads, qk = p.num_heads + p.num_kv_heads;
  const bool turned = 8 * j < p.rot;
  const int c0 = FAR && turned ? 4 * j : 8 * j, c1 = FAR && turned ? p.rot / 2 + 4 * j : 8 * j + 4;
  const bool norm = p.q_w != nullptr;
  u32x2 wq[2] = {}, wk[2] = {};
  if (norm) {
    wq[0] = *reinterpret_cast<const u32x2*>(p.q_w + c0);
    wq[1] = *reinterpret_cast<const u32x2*>(p.q_w + c1);
    wk[0] = *reinterpret_cast<const u32x2*>(p.k_w + c0);
    wk[1] = *reinterpret_cast<const u32x2*>(p.k_w + c1);
  }
  for (int64_t tok = blockIdx.x; tok < p.tokens; tok += gridDim.x) {
    int64_t pos = p.positions[tok];
    const int64_t slot = p.slots[tok];
    const bool store = slot >= 0 && slot < p.num_slots;
    const uint16_t* row = p.qkv + tok * p.qkv_stride;
    pos = pos < 0 ? 0 : (pos >= p.max_position ? p.max_position - 1 : pos);
    f32x4 cs = {1, 1, 1, 1}, sn = {0, 0, 0, 0};
    if (turned) {
      const float* t = p.cos_sin + pos * p.rot + 4 * j;
      cs = *reinterpret_cast<const f32x4*>(t);
      sn = *reinterpret_cast<const f32x4*>(t + p.rot / 2);
    }
    for (int h0 = 0; h0 < heads; h0 += GROUPS * U) {
      u32x2 x[U][2];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = h0 + GROUPS * u + grp;
        // V keeps its order: its lanes hold 8 channels side by side.
        const int a = h < qk ? c0 : 8 * j, b = h < qk ? c1 : 8 * j + 4;
        x[u][0] = x[u][1] = u32x2{0, 0};
        if (h < heads) {
          x[u][0] = *reinterpret_cast<const u32x2*>(row + h * D + a);
          x[u][1] = *reinterpret_cast<const u32x2*>(row + h * D + b);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = h0 + GROUPS * u + grp;
        if (h >= heads) continue;
        int a = 8 * j, b = 8 * j + 4;
        u32x2 o[2] = {x[u][0], x[u][1]};
        if (h < qk) {
          a = c0;
          b = c1;
          float f[8];
          unpack4(x[u][0], f);
          unpack4(x[u][1], f + 4);
          if (norm) {
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(f[i], f[i], ss);
            const float r = __builtin_amdgcn_rsqf(group_sum<LANES>(ss) * (1.0f / D) + p.eps);
            float w[8];
            unpack4(h < p.num_heads ? wq[0] : wk[0], w);
            unpack4(h < p.num_heads ? wq[1] : wk[1], w + 4);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] *= r * w[i];
          }
          if (turned) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int m = FAR ? i : 2 * i, n = FAR ? 4 + i : 2 * i + 1;
              const float s = f[m], t = f[n];
              f[m] = s * cs[i] - t * sn[i];
              f[n] = t * cs[i] + s * sn[i];
            }
          }
          o[0] = u32x2{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3])};
          o[1] = u32x2{pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])};
          uint16_t* out = h < p.num_heads ? p.q_out + (tok * p.num_heads + h) * D
                                          : p.k_out + (tok * p.num_kv_heads + h - p.num_heads) * D;
          *reinterpret_cast<u32x2*>(out + a) = o[0];
          *reinterpret_cast<u32x2*>(out + b) = o[1];
          if (h < p.num_heads) continue;
        }
        if (!store) continue;
        const int kvh = h < qk ? h - p.num_heads : h - qk;
        const int64_t at = (slot * p.num_kv_heads + kvh) * D;
        if (p.kv_dtype == KV_BF16) {
          uint16_t* to = static_cast<uint16_t*>(h < qk ? p.k_cache : p.v_cache) + at;
          *reinterpret_cast<u32x2*>(to + a) = o[0];
          *reinterpret_cast<u32x2*>(to + b) = o[1];
        } else {
          float f[8], scale;
          unpack4(o[0], f);
          unpack4(o[1], f + 4);
          const u32x2 codes = e4m3_encode8<LANES>(f, p.scale_floor, scale);
          uint8_t* to = static_cast<uint8_t*>(h < qk ? p.k_cache : p.v_cache) + at;
          *reinterpret_cast<uint32_t*>(to + a) = codes.x;
          *reinterpret_cast<uint32_t*>(to + b) = codes.y;
          if (j == 0) (h < qk ? p.k_scale : p.v_scale)[slot * p.num_kv_heads + kvh] = scale;
        }
      }
    }
  }
}

// A grid holds less than 2^32 threads: past so many tokens workgroups go round.
constexpr int kGrid = 1 << 20;

template <int D, bool FAR>
void launch_rope(const RopeParams& p, hipStream_t s) {
  const dim3 grid(p.tokens < kGrid ? p.tokens : kGrid);
  if (p.tokens > kMany)
    hipLaunchKernelGGL((rope_store_kernel<D, FAR, kManyThreads, kManyHeads>), grid, dim3(kManyThreads), 0, s, p);
  else
    hipLaunchKernelGGL((rope_store_kernel<D, FAR, kFewThreads, kFewHeads>), grid, dim3(kFewThreads), 0, s, p);
}

template <int D>
void launch_rope(const RopeParams& p, bool interleaved, hipStream_t s) {
  if (interleaved) launch_rope<D, false>(p, s);
  else launch_rope<D, true>(p, s);
}

inline bool unaligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; }

}  // namespace
}  // namespace slo

using namespace slo;

extern "C" int slo_rope_store(const slo_rope_store_args* a, slo_stream_t stream) {
  if (!a) return fail(SLO_ERR_INVALID, "rope_store: null args");
  if (a->num_tokens < 0 || a->num_heads <= 0 || a->num_kv_heads <= 0)
    return fail(SLO_ERR_INVALID, "rope_store: bad token/head count");
  if (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256)
    return fail(SLO_ERR_UNSUPPORTED, "rope_store: head_dim must be 64, 128 or 256");
  if (a->rotary_dim <= 0 || a->rotary_dim > a->head_dim || a->rotary_dim % 8)
    return fail(SLO_ERR_INVALID, "rope_store: rotary_dim must be a multiple of 8 up to head_dim");
  const bool fp8 = a->kv_dtype == KV_FP8_E4M3FN;
  if (a->kv_dtype != KV_BF16 && !fp8) return fail(SLO_ERR_INVALID, "rope_store: bad kv_dtype");
  if (a->max_position <= 0 || a->num_slots < 0)
    return fail(SLO_ERR_INVALID, "rope_store: max_position must be positive and num_slots not negative");
  if ((int64_t)a->num_heads + 2 * (int64_t)a->num_kv_heads > 65536) return fail(SLO_ERR_UNSUPPORTED, "rope_store: too many heads");
  if (!a->q_norm_weight != !a->k_norm_weight) return fail(SLO_ERR_INVALID, "rope_store: weights of both norms, or of neither");
  if (a->q_norm_weight && !(a->eps >= 0.0f)) return fail(SLO_ERR_INVALID, "rope_store: eps must be >= 0");
  if (a->num_tokens == 0) return SLO_OK;
  if (!a->qkv || !a->positions || !a->cos_sin || !a->q_out || !a->k_out || !a->slot_mapping ||
      (a->num_slots && (!a->k_cache || !a->v_cache)))
    return fail(SLO_ERR_INVALID, "rope_store: null pointer");
  if (fp8 && (!a->k_scale || !a->v_scale)) return fail(SLO_ERR_INVALID, "rope_store: FP8 needs scale pools");
  if (fp8 && !(a->scale_floor > 0.0f)) return fail(SLO_ERR_INVALID, "rope_store: scale_floor must be > 0");
  if ((a->qkv_row_stride % 8) || a->qkv_row_stride < ((int64_t)a->num_heads + 2 * (int64_t)a->num_kv_heads) * a->head_dim ||
      unaligned16(a->qkv) || unaligned16(a->q_out) || unaligned16(a->k_out) || unaligned16(a->k_cache) ||
      unaligned16(a->v_cache) || unaligned16(a->cos_sin) || unaligned16(a->q_norm_weight) || unaligned16(a->k_norm_weight))
    return fail(SLO_ERR_INVALID, "rope_store: rows and tables must be 16-byte aligned");
  const RopeParams p = {static_cast<const uint16_t*>(a->qkv), a->qkv_row_stride, a->positions, a->num_tokens, a->num_heads,
                        a->num_kv_heads, static_cast<const uint16_t*>(a->q_norm_weight),
                        static_cast<const uint16_t*>(a->k_norm_weight), a->eps, a->cos_sin, a->max_position, a->rotary_dim,
                        static_cast<uint16_t*>(a->q_out), static_cast<uint16_t*>(a->k_out), a->slot_mapping, a->kv_dtype,
                        a->k_cache, a->v_cache, a->k_scale, a->v_scale, a->num_slots, a->scale_floor};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->head_dim == 64) launch_rope<64>(p, a->interleaved != 0, s);
  else if (a->head_dim == 128) launch_rope<128>(p, a->interleaved != 0, s);
  else launch_rope<256>(p, a->interleaved != 0, s);
  return check_launch("rope_store");
}
