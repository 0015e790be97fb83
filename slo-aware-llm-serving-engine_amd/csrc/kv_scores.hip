// Accumulated attention weights of cached tokens (gfx950).
//
// scores[slot of key j, kv head] += sum over the step's queries i and the
// heads h of the kv head's group of softmax_j(scale q[i, h] . k[j]); the keys
// that the step itself adds start from that sum.  K comes from a bf16, E4M3FN
// or 4-bit pool; V is not read.
//
// S^T = K q^T by v_mfma_f32_16x16x32_bf16 (rows: 16 tokens, columns: 16 (query,
// head) pairs), so a lane has 4 tokens of one column.  A weight needs its row's
// maximum and sum first, so each phase takes two passes:
//
//  * decode rows (one query): the first pass keeps the logits (fp32), the second
//    turns them into weights, so K is read once.  A row's logits stay in LDS if
//    they fit; those of longer rows, and of long ones that are few, go through
//    memory (4 bytes per (head, token): at a group of 4 a sixteenth of bf16 K and
//    a quarter of 4-bit K, at 16 a quarter of the one and all of the other), with
//    each chunk's maximum and sum.
//  * prefill rows: the first pass finds every (query, head)'s log2-sum; the
//    second computes S^T again, 64 keys of a workgroup against all queries,
//    and sums the weights over the queries in registers (writing the scores of
//    a 1,000-query chunk would take more than the two products).
//
// A key's sum over queries is taken in one order, whatever the grid.  Old keys
// get it by fp32 atomic adds, so rows that share a page (a cached prefix) both
// count; only for such a page does the order of its rows' additions vary.
#include "capi_internal.h"
#include "fp4.h"
#include "tile_io.h"

namespace slo {
namespace {

constexpr int HDS = 128;
constexpr float kNone = -1e30f;

struct ScoreParams {
  const uint16_t* q;
  int64_t q_stride;
  int num_q_rows;
  const uint8_t* kc;
  const void* ks;
  int num_blocks, block_size;
  const int32_t* lens;
  const int32_t* cu_q;
  const int32_t* cu_k;
  const int32_t* tables;
  int table_stride, table_width;
  int first_row;
  int hq, hkv, group;
  float scale_log2;  // softmax scale * log2(e)
  float* scores;   // [num_blocks, hkv, block_size]
  float* logits;   // decode: [rows, hq, capacity], log2 units
  float2* partial;  // decode: [rows, hq, splits] (maximum, sum)
  float* lse;      // prefill: [queries, hq], log2 units
  int splits, chunk, capacity;
};

struct Row {
  int64_t q0;
  int lq, lk, prefix;
};

__device__ __forceinline__ Row row_of(const ScoreParams& p, int r) {
  Row g;
  const int cap = p.table_width * p.block_size;
  if (p.lens) {
    g.q0 = p.first_row + r;
    g.lq = 1;
    g.lk = min(max(p.lens[r], 0), cap);
    g.prefix = g.lk - 1;
  } else {
    const int start = p.cu_q[r], k = p.cu_k[r + 1] - p.cu_k[r];
    g.q0 = (int64_t)p.first_row + start;
    g.lq = p.cu_q[r + 1] - start;
    g.prefix = k - g.lq;
    g.lk = min(k, cap);
    if (start < 0 || g.q0 + g.lq > p.num_q_rows) g.lq = 0;
  }
  return g;
}

// Channels of a lane's k-group kg in product i, by how the format's rows load
// in 16-byte pieces: the sum over channels is the same in any order.
template <int KV>
__device__ __forceinline__ int channel_of(int i, int kg) {
  return KV == KV_BF16 ? 32 * i + 8 * kg : KV == KV_FP8_E4M3FN ? 64 * (i >> 1) + 16 * kg + 8 * (i & 1) : 32 * kg + 8 * i;
}

template <int KV>
__device__ __forceinline__ bf16x8 load_q(const ScoreParams& p, int64_t row, int h, int i, int kg, bool live) {
  u32x4 x = {0, 0, 0, 0};
  if (live) x = *reinterpret_cast<const u32x4*>(p.q + row * p.q_stride + h * HDS + channel_of<KV>(i, kg));
  return as_bf16x8(x);
}

// 16 tokens' keys of one kv head as they lie in the pool.
template <int KV>
struct Keys {
  static constexpr int N = KV == KV_BF16 ? 4 : KV == KV_FP8_E4M3FN ? 2 : 1;
  u32x4 w[N];
  float scale[KV == KV_FP8_E4M3FN ? 4 : 1];
  uint32_t code;

  // `block` page, token `off` of it
  template <bool SCALE = true>
  __device__ __forceinline__ void load(const ScoreParams& p, int block, int off, int head, int lane) {
    const int col = lane & 15, kg = lane >> 4;
    if (KV == KV_FP4_E2M1) {
      const int64_t row = ((int64_t)block * p.hkv + head) * p.block_size + off + col;
      w[0] = *reinterpret_cast<const u32x4*>(p.kc + row * 64 + kg * 16);
      code = static_cast<const uint8_t*>(p.ks)[row * 4 + kg];
    } else {
      const int64_t slot = (int64_t)block * p.block_size + off;
      const int rb = KV == KV_BF16 ? 256 : 128;
      const uint8_t* at = p.kc + ((slot + col) * p.hkv + head) * rb + kg * 16;
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = *reinterpret_cast<const u32x4*>(at + i * 64);
      if (KV == KV_FP8_E4M3FN && SCALE) {
        const float* s = static_cast<const float*>(p.ks) + (slot + 4 * kg) * p.hkv + head;
#pragma unroll
        for (int i = 0; i < 4; ++i) scale[i & (sizeof(scale) / 4 - 1)] = s[(int64_t)i * p.hkv];
      }
    }
  }
  __device__ __forceinline__ bf16x8 operand(int i) const {
    if (KV == KV_BF16) return as_bf16x8(w[i & (N - 1)]);
    if (KV == KV_FP8_E4M3FN) {
      const u32x4& x = w[(i >> 1) & (N - 1)];
      const u32x2 a = fp8x4_to_bf16x4(x[2 * (i & 1)]), b = fp8x4_to_bf16x4(x[2 * (i & 1) + 1]);
      return as_bf16x8(u32x4{a.x, a.y, b.x, b.y});
    }
    return as_bf16x8(e2m1_decode8(w[0][i], e8m0(code)));
  }
  // token 4 kg + i's factor of the products
  __device__ __forceinline__ float factor(int i) const { return KV == KV_FP8_E4M3FN ? scale[i & (sizeof(scale) / 4 - 1)] : 1.0f; }
};

__device__ __forceinline__ int page_of(const ScoreParams& p, int r, int token, int& off) {
  const int page = token / p.block_size;
  off = token - page * p.block_size;
  const int b = p.tables[(int64_t)r * p.table_stride + page];
  return b >= 0 && b < p.num_blocks ? b : -1;
}

// (m, l) with the maximum m and the sum l of 2^(x - m); absorbs another pair.
__device__ __forceinline__ void absorb(float& m, float& l, float m2, float l2) {
  const float top = fmaxf(m, m2);
  l = l * __builtin_amdgcn_exp2f(m - top) + l2 * __builtin_amdgcn_exp2f(m2 - top);
  m = top;
}

// Logits (log2 units) of tokens begin, begin + stride, ... < end of a decode
// row, 16 T at a time, the next ones' loads ahead of the products; `put` takes
// four tokens' logits of this lane's column.  Returns the lane's maximum and sum.
template <int KV, typename Put>
__device__ __forceinline__ float2 decode_logits(const ScoreParams& p, const Row& g, int r, int head, int begin, int end,
                                                int stride, int lane, Put put) {
  constexpr int T = KV == KV_FP4_E2M1 ? 4 : 2;
  const int col = lane & 15, kg = lane >> 4;
  float m = kNone, l = 0.0f;
  if (begin >= end) return float2{m, l};
  Keys<KV> k[T];
  auto load = [&](Keys<KV>(&to)[T], int at) {
    int off;
    const int block = page_of(p, r, at, off);
#pragma unroll
    for (int t = 0; t < T; ++t) to[t].load(p, block < 0 ? 0 : block, (block < 0 ? 0 : off) + 16 * t, head, lane);
    return block >= 0;
  };
  bool ok = load(k, begin);
  bf16x8 q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = load_q<KV>(p, g.q0, head * p.group + col, i, kg, col < p.group);
  for (int at = begin; at < end; at += stride) {
    Keys<KV> n[T];
    bool next_ok = false;
    if (at + stride < end) next_ok = load(n, at + stride);
    f32x4 s[T];
    float top = kNone;
#pragma unroll
    for (int t = 0; t < T; ++t) {
      s[t] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < 4; ++i) s[t] = mfma16(k[t].operand(i), q[i], s[t]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[t][i] *= k[t].factor(i) * p.scale_log2;
        if (!ok || at + 16 * t + 4 * kg + i >= g.lk) s[t][i] = -INFINITY;
        top = fmaxf(top, s[t][i]);
      }
      put(at + 16 * t + 4 * kg, s[t]);
    }
    if (__any(top > m + 8.0f)) {  // sums of weights up to 256 round like those below 1
      const float to = fmaxf(m, top);
      l *= __builtin_amdgcn_exp2f(m - to);
      m = to;
    }
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) l += __builtin_amdgcn_exp2f(s[t][i] - m);
#pragma unroll
    for (int t = 0; t < T; ++t) k[t] = n[t];
    ok = next_ok;
  }
  return float2{m, l};
}

__device__ __forceinline__ void add_score(const ScoreParams& p, const Row& g, int block, int off, int head, int token, float w) {
  float* s = p.scores + ((int64_t)block * p.hkv + head) * p.block_size + off;
  if (token >= g.prefix)
    *s = w;
  else
    unsafeAtomicAdd(s, w);
}

// (maximum, sum) of a column over its four lanes, in each of them.
__device__ __forceinline__ float2 column_lse(float2 e) {
  const float m = col_max(e.x);
  return float2{m, col_sum(e.y * __builtin_amdgcn_exp2f(e.x - m))};
}

// Decode rows whose logits fit LDS (by the tables' width, as a captured launch
// knows no more): a workgroup takes a (row, kv head) whole,
// so one launch does, and K is all that moves.  64 rows of 512-4,096 tokens of
// a 4-bit pool, 8 kv heads (86 MB of K): 30 us, against 37 and 11 in two
// launches through memory; 25 without the adds to the scores, 23 without the
// second half.
constexpr int kRowLogits = 16384;
// With fewer (row, kv head) pairs than CUs, rows of 512 KiB of K and more take
// the two launches: a workgroup a pair reads too slowly.  us whole / in two, one
// row and 16 of them, 8 kv heads: bf16, 1,024 tokens 12.2 / 15.6 and 13.7 / 16.0,
// 2,048 18.7 / 15.7 and 21.9 / 20.9, 16,384 (group 1) 120 / 16 and 168 / 142;
// E4M3FN, 2,048 13.6 / 16.3 and 16.8 / 17.7, 4,096 22.3 / 16.2 and 28.3 / 27.5;
// 4 bits, 4,096 14.4 / 17.5 and 20.0 / 21.5, 8,192 23.3 / 17.2 and 34.8 / 32.8.
// 64 rows of 2,048-4,096 tokens fill the CUs: bf16 113 / 154, 4 bits 46 / 65.
constexpr int kFullGroups = 256, kLongRow = 512 << 10;

template <int KV, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, 4)
score_row_kernel(ScoreParams p) {
  __shared__ float logits[kRowLogits];  // [group, capacity]
  __shared__ float sm[WAVES][16], sl[WAVES][16], lse[16];
  const int head = blockIdx.x, r = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15;
  const Row g = row_of(p, r);
  constexpr int SPAN = KV == KV_FP4_E2M1 ? 64 : 32;
  float* mine = logits + col * p.capacity;
  const float2 e = column_lse(decode_logits<KV>(p, g, r, head, wave * SPAN, g.lk, WAVES * SPAN, lane, [&](int at, const f32x4& s) {
    if (col < p.group && at < p.capacity) *reinterpret_cast<f32x4*>(mine + at) = s;
  }));
  if (lane < 16) {
    sm[wave][lane] = e.x;
    sl[wave][lane] = e.y;
  }
  __syncthreads();
  if (wave == 0) {  // lane: column, and a quarter of the wavefronts
    float2 f = {kNone, 0.0f};
#pragma unroll
    for (int w = 0; w < WAVES; w += 4) absorb(f.x, f.y, sm[w + (lane >> 4)][col], sl[w + (lane >> 4)][col]);
    f = column_lse(f);
    if (lane < 16) lse[lane] = f.x + __builtin_amdgcn_logf(f.y);
  }
  __syncthreads();
  // Four tokens a lane: one look into the table for them.
  for (int token = 4 * threadIdx.x; token < g.lk; token += 4 * 64 * WAVES) {
    int off;
    const int block = page_of(p, r, token, off);
    if (block < 0) continue;
    f32x4 w = {0, 0, 0, 0};
    for (int h = 0; h < p.group; ++h) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(logits + h * p.capacity + token);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] += __builtin_amdgcn_exp2f(x[i] - lse[h]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (token + i < g.lk) add_score(p, g, block, off + i, head, token + i, w[i]);
  }
}

// Longer rows, first pass: one chunk of one (row, kv head) per workgroup, its
// four wavefronts every fourth step.
template <int KV>
__global__ void __launch_bounds__(256, 4)
score_logits_kernel(ScoreParams p) {
  __shared__ float sm[4][16], sl[4][16];
  const int head = blockIdx.x, split = blockIdx.y, r = blockIdx.z;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15;
  const Row g = row_of(p, r);
  const int k0 = split * p.chunk, k1 = min(k0 + p.chunk, g.lk);
  if (k0 >= g.lk) return;
  constexpr int SPAN = KV == KV_FP4_E2M1 ? 64 : 32;
  float* logits = p.logits + ((int64_t)r * p.hq + head * p.group + col) * p.capacity;
  const float2 e = column_lse(decode_logits<KV>(p, g, r, head, k0 + wave * SPAN, k1, 4 * SPAN, lane, [&](int at, const f32x4& s) {
    if (col < p.group) *reinterpret_cast<f32x4*>(logits + at) = s;
  }));
  if (lane < 16) {
    sm[wave][lane] = e.x;
    sl[wave][lane] = e.y;
  }
  __syncthreads();
  if (threadIdx.x < p.group) {
    float m = kNone, l = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) absorb(m, l, sm[w][threadIdx.x], sl[w][threadIdx.x]);
    p.partial[((int64_t)r * p.hq + head * p.group + threadIdx.x) * p.splits + split] = float2{m, l};
  }
}

// Second pass: four tokens a lane.
__global__ void __launch_bounds__(256)
score_decode_kernel(ScoreParams p) {
  __shared__ float lse[16];
  const int head = blockIdx.x, r = blockIdx.z;
  const Row g = row_of(p, r);
  if ((int)blockIdx.y * 1024 >= g.lk) return;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int n = (g.lk + p.chunk - 1) / p.chunk;
  for (int h = wave; h < p.group; h += 4) {
    const float2* e = p.partial + ((int64_t)r * p.hq + head * p.group + h) * p.splits;
    float m = kNone, l = 0.0f;
    for (int s = lane; s < n; s += 64) absorb(m, l, e[s].x, e[s].y);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const float m2 = __shfl_xor(m, d, 64), l2 = __shfl_xor(l, d, 64);
      absorb(m, l, m2, l2);
    }
    if (lane == 0) lse[h] = m + __builtin_amdgcn_logf(l);
  }
  __syncthreads();
  const int token = blockIdx.y * 1024 + threadIdx.x * 4;
  if (token >= g.lk) return;
  int off;
  const int block = page_of(p, r, token, off);
  if (block < 0) return;
  const float* x = p.logits + ((int64_t)r * p.hq + head * p.group) * p.capacity + token;
  f32x4 w = {0, 0, 0, 0};
  for (int h = 0; h < p.group; ++h) {
    const f32x4 y = *reinterpret_cast<const f32x4*>(x + (int64_t)h * p.capacity);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] += __builtin_amdgcn_exp2f(y[i] - lse[h]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (token + i < g.lk) add_score(p, g, block, off + i, head, token + i, w[i]);
}

// Sum over 16 lanes by DPP, in each of them.
__device__ __forceinline__ float row_sum16(float x) {
  x += __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0xb1, 0xf, 0xf, false));   // quad_perm 1, 0, 3, 2
  x += __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0x4e, 0xf, 0xf, false));   // quad_perm 2, 3, 0, 1
  x += __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0x141, 0xf, 0xf, false));  // row_half_mirror
  return x + __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0x140, 0xf, 0xf, false));  // row_mirror
}

// Prefill rows, first pass: 16 NT (query, head) columns of one row per
// workgroup, its four wavefronts every fourth pair of 16-token tiles of their
// keys, the next pair's loads ahead of the products.  A lane sums its own
// tokens' weights against a reference of its own, which follows a new maximum
// only where that passes it by 2^8 (sums of weights up to 256 round like those
// below 1); the lanes meet at the end.  1,024 queries on 2,048 keys and 500 on
// 500, 32 heads, E4M3FN: 39 us (45 with two column groups a wavefront, whose
// keys then serve half as many columns), 12 without the loop over the keys;
// matrix cores busy 13% of the time, as in the second pass.
template <int KV, int NT>
__device__ __forceinline__ void find_lse(const ScoreParams& p, const Row& g, int r, int head, int per, int t0) {
  __shared__ float sm[NT][4][16], sl[NT][4][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, kg = lane >> 4;
  const int t1 = min(t0 + per, g.lq);
  const int kend = min(max(g.prefix + t1, 0), g.lk);
  bf16x8 q[NT][4];
  int limit[NT];
  float m[NT], l[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int x = 16 * n + col, tok = t0 + x / p.group;
    const bool live = x < per * p.group && tok < t1;
    limit[n] = live ? min(g.prefix + tok + 1, g.lk) : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) q[n][i] = load_q<KV>(p, g.q0 + tok, head * p.group + x % p.group, i, kg, live);
    // A column of no query has scores of zero: from a reference of zero its
    // weights of 1 do not look like a maximum that moved.
    m[n] = live ? kNone : 0.0f;
    l[n] = 0.0f;
  }
  const int full = min(g.prefix + t0 + 1, g.lk);
  Keys<KV> k[2];
  auto load = [&](int at) {
    int off;
    const int block = page_of(p, r, at, off);
#pragma unroll
    for (int h = 0; h < 2; ++h) k[h].load(p, block < 0 ? 0 : block, (block < 0 ? 0 : off) + 16 * h, head, lane);
    return block >= 0;
  };
  int at = 32 * wave;
  bool ok = at < kend && load(at);
  for (; at < kend; at += 128) {
    bf16x8 a[2][4];
    float f[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[h][i] = k[h].operand(i);
        f[h][i] = k[h].factor(i) * p.scale_log2;
      }
    const bool now = ok;
    if (at + 128 < kend) ok = load(at + 128);
    if (!now) continue;
    // One block of products and weights without a branch, so that the matrix
    // cores work on a column group while the last one's weights are taken.
    f32x4 s[NT][2];
    float sum[NT], most = 0.0f;
    auto weights = [&](bool masked) {
      most = 0.0f;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          e[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][j >> 2][j & 3], f[j >> 2][j & 3], -m[n]));
          if (masked && at + 16 * (j >> 2) + 4 * kg + (j & 3) >= limit[n]) e[j] = 0.0f;
        }
        most = fmaxf(most, fmaxf(fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])), fmaxf(fmaxf(e[4], e[5]), fmaxf(e[6], e[7]))));
        sum[n] = ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
      }
    };
    auto products = [&] {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        s[n][0] = s[n][1] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[n][0] = mfma16(a[0][i], q[n][i], s[n][0]);
          s[n][1] = mfma16(a[1][i], q[n][i], s[n][1]);
        }
      }
    };
    const bool masked = at + 32 > full;
    if (masked) {
      products();
      weights(true);
    } else {
      products();
      weights(false);
    }
    // The weights themselves tell whether a reference has to move.
    if (__any(most > 256.0f)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float top = m[n];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (at + 16 * (j >> 2) + 4 * kg + (j & 3) < limit[n]) top = fmaxf(top, s[n][j >> 2][j & 3] * f[j >> 2][j & 3]);
        l[n] *= __builtin_amdgcn_exp2f(m[n] - top);
        m[n] = top;
      }
      weights(true);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) l[n] += sum[n];
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const float2 e = column_lse(float2{m[n], l[n]});
    if (lane < 16) {
      sm[n][wave][lane] = e.x;
      sl[n][wave][lane] = e.y;
    }
  }
  __syncthreads();
  const int x = threadIdx.x, tok = t0 + x / p.group;
  if (x < per * p.group && tok < t1) {
    float mm = kNone, ll = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) absorb(mm, ll, sm[x >> 4][w][x & 15], sl[x >> 4][w][x & 15]);
    p.lse[(g.q0 - p.first_row + tok) * p.hq + head * p.group + x % p.group] = mm + __builtin_amdgcn_logf(ll);
  }
}

// One tile a workgroup; those of a row with more queries than the launch was
// sized for (max_q) go round.
template <int KV, int NT>
__global__ void __launch_bounds__(256, 2)
score_lse_kernel(ScoreParams p, int tiles) {
  const int head = blockIdx.x, r = blockIdx.z, per = 16 * NT / p.group;
  const Row g = row_of(p, r);
  for (int t0 = (tiles - 1 - (int)blockIdx.y) * per; t0 < g.lq; t0 += tiles * per) {
    find_lse<KV, NT>(p, g, r, head, per, t0);
    __syncthreads();  // the maxima and sums have been read
  }
}

// Prefill rows, second pass: a workgroup takes 64 keys of one (row, kv head),
// held as operands in every wavefront's registers, and its eight wavefronts
// every eighth 16 of the columns that see one of them.  A lane sums its 16
// tokens' weights over its columns; lanes, then wavefronts, are added in order
// at the end.  The same queries and keys: 40 us; three or four steps of columns
// in flight instead of two 40 and 41.  Of 42 before the last change, the loop was
// 27, the exponents alone 2 and the products alone 3.
constexpr int kSumWaves = 8, kSumKeys = 64, kSumDepth = 2;

// 16 columns as their lanes take them: four operands of q, and the log2-sums.
// They arrive by LDS DMA, kSumDepth in flight.
struct Columns {
  u32x4 q[4][64];
  float lse[64];
};

// The keys from token `at` of row r, in page `block` from place `off` on.
template <int KV>
__device__ __forceinline__ void weigh_keys(const ScoreParams& p, const Row& g, int head, int at, int block, int off) {
  __shared__ Columns ring[kSumWaves][kSumDepth];
  __shared__ float sums[kSumWaves][kSumKeys];
  __shared__ f32x4 factors[KV == KV_FP8_E4M3FN ? kSumKeys / 4 : 1];  // E4M3FN scales, in LDS to save registers
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, kg = lane >> 4;
  Keys<KV> keys[4];
#pragma unroll
  for (int h = 0; h < 4; ++h) keys[h].template load<false>(p, block, off + 16 * h, head, lane);
  // This wavefront's columns first + stride i; the next ones' query and head by
  // addition.  A column past the last is read as the last and weighs nothing.
  const int columns = g.lq * p.group, stride = 16 * kSumWaves;
  const int first = max(at - g.prefix, 0) * p.group + 16 * wave;
  const int count = first < columns ? (columns - first + stride - 1) / stride : 0;
  const int dt = stride / p.group, dh = stride - dt * p.group;
  int tok = (first + col) / p.group, hh = first + col - tok * p.group;  // of the columns that are fetched next
  const uint32_t lds = lds_addr(&ring[wave][0]);
  int to = 0;
  auto fetch = [&] {
    const bool live = tok < g.lq;
    const int64_t row = g.q0 + (live ? tok : g.lq - 1);
    const int h = head * p.group + (live ? hh : p.group - 1);
    const uint16_t* q = p.q + row * p.q_stride + h * HDS;
    const uint32_t base = lds + to * (uint32_t)sizeof(Columns);
#pragma unroll
    for (int i = 0; i < 4; ++i) dma16(q + channel_of<KV>(i, kg), base + 1024 * i);
    dma4(p.lse + (row - p.first_row) * p.hq + h, base + 4096);
    to = to == kSumDepth - 1 ? 0 : to + 1;
    tok += dt;
    hh += dh;
    if (hh >= p.group) {
      hh -= p.group;
      ++tok;
    }
  };
  int now_tok = tok, now_hh = hh, sent = 0;
  for (; sent < kSumDepth && sent < count; ++sent) fetch();
  bf16x8 a[4][4];
#pragma unroll
  for (int h = 0; h < 4; ++h) {
#pragma unroll
    for (int i = 0; i < 4; ++i) a[h][i] = keys[h].operand(i);
  }
  if (KV == KV_FP8_E4M3FN) {
    if (threadIdx.x < kSumKeys)
      reinterpret_cast<float*>(factors)[threadIdx.x] =
          static_cast<const float*>(p.ks)[((int64_t)block * p.block_size + off + threadIdx.x) * p.hkv + head] * p.scale_log2;
    __syncthreads();
  }
  float w[4][4] = {};
  // One step ahead: the next columns' products run on the matrix cores while
  // this one's weights are taken.
  f32x4 s[2][4];
  float ref[2];
  int from = 0;
  auto wait = [&](int c) {  // for the columns of step c
    asm volatile("" ::: "memory");
    if (sent - 1 - c >= 1)
      __builtin_amdgcn_s_waitcnt(vmcnt_imm(5));
    else
      __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    asm volatile("" ::: "memory");
  };
  auto products = [&](f32x4(&o)[4], float& l) {
    const Columns& x = ring[wave][from];
#pragma unroll
    for (int h = 0; h < 4; ++h) o[h] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bf16x8 q = as_bf16x8(x.q[i][lane]);
#pragma unroll
      for (int h = 0; h < 4; ++h) o[h] = mfma16(a[h][i], q, o[h]);
    }
    l = x.lse[lane];
  };
  auto add = [&](const f32x4(&x)[4], float l, bool masked, int limit) {
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const f32x4 f = KV == KV_FP8_E4M3FN ? factors[4 * h + kg] : f32x4{p.scale_log2, p.scale_log2, p.scale_log2, p.scale_log2};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(x[h][i], f[i], -l));
        w[h][i] += masked && at + 16 * h + 4 * kg + i >= limit ? 0.0f : e;
      }
    }
  };
  if (count) {
    wait(0);
    products(s[0], ref[0]);
  }
  for (int c0 = 0; c0 < count; c0 += 2) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int c = c0 + u;
      if (c >= count) break;
      from = from == kSumDepth - 1 ? 0 : from + 1;
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the place that the next fetch fills has been read
      if (sent < count) {
        fetch();
        ++sent;
      }
      const int limit = now_tok < g.lq ? min(g.prefix + now_tok + 1, g.lk) : 0;
      now_tok += dt;
      now_hh += dh;
      if (now_hh >= p.group) {
        now_hh -= p.group;
        ++now_tok;
      }
      const bool more = c + 1 < count;
      if (more) wait(c + 1);
      if (!__any(limit < at + kSumKeys) && more) {
        products(s[u ^ 1], ref[u ^ 1]);
        add(s[u], ref[u], false, limit);
      } else {
        if (more) products(s[u ^ 1], ref[u ^ 1]);
        add(s[u], ref[u], true, limit);
      }
    }
  }
#pragma unroll
  for (int h = 0; h < 4; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float e = row_sum16(w[h][i]);
      if (col == 0) sums[wave][16 * h + 4 * kg + i] = e;
    }
  __syncthreads();
  const int token = at + (int)threadIdx.x;
  if (threadIdx.x < kSumKeys && token < g.lk) {
    float e = 0.0f;
#pragma unroll
    for (int v = 0; v < kSumWaves; ++v) e += sums[v][threadIdx.x];
    add_score(p, g, block, off + threadIdx.x, head, token, e);
  }
}

template <int KV>
__global__ void __launch_bounds__(64 * kSumWaves, 2)
score_prefill_kernel(ScoreParams p) {
  const int head = blockIdx.x, r = blockIdx.z;
  int at = blockIdx.y * kSumKeys, off;
  int block = page_of(p, r, at, off);  // inside the tables' width, whatever the row's length
  const Row g = row_of(p, r);
  if (g.lq <= 0) return;
  // 64 keys a workgroup; those of a row with more keys than the launch was sized
  // for (max_k) go round.
  while (at < g.lk) {
    if (block >= 0) weigh_keys<KV>(p, g, head, at, block, off);
    at += gridDim.y * kSumKeys;
    if (at >= g.lk) return;
    block = page_of(p, r, at, off);
    __syncthreads();  // the last keys' sums and factors have been read
  }
}

constexpr int kLseNT = 4;
constexpr int kMostQueries = 1 << 17;  // of a row, where max_q is given
constexpr int kUnbounded = 1 << 15;

struct Plan {
  bool whole;  // decode rows in one launch
  int splits, chunk, tiles, keys;
  size_t logits, partial, lse;
};

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

Plan plan_of(const slo_paged_attention_args* a) {
  Plan n = {false, 1, 1 << 30, 0, 0, 0, 0, 0};
  if (a->num_decode > 0 && (a->phases & SLO_PHASE_DECODE)) {
    const int64_t cap = (int64_t)a->decode_table_width * a->block_size, groups = (int64_t)a->num_decode * a->num_kv_heads;
    const int64_t row = cap * (a->kv_dtype == KV_BF16 ? 256 : a->kv_dtype == KV_FP8_E4M3FN ? 128 : 64);
    n.whole = cap * (a->num_heads / a->num_kv_heads) <= kRowLogits && (groups >= kFullGroups || row < kLongRow);
    const int64_t want = (2048 + groups - 1) / groups;
    int64_t c = ((cap + want - 1) / want + 127) / 128 * 128;
    if (c < 256) c = 256;
    n.chunk = (int)c;
    n.splits = (int)((cap + c - 1) / c);
    if (!n.whole) n.logits = up256((size_t)a->num_decode * a->num_heads * cap * 4);
    if (!n.whole) n.partial = up256((size_t)a->num_decode * a->num_heads * n.splits * 8);
  }
  if (a->num_prefill > 0 && (a->phases & SLO_PHASE_PREFILL) && a->num_q_rows > a->num_decode) {
    // max_q and max_k size the two launches, whose workgroups go round where a
    // row is longer.  Without them the queries and the tables' width bound a row,
    // and a launch has kUnbounded workgroups or 16 a (row, kv head).
    const int per = 16 * kLseNT / (a->num_heads / a->num_kv_heads), all = a->num_q_rows - a->num_decode;
    const int64_t pairs = (int64_t)a->num_prefill * a->num_kv_heads, few = kUnbounded / pairs > 16 ? kUnbounded / pairs : 16;
    const int64_t cap = (int64_t)a->prefill_table_width * a->block_size / kSumKeys;
    const int64_t tiles = ((a->max_q > 0 && a->max_q < all ? a->max_q : all) + per - 1) / per;
    const int64_t keys = a->max_k > 0 ? ((int64_t)a->max_k + kSumKeys - 1) / kSumKeys : few;
    n.tiles = (int)(a->max_q > 0 || tiles < few ? tiles : few);
    n.keys = (int)(keys < cap ? keys : cap);
    n.lse = up256((size_t)all * a->num_heads * 4);
  }
  return n;
}

int check_args(const slo_paged_attention_args* a) {
  if (!a) return fail(SLO_ERR_INVALID, "accumulate_attention: null args");
  if (a->head_dim != HDS) return fail(SLO_ERR_UNSUPPORTED, "accumulate_attention: head_dim must be 128");
  if (a->num_heads <= 0 || a->num_kv_heads <= 0 || a->num_heads % a->num_kv_heads)
    return fail(SLO_ERR_INVALID, "accumulate_attention: num_heads must be a multiple of num_kv_heads");
  if (a->num_heads / a->num_kv_heads > 16)
    return fail(SLO_ERR_UNSUPPORTED, "accumulate_attention: at most 16 query heads per kv head");
  if (a->kv_dtype < KV_BF16 || a->kv_dtype > KV_FP4_E2M1) return fail(SLO_ERR_INVALID, "accumulate_attention: bad kv_dtype");
  if (a->num_q_rows < 0 || a->num_decode < 0 || a->num_prefill < 0 || a->num_decode > a->num_q_rows)
    return fail(SLO_ERR_INVALID, "accumulate_attention: bad row counts");
  if (!(a->softmax_scale != 0.0f) || a->softmax_scale - a->softmax_scale != 0.0f)
    return fail(SLO_ERR_INVALID, "accumulate_attention: softmax_scale must be finite and not zero");
  if (a->num_decode > 32768 || a->num_prefill > 32768)
    return fail(SLO_ERR_UNSUPPORTED, "accumulate_attention: more than 32768 rows");
  const bool dec = a->num_decode > 0 && (a->phases & SLO_PHASE_DECODE);
  const bool pre = a->num_prefill > 0 && (a->phases & SLO_PHASE_PREFILL);
  if (!dec && !pre) return SLO_OK;
  if (!a->q) return fail(SLO_ERR_INVALID, "accumulate_attention: null pointer");
  if ((a->q_row_stride % 8) || a->q_row_stride < a->num_heads * HDS || (reinterpret_cast<uintptr_t>(a->q) % 16))
    return fail(SLO_ERR_INVALID, "accumulate_attention: q rows must be 16-byte aligned");
  if (!a->k_cache || a->num_blocks <= 0) return fail(SLO_ERR_INVALID, "accumulate_attention: no KV pool");
  if (a->kv_dtype != KV_BF16 && !a->k_scale) return fail(SLO_ERR_INVALID, "accumulate_attention: a quantised pool needs k_scale");
  if (reinterpret_cast<uintptr_t>(a->k_cache) % 16)
    return fail(SLO_ERR_INVALID, "accumulate_attention: the pool must be 16-byte aligned");
  if (a->block_size <= 0 || a->block_size % 64)
    return fail(SLO_ERR_UNSUPPORTED, "accumulate_attention: block_size must be a multiple of 64");
  if (pre && a->max_q > kMostQueries) return fail(SLO_ERR_UNSUPPORTED, "accumulate_attention: more than 2^17 queries a row");
  if (dec && (!a->decode_lens || !a->decode_tables || a->decode_table_width <= 0))
    return fail(SLO_ERR_INVALID, "accumulate_attention: missing decode metadata");
  if (pre && (!a->prefill_cu_q || !a->prefill_cu_k || !a->prefill_tables || a->prefill_table_width <= 0))
    return fail(SLO_ERR_INVALID, "accumulate_attention: missing prefill metadata");
  if ((dec && (int64_t)a->decode_table_width * a->block_size > (1 << 21)) ||
      (pre && (int64_t)a->prefill_table_width * a->block_size > (1 << 21)))
    return fail(SLO_ERR_UNSUPPORTED, "accumulate_attention: tables span more than 2^21 tokens");
  return SLO_OK;
}

template <int KV>
void launch(const ScoreParams& d, const ScoreParams& f, const slo_paged_attention_args* a, const Plan& n, hipStream_t s) {
  // Two workgroups fit a CU (64 KiB of logits): where there are few rows, each
  // gets sixteen wavefronts instead of eight.
  if (n.whole && a->num_decode * d.hkv <= 256)
    hipLaunchKernelGGL((score_row_kernel<KV, 16>), dim3(d.hkv, a->num_decode), dim3(1024), 0, s, d);
  else if (n.whole)
    hipLaunchKernelGGL((score_row_kernel<KV, 8>), dim3(d.hkv, a->num_decode), dim3(512), 0, s, d);
  if (n.logits) {
    hipLaunchKernelGGL(score_logits_kernel<KV>, dim3(d.hkv, d.splits, a->num_decode), dim3(256), 0, s, d);
    hipLaunchKernelGGL(score_decode_kernel, dim3(d.hkv, (d.capacity + 1023) / 1024, a->num_decode), dim3(256), 0, s, d);
  }
  if (n.tiles) {
    hipLaunchKernelGGL((score_lse_kernel<KV, kLseNT>), dim3(f.hkv, n.tiles, a->num_prefill), dim3(256), 0, s, f, n.tiles);
    hipLaunchKernelGGL(score_prefill_kernel<KV>, dim3(f.hkv, n.keys, a->num_prefill), dim3(64 * kSumWaves), 0, s, f);
  }
}

}  // namespace
}  // namespace slo

using namespace slo;

extern "C" int slo_accumulate_attention_workspace_bytes(const slo_paged_attention_args* a, size_t* bytes) {
  if (!bytes) return fail(SLO_ERR_INVALID, "accumulate_attention: null pointer");
  const int rc = check_args(a);
  if (rc) return rc;
  const Plan n = plan_of(a);
  *bytes = n.logits + n.partial + n.lse;
  return SLO_OK;
}

extern "C" int slo_accumulate_attention(const slo_paged_attention_args* a, float* scores, slo_stream_t stream) {
  const int rc = check_args(a);
  if (rc) return rc;
  const Plan n = plan_of(a);
  const size_t need = n.logits + n.partial + n.lse;
  if (!need && !n.whole) return SLO_OK;
  if (!scores) return fail(SLO_ERR_INVALID, "accumulate_attention: null pointer");
  if (need && (!a->workspace || a->workspace_bytes < need || reinterpret_cast<uintptr_t>(a->workspace) % 16))
    return fail(SLO_ERR_WORKSPACE, "accumulate_attention: workspace smaller than slo_accumulate_attention_workspace_bytes");
  ScoreParams p = {};
  p.q = static_cast<const uint16_t*>(a->q);
  p.q_stride = a->q_row_stride;
  p.num_q_rows = a->num_q_rows;
  p.kc = static_cast<const uint8_t*>(a->k_cache);
  p.ks = a->k_scale;
  p.num_blocks = a->num_blocks;
  p.block_size = a->block_size;
  p.hq = a->num_heads;
  p.hkv = a->num_kv_heads;
  p.group = a->num_heads / a->num_kv_heads;
  p.scale_log2 = a->softmax_scale * kLog2e;
  p.scores = scores;
  char* ws = static_cast<char*>(a->workspace);
  ScoreParams d = p, f = p;
  d.lens = a->decode_lens;
  d.tables = a->decode_tables;
  d.table_stride = a->decode_table_stride;
  d.table_width = a->decode_table_width;
  d.splits = n.splits;
  d.chunk = n.chunk;
  d.capacity = a->decode_table_width * a->block_size;
  d.logits = reinterpret_cast<float*>(ws);
  d.partial = reinterpret_cast<float2*>(ws + n.logits);
  f.cu_q = a->prefill_cu_q;
  f.cu_k = a->prefill_cu_k;
  f.tables = a->prefill_tables;
  f.table_stride = a->prefill_table_stride;
  f.table_width = a->prefill_table_width;
  f.first_row = a->num_decode;
  f.lse = reinterpret_cast<float*>(ws + n.logits + n.partial);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->kv_dtype == KV_BF16)
    launch<KV_BF16>(d, f, a, n, s);
  else if (a->kv_dtype == KV_FP8_E4M3FN)
    launch<KV_FP8_E4M3FN>(d, f, a, n, s);
  else
    launch<KV_FP4_E2M1>(d, f, a, n, s);
  return check_launch("accumulate_attention");
}
