// Ragged paged attention with a sliding window and a few first tokens that
// stay visible (gfx950).
//
// out[t, h] = sum_j softmax_j(scale q[t, h] . k[j]) v[j] over the keys j that
// the query at position t of its row sees: j <= t and (j > t - window or
// j < sinks).  One pass over those keys with a running maximum and sum per
// (query, head); pages and steps without a visible key are not read, so that a
// row costs what its window does, however long it is.
//
//   S^T = K q^T      A = K (rows: 16 tokens), B = q (columns: 16 queries or heads)
//   O^T += V^T P^T   A = V^T (rows: 16 channels), B = P (columns: the same 16)
//
// Transposed products keep a column's statistics in the lanes that hold its
// scores and outputs.  Lane (c, kg), c = lane % 16 and kg = lane / 16, has of
// each 16 tokens K's channels 32 kg .. 32 kg + 31 of token c (four operands of
// 8), and V's channels 8 c .. 8 c + 7 of tokens 4 kg .. 4 kg + 3, of which two
// v_perm_b32 per channel pair make the operand that has those tokens side by
// side; a lane's scores are of tokens 4 kg .. 4 kg + 3 and are, exponentiated,
// the other operand as they lie.  Codes are converted to bf16 operands exactly
// (E4M3FN scales multiply scores and weights, E8M0 ones go in with the
// conversion).  Only bf16 prefill rows, which need no conversion, have another
// order of the channels, that of their way through LDS.
// Sums, maxima and outputs are fp32 until the one rounding at the end.  Weights
// are rounded to bf16 for the second product: in two terms, which carry them to
// 2^-17, for decode rows, whose outputs are then off by the output's rounding alone
// (0.0016-0.0017 of their size); in one for prefill rows (0.0020-0.0023), where a
// second term would double that product.  Prefill rows divide by the sum of the
// rounded weights (one more row of the second product), so that a weight's rounding
// cancels where one key dominates.
#include "capi_internal.h"
#include "fp4.h"
#include "tile_io.h"
#include <algorithm>
#include <type_traits>

namespace slo {
namespace {

constexpr int RECORD = HD + 4;   // floats of a decode chunk's partial result: outputs, maximum, sum, 2 unused
constexpr float kNone = -1e30f;  // running maximum before the first key
// Largest weight of a prefill lane in a step before its column's reference moves to
// the step's maximum, so that most steps need no maximum over the column: weights
// keep their relative rounding up to there, sums far from overflow.
constexpr float kMost = 224.0f;
// E4M3FN V scales below this count as zero in prefill rows (their reciprocals and the
// weights that they multiply stay in range): values of less than 448 x 2^-100.
constexpr float kSmallScale = 0x1p-100f;
constexpr int NT = 2;            // 16-column blocks of a prefill wavefront
constexpr int kWaves = 4;        // wavefronts that run a tile

// Partial result of a part of a prefill tile, as it lies in the registers of
// its lanes (four channels a piece).
struct Part {
  f32x4 o[kWaves * NT][8][64];
  float m[64 * NT], l[64 * NT];
};

struct WinParams {
  const uint16_t* q;
  int64_t q_stride;
  uint16_t* out;
  int64_t out_stride;
  int num_q_rows;
  const uint8_t *kc, *vc;  // pool, or the step's own rows (no prefill tables)
  const void *ks, *vs;
  int num_blocks, block_size;
  uint32_t tpb, tpb_inv;  // 64-token tiles per block, ceil(2^32 / tpb)
  int hq, hkv, group;
  uint32_t group_inv;  // ceil(2^16 / group)
  float scale_log2;  // |softmax scale| * log2(e)
  uint32_t q_sign;   // 0x80008000 where the scale is negative
  int window, sinks;
  // decode rows
  const int32_t* lens;
  const int32_t* dtables;
  int dstride, dwidth, drows, chunks;
  float* records;  // [rows, kv heads, chunks, group] records
  // prefill rows
  const int32_t* cu_q;
  const int32_t* cu_k;
  const int32_t* ptables;
  int pstride, pwidth, prows, splits, items;
  Part* parts;  // [items, kv heads, splits]
  const uint8_t *rk, *rv;  // without tables: bf16 rows, byte strides
  int64_t rk_stride, rv_stride;
  int num_kv_rows;
  int first_row;  // query row of the first prefill row's first query
  // Query rows from first_idle + (ends ? *ends : 0) on belong to no row (the
  // capacity padding of a captured step) and are given zeros.
  const int32_t* ends;
  int first_idle;
  bool idle;
};

__device__ __forceinline__ void clear_idle(const WinParams& p) {
  const int64_t from = (int64_t)p.first_idle + (p.ends ? max(*p.ends, 0) : 0);
  const int per = p.hq * (HD / 8);  // 16-byte pieces of a row
  const int64_t pieces = (p.num_q_rows - from) * per, stride = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < pieces; i += stride)
    *reinterpret_cast<u32x4*>(p.out + (from + i / per) * p.out_stride + 8 * (i % per)) = u32x4{0, 0, 0, 0};
}

// The steps of T keys that hold what queries at positions [x0, x1] see of a
// row of lk keys: `sink` steps from key 0 on, then those from key `start` on.
struct Span {
  int first, end;  // keys of the window part
  int sink, start, steps;
};
template <int T>
__device__ __forceinline__ Span span_of(const WinParams& p, int x0, int x1, int lk) {
  Span s;
  s.end = max(min(x1 + 1, lk), 0);
  s.first = max(x0 - p.window + 1, 0);
  const int f = s.first / T;
  s.sink = min((min(p.sinks, s.end) + T - 1) / T, f);
  s.start = f * T;
  s.steps = s.sink + max((s.end + T - 1) / T - f, 0);
  // (Said to be uniform, or what follows from them is computed lane by lane.)
  s.first = __builtin_amdgcn_readfirstlane(s.first);
  s.end = __builtin_amdgcn_readfirstlane(s.end);
  s.sink = __builtin_amdgcn_readfirstlane(s.sink);
  s.start = __builtin_amdgcn_readfirstlane(s.start);
  s.steps = __builtin_amdgcn_readfirstlane(s.steps);
  return s;
}
template <int T>
__device__ __forceinline__ int key_of(const Span& s, int i) {
  return i < s.sink ? i * T : s.start + (i - s.sink) * T;
}

// The pool row (token * kv heads, or the head's own token) of a row's key.
__device__ __forceinline__ const __attribute__((address_space(4))) int32_t* scalar(const int32_t* x) {
  return (const __attribute__((address_space(4))) int32_t*)(uintptr_t)x;
}
template <int F>
__device__ __forceinline__ int64_t pool_row(const WinParams& p, const int32_t* table, int head, int key, int& ok) {
  const uint32_t t = (uint32_t)key / 64;
  const int page = p.tpb == 1 ? (int)t : (int)__umulhi(t, p.tpb_inv);
  const int b = scalar(table)[page], off = key - page * p.block_size;
  ok = b >= 0 && b < p.num_blocks;
  const int64_t block = ok ? b : 0;
  if (F == KV_FP4_E2M1) return (block * p.hkv + head) * p.block_size + off;
  return (block * p.block_size + off) * p.hkv + head;
}

// Four operands of a query, channels 32 kg .. 32 kg + 31, or with ROWS 8 kg ..
// 8 kg + 7 of each 32 (zeros where not live):
// the load, and, once what else is to be loaded is on its way, the sign.
template <bool ROWS = false>
__device__ __forceinline__ void load_q(u32x4 (&x)[4], const WinParams& p, int64_t row, int h, int kg, bool live) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = u32x4{0, 0, 0, 0};
  if (live) {
    const uint16_t* from = p.q + row * p.q_stride + h * HD + (ROWS ? 8 : 32) * kg;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = ld16(from + (ROWS ? 32 : 8) * i);
  }
}
__device__ __forceinline__ void operands(bf16x8 (&q)[4], u32x4 (&x)[4], const WinParams& p) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[i][j] ^= p.q_sign;
    q[i] = as_bf16x8(x[i]);
  }
}

// Four tokens' channel pairs as two channels' token quadruples.
__device__ __forceinline__ u32x2 evens(const uint32_t (&w)[4]) {
  return u32x2{__builtin_amdgcn_perm(w[1], w[0], 0x05040100u), __builtin_amdgcn_perm(w[3], w[2], 0x05040100u)};
}
__device__ __forceinline__ u32x2 odds(const uint32_t (&w)[4]) {
  return u32x2{__builtin_amdgcn_perm(w[1], w[0], 0x07060302u), __builtin_amdgcn_perm(w[3], w[2], 0x07060302u)};
}

// ------------------------------------------------------------- decode rows
// A wavefront's steps of T tokens arrive in LDS by non-temporal DMA, two in
// flight, as their lanes fetch them: 16-byte pieces of K's rows in an order
// that spreads the operands' reads over the banks, V's rows as they are.
template <int F> struct Step;
template <> struct Step<KV_BF16> {
  static constexpr int T = 16, LOADS = 8;
  uint8_t k[T * 256], v[T * 256];
};
template <> struct Step<KV_FP8_E4M3FN> {
  static constexpr int T = 32, LOADS = 9;
  uint8_t k[T * 128], v[T * 128];
  float s[2 * T];
};
template <> struct Step<KV_FP4_E2M1> {
  static constexpr int T = 32, LOADS = 5;
  uint8_t k[T * 64], v[T * 64], ks[T * 4], vs[T * 4];
};

template <int F>
__device__ __forceinline__ void fetch(const WinParams& p, int64_t row, uint32_t to, int lane) {
  if constexpr (F == KV_BF16) {
    const uint32_t stride = p.hkv * 256, r = lane >> 4, c = lane & 15;
    const uint8_t *k = p.kc + row * 256, *v = p.vc + row * 256;
#pragma unroll
    for (int i = 0; i < 4; ++i) dma16_nt_at(k, (4 * i + r) * stride + 16 * (c ^ (4 * i + r)), to + 1024 * i);
#pragma unroll
    for (int i = 0; i < 4; ++i) dma16_nt_at(v, (4 * i + r) * stride + 16 * c, to + 4096 + 1024 * i);
  } else if constexpr (F == KV_FP8_E4M3FN) {
    const uint32_t stride = p.hkv * 128, r = lane >> 3, c = lane & 7;
    const uint8_t *k = p.kc + row * 128, *v = p.vc + row * 128;
#pragma unroll
    for (int i = 0; i < 4; ++i) dma16_nt_at(k, (8 * i + r) * stride + 16 * (c ^ r), to + 1024 * i);
#pragma unroll
    for (int i = 0; i < 4; ++i) dma16_nt_at(v, (8 * i + r) * stride + 16 * c, to + 4096 + 1024 * i);
    dma4(static_cast<const float*>(lane < 32 ? p.ks : p.vs) + row + (int64_t)(lane & 31) * p.hkv, to + 8192);
  } else {
    // Of K, 16-byte part x of token t lies at part x ^ (t / 4 mod 4) of its
    // place; of V, token t lies at place t ^ (t / 4 mod 4).
    const uint32_t t = lane >> 2, x = (lane >> 4) & 3;
    const uint32_t ko = t * 64 + ((lane & 3) ^ x) * 16, vo = (t ^ x) * 64 + (lane & 3) * 16;
    const uint8_t *k = p.kc + row * 64, *v = p.vc + row * 64;
    dma16_nt_at(k, ko, to);
    dma16_nt_at(k, ko + 1024, to + 1024);
    dma16_nt_at(v, vo, to + 2048);
    dma16_nt_at(v, vo + 1024, to + 2048 + 1024);
    dma4(static_cast<const uint8_t*>(lane < 32 ? p.ks : p.vs) + row * 4 + (lane & 31) * 4, to + 4096);
  }
}

struct DecodeAcc {
  f32x4 o[8];
  float m, l;  // l: this lane's own tokens
};

// Weights of H x 4 scores (log2 domain) of a lane's tokens; the reference of
// the column moves only where a score passes it by 2^8.
template <int H>
__device__ __forceinline__ void weigh(f32x4 (&s)[H], DecodeAcc& a) {
  float top = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3]));
  if constexpr (H == 2) top = fmaxf(top, fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
  if (__any(top > a.m + 8.0f)) {
    const float m = fmaxf(a.m, col_max(top)), w = __builtin_amdgcn_exp2f(a.m - m);
    a.m = m;
    a.l *= w;
#pragma unroll
    for (int e = 0; e < 8; ++e) a.o[e] *= w;
  }
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[h][i] = __builtin_amdgcn_exp2f(s[h][i] - a.m);
      a.l += s[h][i];
    }
}

// A weight as two bf16 terms, which carry it to 2^-17: the decode steps wait
// for memory, not for the second product.
template <int H>
__device__ __forceinline__ void split(const f32x4 (&e)[H], uint32_t (&hi)[2 * H], uint32_t (&lo)[2 * H]) {
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float x = e[h][2 * i], y = e[h][2 * i + 1];
      const uint32_t w = pack_bf16x2(x, y);
      hi[2 * h + i] = w;
      lo[2 * h + i] = pack_bf16x2(x - __uint_as_float(w << 16), y - __uint_as_float(w & 0xffff0000u));
    }
}

// One landed step: token i of half h of a lane is seen where bit 4 h + i of
// `seen` is set.  (A token that is not seen may be anything in the pages.)
template <int F>
__device__ __forceinline__ void decode_step(const WinParams& p, const Step<F>& st, uint32_t seen, const bf16x8 (&q)[4],
                                            DecodeAcc& a, int lane) {
  constexpr int H = Step<F>::T / 16;
  const int c = lane & 15, kg = lane >> 4;
  const bool masked = __any(seen != (1u << (4 * H)) - 1);
  f32x4 s[H];
  if constexpr (F == KV_BF16) {
    u32x4 k[4], v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) k[i] = ld16(st.k + c * 256 + 16 * ((4 * kg + i) ^ c));
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = ld16(st.v + (4 * kg + i) * 256 + 16 * c);
#pragma unroll
    for (int i = 0; i < 4; ++i) s[0] = mfma16(as_bf16x8(k[i]), q[i], i ? s[0] : f32x4{0, 0, 0, 0});
    s[0] *= p.scale_log2;
    if (masked) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (!(seen >> i & 1)) {
          s[0][i] = -INFINITY;
          v[i] = u32x4{0, 0, 0, 0};
        }
    }
    weigh<1>(s, a);
    uint32_t hi[2], lo[2];
    split<1>(s, hi, lo);
    const s16x4 ph = __builtin_bit_cast(s16x4, u32x2{hi[0], hi[1]}), pl = __builtin_bit_cast(s16x4, u32x2{lo[0], lo[1]});
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const uint32_t w[4] = {v[0][b], v[1][b], v[2][b], v[3][b]};
      const s16x4 e = __builtin_bit_cast(s16x4, evens(w)), o = __builtin_bit_cast(s16x4, odds(w));
      a.o[2 * b] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(e, ph, a.o[2 * b], 0, 0, 0);
      a.o[2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(o, ph, a.o[2 * b + 1], 0, 0, 0);
      a.o[2 * b] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(e, pl, a.o[2 * b], 0, 0, 0);
      a.o[2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(o, pl, a.o[2 * b + 1], 0, 0, 0);
    }
  } else {
    u32x4 v[8];  // 8 channels of 8 tokens: 4 kg + i and 16 + 4 kg + i
    f32x4 vs[2];
    if constexpr (F == KV_FP8_E4M3FN) {
      u32x2 raw[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const u32x4 k = ld16(st.k + (16 * h + c) * 128 + 16 * ((2 * kg + i) ^ (c & 7)));
          s[h] = mfma16(as_bf16x8(fp8x8_to_bf16x8(u32x2{k[0], k[1]})), q[2 * i], i ? s[h] : f32x4{0, 0, 0, 0});
          s[h] = mfma16(as_bf16x8(fp8x8_to_bf16x8(u32x2{k[2], k[3]})), q[2 * i + 1], s[h]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) raw[4 * h + i] = ld8(st.v + (16 * h + 4 * kg + i) * 128 + 8 * c);
      }
      const f32x4* ks = reinterpret_cast<const f32x4*>(st.s);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s[h] *= p.scale_log2 * ks[4 * h + kg];
        vs[h] = ks[8 + 4 * h + kg];
      }
      if (masked) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (!(seen >> j & 1)) {
            raw[j] = u32x2{0, 0};
            vs[j >> 2][j & 3] = 0.0f;
          }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = fp8x8_to_bf16x8(raw[j]);
    } else {
      uint32_t raw[8];
      float sc[8];
      const int turn = (9 + 8 * (c >> 2)) & 31;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u32x4 k = ld16(st.k + h * 1024 + c * 64 + (kg ^ (c >> 2)) * 16);
        const float ks = e8m0(st.ks[h * 64 + c * 4 + kg]);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[h] = mfma16(as_bf16x8(e2m1_decode8(k[i], ks)), q[i], i ? s[h] : f32x4{0, 0, 0, 0});
        s[h] *= p.scale_log2;
        // The conversion reads nothing but the exponent of its scale.
        const u32x4 x = ld16(st.vs + h * 64 + kg * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          raw[4 * h + i] = *reinterpret_cast<const uint32_t*>(st.v + h * 1024 + kg * 256 + (i ^ kg) * 64 + c * 4);
          sc[4 * h + i] = __uint_as_float(__builtin_amdgcn_alignbit(x[i], x[i], turn));
        }
      }
      if (masked) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (!(seen >> j & 1)) sc[j] = 0.0f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = e2m1_decode8(raw[j], sc[j]);
    }
    if (masked) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (!(seen >> j & 1)) s[j >> 2][j & 3] = -INFINITY;
    }
    weigh<2>(s, a);
    if constexpr (F == KV_FP8_E4M3FN) {
      s[0] *= vs[0];
      s[1] *= vs[1];
    }
    uint32_t hi[4], lo[4];
    split<2>(s, hi, lo);
    const bf16x8 ph = as_bf16x8(u32x4{hi[0], hi[1], hi[2], hi[3]}), pl = as_bf16x8(u32x4{lo[0], lo[1], lo[2], lo[3]});
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const uint32_t w0[4] = {v[0][b], v[1][b], v[2][b], v[3][b]}, w1[4] = {v[4][b], v[5][b], v[6][b], v[7][b]};
      const u32x2 e0 = evens(w0), e1 = evens(w1), o0 = odds(w0), o1 = odds(w1);
      const bf16x8 e = as_bf16x8(u32x4{e0.x, e0.y, e1.x, e1.y}), o = as_bf16x8(u32x4{o0.x, o0.y, o1.x, o1.y});
      a.o[2 * b] = mfma16(e, ph, a.o[2 * b]);
      a.o[2 * b + 1] = mfma16(o, ph, a.o[2 * b + 1]);
      a.o[2 * b] = mfma16(e, pl, a.o[2 * b]);
      a.o[2 * b + 1] = mfma16(o, pl, a.o[2 * b + 1]);
    }
  }
}

// A decode row's chunks: `count` of equal steps, no shorter than 256 keys.
template <int F>
struct Chunks {
  Span s;
  int len, count, per;
};
template <int F>
__device__ __forceinline__ Chunks<F> chunks_of(const WinParams& p, int r) {
  constexpr int T = Step<F>::T;
  Chunks<F> c;
  c.len = min(max(scalar(p.lens)[r], 0), p.dwidth * p.block_size);
  c.s = span_of<T>(p, c.len - 1, c.len - 1, c.len);
  c.count = max(1, min(p.chunks, (c.s.steps * T + 255) / 256));
  c.per = (c.s.steps + c.count - 1) / c.count;
  return c;
}

template <int F, int WAVES>
struct DecodeLds {
  union {
    Step<F> steps[2];
    float o[16][HD];
  } ring[WAVES];
  float m[WAVES][16], l[WAVES][16];
};

// One chunk of one (row, kv head) a workgroup, its wavefronts a step each in
// turn, all heads of the group as columns.  Each wavefront fetches its own
// steps, so the loop has no barrier; the wavefronts' results meet in LDS.
// Bound by the read: 64 rows under 1,024 keys and 4 sinks, 8 kv heads of bf16
// (268 MB), 47.5 us or 5.6 TB/s, 47.0 with the arithmetic left out and about 4 of
// them before the first key (length, page, key); E4M3FN 33.9 (32.2); 4 bits under
// 2,048 keys (138 MB) 32.5 (28.6).  Eight wavefronts: bf16 49.4, 4 bits 34; four of
// the 4-bit steps in flight 35.5.
template <int F, int WAVES>
__device__ void decode_item(const WinParams& p, DecodeLds<F, WAVES>& lds, int r, int chunk, int head) {
  constexpr int T = Step<F>::T, H = T / 16;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, kg = lane >> 4;
  u32x4 raw[4];
  load_q(raw, p, r, head * p.group + c, kg, c < p.group);
  const Chunks<F> ch = chunks_of<F>(p, r);
  if (chunk >= ch.count) return;
  bf16x8 q[4];
  operands(q, raw, p);
  const int begin = chunk * ch.per + wave, end = min((chunk + 1) * ch.per, ch.s.steps);
  DecodeAcc a;
#pragma unroll
  for (int e = 0; e < 8; ++e) a.o[e] = f32x4{0, 0, 0, 0};
  a.m = kNone;
  a.l = 0.0f;
  const int steps = end > begin ? (end - begin + WAVES - 1) / WAVES : 0;
  if (steps > 0) {
    const int32_t* table = p.dtables + (int64_t)r * p.dstride;
    const uint32_t ring = lds_addr(&lds.ring[wave]);
    int key[2];   // of the steps in flight; past every key where the page is not in the pool
    auto send = [&](int i) {
      int ok;
      const int k = key_of<T>(ch.s, begin + WAVES * i);
      const int64_t row = pool_row<F>(p, table, head, k, ok);
      fetch<F>(p, row, ring + (i & 1) * (uint32_t)sizeof(Step<F>), lane);
      return ok ? k : ch.len;
    };
    key[1] = send(0);
    for (int i = 0; i < steps; ++i) {
      key[0] = key[1];
      // The place that the next fetch fills was read in the last iteration; its
      // reads have returned.
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
      const bool more = i + 1 < steps;
      if (more) key[1] = send(i + 1);
      asm volatile("" ::: "memory");
      if (more)
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(Step<F>::LOADS));
      else
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
      asm volatile("" ::: "memory");
      uint32_t seen = 0;
#pragma unroll
      for (int j = 0; j < 4 * H; ++j) {
        const int k = key[0] + 16 * (j >> 2) + 4 * kg + (j & 3);
        seen |= (uint32_t)(k < ch.len && (k >= ch.s.first || k < p.sinks)) << j;
      }
      decode_step<F>(p, lds.ring[wave].steps[i & 1], seen, q, a, lane);
    }
  }
  a.l = col_sum(a.l);
  if (c < p.group) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 8; e += 4)
        *reinterpret_cast<f32x4*>(&lds.ring[wave].o[c][32 * kg + 8 * i + e]) =
            f32x4{a.o[e][i], a.o[e + 1][i], a.o[e + 2][i], a.o[e + 3][i]};
    if (kg == 0) {
      lds.m[wave][c] = a.m;
      lds.l[wave][c] = a.l;
    }
  }
  __syncthreads();
  for (int x = threadIdx.x; x < p.group * (HD / 4); x += 64 * WAVES) {
    const int h = x >> 5, d = (x & 31) * 4;
    float m = lds.m[0][h];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) m = fmaxf(m, lds.m[w][h]);
    f32x4 o = {0, 0, 0, 0};
    float l = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float f = __builtin_amdgcn_exp2f(lds.m[w][h] - m);
      o += *reinterpret_cast<const f32x4*>(&lds.ring[w].o[h][d]) * f;
      l += lds.l[w][h] * f;
    }
    if (ch.count == 1) {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      *reinterpret_cast<u32x2*>(p.out + (int64_t)r * p.out_stride + (head * p.group + h) * HD + d) =
          u32x2{pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv)};
    } else {
      float* rec = p.records + ((((int64_t)r * p.hkv + head) * p.chunks + chunk) * p.group + h) * RECORD;
      *reinterpret_cast<f32x4*>(rec + d) = o;
      if (d == 0) {
        rec[HD] = m;
        rec[HD + 1] = l;
      }
    }
  }
}

// ------------------------------------------------------------ prefill rows
// One 64-token step of a workgroup in LDS.  Quantised: as bf16 operands in the
// order in which lanes read them (16 bytes a lane, no bank twice): K's four
// operands of each 16 tokens, V's eight of each 32 tokens, and E4M3FN's scales.
template <int F>
struct Stage {
  u32x4 k[4][4][64], v[2][8][64];
};
template <> struct Stage<KV_FP8_E4M3FN> {
  u32x4 k[4][4][64], v[2][8][64];
  float s[2][64];
  uint16_t r[3][64];  // 1 / V scale as three bf16 terms
};
// bf16 needs no conversion: rows as they are, sent there by the memory system in
// whole rows, 16-byte part x of token t at part x ^ (t mod 16) so that no read has
// a bank twice, V turned as it is read.  (By way of registers, a lane 64 bytes of a
// K row and 16 of four V rows, 4,096 queries under 4,096 keys took 276 us for 258, cold
// rows of 7,733 tokens 149 for 137, 24 decode rows and two chunks of 512 28.9 for 26.5.)
template <> struct Stage<KV_BF16> {
  u32x4 k[64][16], v[64][16];
};

// A wavefront's quarter of a step, 16 tokens, as loaded.
template <int F> struct Quarter {};
template <> struct Quarter<KV_FP8_E4M3FN> {
  u32x4 k[2];
  u32x2 v[4];
  float ks, vs;  // of token c
};
template <> struct Quarter<KV_FP4_E2M1> {
  u32x4 k, vs;
  uint32_t ks, v[4];
};

// x / group of a tile's column (x < 64).
__device__ __forceinline__ int by_group(const WinParams& p, int x) { return x * p.group_inv >> 16; }

struct PrefillRow {
  int q0;  // first query row of the row
  int lq, lk, prefix, k0;
};

__device__ __forceinline__ PrefillRow prefill_row(const WinParams& p, int r) {
  PrefillRow g;
  const int start = p.cu_q[r], k0 = p.cu_k[r], k = p.cu_k[r + 1] - k0;
  g.q0 = p.first_row + start;
  g.lq = p.cu_q[r + 1] - start;
  g.prefix = k - g.lq;
  g.k0 = k0;
  g.lk = p.ptables ? min(k, p.pwidth * p.block_size) : k0 < 0 ? 0 : min(k, p.num_kv_rows - k0);
  if (start < 0 || (int64_t)g.q0 + g.lq > p.num_q_rows) g.lq = 0;
  return g;
}

// Byte offsets of a lane's pieces (of V, of the first of its four tokens) from
// its step's first token: the same at every step, so that a load is a uniform
// base and one of these.
template <int F> struct Lanes {
  uint32_t k, v;
};
template <> struct Lanes<KV_BF16> {
  int k[4], v[4];  // of tokens kg, kg + 4, .. of 16, whole rows by 16 lanes (see dma16x4_at)
};
template <int F>
__device__ __forceinline__ Lanes<F> lanes_of(const WinParams& p, int wave, int lane) {
  const uint32_t c = lane & 15, kg = lane >> 4, row = F == KV_BF16 ? 256 : F == KV_FP8_E4M3FN ? 128 : 64;
  const uint32_t stride = F == KV_FP4_E2M1 ? row : p.hkv * row;
  Lanes<F> l;
  if constexpr (F == KV_BF16) {
    const uint32_t ks = p.ptables ? stride : (uint32_t)p.rk_stride, vs = p.ptables ? stride : (uint32_t)p.rv_stride;
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // (a row is 256 bytes or more from the next: none is negative)
      const uint32_t t = 16 * wave + 4 * i + kg, part = 16 * (c ^ (4 * i + kg));
      l.k[i] = t * ks + part - 1024 * i;
      l.v[i] = t * vs + part - 1024 * i;
    }
  } else {
    l.k = (16 * wave + c) * stride + kg * (row / 4);
    l.v = (16 * wave + 4 * kg) * stride + c * (row / 16);
  }
  return l;
}

// A load at a uniform base plus a lane's 32-bit offset.  (The offset is found
// again at each step: extended to 64 bits before the loop, it would take two
// registers and the load a lane address.)
template <typename T>
__device__ __forceinline__ T load(const void* base, uint32_t off, int more = 0) {
  asm("" : "+v"(off));
  return *reinterpret_cast<const T*>(static_cast<const uint8_t*>(base) + off + more);
}

// This wavefront's 16 of the 64 tokens from `key` on, bf16, straight to LDS.
__device__ __forceinline__ void send_quarter(Stage<KV_BF16>& s, const WinParams& p, const PrefillRow& g, const int32_t* table,
                                             int head, int key, const Lanes<KV_BF16>& l, int wave, int lane, int& ok) {
  const uint32_t tk = lds_addr(&s.k[16 * wave]), tv = lds_addr(&s.v[16 * wave]);
  const uint8_t *k, *v;
  ok = true;
  if (p.ptables) {
    const int64_t row = pool_row<KV_BF16>(p, table, head, key, ok);
    k = p.kc + row * 256;
    v = p.vc + row * 256;
  } else {
    const int64_t row = (int64_t)g.k0 + key;
    k = p.rk + row * p.rk_stride + head * 256;
    v = p.rv + row * p.rv_stride + head * 256;
    const int last = g.lk - 1 - key;
    if (last < 63) {  // nothing is read past the rows' end
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int x = 4 * i + (lane >> 4), part = 16 * ((lane & 15) ^ x);
        const uint32_t t = min(16 * wave + x, last);
        dma16(k + t * (uint32_t)p.rk_stride + part, tk + 1024 * i);
        dma16(v + t * (uint32_t)p.rv_stride + part, tv + 1024 * i);
      }
      return;
    }
  }
  dma16x4_at(k, l.k, tk);
  dma16x4_at(v, l.v, tv);
}

// This wavefront's 16 of the 64 tokens from `key` on.
template <int F>
__device__ __forceinline__ void load_quarter(Quarter<F>& t, const WinParams& p, const int32_t* table, int head, int key,
                                             const Lanes<F>& l, int wave, int lane, int& ok) {
  const int c = lane & 15, kg = lane >> 4;
  if constexpr (F == KV_FP8_E4M3FN) {
    const int64_t row = pool_row<F>(p, table, head, key, ok);
    const uint8_t *k = p.kc + row * 128, *v = p.vc + row * 128;
#pragma unroll
    for (int i = 0; i < 2; ++i) t.k[i] = load<u32x4>(k, l.k, 16 * i);
#pragma unroll
    for (int i = 0; i < 4; ++i) t.v[i] = load<u32x2>(v + i * (uint32_t)(p.hkv * 128), l.v);
    const uint32_t at = 4 * (16 * wave + c) * p.hkv;
    t.ks = load<float>(static_cast<const float*>(p.ks) + row, at);
    t.vs = load<float>(static_cast<const float*>(p.vs) + row, at);
  } else {
    const int64_t row = pool_row<F>(p, table, head, key, ok);
    const uint8_t *ks = static_cast<const uint8_t*>(p.ks) + row * 4, *vs = static_cast<const uint8_t*>(p.vs) + row * 4;
    t.k = load<u32x4>(p.kc + row * 64, l.k);
    t.ks = load<uint8_t>(ks, 64 * wave + c * 4 + kg);
    t.vs = load<u32x4>(vs, 64 * wave + kg * 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) t.v[i] = load<uint32_t>(p.vc + row * 64, l.v, 64 * i);
  }
}

// Clears the V tokens that none of the tile's queries sees, of a step from
// `key` on that may hold some.  They may be anything in the pages, and a weight
// of zero must not make that a NaN.
__device__ __forceinline__ void clear_unseen(Stage<KV_BF16>& s, int key, int first, int end, int sinks, int wave, int lane) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = 16 * wave + 4 * i + (lane >> 4), k = key + t;
    if (!((k < end) & ((k >= first) | (k < sinks)))) s.v[t][lane & 15] = u32x4{0, 0, 0, 0};
  }
}
template <int F>
__device__ __forceinline__ void clear_unseen(Quarter<F>& t, int key, int first, int end, int sinks, int wave, int lane) {
  const int k = key + 16 * wave + 4 * (lane >> 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool seen = (k + i < end) & ((k + i >= first) | (k + i < sinks));
    if constexpr (F == KV_FP8_E4M3FN) {
      t.v[i] = seen ? t.v[i] : u32x2{0, 0};
    } else {
      t.vs[i] = seen ? t.vs[i] : 0;
    }
  }
  if constexpr (F == KV_FP8_E4M3FN) {
    const int k = key + 16 * wave + (lane & 15);
    if (!((k < end) & ((k >= first) | (k < sinks)))) t.vs = 1.0f;
  }
}

template <int F>
__device__ __forceinline__ void stage(Stage<F>& s, const Quarter<F>& t, int wave, int lane) {
  const int c = lane & 15;
  u32x4 v[4];
  if constexpr (F == KV_FP8_E4M3FN) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s.k[wave][2 * i][lane] = fp8x8_to_bf16x8(u32x2{t.k[i][0], t.k[i][1]});
      s.k[wave][2 * i + 1][lane] = fp8x8_to_bf16x8(u32x2{t.k[i][2], t.k[i][3]});
    }
    u32x2 codes[4] = {t.v[0], t.v[1], t.v[2], t.v[3]};
    float vs = t.vs;
    const bool small = __builtin_fabsf(vs) < kSmallScale;
    if (__any(small)) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (__shfl((int)small, 4 * (lane >> 4) + i)) codes[i] = u32x2{0, 0};
      if (small) vs = 1.0f;
    }
    if (lane < 16) {
      s.s[0][16 * wave + c] = t.ks;
      s.s[1][16 * wave + c] = vs;
      float rest = __builtin_amdgcn_rcpf(vs);
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        const uint32_t term = pack_bf16x2(rest, 0.0f);
        s.r[i][16 * wave + c] = (uint16_t)term;
        rest -= __uint_as_float(term << 16);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = fp8x8_to_bf16x8(codes[i]);
  } else {
    const float sc = e8m0(t.ks);
#pragma unroll
    for (int i = 0; i < 4; ++i) s.k[wave][i][lane] = e2m1_decode8(t.k[i], sc);
    const int turn = (9 + 8 * (c >> 2)) & 31;  // the lane's scale byte to the exponent's place
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = e2m1_decode8(t.v[i], __uint_as_float(__builtin_amdgcn_alignbit(t.vs[i], t.vs[i], turn)));
  }
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const uint32_t w[4] = {v[0][b], v[1][b], v[2][b], v[3][b]};
    reinterpret_cast<u32x2*>(&s.v[wave >> 1][2 * b][lane])[wave & 1] = evens(w);
    reinterpret_cast<u32x2*>(&s.v[wave >> 1][2 * b + 1][lane])[wave & 1] = odds(w);
  }
}

// K's operand i of 16 tokens t, V's operand i of 32 tokens g.  (bf16 K's channels
// are 32 i + 8 kg on: with 32 kg + 8 i lanes that are served together meet a bank
// twice, a third of LDS's time.)
template <int F>
__device__ __forceinline__ bf16x8 k_operand(const Stage<F>& s, int t, int i, int lane) {
  if constexpr (F == KV_BF16) return as_bf16x8(s.k[16 * t + (lane & 15)][(4 * i + (lane >> 4)) ^ (lane & 15)]);
  else return as_bf16x8(s.k[t][i][lane]);
}
template <int F>
__device__ __forceinline__ bf16x8 v_operand(const Stage<F>& s, int g, int i, int lane) {
  if constexpr (F == KV_BF16) {
    // The lanes of a column group read 4 tokens' 8 channels at 8 i and 64 + 8 i
    // and receive a channel's 4 tokens each.
    const int t = 4 * (lane >> 4) + ((lane & 15) >> 2), x = (4 * (lane & 2) + i) ^ t;
    const uint8_t* from = reinterpret_cast<const uint8_t*>(&s.v[32 * g + t][x]) + 8 * (lane & 1);
    return join_tr(lds_tr16(from), lds_tr16(from + 16 * 256));
  } else {
    return as_bf16x8(s.v[g][i][lane]);
  }
}

// The row of the second product that sums 32 tokens' weights, as they were rounded
// for it: ones, or for E4M3FN, whose weights carry V's scales, the scales'
// reciprocals, a term in each of the first three rows.  us against lanes' own sums of
// the unrounded weights: 4,096 queries under 4,096 keys 252.6 / 250.0, cold rows of
// 7,733 tokens 126.9 / 126.4, three E4M3FN chunks of 1,377 38.0 / 36.8, 24 decode rows
// and two chunks of 512 24.2 / 24.2 (260.4, 128.4, 37.8 and 24.5 with those sums kept
// for the test of the reference, which takes the largest weight instead).
template <int F>
__device__ __forceinline__ bf16x8 sum_operand(const Stage<F>& s, int g, int lane) {
  if constexpr (F == KV_FP8_E4M3FN) {
    const int c = lane & 15, t = 32 * g + 4 * (lane >> 4);
    const u32x2 x = ld8(&s.r[c < 3 ? c : 0][t]), y = ld8(&s.r[c < 3 ? c : 0][t + 16]);
    return as_bf16x8(c < 3 ? u32x4{x.x, x.y, y.x, y.y} : u32x4{0, 0, 0, 0});
  } else {
    return as_bf16x8(u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});
  }
}

struct Acc {
  f32x4 o[NT][8];
  f32x4 l[NT];    // sums of the rounded weights (see sum_operand): four times, or in its first rows
  float ncm[NT];  // minus the reference in the log2 domain (+inf before the first key)
};
// A column's sum, in each of its lanes.
template <int F>
__device__ __forceinline__ float column_sum(const f32x4& l) {
  return F == KV_FP8_E4M3FN ? col_sum(l[0] + l[1] + l[2]) : l[0];
}

// 64 tokens from `key` on of a wavefront's columns against the staged operands,
// read four ahead of the products.  A wavefront at its score products goes before
// the other one of its SIMD, so that the two do not fall into step (4,096 queries
// under 4,096 keys 252 us; without priorities 264).  at[n]: position of
// column block n's query; keys from `kend` on are not the row's.  A step before the
// window part (`sink`) shows a query nothing but sinks.
template <int F>
__device__ __forceinline__ void staged_step(const WinParams& p, const Stage<F>& st, bool masked, bool sink, const bf16x8 (&q)[NT][4],
                                            Acc& a, int key, const int (&at)[NT], int kend, int lane) {
  const int kg = lane >> 4;
  __builtin_amdgcn_s_setprio(1);
  f32x4 s[NT][4];
  bf16x8 x[2][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[0][i] = k_operand<F>(st, 0, i, lane);
#pragma unroll
  for (int t = 0; t < 4; ++t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[(t + 1) & 1][i] = t < 3 ? k_operand<F>(st, t + 1, i, lane) : v_operand<F>(st, 0, i, lane);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n][t] = mfma16(x[t & 1][i], q[n][i], i ? s[n][t] : f32x4{0, 0, 0, 0});
    __builtin_amdgcn_sched_barrier(0);
  }
  __builtin_amdgcn_s_setprio(0);
  // A reference that is too low shows in the largest of a lane's weights (inf or
  // NaN while it is unset).  Only then are the columns' maxima found and the
  // weights taken again.
  const float c = p.scale_log2;
  const int few = sink ? 0 : p.sinks - key;  // sinks among the window part's keys
  // Column blocks are taken together (4,096 queries under 4,096 keys 252 us, one after
  // the other 254, cold rows of 7,733 tokens 124 and 128, 960 queries under 1,024 keys
  // 29.7 and 30.8, on a 4-bit pool the same); E4M3FN's scales leave no registers for it.
  constexpr int COLS = F == KV_FP8_E4M3FN ? 1 : NT;
  bf16x8 pr[NT][2];
#pragma unroll
  for (int n0 = 0; n0 < NT; n0 += COLS) {
#pragma unroll
    for (int n = n0; n < n0 + COLS; ++n) {
      if constexpr (F == KV_FP8_E4M3FN) {
#pragma unroll
        for (int t = 0; t < 4; ++t) s[n][t] *= *reinterpret_cast<const f32x4*>(&st.s[0][16 * t + 4 * kg]);
      }
      if (!masked) continue;
      const int hi = min(at[n], (sink ? min(kend, p.sinks) : kend) - 1) - key - 4 * kg;
      const int lo = (sink ? 0 : max(at[n] - p.window + 1 - key, 0)) - 4 * kg;
      if (few <= 0) {
        const uint32_t span = max(hi - lo + 1, 0), from = -lo;  // tokens below lo wrap past every span
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][t][i] = from + (16 * t + i) < span ? s[n][t][i] : -INFINITY;
      } else {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int k = 16 * t + i;
            s[n][t][i] = (k <= hi) & ((k >= lo) | (k < few - 4 * kg)) ? s[n][t][i] : -INFINITY;
          }
      }
    }
    f32x4 e[COLS][4];
    auto exponents = [&](int n, float ncm) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) e[n - n0][t][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][t][i], c, ncm));
    };
    bool low = false;
#pragma unroll
    for (int n = n0; n < n0 + COLS; ++n) {
      exponents(n, a.ncm[n]);
      const f32x4(&x)[4] = e[n - n0];
      float top = x[0][0];
#pragma unroll
      for (int i = 1; i < 15; i += 2) top = fmaxf(fmaxf(top, x[i >> 2][i & 3]), x[(i + 1) >> 2][(i + 1) & 3]);
      top = fmaxf(top, x[3][3]);
      low |= !(top <= kMost);
    }
    if (__any(low)) {
#pragma unroll
      for (int n = n0; n < n0 + COLS; ++n) {
        float top = s[n][0][0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, s[n][i >> 2][i & 3]);
        const float next = fminf(a.ncm[n], -c * col_max(top)), use = next == INFINITY ? 0.0f : next;  // no key yet: weights of zero
        const float w = __builtin_amdgcn_exp2f(use - a.ncm[n]);
        exponents(n, use);
        a.l[n] *= w;
#pragma unroll
        for (int i = 0; i < 8; ++i) a.o[n][i] *= w;
        a.ncm[n] = next;
      }
    }
#pragma unroll
    for (int n = n0; n < n0 + COLS; ++n) {
      f32x4(&x)[4] = e[n - n0];
      if constexpr (F == KV_FP8_E4M3FN) {
#pragma unroll
        for (int t = 0; t < 4; ++t) x[t] *= *reinterpret_cast<const f32x4*>(&st.s[1][16 * t + 4 * kg]);
      }
#pragma unroll
      for (int g = 0; g < 2; ++g)
        pr[n][g] = as_bf16x8(u32x4{pack_bf16x2(x[2 * g][0], x[2 * g][1]), pack_bf16x2(x[2 * g][2], x[2 * g][3]),
                                   pack_bf16x2(x[2 * g + 1][0], x[2 * g + 1][1]), pack_bf16x2(x[2 * g + 1][2], x[2 * g + 1][3])});
    }
    __builtin_amdgcn_sched_barrier(0);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {  // V's operands, four at a time
    const int g = j >> 1;
    if (j < 3) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[(j + 1) & 1][i] = v_operand<F>(st, (j + 1) >> 1, 4 * ((j + 1) & 1) + i, lane);
    }
    const bf16x8 ones = sum_operand<F>(st, g, lane);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n) a.o[n][4 * (j & 1) + i] = mfma16(x[j & 1][i], pr[n][g], a.o[n][4 * (j & 1) + i]);
    if (j & 1) {
#pragma unroll
      for (int n = 0; n < NT; ++n) a.l[n] = mfma16(ones, pr[n][g], a.l[n]);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Item i's row and tile: the rows' tiles in order, each row's last one (the
// longest, where the window has not filled) first.
__device__ __forceinline__ bool find_tile(const WinParams& p, int per, int item, int lane, int& row, int& tile, PrefillRow& g) {
  int before = 0;
  for (int base = 0; base < p.prows; base += 64) {
    int n = 0;
    PrefillRow x = {};
    if (base + lane < p.prows) {
      x = prefill_row(p, base + lane);
      n = x.lq > 0 ? (int)((uint32_t)(x.lq + per - 1) / (uint32_t)per) : 0;
    }
    const int upto = wave_scan(n);
    const uint64_t past = __ballot(before + upto > item);
    if (past) {
      const int at = __builtin_amdgcn_readfirstlane(__builtin_ctzll(past));
      auto of = [&](int v) { return __builtin_amdgcn_readfirstlane(__builtin_amdgcn_readlane(v, at)); };
      row = __builtin_amdgcn_readfirstlane(base + at);
      tile = __builtin_amdgcn_readfirstlane(before + __builtin_amdgcn_readlane(upto, at) - 1 - item);
      g.q0 = of(x.q0);
      g.lq = of(x.lq);
      g.lk = of(x.lk);
      g.prefix = of(x.prefix);
      g.k0 = of(x.k0);
      return true;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

// What a second half of a workgroup leaves for the first.
struct Half {
  f32x4 o[kWaves][NT][8][64];
  float ncm[kWaves][NT][64], l[kWaves][NT][64];
};
template <int F, int HALVES>
union PrefillLds {
  Stage<F> st[HALVES][2];
  std::conditional_t<HALVES == 2, Half, char> half;
};

// Tile `item`, part `part` of its steps, kv head `head`.  Four wavefronts turn a
// step into operands together, a quarter each, and each runs 16 NT columns,
// (query, head of the group) pairs of consecutive queries, over them; the next
// step loads meanwhile.  With two halves of four wavefronts each half takes
// every other step.  4,096 queries of 32 heads under 4,096 keys run 250-264 us by the
// card, 1,050-1,100 TFLOP/s (a library product of 8,192^3: 1,406): matrix cores and lane
// operations (exponents, masks, packing) are busy about half of the time each and the
// two wavefronts of a SIMD hardly overlap them.  Weights taken between the products,
// one by one, came to the same (258 for 260 before the sums' row; E4M3FN rows 36 for
// 39, mixed steps 28 for 26), pages looked up a step ahead too; four column blocks a
// wavefront and one wavefront a SIMD took twice as long.  A launch of few steps mostly waits: 2.5 us
// to the tile, 3.2 for queries and output, 2.5 for page and first keys, 2.8 for the
// first step, 1 of them for the first maximum.
template <int F, int HALVES>
__device__ void prefill_item(const WinParams& p, PrefillLds<F, HALVES>& lds, int item, int part, int head) {
  const int lane = threadIdx.x & 63, any = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = any & (kWaves - 1), half = any / kWaves;
  const int c = lane & 15, kg = lane >> 4;
  const int each = by_group(p, 16 * NT), per = kWaves * each;  // queries of a wavefront, of a tile
  int r = 0, tile = 0;
  PrefillRow g;
  if (!find_tile(p, per, item, lane, r, tile, g)) return;
  const int w0 = tile * per, w1 = min(w0 + per, g.lq);
  const Span s = span_of<64>(p, g.prefix + w0, g.prefix + w1 - 1, g.lk);
  // (At most 2^18 steps, 512 parts.)
  const int from = __builtin_amdgcn_readfirstlane((uint32_t)s.steps * part / p.splits);
  const int to = __builtin_amdgcn_readfirstlane((uint32_t)s.steps * (part + 1) / p.splits);
  // Queries of this wavefront [t0, t1); columns past them repeat the last one's
  // mask with a query of zeros.
  const int t0 = min(w0 + wave * each, w1 - 1), t1 = max(min(w0 + wave * each + each, w1), t0 + 1);
  int at[NT];
  u32x4 raw[NT][4];
  Acc a;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int x = 16 * n + c, y = by_group(p, x), tok = w0 + wave * each + y;
    at[n] = g.prefix + min(tok, t1 - 1);
    load_q<F == KV_BF16>(raw[n], p, g.q0 + tok, head * p.group + x - y * p.group, kg, y < each && tok < w1);
#pragma unroll
    for (int i = 0; i < 8; ++i) a.o[n][i] = f32x4{0, 0, 0, 0};
    a.ncm[n] = INFINITY;
    a.l[n] = f32x4{0, 0, 0, 0};
  }
  if (from < to) {
    const int32_t* table = p.ptables ? p.ptables + (int64_t)r * p.pstride : nullptr;
    const int x0 = g.prefix + t0, x1 = g.prefix + t1 - 1;
    const Lanes<F> lanes = lanes_of<F>(p, wave, lane);
    Quarter<F> t;
    int in = 0;
    auto get = [&](int i, int to_buffer) {
      if constexpr (F == KV_BF16) send_quarter(lds.st[half][to_buffer], p, g, table, head, key_of<64>(s, i), lanes, wave, lane, in);
      else load_quarter<F>(t, p, table, head, key_of<64>(s, i), lanes, wave, lane, in);
    };
    if (from + half < to) get(from + half, 0);
    bf16x8 q[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) operands(q[n], raw[n], p);
    for (int i = from + half; i < to + half; i += HALVES) {
      const int buffer = (i - from) / HALVES & 1;
      Stage<F>& st = lds.st[half][buffer];
      const bool mine = HALVES == 1 || i < to;  // the last turn may have steps for one half only
      const int key = key_of<64>(s, i);
      const int ok = in;  // whether the step's page is in the pool
      if (mine) {
        const bool unseen = !ok || key + 64 > s.end || (key < s.first && key + 64 > p.sinks);
        if constexpr (F == KV_BF16) {
          __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // this wavefront's quarter has come
          if (unseen) clear_unseen(st, key, s.first, ok ? s.end : 0, p.sinks, wave, lane);
        } else {
          if (unseen) clear_unseen<F>(t, key, s.first, ok ? s.end : 0, p.sinks, wave, lane);
          stage<F>(st, t, wave, lane);
          if (i + HALVES < to) get(i + HALVES, 0);
        }
      }
      // Two buffers: a wavefront comes to fill this one again only past the
      // next step's barrier, when every wavefront has left it.  The barrier
      // waits for LDS only: the loads of the next step stay in flight.
      lds_sync();
      if (mine) {
        if constexpr (F == KV_BF16) {
          if (i + HALVES < to) get(i + HALVES, buffer ^ 1);
        }
        const bool all = ok && key + 63 <= x0 && key + 64 <= g.lk && (key > x1 - p.window || key + 64 <= p.sinks);
        staged_step<F>(p, st, !all, i < s.sink, q, a, key, at, ok ? g.lk : 0, lane);
      }
    }
  }
  float l[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) l[n] = column_sum<F>(a.l[n]);
  if constexpr (HALVES == 2) {
    Half& h = lds.half;
    __syncthreads();
    if (half == 1) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 8; ++e) h.o[wave][n][e][lane] = a.o[n][e];
        h.ncm[wave][n][lane] = a.ncm[n];
        h.l[wave][n][lane] = l[n];
      }
    }
    __syncthreads();
    if (half == 1) return;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float other = h.ncm[wave][n][lane], ncm = fminf(a.ncm[n], other);
      const float mine = a.ncm[n] == INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ncm - a.ncm[n]);
      const float w = other == INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ncm - other);
      a.ncm[n] = ncm;
      l[n] = l[n] * mine + h.l[wave][n][lane] * w;
#pragma unroll
      for (int e = 0; e < 8; ++e) a.o[n][e] = a.o[n][e] * mine + h.o[wave][n][e][lane] * w;
    }
  }
  int col = lane & 15;
  asm("" : "+v"(col));  // found again here, so that the loop need not hold what follows from it in registers
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if (p.splits == 1) {
      const int x = 16 * n + col, y = by_group(p, x), tok = w0 + wave * each + y, h = head * p.group + x - y * p.group;
      const bool live = y < each && tok < w1;
      const float inv = l[n] == 0.0f ? 0.0f : 1.0f / l[n];
      uint16_t* out = p.out + (int64_t)(g.q0 + tok) * p.out_stride + h * HD;
      if constexpr (F == KV_BF16) {
        // A lane's 4 channels at 64 (kg / 2) + 8 e + 4 (kg mod 2): lanes of
        // neighbouring kg exchange theirs of two e.
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const f32x4 v = a.o[n][e] * inv, w = a.o[n][e + 1] * inv;
          const auto x = __builtin_amdgcn_permlane16_swap(pack_bf16x2(v[0], v[1]), pack_bf16x2(w[0], w[1]), false, false);
          const auto y = __builtin_amdgcn_permlane16_swap(pack_bf16x2(v[2], v[3]), pack_bf16x2(w[2], w[3]), false, false);
          if (live) *reinterpret_cast<u32x4*>(out + 64 * (kg >> 1) + 8 * (e + (kg & 1))) = u32x4{x[0], y[0], x[1], y[1]};
        }
        continue;
      }
      if (!live) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<u32x4*>(out + 32 * kg + 8 * i) =
            u32x4{pack_bf16x2(a.o[n][0][i] * inv, a.o[n][1][i] * inv), pack_bf16x2(a.o[n][2][i] * inv, a.o[n][3][i] * inv),
                  pack_bf16x2(a.o[n][4][i] * inv, a.o[n][5][i] * inv), pack_bf16x2(a.o[n][6][i] * inv, a.o[n][7][i] * inv)};
    } else {
      Part& out = p.parts[((int64_t)item * p.hkv + head) * p.splits + part];
      const int block = NT * wave + n;
      if constexpr (F == KV_BF16) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          out.o[block][2 * (e & 3) + (kg & 1)][col + 16 * (2 * (kg >> 1) + (e >> 2))] = a.o[n][e];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 8; e += 4)
            out.o[block][2 * i + (e >> 2)][lane] = f32x4{a.o[n][e][i], a.o[n][e + 1][i], a.o[n][e + 2][i], a.o[n][e + 3][i]};
      }
      if (kg == 0) {
        out.m[16 * block + col] = a.ncm[n] == INFINITY ? kNone : -a.ncm[n];
        out.l[16 * block + col] = l[n];
      }
    }
  }
}

// Both phases in one launch, prefill items first.
template <int F, int HALVES>
__global__ void __launch_bounds__(64 * kWaves * HALVES, 2)
window_attention_kernel(WinParams p) {
  __shared__ union {
    PrefillLds<F, HALVES> pre;
    DecodeLds<F, kWaves * HALVES> dec;
  } lds;
  // (Quotients are said to be uniform, or what follows from them is computed
  // lane by lane.)
  auto div = [](uint32_t x, uint32_t y) { return (int)__builtin_amdgcn_readfirstlane(x / y); };
  int i = div(blockIdx.x, p.hkv);
  const int head = blockIdx.x - i * p.hkv, prefill = p.items * p.splits;
  if (i < prefill) {
    const int item = div(i, p.splits);
    prefill_item<F, HALVES>(p, lds.pre, item, i - item * p.splits, head);
  } else {
    i -= prefill;
    const int r = div(i, p.chunks);
    decode_item<F, kWaves * HALVES>(p, lds.dec, r, i - r * p.chunks, head);
  }
  if (p.idle) clear_idle(p);
}

// Decode rows alone.
template <int F>
__global__ void __launch_bounds__(64 * kWaves, 2)
window_decode_kernel(WinParams p) {
  __shared__ DecodeLds<F, kWaves> lds;
  auto div = [](uint32_t x, uint32_t y) { return (int)__builtin_amdgcn_readfirstlane(x / y); };
  const int i = div(blockIdx.x, p.hkv), r = div(i, p.chunks);
  decode_item<F, kWaves>(p, lds, r, i - r * p.chunks, blockIdx.x - i * p.hkv);
  if (p.idle) clear_idle(p);
}

// Joins the chunks of decode row r, query head h: half wavefront i takes chunks
// i, i + 8, ..., four channels a lane, and the eight sums meet in LDS in order.
template <int F>
__device__ __forceinline__ void join_decode(const WinParams& p, int r, int h) {
  __shared__ f32x4 so[8][32];
  __shared__ float sl[8];
  const int lane = threadIdx.x & 31, i = threadIdx.x >> 5, head = h / p.group;
  const int count = chunks_of<F>(p, r).count;
  if (count == 1) return;  // written by its only chunk
  const float* rec = p.records + (((int64_t)r * p.hkv + head) * p.chunks * p.group + h - head * p.group) * RECORD;
  const int64_t stride = (int64_t)p.group * RECORD;
  float m = kNone;
  for (int s = lane; s < count; s += 32) m = fmaxf(m, rec[s * stride + HD]);
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) m = wave_max_xor(m, d);
  f32x4 o = {0, 0, 0, 0};
  float l = 0;
#pragma unroll 4
  for (int s = i; s < count; s += 8) {
    const float* e = rec + s * stride;
    const float w = __builtin_amdgcn_exp2f(e[HD] - m);
    o += *reinterpret_cast<const f32x4*>(e + 4 * lane) * w;
    l += e[HD + 1] * w;
  }
  so[i][lane] = o;
  if (lane == 0) sl[i] = l;
  __syncthreads();
  if (i) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) {
    o += so[k][lane];
    l += sl[k];
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  *reinterpret_cast<u32x2*>(p.out + (int64_t)r * p.out_stride + h * HD + 4 * lane) =
      u32x2{pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv)};
}

// Joins the chunks of decode rows (workgroups below `decode`, one per row and
// query head) and the parts of prefill tiles (one per item, kv head and 16
// columns).
template <int F>
__global__ void __launch_bounds__(256)
window_join_kernel(WinParams p, int decode) {
  int i = blockIdx.x;
  if (i < decode) {
    const int r = i / p.hq;
    join_decode<F>(p, r, i - r * p.hq);
    return;
  }
  i -= decode;
  const int block = i % (kWaves * NT), head = i / (kWaves * NT) % p.hkv, item = i / (kWaves * NT) / p.hkv;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, kg = lane >> 4;
  const int each = by_group(p, 16 * NT), per = kWaves * each;
  int r = 0, tile = 0;
  PrefillRow g;
  if (!find_tile(p, per, item, lane, r, tile, g)) return;
  const int x = 16 * (block % NT) + c, y = by_group(p, x), tok = tile * per + block / NT * each + y;
  if (y >= each || tok >= g.lq) return;
  const Part* part = p.parts + ((int64_t)item * p.hkv + head) * p.splits;
  const int at = 16 * block + c;
  float m = kNone;
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, part[s].m[at]);
  f32x4 o[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
  float l = 0;
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const float w = __builtin_amdgcn_exp2f(part[s].m[at] - m);
#pragma unroll
    for (int j = 0; j < 2; ++j) o[j] += part[s].o[block][wave + 4 * j][lane] * w;
    l += part[s].l[at] * w;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint16_t* out = p.out + (int64_t)(g.q0 + tok) * p.out_stride + (head * p.group + x - y * p.group) * HD + 32 * kg;
#pragma unroll
  for (int j = 0; j < 2; ++j)
    *reinterpret_cast<u32x2*>(out + 4 * (wave + 4 * j)) =
        u32x2{pack_bf16x2(o[j][0] * inv, o[j][1] * inv), pack_bf16x2(o[j][2] * inv, o[j][3] * inv)};
}

// ------------------------------------------------------------------- launch
constexpr int kMaxPrefillRows = 1024;
constexpr int kSlots = 512;  // two workgroups fit a CU

struct Plan {
  bool dwork, pwork;
  int halves, chunks, items, splits;
  size_t dbytes, pbytes;
};

// Steps of 64 keys that queries at `n` consecutive positions may need.
int64_t most_steps(int64_t window, int64_t sinks, int64_t n, int64_t cap) {
  const int64_t keys = std::min(window + n, cap);
  return std::min((keys + 63) / 64 + 1 + (sinks + 63) / 64, (cap + 63) / 64);
}

// Chunks of a decode row that sees up to so many keys, by the (row, kv head)
// pairs.  A cut spreads few pairs over the GPU and costs the join (4-5 us).  us
// in 1, 2, 3, 4, 6 and 8 chunks:
//   8 pairs, 1,028 keys, bf16        13.4  11.7  10.1   9.4   9.0   9.0
//   16 pairs, 8,196 keys, bf16       90.5  51.2  37.5  30.6  23.8  20.5
//   64 pairs, 1,028 keys, bf16       16.5  15.0  13.0  12.4  14.5  14.4
//   128 pairs, 1,028 keys, bf16      20.5  19.1  20.9  19.3  20.8  20.9
//   128 pairs, 516 keys, bf16        11.8  13.3  14.8  15.0
//   320 pairs, 4,100 keys, E4M3FN    94.6  85.2  82.3  80.7  84.2  85.9
//   512 pairs, 4,100 keys, bf16       163   171   173   175   180   186
// 32 pairs of 8,256 keys, E4M3FN: 8 chunks 22.4, 16 24.6, 32 32.3.
int decode_chunks(int64_t pairs, int64_t keys) {
  if (pairs >= kSlots) return 1;
  const int64_t wanted = pairs >= 128 && keys >= 2048 ? 768 : 256;
  const int64_t chunks = std::min((wanted + pairs - 1) / pairs, (keys + 255) / 256);
  return chunks > 1 && keys - keys / chunks >= 512 ? (int)chunks : 1;
}

// Where all tiles fit one to a CU, beside the decode rows' workgroups, a second
// half of each takes every other step: no records and no join.  us with one
// half / two, 32 and 8 heads of bf16 behind 6,000 keys: 512 queries under 512 keys
// 21.6 / 20.2, under 1,024 32.6 / 28.1, 960 under 1,024 34.1 / 29.7 (4 bits 36.6 /
// 32.2), 2,000 (504 tiles) 45.6 / 55.6; 24 decode rows and two chunks of 512 24.9 / 30.5.
// Few tiles are cut into parts besides, as far as CUs are left: of 4 steps or
// more where there is room for four parts (32 queries, 8 tiles: under 512 keys whole
// 18.7, so 17.3; under 1,024 26.6, parts of 8, 6, 4 steps 21.4, 18.9, 17.2; under
// 4,096 76.0, parts of at least 8, 6, 4 steps 24.0, 23.8, 23.6), else of 12 (512
// queries, 128 tiles: under 512 keys whole 20.0, parts of 4 steps 27.2; under 1,024
// 28.0, parts of 6 31.5; under 4,096 whole 75.1, in two 54.4).
int tile_parts(int64_t tiles, int64_t steps) {
  return (int)std::max<int64_t>(1, std::min(kSlots / 2 / tiles, steps / (4 * tiles <= kSlots / 2 ? 4 : 12)));
}

Plan plan_of(const slo_paged_attention_args* a, int window, int sinks) {
  Plan n = {false, false, 1, 0, 0, 1, 0, 0};
  const int group = a->num_heads / a->num_kv_heads;
  if (a->num_decode > 0 && (a->phases & SLO_PHASE_DECODE)) {
    n.dwork = true;
    n.chunks = decode_chunks((int64_t)a->num_decode * a->num_kv_heads,
                             64 * most_steps(window, sinks, 1, (int64_t)a->decode_table_width * a->block_size));
    if (n.chunks > 1) n.dbytes = (size_t)a->num_decode * a->num_heads * n.chunks * RECORD * 4;
  }
  if (a->num_prefill > 0 && (a->phases & SLO_PHASE_PREFILL)) {
    n.pwork = true;
    // The rows' queries together bound the tiles.
    const int per = kWaves * (16 * NT / group);
    const int64_t tokens = a->num_q_rows - a->num_decode;
    n.items = (int)(tokens / per + a->num_prefill);
    const int64_t cap = a->prefill_tables ? (int64_t)a->prefill_table_width * a->block_size : a->num_kv_rows;
    const int64_t steps = most_steps(window, sinks, per, cap);
    // About the tiles there are; workgroups past the last one end at once.
    const int64_t tiles = std::max<int64_t>(a->num_prefill, (tokens + per - 1) / per) * a->num_kv_heads;
    n.halves = tiles + (n.dwork ? (int64_t)a->num_decode * a->num_kv_heads : 0) <= kSlots / 2 ? 2 : 1;
    if (n.halves == 2) n.splits = tile_parts(tiles, steps);
    if (n.splits > 1) n.pbytes = (size_t)n.items * a->num_kv_heads * n.splits * sizeof(Part);
  }
  return n;
}

int64_t workgroups(const slo_paged_attention_args* a, const Plan& n) {
  const int64_t heads = a->num_kv_heads;
  const int64_t joined = (n.chunks > 1 ? (int64_t)a->num_decode * a->num_heads : 0) + (n.splits > 1 ? n.items * heads * kWaves * NT : 0);
  return std::max((int64_t)n.items * n.splits * heads * n.halves + (int64_t)a->num_decode * n.chunks * heads * n.halves, joined);
}

int check_args(const slo_paged_attention_args* a, int window, int sinks) {
  if (!a) return fail(SLO_ERR_INVALID, "paged_attention_window: null args");
  if (window <= 0 || sinks < 0) return fail(SLO_ERR_INVALID, "paged_attention_window: window must be positive and sinks not negative");
  if (a->head_dim != HD) return fail(SLO_ERR_UNSUPPORTED, "paged_attention_window: head_dim must be 128");
  if (a->num_heads <= 0 || a->num_kv_heads <= 0 || a->num_heads % a->num_kv_heads)
    return fail(SLO_ERR_INVALID, "paged_attention_window: num_heads must be a multiple of num_kv_heads");
  if (a->num_heads / a->num_kv_heads > 16)
    return fail(SLO_ERR_UNSUPPORTED, "paged_attention_window: at most 16 query heads per kv head");
  if (a->num_kv_heads > 4096) return fail(SLO_ERR_UNSUPPORTED, "paged_attention_window: more than 4096 kv heads");
  if (a->kv_dtype < KV_BF16 || a->kv_dtype > KV_FP4_E2M1) return fail(SLO_ERR_INVALID, "paged_attention_window: bad kv_dtype");
  if (a->num_q_rows < 0 || a->num_decode < 0 || a->num_prefill < 0 || a->num_decode > a->num_q_rows)
    return fail(SLO_ERR_INVALID, "paged_attention_window: bad row counts");
  if (!(a->softmax_scale != 0.0f) || a->softmax_scale - a->softmax_scale != 0.0f)
    return fail(SLO_ERR_INVALID, "paged_attention_window: softmax_scale must be finite and not zero");
  if (a->store_slot_mapping) return fail(SLO_ERR_INVALID, "paged_attention_window: store the new rows first");
  if (a->num_decode > 32768 || a->num_prefill > kMaxPrefillRows)
    return fail(SLO_ERR_UNSUPPORTED, "paged_attention_window: more than 32768 decode or 1024 prefill rows");
  const bool dec = a->num_decode > 0 && (a->phases & SLO_PHASE_DECODE);
  const bool pre = a->num_prefill > 0 && (a->phases & SLO_PHASE_PREFILL);
  if (!dec && !pre) return SLO_OK;
  if (!a->q || !a->out) return fail(SLO_ERR_INVALID, "paged_attention_window: null pointer");
  if ((a->q_row_stride % 8) || (a->out_row_stride % 8) || a->q_row_stride < a->num_heads * HD ||
      a->out_row_stride < a->num_heads * HD || (reinterpret_cast<uintptr_t>(a->q) % 16) ||
      (reinterpret_cast<uintptr_t>(a->out) % 16))
    return fail(SLO_ERR_INVALID, "paged_attention_window: q and out rows must be 16-byte aligned");
  if (dec || (pre && a->prefill_tables)) {
    const bool scaled = a->kv_dtype != KV_BF16;
    if (!a->k_cache || !a->v_cache || a->num_blocks <= 0 || (scaled && (!a->k_scale || !a->v_scale)))
      return fail(SLO_ERR_INVALID, "paged_attention_window: no KV pool or no scales");
    if ((reinterpret_cast<uintptr_t>(a->k_cache) % 16) || (reinterpret_cast<uintptr_t>(a->v_cache) % 16) ||
        (scaled && ((reinterpret_cast<uintptr_t>(a->k_scale) % 16) || (reinterpret_cast<uintptr_t>(a->v_scale) % 16))))
      return fail(SLO_ERR_INVALID, "paged_attention_window: pools and scales must be 16-byte aligned");
    if (a->block_size <= 0 || a->block_size % 64)
      return fail(SLO_ERR_UNSUPPORTED, "paged_attention_window: block_size must be a multiple of 64");
  }
  if (dec && (!a->decode_lens || !a->decode_tables || a->decode_table_width <= 0))
    return fail(SLO_ERR_INVALID, "paged_attention_window: missing decode metadata");
  if (pre && (!a->prefill_cu_q || !a->prefill_cu_k || (a->prefill_tables && a->prefill_table_width <= 0)))
    return fail(SLO_ERR_INVALID, "paged_attention_window: missing prefill metadata");
  if (pre && !a->prefill_tables) {
    if (!a->k || !a->v || a->num_kv_rows <= 0) return fail(SLO_ERR_INVALID, "paged_attention_window: prefill rows without tables need k and v");
    if ((a->k_row_stride % 8) || (a->v_row_stride % 8) || a->k_row_stride < a->num_kv_heads * HD ||
        a->v_row_stride < a->num_kv_heads * HD || a->k_row_stride >= 1 << 25 || a->v_row_stride >= 1 << 25 ||
        (reinterpret_cast<uintptr_t>(a->k) % 16) || (reinterpret_cast<uintptr_t>(a->v) % 16))
      return fail(SLO_ERR_INVALID, "paged_attention_window: k and v rows must be 16-byte aligned, from num_kv_heads * 128 to 2^25 elements apart");
  }
  if ((dec && (int64_t)a->decode_table_width * a->block_size > (1 << 22)) ||
      (pre && a->prefill_tables && (int64_t)a->prefill_table_width * a->block_size > (1 << 22)) ||
      (pre && !a->prefill_tables && a->num_kv_rows > (1 << 24)))
    return fail(SLO_ERR_UNSUPPORTED, "paged_attention_window: tables span more than 2^22 tokens, or more than 2^24 k rows");
  // A grid holds less than 2^32 threads.
  if (workgroups(a, plan_of(a, window, sinks)) >= 1 << 24)
    return fail(SLO_ERR_UNSUPPORTED, "paged_attention_window: too many rows times kv heads in one call");
  return SLO_OK;
}

template <int F>
void launch(const WinParams& p, int halves, hipStream_t s) {
  const unsigned blocks = (unsigned)(((int64_t)p.items * p.splits + (int64_t)p.drows * p.chunks) * p.hkv);
  if (!p.items)
    hipLaunchKernelGGL(window_decode_kernel<F>, dim3(blocks), dim3(64 * kWaves), 0, s, p);
  else if (halves == 2)
    hipLaunchKernelGGL((window_attention_kernel<F, 2>), dim3(blocks), dim3(64 * kWaves * 2), 0, s, p);
  else
    hipLaunchKernelGGL((window_attention_kernel<F, 1>), dim3(blocks), dim3(64 * kWaves), 0, s, p);
  const int decode = p.chunks > 1 ? p.drows * p.hq : 0;
  const int prefill = p.splits > 1 ? p.items * p.hkv * kWaves * NT : 0;
  if (decode + prefill) hipLaunchKernelGGL(window_join_kernel<F>, dim3(decode + prefill), dim3(256), 0, s, p, decode);
}

}  // namespace
}  // namespace slo

using namespace slo;

extern "C" int slo_paged_attention_window_workspace_bytes(const slo_paged_attention_args* a, int32_t window, int32_t sinks,
                                                          size_t* bytes) {
  if (!bytes) return fail(SLO_ERR_INVALID, "paged_attention_window: null pointer");
  const int rc = check_args(a, window, sinks);
  if (rc) return rc;
  const Plan n = plan_of(a, window, sinks);
  *bytes = n.dbytes + n.pbytes;
  return SLO_OK;
}

extern "C" int slo_paged_attention_window(const slo_paged_attention_args* a, int32_t window, int32_t sinks,
                                          slo_stream_t stream) {
  const int rc = check_args(a, window, sinks);
  if (rc) return rc;
  const Plan n = plan_of(a, window, sinks);
  if (n.dbytes + n.pbytes > 0 && (!a->workspace || a->workspace_bytes < n.dbytes + n.pbytes ||
                                  reinterpret_cast<uintptr_t>(a->workspace) % 16))
    return fail(SLO_ERR_WORKSPACE, "paged_attention_window: workspace smaller than slo_paged_attention_window_workspace_bytes");
  if (!n.dwork && !n.pwork) return SLO_OK;
  WinParams p = {};
  p.q = static_cast<const uint16_t*>(a->q);
  p.q_stride = a->q_row_stride;
  p.out = static_cast<uint16_t*>(a->out);
  p.out_stride = a->out_row_stride;
  p.num_q_rows = a->num_q_rows;
  p.kc = static_cast<const uint8_t*>(a->k_cache);
  p.vc = static_cast<const uint8_t*>(a->v_cache);
  p.ks = a->k_scale;
  p.vs = a->v_scale;
  p.num_blocks = a->num_blocks;
  p.block_size = a->block_size;
  p.tpb = a->block_size > 0 ? a->block_size / 64 : 1;
  p.tpb_inv = (uint32_t)((0xffffffffull + p.tpb) / p.tpb);
  p.hq = a->num_heads;
  p.hkv = a->num_kv_heads;
  p.group = a->num_heads / a->num_kv_heads;
  p.group_inv = ((1 << 16) + p.group - 1) / p.group;
  p.scale_log2 = (a->softmax_scale < 0 ? -a->softmax_scale : a->softmax_scale) * kLog2e;
  p.q_sign = a->softmax_scale < 0 ? 0x80008000u : 0u;
  p.window = std::min(window, 1 << 26);
  p.sinks = std::min(sinks, 1 << 26);
  const bool rows = a->num_prefill > 0 && a->prefill_cu_q;  // whatever the phases
  p.ends = rows ? a->prefill_cu_q + a->num_prefill : nullptr;
  p.first_idle = p.first_row = a->num_decode;
  p.idle = n.pwork || a->num_q_rows > a->num_decode;
  p.chunks = p.splits = 1;
  if (n.dwork) {
    p.lens = a->decode_lens;
    p.dtables = a->decode_tables;
    p.dstride = a->decode_table_stride;
    p.dwidth = a->decode_table_width;
    p.drows = a->num_decode;
    p.chunks = n.chunks;
    p.records = static_cast<float*>(a->workspace);
  }
  if (n.pwork) {
    p.cu_q = a->prefill_cu_q;
    p.cu_k = a->prefill_cu_k;
    p.ptables = a->prefill_tables;
    p.pstride = a->prefill_table_stride;
    p.pwidth = a->prefill_table_width;
    p.prows = a->num_prefill;
    p.items = n.items;
    p.splits = n.splits;
    p.parts = reinterpret_cast<Part*>(static_cast<char*>(a->workspace) + n.dbytes);
    p.rk = static_cast<const uint8_t*>(a->k);
    p.rv = static_cast<const uint8_t*>(a->v);
    p.rk_stride = 2 * a->k_row_stride;
    p.rv_stride = 2 * a->v_row_stride;
    p.num_kv_rows = a->num_kv_rows;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (n.pwork && !p.ptables && a->kv_dtype != KV_BF16) {
    // The step's own rows are bf16 whatever the pool's format.
    WinParams cold = p;
    cold.drows = 0;
    launch<KV_BF16>(cold, n.halves, s);
    p.items = 0;
    p.splits = 1;
    p.idle = false;
  }
  if (p.items || p.drows) {
    if (a->kv_dtype == KV_BF16) launch<KV_BF16>(p, n.halves, s);
    else if (a->kv_dtype == KV_FP8_E4M3FN) launch<KV_FP8_E4M3FN>(p, n.halves, s);
    else launch<KV_FP4_E2M1>(p, n.halves, s);
  }
  return check_launch("paged_attention_window");
}
