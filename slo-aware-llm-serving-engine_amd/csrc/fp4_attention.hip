// Ragged paged attention over a 4-bit KV pool (gfx950).
//
// out[i, h] = sum_j softmax_j(scale q[i, h] . k[j]) v[j] over the keys j that
// query i sees, with K and V read from 4-bit pages (fp4.h).  One pass over the
// keys with a running maximum and sum per (query, head):
//
//   S^T = K q^T      A = K (rows: 16 tokens), B = q (columns: 16 queries or heads)
//   O^T += V^T P^T   A = V^T (rows: 16 channels), B = P (columns: the same 16)
//
// Transposed products keep a column's statistics in the lanes that hold its
// scores and its outputs, and the 8 probabilities that a lane has of two
// 16-token tiles (tokens 4 kg + i and 16 + 4 kg + i, kg = lane / 16) are, as
// they lie, the operand of the second product for that order of its 32 tokens.
// Codes become bf16 operands by v_cvt_scalef32_pk_bf16_fp4, exactly, scale
// included: two channels of a token per instruction.  For K that is the
// operand's order (lane: one token, the 32 channels of one scale, 16 bytes);
// for V (lane: 8 tokens, 8 channels, 4 bytes each) two v_perm_b32 per two pairs
// turn channel pairs into token pairs.  Probabilities are rounded to bf16 and
// their sum is taken of the rounded values (one more row of the second
// product, of ones), so a weight's rounding cancels where one key dominates.
// Sums, maxima and outputs are fp32 until the one rounding at the end.
#include "capi_internal.h"
#include "fp4.h"
#include "tile_io.h"
#include <type_traits>

namespace slo {
namespace {

constexpr int HD4 = 128;        // head_dim
constexpr int KT = 32;          // tokens per step of a wavefront
constexpr int RECORD = HD4 + 4;  // floats of a partial result: outputs, maximum, sum, 2 unused
constexpr float kNone = -1e30f;  // running maximum before the first key

struct Fp4Params {
  const uint16_t* q;
  int64_t q_stride;
  uint16_t* out;
  int64_t out_stride;
  int num_q_rows;
  const uint8_t *kc, *vc, *ks, *vs;
  int num_blocks, block_size;
  const int32_t* lens;  // decode rows: key counts; null for prefill rows
  const int32_t* cu_q;
  const int32_t* cu_k;
  const int32_t* tables;
  int table_stride, table_width;
  int first_row;  // query row of the phase's first query
  int hq, hkv, group;
  float scale_log2;  // |softmax scale| * log2(e)
  uint32_t q_sign;   // 0x80008000 where the scale is negative
  float* partial;    // prefill rows: [queries, hq, splits] records when splits > 1; decode rows: [chunks, hq]
  int splits, chunk;  // prefill rows
  int rows, budget;   // decode rows: about so many chunks over all rows
};

struct Row {
  int64_t q0;  // first query row
  int lq, lk, prefix;
};

__device__ __forceinline__ Row row_of(const Fp4Params& p, int r) {
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

// The chunks of the decode rows, found on the GPU from the rows' lengths (a
// captured launch knows no more of them than its tables' width): chunks of one
// length over all rows, in units of 128 tokens, such that there are about
// `budget`; a row's own are equal.  Every wavefront works it out for itself, 64
// rows at a time.
struct Chunk {
  int row, index, count;  // the row's chunk `index` of `count`
  int first;              // number of the row's first chunk
  int k0, k1;
};

__device__ __forceinline__ int units_of(const Fp4Params& p, int r) {
  const int cap = p.table_width * p.block_size;
  return r < p.rows ? (min(max(p.lens[r], 0), cap) + 127) >> 7 : 0;
}

// Inclusive sum over the wavefront by DPP: within rows of 16 lanes, then the
// rows' last lanes onto the rows behind them.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr 1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast 15
  return x + __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast 31
}

__device__ __forceinline__ int chunk_units(const Fp4Params& p, int lane) {
  int total = 0;  // at most 65,535 rows of 2^15 units
  for (int r = lane; r < p.rows; r += 64) total += units_of(p, r);
  total = __builtin_amdgcn_readlane(wave_scan(total), 63);
  return max((total + p.budget - 1) / p.budget, 2);
}

// Chunk number i (by_row: the first one of row i); false past the last.
__device__ __forceinline__ bool find_chunk(const Fp4Params& p, int i, bool by_row, int lane, Chunk& c) {
  const int per = chunk_units(p, lane);
  int before = 0;
  for (int base = 0; base < p.rows; base += 64) {
    const int u = units_of(p, base + lane), n = base + lane < p.rows ? max(1, (u + per - 1) / per) : 0;
    const int upto = wave_scan(n);
    const uint64_t past = __ballot(by_row ? base + lane >= i : before + upto > i);
    const int at = past ? __builtin_ctzll(past) : 64;
    if (at < 64 && base + at < p.rows) {
      c.row = base + at;
      c.count = __builtin_amdgcn_readlane(n, at);
      c.first = before + __builtin_amdgcn_readlane(upto, at) - c.count;
      c.index = by_row ? 0 : i - c.first;
      const int mine = (__builtin_amdgcn_readlane(u, at) + c.count - 1) / c.count * 128;
      c.k0 = c.index * mine;
      c.k1 = c.k0 + mine;
      return true;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

// A decode wavefront's steps arrive in LDS by DMA, kDepth in flight.  Codes
// land as their lanes fetch them, so the lanes fetch in an order that lets both
// operands be read without a bank conflict: of K, 16-byte part p of token t
// lies at part p ^ (t / 4 mod 4) of its place; of V, token t lies at place
// t ^ (t / 4 mod 4).  Both stay within the 256 bytes of four tokens, so a
// fetch still takes whole lines.
struct Step {
  uint8_t k[2048], v[2048], ks[128], vs[128];
};
constexpr int kDepth = 2, kStepLoads = 5;

__device__ __forceinline__ void fetch(const Fp4Params& p, int64_t row, uint32_t to, int lane) {
  const uint32_t t = lane >> 2, x = (lane >> 4) & 3;
  const uint32_t ko = t * 64 + ((lane & 3) ^ x) * 16, vo = (t ^ x) * 64 + (lane & 3) * 16;
  const uint8_t *k = p.kc + row * 64, *v = p.vc + row * 64;
  dma16_nt_at(k, ko, to);
  dma16_nt_at(k, ko + 1024, to + 1024);
  dma16_nt_at(v, vo, to + 2048);
  dma16_nt_at(v, vo + 1024, to + 3072);
  dma4((lane < 32 ? p.ks : p.vs) + row * 4 + (lane & 31) * 4, to + 4096);
}

struct Tile {
  u32x4 k[2], vs[2];
  uint32_t v[8], ks[2];
};

__device__ __forceinline__ void read_step(Tile& t, const Step& s, int lane) {
  const int c = lane & 15, kg = lane >> 4;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    t.k[h] = *reinterpret_cast<const u32x4*>(s.k + h * 1024 + c * 64 + (kg ^ (c >> 2)) * 16);
    t.ks[h] = s.ks[h * 64 + c * 4 + kg];
    t.vs[h] = *reinterpret_cast<const u32x4*>(s.vs + h * 64 + kg * 16);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      t.v[4 * h + i] = *reinterpret_cast<const uint32_t*>(s.v + h * 1024 + kg * 256 + (i ^ kg) * 64 + c * 4);
  }
}

template <int NT>
struct Acc {
  f32x4 o[NT][8], l[NT];
  float m[NT];
};

__device__ __forceinline__ float column_max(float x) {  // over the four lanes of a column
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// The reference of column n's weights follows a new maximum only where a score
// passes it by 2^8: weights up to 256 round like those below 1, and the
// rescaling of the outputs is rare.
template <int NT>
__device__ __forceinline__ void move_reference(Acc<NT>& a, int n, float top) {
  if (__any(top > a.m[n] + 8.0f)) {
    const float m = fmaxf(a.m[n], column_max(top));
    const float w = __builtin_amdgcn_exp2f(a.m[n] - m);
    a.m[n] = m;
#pragma unroll
    for (int e = 0; e < 8; ++e) a.o[n][e] *= w;
    a.l[n] *= w;
  }
}

__device__ __forceinline__ bf16x8 ones() {
  return as_bf16x8(u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});
}

template <int NT>
__device__ __forceinline__ void step(const Tile& t, bool masked, const bf16x8 (&q)[NT][4], Acc<NT>& a, float c, int kv0,
                                     const int (&limit)[NT], int kend, int lane) {
  const int kg = lane >> 4;
  f32x4 s[NT][2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float sc = e8m0(t.ks[h]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bf16x8 k = as_bf16x8(e2m1_decode8(t.k[h][i], sc));
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n][h] = mfma16(k, q[n][i], i ? s[n][h] : f32x4{0, 0, 0, 0});
    }
  }
  bf16x8 pr[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if (masked) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (kv0 + 16 * h + 4 * kg + i >= limit[n]) s[n][h][i] = -INFINITY;
    }
    float top = fmaxf(s[n][0][0], s[n][0][1]);
#pragma unroll
    for (int i = 2; i < 8; ++i) top = fmaxf(top, s[n][i >> 2][i & 3]);
    move_reference(a, n, top * c);
    u32x4 b;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      b[i] = pack_bf16x2(__builtin_amdgcn_exp2f(__builtin_fmaf(s[n][i >> 1][2 * (i & 1)], c, -a.m[n])),
                         __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][i >> 1][2 * (i & 1) + 1], c, -a.m[n])));
    pr[n] = as_bf16x8(b);
  }
  // The lane's scale byte of each token, rotated to the exponent's place: the
  // conversion reads nothing but the exponent of its scale (all mantissas and
  // both signs give the same bits, checked on gfx950).
  float vs[8];
  const int turn = (9 + 8 * ((lane & 15) >> 2)) & 31;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t x = t.vs[j >> 2][j & 3];
    vs[j] = __uint_as_float(__builtin_amdgcn_alignbit(x, x, turn));
  }
  // A token past the row's keys may be anything in the pages: its weight is
  // zero, and its scale must not make that a NaN.
  if (masked) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (kv0 + 16 * (j >> 2) + 4 * kg + (j & 3) >= kend) vs[j] = 0.0f;
  }
  auto pair = [&](auto sel) {
    constexpr int B = decltype(sel)::value;
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = e2m1_pair<B>(t.v[j], vs[j]);
    u32x4 lo, hi;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lo[i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x05040100u);
      hi[i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x07060302u);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      a.o[n][2 * B] = mfma16(as_bf16x8(lo), pr[n], a.o[n][2 * B]);
      a.o[n][2 * B + 1] = mfma16(as_bf16x8(hi), pr[n], a.o[n][2 * B + 1]);
    }
  };
#pragma unroll
  for (int n = 0; n < NT; ++n) a.l[n] = mfma16(ones(), pr[n], a.l[n]);
  pair(std::integral_constant<int, 0>{});
  pair(std::integral_constant<int, 1>{});
  pair(std::integral_constant<int, 2>{});
  pair(std::integral_constant<int, 3>{});
}

// Walks a row's tokens in steps of `stride` through its table; pages that are
// not in the pool count as unseen keys.
struct Walk {
  const __attribute__((address_space(4))) int32_t* table;  // read by scalar loads
  int page, off, block_size, num_blocks, hkv, head;
  __device__ __forceinline__ void advance(int by) {
    off += by;
    while (off >= block_size) {
      off -= block_size;
      ++page;
    }
  }
  __device__ __forceinline__ int64_t row(bool& ok) const {
    const int b = table[page];
    ok = b >= 0 && b < num_blocks;
    return ((int64_t)(ok ? b : 0) * hkv + head) * block_size + off;
  }
};

__device__ __forceinline__ const __attribute__((address_space(4))) int32_t* row_table(const Fp4Params& p, int r) {
  return (const __attribute__((address_space(4))) int32_t*)(uintptr_t)(p.tables + (int64_t)r * p.table_stride);
}

__device__ __forceinline__ bf16x8 load_q(const Fp4Params& p, int64_t row, int h, int channel, bool live) {
  u32x4 x = {0, 0, 0, 0};
  if (live) x = *reinterpret_cast<const u32x4*>(p.q + row * p.q_stride + h * HD4 + channel);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] ^= p.q_sign;
  return as_bf16x8(x);
}

template <int NT>
__device__ __forceinline__ void clear(Acc<NT>& a) {
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int e = 0; e < 8; ++e) a.o[n][e] = f32x4{0, 0, 0, 0};
    a.l[n] = f32x4{0, 0, 0, 0};
    a.m[n] = kNone;
  }
}

// Decode rows: a workgroup takes one chunk of one (row, kv head), its four
// wavefronts every fourth 32-token step, all heads of the group as columns.
// Each wavefront fetches its own steps, so the loop has no barrier; the
// wavefronts' results meet in LDS.
template <int WAVES>
__global__ void __launch_bounds__(64 * WAVES, 4)
fp4_decode_kernel(Fp4Params p) {
  __shared__ union {
    Step steps[kDepth];
    float o[16][HD4];
  } ring[WAVES];
  __shared__ float sm[WAVES][16], sl[WAVES][16];
  const int head = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Chunk chunk;
  if (!find_chunk(p, blockIdx.y, false, lane, chunk)) return;
  const int r = chunk.row;
  const Row g = row_of(p, r);
  const int k0 = chunk.k0, k1 = min(chunk.k1, g.lk);
  const int col = lane & 15, kg = lane >> 4;
  bf16x8 q[1][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) q[0][i] = load_q(p, g.q0, head * p.group + col, 32 * kg + 8 * i, col < p.group);
  Acc<1> a;
  clear(a);
  const int limit[1] = {g.lk};
  const int begin = k0 + wave * KT, steps = (k1 - begin + WAVES * KT - 1) / (WAVES * KT);
  if (steps > 0) {
    Walk w{row_table(p, r), begin / p.block_size, 0, p.block_size, p.num_blocks, p.hkv, head};
    w.off = begin - w.page * p.block_size;
    const uint32_t lds = lds_addr(&ring[wave]);
    uint32_t ok = 0;  // bit i: the step that lies i steps ahead reads a page of the pool
    int sent = 0, to = 0;
    auto send = [&] {
      bool in;
      const int64_t row = w.row(in);
      ok |= (uint32_t)in << (kDepth - 1);
      fetch(p, row, lds + to * (uint32_t)sizeof(Step), lane);
      to = to == kDepth - 1 ? 0 : to + 1;
      if (++sent < steps) w.advance(WAVES * KT);
    };
    for (int i = 0; i < kDepth - 1; ++i) {
      ok >>= 1;
      if (sent < steps) send();
    }
    int from = 0;
    for (int i = 0; i < steps; ++i) {
      // Bit 0 is now step i's.  The place that the next fetch fills was read in
      // the last iteration; its reads have returned.
      ok >>= 1;
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
      if (sent < steps) send();
      const int ahead = sent - 1 - i;
      asm volatile("" ::: "memory");
      if (ahead >= 2)
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * kStepLoads));
      else if (ahead == 1)
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(kStepLoads));
      else
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
      asm volatile("" ::: "memory");
      Tile t;
      read_step(t, ring[wave].steps[from], lane);
      from = from == kDepth - 1 ? 0 : from + 1;
      const int at = begin + WAVES * KT * i;
      if (ok & 1) step<1>(t, at + KT > g.lk, q, a, p.scale_log2, at, limit, g.lk, lane);
    }
  }
  auto& so = ring;
  if (col < p.group) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 8; e += 4)
        *reinterpret_cast<f32x4*>(&so[wave].o[col][32 * kg + 8 * i + e]) =
            f32x4{a.o[0][e][i], a.o[0][e + 1][i], a.o[0][e + 2][i], a.o[0][e + 3][i]};
    if (kg == 0) {
      sm[wave][col] = a.m[0];
      sl[wave][col] = a.l[0][0];
    }
  }
  __syncthreads();
  for (int x = threadIdx.x; x < p.group * (HD4 / 4); x += 64 * WAVES) {
    const int h = x >> 5, d = (x & 31) * 4;
    float m = sm[0][h];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) m = fmaxf(m, sm[w][h]);
    f32x4 o = {0, 0, 0, 0};
    float l = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float f = __builtin_amdgcn_exp2f(sm[w][h] - m);
      o += *reinterpret_cast<const f32x4*>(&so[w].o[h][d]) * f;
      l += sl[w][h] * f;
    }
    if (chunk.count == 1) {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      *reinterpret_cast<u32x2*>(p.out + g.q0 * p.out_stride + (head * p.group + h) * HD4 + d) =
          u32x2{pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv)};
    } else {
      float* rec = p.partial + ((int64_t)blockIdx.y * p.hq + head * p.group + h) * RECORD;
      *reinterpret_cast<f32x4*>(rec + d) = o;
      if (d == 0) {
        rec[HD4] = m;
        rec[HD4 + 1] = l;
      }
    }
  }
}

// One 64-token step of a workgroup as bf16 operands in LDS, in the order in
// which lanes read them (16 bytes a lane, no bank twice): K's four operands of
// each 16 tokens, V's eight of each 32 tokens.
struct Stage {
  u32x4 k[4][4][64], v[2][8][64];
};

// A wavefront's quarter of a step: 16 tokens of K, and four channels of every
// lane's eight of 32 tokens of V.
struct Quarter {
  u32x4 k, vs[2];
  uint32_t ks;
  uint16_t v[8];
};

__device__ __forceinline__ void load_quarter(Quarter& t, const Fp4Params& p, int64_t row, int wave, int lane) {
  const uint32_t c = lane & 15, kg = lane >> 4;
  const uint8_t *k = p.kc + (row + 16 * wave) * 64, *ks = p.ks + (row + 16 * wave) * 4;
  const int64_t vrow = row + 32 * (wave >> 1);
  const uint8_t *v = p.vc + vrow * 64 + 2 * (wave & 1), *vs = p.vs + vrow * 4;
  const uint32_t ko = c * 64 + kg * 16, kso = c * 4 + kg, vo = kg * 256 + c * 4, vso = kg * 16;
  t.k = *reinterpret_cast<const u32x4*>(k + ko);
  t.ks = ks[kso];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    t.vs[h] = *reinterpret_cast<const u32x4*>(vs + (vso + h * 64));
#pragma unroll
    for (int i = 0; i < 4; ++i) t.v[4 * h + i] = *reinterpret_cast<const uint16_t*>(v + (vo + h * 1024 + i * 64));
  }
}

// `left`: tokens of the step that belong to the row; V's scales past them are
// cleared (see step).
__device__ __forceinline__ void stage(Stage& s, const Quarter& t, int left, int wave, int lane) {
  const int c = lane & 15, kg = lane >> 4;
  const float sc = e8m0(t.ks);
#pragma unroll
  for (int i = 0; i < 4; ++i) s.k[wave][i][lane] = e2m1_decode8(t.k[i], sc);
  float vs[8];
  const int turn = (9 + 8 * (c >> 2)) & 31;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t x = t.vs[j >> 2][j & 3];
    vs[j] = __uint_as_float(__builtin_amdgcn_alignbit(x, x, turn));
  }
  if (left < 64) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (32 * (wave >> 1) + 16 * (j >> 2) + 4 * kg + (j & 3) >= left) vs[j] = 0.0f;
  }
  u32x4 o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t a0 = e2m1_pair<0>(t.v[2 * i], vs[2 * i]), b0 = e2m1_pair<0>(t.v[2 * i + 1], vs[2 * i + 1]);
    const uint32_t a1 = e2m1_pair<1>(t.v[2 * i], vs[2 * i]), b1 = e2m1_pair<1>(t.v[2 * i + 1], vs[2 * i + 1]);
    o[0][i] = __builtin_amdgcn_perm(b0, a0, 0x05040100u);
    o[1][i] = __builtin_amdgcn_perm(b0, a0, 0x07060302u);
    o[2][i] = __builtin_amdgcn_perm(b1, a1, 0x05040100u);
    o[3][i] = __builtin_amdgcn_perm(b1, a1, 0x07060302u);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) s.v[wave >> 1][4 * (wave & 1) + e][lane] = o[e];
}

// 64 tokens of a wavefront's columns against the staged operands.
template <int NT>
__device__ __forceinline__ void staged_step(const Stage& st, bool masked, const bf16x8 (&q)[NT][4], Acc<NT>& a, float c, int kv0,
                                            const int (&limit)[NT], int lane) {
  const int kg = lane >> 4;
  f32x4 s[NT][4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bf16x8 k = as_bf16x8(st.k[t][i][lane]);
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n][t] = mfma16(k, q[n][i], i ? s[n][t] : f32x4{0, 0, 0, 0});
    }
  }
  bf16x8 pr[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if (masked) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (kv0 + 16 * t + 4 * kg + i >= limit[n]) s[n][t][i] = -INFINITY;
    }
    float top = fmaxf(s[n][0][0], s[n][0][1]);
#pragma unroll
    for (int i = 2; i < 16; ++i) top = fmaxf(top, s[n][i >> 2][i & 3]);
    move_reference(a, n, top * c);
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      u32x4 b;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4& x = s[n][2 * g + (i >> 1)];
        b[i] = pack_bf16x2(__builtin_amdgcn_exp2f(__builtin_fmaf(x[2 * (i & 1)], c, -a.m[n])),
                           __builtin_amdgcn_exp2f(__builtin_fmaf(x[2 * (i & 1) + 1], c, -a.m[n])));
      }
      pr[n][g] = as_bf16x8(b);
    }
  }
#pragma unroll
  for (int g = 0; g < 2; ++g) {
#pragma unroll
    for (int n = 0; n < NT; ++n) a.l[n] = mfma16(ones(), pr[n][g], a.l[n]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bf16x8 v = as_bf16x8(st.v[g][e][lane]);
#pragma unroll
      for (int n = 0; n < NT; ++n) a.o[n][e] = mfma16(v, pr[n][g], a.o[n][e]);
    }
  }
}

// Prefill rows: a workgroup takes 64 NT columns, (query, head of the group)
// pairs of consecutive queries of one row, over its keys (or one chunk of
// them), the latest queries first.  Its four wavefronts turn each 64-token
// step's codes into operands together, each a quarter, one step ahead of the
// products, and each runs 16 NT columns over them.
template <int NT>
__global__ void __launch_bounds__(256, 2)
fp4_prefill_kernel(Fp4Params p, int tiles) {
  __shared__ Stage st[2];
  const int head = blockIdx.x, r = blockIdx.z;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int split = blockIdx.y % p.splits;
  const int per = 16 * NT / p.group;  // queries of a wavefront
  const Row g = row_of(p, r);
  const int w0 = (tiles - 1 - (int)(blockIdx.y / p.splits)) * 4 * per;  // the workgroup's first query
  if (w0 >= g.lq) return;
  const int all = min(max(g.prefix + min(w0 + 4 * per, g.lq), 0), g.lk);  // keys that one of its queries sees
  const int k0 = split * p.chunk, k1 = p.splits == 1 ? all : min(k0 + p.chunk, all);
  if (split && k0 >= all) return;
  const int t0 = w0 + wave * per, t1 = min(t0 + per, g.lq);
  const int kend = t0 < g.lq ? min(max(g.prefix + t1, 0), g.lk) : 0;  // that one of the wavefront's sees
  const int full = min(g.prefix + t0 + 1, g.lk);                      // that all of them see
  const int col = lane & 15, kg = lane >> 4;
  bf16x8 q[NT][4];
  int limit[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int x = 16 * n + col, tok = t0 + x / p.group;
    const bool live = x < per * p.group && tok < t1;
    limit[n] = live ? min(g.prefix + tok + 1, g.lk) : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) q[n][i] = load_q(p, g.q0 + tok, head * p.group + x % p.group, 32 * kg + 8 * i, live);
  }
  Acc<NT> a;
  clear(a);
  if (k0 < k1) {
    Walk w{row_table(p, r), k0 / p.block_size, 0, p.block_size, p.num_blocks, p.hkv, head};
    w.off = k0 - w.page * p.block_size;
    Quarter t;
    bool ok, next_ok = false;
    load_quarter(t, p, w.row(ok), wave, lane);
    for (int at = k0, b = 0; at < k1; at += 64, b ^= 1) {
      stage(st[b], t, all - at, wave, lane);
      if (at + 64 < k1) {
        w.advance(64);
        load_quarter(t, p, w.row(next_ok), wave, lane);
      }
      // Two buffers: a wavefront comes to write this one again only past the
      // next step's barrier, when every wavefront has left it.
      __syncthreads();
      if (ok && at < kend) staged_step<NT>(st[b], at + 64 > full, q, a, p.scale_log2, at, limit, lane);
      ok = next_ok;
    }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    int x = 16 * n + col;
    asm("" : "+v"(x));  // found again here, so that the loop need not hold it in registers
    const int tok = t0 + x / p.group, h = head * p.group + x % p.group;
    if (x >= per * p.group || tok >= t1) continue;
    if (p.splits == 1) {
      const float inv = a.l[n][0] == 0.0f ? 0.0f : 1.0f / a.l[n][0];
      uint16_t* out = p.out + (g.q0 + tok) * p.out_stride + h * HD4 + 32 * kg;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<u32x4*>(out + 8 * i) =
            u32x4{pack_bf16x2(a.o[n][0][i] * inv, a.o[n][1][i] * inv), pack_bf16x2(a.o[n][2][i] * inv, a.o[n][3][i] * inv),
                  pack_bf16x2(a.o[n][4][i] * inv, a.o[n][5][i] * inv), pack_bf16x2(a.o[n][6][i] * inv, a.o[n][7][i] * inv)};
    } else {
      float* rec = p.partial + (((g.q0 - p.first_row + tok) * p.hq + h) * p.splits + split) * RECORD;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 8; e += 4)
          *reinterpret_cast<f32x4*>(rec + 32 * kg + 8 * i + e) =
              f32x4{a.o[n][e][i], a.o[n][e + 1][i], a.o[n][e + 2][i], a.o[n][e + 3][i]};
      if (kg == 0) {
        rec[HD4] = a.m[n];
        rec[HD4 + 1] = a.l[n][0];
      }
    }
  }
}

// Joins the partial results of the phase's chunks: a workgroup of W half
// wavefronts per (query, head), four channels a lane.  Half wavefront i takes
// chunks i, i + W, ... and the W sums meet in LDS in that order.
template <int W>
__global__ void __launch_bounds__(32 * W < 256 ? 256 : 32 * W)
fp4_join_kernel(Fp4Params p) {
  constexpr int UNITS = 32 * W < 256 ? 8 / W : 1;  // (query, head) pairs of a workgroup
  __shared__ f32x4 so[UNITS][W][32];
  __shared__ float sl[UNITS][W];
  const int lane = threadIdx.x & 31, i = (threadIdx.x >> 5) % W, u = (threadIdx.x >> 5) / W;
  const int r = blockIdx.y;
  const Row g = row_of(p, r);
  const int unit = (int)blockIdx.x * UNITS + u, query = unit / p.hq, h = unit - query * p.hq;
  bool live = query < g.lq;
  int n = 0;
  const float* rec = p.partial;
  int64_t stride = RECORD;
  if (p.lens) {
    Chunk c;
    find_chunk(p, r, true, threadIdx.x & 63, c);
    if (c.count == 1) return;  // written by its only chunk
    n = live ? c.count : 0;
    rec += ((int64_t)c.first * p.hq + h) * RECORD;
    stride = (int64_t)p.hq * RECORD;
  } else if (live) {
    const int kend = min(max(g.prefix + query + 1, 0), g.lk);
    n = min(max(1, (kend + p.chunk - 1) / p.chunk), p.splits);
    rec += ((g.q0 - p.first_row + query) * p.hq + h) * (int64_t)p.splits * RECORD;
  }
  float m = kNone;
  for (int s = lane; s < n; s += 32) m = fmaxf(m, rec[s * stride + HD4]);
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) m = wave_max_xor(m, d);
  f32x4 o = {0, 0, 0, 0};
  float l = 0;
#pragma unroll 4
  for (int s = i; s < n; s += W) {
    const float* e = rec + s * stride;
    const float w = __builtin_amdgcn_exp2f(e[HD4] - m);
    o += *reinterpret_cast<const f32x4*>(e + 4 * lane) * w;
    l += e[HD4 + 1] * w;
  }
  if (W > 1) {
    so[u][i][lane] = o;
    if (lane == 0) sl[u][i] = l;
    __syncthreads();
    if (i) return;
#pragma unroll
    for (int k = 1; k < W; ++k) {
      o += so[u][k][lane];
      l += sl[u][k];
    }
  }
  if (!live) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  *reinterpret_cast<u32x2*>(p.out + (g.q0 + query) * p.out_stride + h * HD4 + 4 * lane) =
      u32x2{pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv)};
}

constexpr int kPrefillNT = 2;
constexpr int kPrefillTarget = 1024;
// Chunks of all decode rows and heads together: one for each of the four
// workgroups that a CU holds.  64 rows of 512-4,096 tokens, 8 kv heads: 36.6 us
// and 5.1 us to join them, 38.1 + 6.6 with twice as many, 42.1 + 6.8 with four
// times; three rows of 20,000-60,000 30.2 + 4.2, 32.1 + 5.8, 35.9 + 7.2.
constexpr int kDecodeChunks = 1024;
// Rows of at most this many tokens are not cut, and eight wavefronts take each:
// one row of 1,000 6.7 us, 5.4 + 4.4 us as two chunks and their join.
constexpr int kWholeRow = 1024;

// Chunks of `capacity` keys for a launch of so many workgroups per chunk:
// enough for `target` workgroups, at least `least` keys each.
int splits_of(int64_t groups, int64_t capacity, int least, int target, int& chunk) {
  const int64_t want = groups > 0 ? (target + groups - 1) / groups : 1;
  int64_t c = ((capacity + want - 1) / want + 127) / 128 * 128;
  if (c < least) c = least;
  chunk = (int)c;
  const int64_t n = (capacity + c - 1) / c;
  return n < 1 ? 1 : (int)n;
}

struct Plan {
  bool dwork, joined;
  int budget, psplits, pchunk, ptiles;
  size_t dbytes, pbytes;
};

Plan plan_of(const slo_paged_attention_args* a) {
  Plan n = {false, false, 0, 1, 1 << 30, 0, 0, 0};
  if (a->num_decode > 0 && (a->phases & SLO_PHASE_DECODE)) {
    n.dwork = true;
    n.joined = (int64_t)a->decode_table_width * a->block_size > kWholeRow;
    n.budget = n.joined ? (kDecodeChunks + a->num_kv_heads - 1) / a->num_kv_heads : 0;
    if (n.joined) n.dbytes = (size_t)(n.budget + a->num_decode) * a->num_heads * RECORD * 4;
  }
  if (a->num_prefill > 0 && (a->phases & SLO_PHASE_PREFILL) && a->max_q > 0) {
    const int per = 16 * kPrefillNT / (a->num_heads / a->num_kv_heads);
    n.ptiles = ((a->max_q + per - 1) / per + 3) / 4;
    const int64_t cap = (int64_t)a->prefill_table_width * a->block_size;
    // The rows' queries together, not every row's maximum, make the workgroups.
    const int64_t tiles = (a->num_q_rows - a->num_decode) / (4 * per) + a->num_prefill;
    n.psplits = splits_of(tiles * a->num_kv_heads, cap < a->max_k ? cap : a->max_k, 512, kPrefillTarget, n.pchunk);
    if (n.psplits > 1) n.pbytes = (size_t)(a->num_q_rows - a->num_decode) * a->num_heads * n.psplits * RECORD * 4;
  }
  return n;
}

int check_args(const slo_paged_attention_args* a) {
  if (!a) return fail(SLO_ERR_INVALID, "paged_attention_fp4: null args");
  if (a->head_dim != HD4) return fail(SLO_ERR_UNSUPPORTED, "paged_attention_fp4: head_dim must be 128");
  if (a->num_heads <= 0 || a->num_kv_heads <= 0 || a->num_heads % a->num_kv_heads)
    return fail(SLO_ERR_INVALID, "paged_attention_fp4: num_heads must be a multiple of num_kv_heads");
  if (a->num_heads / a->num_kv_heads > 16)
    return fail(SLO_ERR_UNSUPPORTED, "paged_attention_fp4: at most 16 query heads per kv head");
  if (a->kv_dtype != KV_FP4_E2M1) return fail(SLO_ERR_INVALID, "paged_attention_fp4: kv_dtype must be SLO_KV_FP4_E2M1");
  if (a->num_q_rows < 0 || a->num_decode < 0 || a->num_prefill < 0 || a->num_decode > a->num_q_rows)
    return fail(SLO_ERR_INVALID, "paged_attention_fp4: bad row counts");
  if (!(a->softmax_scale != 0.0f) || a->softmax_scale - a->softmax_scale != 0.0f)
    return fail(SLO_ERR_INVALID, "paged_attention_fp4: softmax_scale must be finite and not zero");
  if (a->store_slot_mapping) return fail(SLO_ERR_INVALID, "paged_attention_fp4: store the new rows first");
  if (a->num_decode > 65535 || a->num_prefill > 65535)
    return fail(SLO_ERR_UNSUPPORTED, "paged_attention_fp4: more than 65535 rows");
  const bool dec = a->num_decode > 0 && (a->phases & SLO_PHASE_DECODE);
  const bool pre = a->num_prefill > 0 && (a->phases & SLO_PHASE_PREFILL);
  if (!dec && !pre) return SLO_OK;
  if (!a->q || !a->out) return fail(SLO_ERR_INVALID, "paged_attention_fp4: null pointer");
  if ((a->q_row_stride % 8) || (a->out_row_stride % 8) || a->q_row_stride < a->num_heads * HD4 ||
      a->out_row_stride < a->num_heads * HD4 || (reinterpret_cast<uintptr_t>(a->q) % 16) ||
      (reinterpret_cast<uintptr_t>(a->out) % 16))
    return fail(SLO_ERR_INVALID, "paged_attention_fp4: q and out rows must be 16-byte aligned");
  if (!a->k_cache || !a->v_cache || !a->k_scale || !a->v_scale || a->num_blocks <= 0)
    return fail(SLO_ERR_INVALID, "paged_attention_fp4: no KV pool or no scales");
  if ((reinterpret_cast<uintptr_t>(a->k_cache) % 16) || (reinterpret_cast<uintptr_t>(a->v_cache) % 16) ||
      (reinterpret_cast<uintptr_t>(a->k_scale) % 16) || (reinterpret_cast<uintptr_t>(a->v_scale) % 16))
    return fail(SLO_ERR_INVALID, "paged_attention_fp4: pools and scales must be 16-byte aligned");
  if (a->block_size <= 0 || a->block_size % 64)
    return fail(SLO_ERR_UNSUPPORTED, "paged_attention_fp4: block_size must be a multiple of 64");
  if (dec && (!a->decode_lens || !a->decode_tables || a->decode_table_width <= 0))
    return fail(SLO_ERR_INVALID, "paged_attention_fp4: missing decode metadata");
  if (pre && (!a->prefill_cu_q || !a->prefill_cu_k || !a->prefill_tables || a->prefill_table_width <= 0))
    return fail(SLO_ERR_INVALID, "paged_attention_fp4: missing prefill metadata");
  if ((dec && (int64_t)a->decode_table_width * a->block_size > (1 << 22)) ||
      (pre && (int64_t)a->prefill_table_width * a->block_size > (1 << 22)))
    return fail(SLO_ERR_UNSUPPORTED, "paged_attention_fp4: tables span more than 2^22 tokens");
  return SLO_OK;
}

}  // namespace
}  // namespace slo

using namespace slo;

extern "C" int slo_paged_attention_fp4_workspace_bytes(const slo_paged_attention_args* a, size_t* bytes) {
  if (!bytes) return fail(SLO_ERR_INVALID, "paged_attention_fp4: null pointer");
  const int rc = check_args(a);
  if (rc) return rc;
  const Plan n = plan_of(a);
  *bytes = n.dbytes + n.pbytes;
  return SLO_OK;
}

extern "C" int slo_paged_attention_fp4(const slo_paged_attention_args* a, slo_stream_t stream) {
  const int rc = check_args(a);
  if (rc) return rc;
  const Plan n = plan_of(a);
  if (n.dbytes + n.pbytes > 0 && (!a->workspace || a->workspace_bytes < n.dbytes + n.pbytes ||
                                  reinterpret_cast<uintptr_t>(a->workspace) % 16))
    return fail(SLO_ERR_WORKSPACE, "paged_attention_fp4: workspace smaller than slo_paged_attention_fp4_workspace_bytes");
  if (!n.dwork && !n.ptiles) return SLO_OK;
  hipStream_t s = static_cast<hipStream_t>(stream);
  Fp4Params p = {};
  p.q = static_cast<const uint16_t*>(a->q);
  p.q_stride = a->q_row_stride;
  p.out = static_cast<uint16_t*>(a->out);
  p.out_stride = a->out_row_stride;
  p.num_q_rows = a->num_q_rows;
  p.kc = static_cast<const uint8_t*>(a->k_cache);
  p.vc = static_cast<const uint8_t*>(a->v_cache);
  p.ks = reinterpret_cast<const uint8_t*>(a->k_scale);
  p.vs = reinterpret_cast<const uint8_t*>(a->v_scale);
  p.num_blocks = a->num_blocks;
  p.block_size = a->block_size;
  p.hq = a->num_heads;
  p.hkv = a->num_kv_heads;
  p.group = a->num_heads / a->num_kv_heads;
  p.scale_log2 = (a->softmax_scale < 0 ? -a->softmax_scale : a->softmax_scale) * kLog2e;
  p.q_sign = a->softmax_scale < 0 ? 0x80008000u : 0u;
  if (n.dwork) {
    p.lens = a->decode_lens;
    p.tables = a->decode_tables;
    p.table_stride = a->decode_table_stride;
    p.table_width = a->decode_table_width;
    p.first_row = 0;
    p.rows = a->num_decode;
    p.budget = n.joined ? n.budget : 1;
    p.partial = static_cast<float*>(a->workspace);
    if (n.joined) {
      hipLaunchKernelGGL(fp4_decode_kernel<4>, dim3(p.hkv, n.budget + p.rows), dim3(256), 0, s, p);
      hipLaunchKernelGGL(fp4_join_kernel<8>, dim3(p.hq, p.rows), dim3(256), 0, s, p);
    } else {
      hipLaunchKernelGGL(fp4_decode_kernel<8>, dim3(p.hkv, p.rows), dim3(512), 0, s, p);
    }
  }
  if (n.ptiles) {
    p.lens = nullptr;
    p.cu_q = a->prefill_cu_q;
    p.cu_k = a->prefill_cu_k;
    p.tables = a->prefill_tables;
    p.table_stride = a->prefill_table_stride;
    p.table_width = a->prefill_table_width;
    p.first_row = a->num_decode;
    p.splits = n.psplits;
    p.chunk = n.pchunk;
    p.partial = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + n.dbytes);
    hipLaunchKernelGGL(fp4_prefill_kernel<kPrefillNT>, dim3(p.hkv, n.ptiles * p.splits, a->num_prefill), dim3(256), 0, s, p,
                       n.ptiles);
    if (p.splits > 1)
      hipLaunchKernelGGL(fp4_join_kernel<1>, dim3((unsigned)(((int64_t)a->max_q * p.hq + 7) / 8), a->num_prefill), dim3(256),
                         0, s, p);
  }
  return check_launch("paged_attention_fp4");
}
