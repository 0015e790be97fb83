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
// The rounding is the matrix operand's, and that of the attention over the other
// pools: outputs are off by 0.0020-0.0023 of their size where 32-bit
// probabilities leave 0.0016-0.0017, the rounding of the output alone; a second
// operand with what was rounded off would double the second product.
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

// What a prefill workgroup leaves for the join: the two tiles that it may have
// shared with its neighbours, the first and the last of its share, as they lie
// in the registers of its lanes (16 NT columns of a wavefront; four channels
// a piece), and where the last one's other parts are.
constexpr int kPrefillNT = 2;
struct Part {
  f32x4 o[2][4 * kPrefillNT][8][64];
  float m[2][64 * kPrefillNT], l[2][64 * kPrefillNT];
  int32_t row, tile, count, unused;  // count > 0: the last tile goes on in the next count - 1 shares
};

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
  // Query rows from first_idle + (ends ? *ends : 0) on belong to no row (the
  // capacity padding of a captured step); the launch that has `idle` set gives
  // them zeros, so every output row is defined.
  const int32_t* ends;
  int first_idle;
  bool idle;
  int rows;
  int budget;      // decode rows: about so many chunks over all rows
  float* partial;  // decode rows: [chunks, hq] records
  int shares;      // prefill rows: workgroups per kv head
  Part* parts;     // prefill rows: [shares, hkv]
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

__device__ __forceinline__ int chunk_units(const Fp4Params& p, int lane) {
  int total = 0;  // at most 2^15 rows of 2^15 units
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
// land as their lanes fetch them, so the lanes fetch in an order that spreads
// both operands' reads over the banks (of about 47 LDS cycles a step 9 are
// conflicts; the other conflicts are where the wavefronts meet): of K, 16-byte part p of token t
// lies at part p ^ (t / 4 mod 4) of its place; of V, token t lies at place
// t ^ (t / 4 mod 4).  Both stay within the 256 bytes of four tokens, so a
// fetch still takes whole lines.
struct Step {
  uint8_t k[2048], v[2048], ks[128], vs[128];
};
// Two in flight leave room for four workgroups on a CU; three for three, which
// took 43.9 us where two took 39.6 (the 64 rows below, by the same rule).
constexpr int kDepth = 2, kStepLoads = 5;

__device__ __forceinline__ void fetch(const Fp4Params& p, int64_t row, uint32_t to, int lane) {
  const uint32_t t = lane >> 2, x = (lane >> 4) & 3;
  const uint32_t ko = t * 64 + ((lane & 3) ^ x) * 16, vo = (t ^ x) * 64 + (lane & 3) * 16;
  const uint8_t *k = p.kc + row * 64, *v = p.vc + row * 64;
  dma16_nt_at(k, ko, to);
  dma16_nt_at(k, ko + 1024, to + 1024);
  dma16_nt_at(v, vo, to + 2 * 1024);
  dma16_nt_at(v, vo + 1024, to + 2 * 1024 + 1024);
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

__device__ __forceinline__ void clear_idle(const Fp4Params& p) {
  const int64_t from = (int64_t)p.first_idle + (p.ends ? max(*p.ends, 0) : 0);
  const int per = p.hq * (HD4 / 8);  // 16-byte pieces of a row
  const int64_t pieces = (p.num_q_rows - from) * per, stride = (int64_t)gridDim.x * gridDim.y * blockDim.x;
  for (int64_t i = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * blockDim.x + threadIdx.x; i < pieces; i += stride)
    *reinterpret_cast<u32x4*>(p.out + (from + i / per) * p.out_stride + 8 * (i % per)) = u32x4{0, 0, 0, 0};
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
// wavefronts' results meet in LDS.  Bound by the read: 64 rows of 512-4,096
// tokens and 8 kv heads, 172 MB, 36.5 us or 4.7 TB/s (31.5 us with the
// arithmetic left out, 39.4 with the default cache policy).  With chunks of
// another rule, steps in registers instead of LDS took 53 us where LDS took 40.
// 172.6 MB are fetched for 170.9 of codes and scales.
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
  if (p.idle) clear_idle(p);
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
      if (ahead == 1)
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(kStepLoads));
      else
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
      asm volatile("" ::: "memory");
      Tile t;
      read_step(t, ring[wave].steps[from], lane);
      from = from == kDepth - 1 ? 0 : from + 1;
      const int at = begin + WAVES * KT * i;
      // Every step runs, so that the accumulators stay where they are: one whose
      // page is not in the pool has no keys.
      const bool in = ok & 1;
      step<1>(t, !in || at + KT > g.lk, q, a, p.scale_log2, in ? at : 1 << 30, limit, g.lk, lane);
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
// each 16 tokens, V's eight of each 32 tokens.  Half a V operand is written at a
// time, two lanes to a bank: 32 of a step's 226 LDS cycles.
struct Stage {
  u32x4 k[4][4][64], v[2][8][64];
};

// A wavefront's quarter of a step: 16 tokens of K, and of V.
struct Quarter {
  u32x4 k, vs;
  uint32_t ks, v[4];
};

__device__ __forceinline__ void load_quarter(Quarter& t, const Fp4Params& p, int64_t row, int wave, int lane) {
  const uint32_t c = lane & 15, kg = lane >> 4;
  row += 16 * wave;
  const uint8_t *k = p.kc + row * 64, *v = p.vc + row * 64, *ks = p.ks + row * 4, *vs = p.vs + row * 4;
  t.k = *reinterpret_cast<const u32x4*>(k + (c * 64 + kg * 16));
  t.ks = ks[c * 4 + kg];
  t.vs = *reinterpret_cast<const u32x4*>(vs + kg * 16);
#pragma unroll
  for (int i = 0; i < 4; ++i) t.v[i] = *reinterpret_cast<const uint32_t*>(v + (kg * 256 + c * 4 + i * 64));
}

// `left`: tokens of the step that belong to the row; V's scales past them are
// cleared (see step).
__device__ __forceinline__ void stage(Stage& s, const Quarter& t, int left, int wave, int lane) {
  const int c = lane & 15, kg = lane >> 4;
  const float sc = e8m0(t.ks);
#pragma unroll
  for (int i = 0; i < 4; ++i) s.k[wave][i][lane] = e2m1_decode8(t.k[i], sc);
  float vs[4];
  const int turn = (9 + 8 * (c >> 2)) & 31;
#pragma unroll
  for (int i = 0; i < 4; ++i) vs[i] = __uint_as_float(__builtin_amdgcn_alignbit(t.vs[i], t.vs[i], turn));
  if (left < 64) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (16 * wave + 4 * kg + i >= left) vs[i] = 0.0f;
  }
  // Tokens 4 kg + i of the wavefront's 16: half of a lane's 32-token operands.
  auto pair = [&](auto sel) {
    constexpr int B = decltype(sel)::value;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = e2m1_pair<B>(t.v[i], vs[i]);
    u32x2* lo = reinterpret_cast<u32x2*>(&s.v[wave >> 1][2 * B][lane]) + (wave & 1);
    u32x2* hi = reinterpret_cast<u32x2*>(&s.v[wave >> 1][2 * B + 1][lane]) + (wave & 1);
    *lo = u32x2{__builtin_amdgcn_perm(w[1], w[0], 0x05040100u), __builtin_amdgcn_perm(w[3], w[2], 0x05040100u)};
    *hi = u32x2{__builtin_amdgcn_perm(w[1], w[0], 0x07060302u), __builtin_amdgcn_perm(w[3], w[2], 0x07060302u)};
  };
  pair(std::integral_constant<int, 0>{});
  pair(std::integral_constant<int, 1>{});
  pair(std::integral_constant<int, 2>{});
  pair(std::integral_constant<int, 3>{});
}

// 64 tokens of a wavefront's columns against the staged operands, read four
// ahead of the products.
template <int NT>
__device__ __forceinline__ void staged_step(const Stage& st, bool masked, const bf16x8 (&q)[NT][4], Acc<NT>& a, float c, int kv0,
                                            const int (&limit)[NT], int lane) {
  const int kg = lane >> 4;
  f32x4 s[NT][4];
  bf16x8 x[2][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[0][i] = as_bf16x8(st.k[0][i][lane]);
#pragma unroll
  for (int t = 0; t < 4; ++t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[(t + 1) & 1][i] = as_bf16x8(t < 3 ? st.k[t + 1][i][lane] : st.v[0][i][lane]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n][t] = mfma16(x[t & 1][i], q[n][i], i ? s[n][t] : f32x4{0, 0, 0, 0});
    __builtin_amdgcn_sched_barrier(0);
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
        const f32x4& e = s[n][2 * g + (i >> 1)];
        b[i] = pack_bf16x2(__builtin_amdgcn_exp2f(__builtin_fmaf(e[2 * (i & 1)], c, -a.m[n])),
                           __builtin_amdgcn_exp2f(__builtin_fmaf(e[2 * (i & 1) + 1], c, -a.m[n])));
      }
      pr[n][g] = as_bf16x8(b);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {  // V's operands, four at a time
    const int g = j >> 1;
    if (j < 3) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[(j + 1) & 1][i] = as_bf16x8(st.v[(j + 1) >> 1][4 * ((j + 1) & 1) + i][lane]);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n) a.o[n][4 * (j & 1) + i] = mfma16(x[j & 1][i], pr[n][g], a.o[n][4 * (j & 1) + i]);
    if (j & 1) {
#pragma unroll
      for (int n = 0; n < NT; ++n) a.l[n] = mfma16(ones(), pr[n][g], a.l[n]);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Prefill rows.  A tile is 64 NT columns, (query, head of the group) pairs of
// consecutive queries of one row, and has as many 64-token steps as its last
// query sees.  All tiles' steps, in row order, are cut into equal shares, one
// for each workgroup of a kv head: causal tiles differ in length, a row may be
// long and its queries few, and the lengths are known on the GPU only.  A tile
// that lies in one share is written out; the parts of one that is cut meet in
// fp4_join_kernel.
__device__ __forceinline__ int tiles_of(const Fp4Params& p, int per, int r) {
  const Row g = row_of(p, r);
  return g.lq > 0 ? (g.lq + per - 1) / per : 0;
}

__device__ __forceinline__ int steps_of(int lq, int prefix, int lk, int per, int t) {
  return (max(min(prefix + min((t + 1) * per, lq), lk), 1) + 63) >> 6;
}

// Sum over a 256-thread workgroup, before this thread and in all.
__device__ __forceinline__ int group_scan(int x, int* sums, int& total) {
  const int wave = threadIdx.x >> 6;
  const int upto = wave_scan(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) sums[wave] = upto;
  __syncthreads();
  total = sums[0] + sums[1] + sums[2] + sums[3];
  int before = upto - x;
#pragma unroll
  for (int w = 0; w < 3; ++w) before += w < wave ? sums[w] : 0;
  return before;
}

constexpr int kMaxPrefillRows = 1024;
constexpr int kLeastSteps = 4;  // of a share

struct Rows {
  int first[kMaxPrefillRows + 1];  // number of each row's first tile
  int lq[kMaxPrefillRows], prefix[kMaxPrefillRows], lk[kMaxPrefillRows];
  int sums[4];
  int row, tile, skip;
};

// A workgroup's share: where it begins, its steps, and those of a whole one.
struct Share {
  int row, tile, skip, steps, each;
};

__device__ __forceinline__ Share find_share(const Fp4Params& p, int per, int share, Rows& s) {
  const int tid = threadIdx.x;
  int tiles = 0;
  for (int base = 0; base < p.rows; base += 256) {
    const int r = base + tid;
    int all, n = 0;
    if (r < p.rows) {
      const Row g = row_of(p, r);
      s.lq[r] = g.lq;
      s.prefix[r] = g.prefix;
      s.lk[r] = g.lk;
      n = g.lq > 0 ? (g.lq + per - 1) / per : 0;
    }
    const int before = group_scan(n, s.sums, all);
    if (r < p.rows) s.first[r] = tiles + before;
    tiles += all;
  }
  if (tid == 0) s.first[p.rows] = tiles;
  __syncthreads();
  // Tile i's row (first[row] <= i < first[row + 1]) and steps.
  auto steps = [&](int i, int& row) {
    if (i >= tiles) return 0;
    int lo = 0, hi = p.rows;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s.first[mid] <= i) lo = mid; else hi = mid;
    }
    row = lo;
    return steps_of(s.lq[lo], s.prefix[lo], s.lk[lo], per, i - s.first[lo]);
  };
  int row = 0, own = steps(tid, row), mine = own, total, at;
  if (tiles > 256) {
    int ignored;
    for (int i = tid + 256; i < tiles; i += 256) mine += steps(i, ignored);
  }
  at = group_scan(mine, s.sums, total);
  Share c = {0, 0, 0, 0, max((total + p.shares - 1) / p.shares, kLeastSteps)};
  const int begin = share * c.each;
  if (begin >= total) return c;
  if (tiles <= 256) {
    if (at <= begin && begin < at + own) {
      s.row = row;
      s.tile = tid - s.first[row];
      s.skip = begin - at;
    }
  } else {
    int before = 0;
    for (int base = 0; base < tiles && before <= begin; base += 256) {
      int all;
      const int n = steps(base + tid, row);
      at = before + group_scan(n, s.sums, all);
      if (at <= begin && begin < at + n) {
        s.row = row;
        s.tile = base + tid - s.first[row];
        s.skip = begin - at;
      }
      before += all;
    }
  }
  __syncthreads();
  c.row = s.row;
  c.tile = s.tile;
  c.skip = s.skip;
  c.steps = min(c.each, total - begin);
  __syncthreads();  // the steps' operands take this memory next
  return c;
}

// Steps [from, to) of one tile for this wavefront's columns.
template <int NT>
__device__ __forceinline__ void run_tile(const Fp4Params& p, const Row& g, int r, int head, int w0, int from, int to,
                                         Stage (&st)[2], int& buf, bf16x8 (&q)[NT][4], Acc<NT>& a, int wave, int lane) {
  const int per = 16 * NT / p.group;
  const int t0 = w0 + wave * per, t1 = min(t0 + per, g.lq);
  const int all = min(max(g.prefix + min(w0 + 4 * per, g.lq), 0), g.lk);  // keys that one of the queries sees
  const int full = min(g.prefix + t0 + 1, g.lk);                          // that all of the wavefront's see
  const int col = lane & 15, kg = lane >> 4;
  int limit[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int x = 16 * n + col, tok = t0 + x / p.group;
    const bool live = x < per * p.group && tok < t1;
    limit[n] = live ? min(g.prefix + tok + 1, g.lk) : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) q[n][i] = load_q(p, g.q0 + tok, head * p.group + x % p.group, 32 * kg + 8 * i, live);
  }
  clear(a);
  const int k0 = from * 64, k1 = min(to * 64, all);
  if (k0 >= k1) return;
  Walk w{row_table(p, r), k0 / p.block_size, 0, p.block_size, p.num_blocks, p.hkv, head};
  w.off = k0 - w.page * p.block_size;
  Quarter t;
  bool ok, next_ok = false;
  load_quarter(t, p, w.row(ok), wave, lane);
  for (int at = k0; at < k1; at += 64, buf ^= 1) {
    // Every step runs, so that the accumulators stay where they are: one whose
    // page is not in the pool has no keys.
    stage(st[buf], t, ok ? all - at : 0, wave, lane);
    if (at + 64 < k1) {
      w.advance(64);
      load_quarter(t, p, w.row(next_ok), wave, lane);
    }
    // Two buffers: a wavefront comes to write this one again only past the
    // next step's barrier, when every wavefront has left it.  The barrier
    // waits for LDS only: the loads of the next step stay in flight.
    lds_sync();
    staged_step<NT>(st[buf], !ok || at + 64 > full, q, a, p.scale_log2, ok ? at : 1 << 30, limit, lane);
    ok = next_ok;
  }
}

// A workgroup's four wavefronts turn each step's codes into operands together,
// each a quarter, and each runs 16 NT columns over them; the next step's codes
// load meanwhile.  Chunks of 1,000, 300 and 77 queries on 3,500, 1,000 and
// 3,077 keys, 16 query heads: every wavefront converting for itself 175 us,
// staged 80, with equal shares 51.  Of the last, copies with a part removed save
// 36 us without the steps, 9 without the operand reads from LDS, 6 without the
// output products, 4 without the exponents, 5 without the conversion.
template <int NT>
__global__ void __launch_bounds__(256, 2)
fp4_prefill_kernel(Fp4Params p) {
  __shared__ union {
    Stage st[2];
    Rows rows;
  } lds;
  const int head = blockIdx.x, share = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per = 4 * (16 * NT / p.group);
  Part& part = p.parts[(int64_t)share * p.hkv + head];
  const Share mine = find_share(p, per, share, lds.rows);
  int left = __builtin_amdgcn_readfirstlane(mine.steps), r = __builtin_amdgcn_readfirstlane(mine.row);
  int tile = __builtin_amdgcn_readfirstlane(mine.tile), from = __builtin_amdgcn_readfirstlane(mine.skip), buf = 0;
  const int each = __builtin_amdgcn_readfirstlane(mine.each);
  int open_row = 0, open_tile = 0, open = 0;
  while (left > 0) {
    const Row g = row_of(p, r);
    const int steps = steps_of(g.lq, g.prefix, g.lk, per, tile), to = min(steps, from + left);
    bf16x8 q[NT][4];
    Acc<NT> a;
    run_tile<NT>(p, g, r, head, tile * per, from, to, lds.st, buf, q, a, wave, lane);
    int c = lane & 15;
    asm("" : "+v"(c));  // found again here, so that the loop need not hold it in registers
    const int kg = lane >> 4;
    if (from == 0 && to == steps) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int x = 16 * n + c, tok = tile * per + wave * (per >> 2) + x / p.group, h = head * p.group + x % p.group;
        if (x >= (per >> 2) * p.group || tok >= g.lq) continue;
        const float inv = a.l[n][0] == 0.0f ? 0.0f : 1.0f / a.l[n][0];
        uint16_t* out = p.out + (g.q0 + tok) * p.out_stride + h * HD4 + 32 * kg;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<u32x4*>(out + 8 * i) =
              u32x4{pack_bf16x2(a.o[n][0][i] * inv, a.o[n][1][i] * inv), pack_bf16x2(a.o[n][2][i] * inv, a.o[n][3][i] * inv),
                    pack_bf16x2(a.o[n][4][i] * inv, a.o[n][5][i] * inv), pack_bf16x2(a.o[n][6][i] * inv, a.o[n][7][i] * inv)};
      }
    } else {
      // A part that does not begin its tile is its share's first.
      const int k = from == 0;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int block = NT * wave + n;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 8; e += 4)
            part.o[k][block][2 * i + (e >> 2)][lane] = f32x4{a.o[n][e][i], a.o[n][e + 1][i], a.o[n][e + 2][i], a.o[n][e + 3][i]};
        if (kg == 0) {
          part.m[k][16 * block + c] = a.m[n];
          part.l[k][16 * block + c] = a.l[n][0];
        }
      }
      if (k) {
        open_row = r;
        open_tile = tile;
        open = steps - to;
      }
    }
    left -= to - from;
    from = 0;
    if (left > 0 && ++tile >= (g.lq + per - 1) / per) {
      tile = 0;
      do ++r;
      while (tiles_of(p, per, r) == 0);
    }
  }
  if (p.idle) clear_idle(p);
  if (threadIdx.x == 0) {
    part.row = open_row;
    part.tile = open_tile;
    part.count = open ? 1 + (open + each - 1) / each : 0;
  }
}

// Joins the partial results of decode row r's chunks: a workgroup per (row,
// head), four channels a lane.  Half wavefront i takes chunks i, i + 8, ... and
// the eight sums meet in LDS in that order.
__device__ __forceinline__ void join_decode(const Fp4Params& p, int r, int h) {
  __shared__ f32x4 so[8][32];
  __shared__ float sl[8];
  const int lane = threadIdx.x & 31, i = threadIdx.x >> 5;
  Chunk c;
  find_chunk(p, r, true, threadIdx.x & 63, c);
  if (c.count == 1) return;  // written by its only chunk
  const float* rec = p.partial + ((int64_t)c.first * p.hq + h) * RECORD;
  const int64_t stride = (int64_t)p.hq * RECORD;
  float m = kNone;
  for (int s = lane; s < c.count; s += 32) m = fmaxf(m, rec[s * stride + HD4]);
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) m = wave_max_xor(m, d);
  f32x4 o = {0, 0, 0, 0};
  float l = 0;
#pragma unroll 4
  for (int s = i; s < c.count; s += 8) {
    const float* e = rec + s * stride;
    const float w = __builtin_amdgcn_exp2f(e[HD4] - m);
    o += *reinterpret_cast<const f32x4*>(e + 4 * lane) * w;
    l += e[HD4 + 1] * w;
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
  *reinterpret_cast<u32x2*>(p.out + (int64_t)r * p.out_stride + h * HD4 + 4 * lane) =
      u32x2{pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv)};
}

// Joins the parts of the tile that a share leaves open, in order: a workgroup
// per 16 of its columns.
template <int NT>
__device__ __forceinline__ void join_prefill(const Fp4Params& p, int share, int head, int block) {
  const Part* part = p.parts + (int64_t)share * p.hkv + head;
  const int count = part->count;
  if (count == 0) return;
  const Row g = row_of(p, part->row);
  const int quarter = 16 * NT / p.group;
  const int lane = threadIdx.x & 63, col = lane & 15, kg = lane >> 4;
  const int x = 16 * (block % NT) + col, tok = (part->tile * 4 + block / NT) * quarter + x / p.group;
  if (x >= quarter * p.group || tok >= g.lq) return;
  const int at = 16 * block + col;
  float m = part->m[1][at];
  for (int s = 1; s < count; ++s) m = fmaxf(m, part[(int64_t)s * p.hkv].m[0][at]);
  f32x4 o[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
  float l = 0;
#pragma unroll 2
  for (int s = 0; s < count; ++s) {
    const Part& e = part[(int64_t)s * p.hkv];
    const int k = s == 0;
    const float w = __builtin_amdgcn_exp2f(e.m[k][at] - m);
#pragma unroll
    for (int j = 0; j < 2; ++j) o[j] += e.o[k][block][(threadIdx.x >> 6) + 4 * j][lane] * w;
    l += e.l[k][at] * w;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint16_t* out = p.out + (g.q0 + tok) * p.out_stride + (head * p.group + x % p.group) * HD4 + 32 * kg;
#pragma unroll
  for (int j = 0; j < 2; ++j)
    *reinterpret_cast<u32x2*>(out + 4 * ((threadIdx.x >> 6) + 4 * j)) =
        u32x2{pack_bf16x2(o[j][0] * inv, o[j][1] * inv), pack_bf16x2(o[j][2] * inv, o[j][3] * inv)};
}

// One launch joins both phases: workgroups below `decode` take decode rows.
__global__ void __launch_bounds__(256)
fp4_join_kernel(Fp4Params d, Fp4Params f, int decode) {
  int i = blockIdx.x;
  if (i < decode) {
    join_decode(d, i / d.hq, i % d.hq);
    return;
  }
  i -= decode;
  const int blocks = 4 * kPrefillNT, block = i % blocks;
  i /= blocks;
  join_prefill<kPrefillNT>(f, i / f.hkv, i % f.hkv, block);
}

// Two prefill workgroups fit a CU (64 KiB of LDS and 256 registers each); all
// heads' shares together are one for each.  The chunks above: 52 us so, 62, 60
// and 58 with 256, 384 and 1,024 shares; the join 12.5, 9.8, 11.7 and 16.2.
constexpr int kPrefillShares = 512;

// Chunks of all decode rows and heads together: one for each of the four
// workgroups that a CU holds.  64 rows of 512-4,096 tokens, 8 kv heads: 36.6 us
// and 5.1 us to join them, 38.1 + 6.6 with twice as many, 42.1 + 6.8 with four
// times; three rows of 20,000-60,000 30.2 + 4.2, 32.1 + 5.8, 35.9 + 7.2.
constexpr int kDecodeChunks = 1024;
// Where the tables span at most this many tokens rows are not cut, and eight
// wavefronts take each: one row of 1,000 6.7 us, 5.4 + 4.4 us as two chunks and
// their join.  The launch knows the tables' width only, so in wider tables (a
// captured step's) such a row is cut into chunks of 256 tokens and more and
// joined: 20.9 us a call in tables of 4,096 and of 40,960 tokens, 15.9 in 1,024.
constexpr int kWholeRow = 1024;

struct Plan {
  bool dwork, joined;
  int budget, shares;
  size_t dbytes, pbytes;
};

// Prefill rows' shares are numbered steps of all tiles together, in 32 bits on
// the GPU (find_share adds up to two shares' steps to their sum).
constexpr int64_t kMaxSteps = 1 << 30;

int64_t prefill_tiles(const slo_paged_attention_args* a) {
  // The rows' queries together bound the tiles.
  const int per = 4 * (16 * kPrefillNT / (a->num_heads / a->num_kv_heads));
  return (int64_t)(a->num_q_rows - a->num_decode) / per + a->num_prefill;
}

Plan plan_of(const slo_paged_attention_args* a) {
  Plan n = {false, false, 0, 0, 0, 0};
  if (a->num_decode > 0 && (a->phases & SLO_PHASE_DECODE)) {
    n.dwork = true;
    n.joined = (int64_t)a->decode_table_width * a->block_size > kWholeRow;
    n.budget = n.joined ? (kDecodeChunks + a->num_kv_heads - 1) / a->num_kv_heads : 0;
    if (n.joined) n.dbytes = (size_t)(n.budget + a->num_decode) * a->num_heads * RECORD * 4;
  }
  if (a->num_prefill > 0 && (a->phases & SLO_PHASE_PREFILL)) {
    // max_k only keeps the shares of short rows in wide tables few: any number
    // of them covers all steps, and without it the tables' width bounds the keys.
    const int64_t cap = (int64_t)a->prefill_table_width * a->block_size, keys = a->max_k > 0 && a->max_k < cap ? a->max_k : cap;
    // No more shares than steps / kLeastSteps.
    const int64_t steps = prefill_tiles(a) * ((keys + 63) / 64);
    const int64_t most = (steps + kLeastSteps - 1) / kLeastSteps, full = (kPrefillShares + a->num_kv_heads - 1) / a->num_kv_heads;
    n.shares = (int)(most < 1 ? 1 : most < full ? most : full);
    n.pbytes = (size_t)n.shares * a->num_kv_heads * sizeof(Part);
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
  if (a->num_decode > 32768 || a->num_prefill > kMaxPrefillRows)
    return fail(SLO_ERR_UNSUPPORTED, "paged_attention_fp4: more than 32768 decode or 1024 prefill rows");
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
  if (pre && prefill_tiles(a) * ((int64_t)a->prefill_table_width * a->block_size / 64) > kMaxSteps)
    return fail(SLO_ERR_UNSUPPORTED, "paged_attention_fp4: prefill queries times the tables' tokens past 2^30 steps of a tile");
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
  if (!n.dwork && !n.shares) return SLO_OK;
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
  const bool rows = a->num_prefill > 0 && a->prefill_cu_q;  // whatever the phases
  p.ends = rows ? a->prefill_cu_q + a->num_prefill : nullptr;
  p.first_idle = a->num_decode;
  Fp4Params d = p, f = p;
  d.idle = !n.shares && a->num_q_rows > a->num_decode;
  f.idle = true;
  if (n.dwork) {
    d.lens = a->decode_lens;
    d.tables = a->decode_tables;
    d.table_stride = a->decode_table_stride;
    d.table_width = a->decode_table_width;
    d.rows = a->num_decode;
    d.budget = n.joined ? n.budget : 1;
    d.partial = static_cast<float*>(a->workspace);
    if (n.joined)
      hipLaunchKernelGGL(fp4_decode_kernel<4>, dim3(d.hkv, n.budget + d.rows), dim3(256), 0, s, d);
    else
      hipLaunchKernelGGL(fp4_decode_kernel<8>, dim3(d.hkv, d.rows), dim3(512), 0, s, d);
  }
  if (n.shares) {
    f.cu_q = a->prefill_cu_q;
    f.cu_k = a->prefill_cu_k;
    f.tables = a->prefill_tables;
    f.table_stride = a->prefill_table_stride;
    f.table_width = a->prefill_table_width;
    f.first_row = a->num_decode;
    f.rows = a->num_prefill;
    f.shares = n.shares;
    f.parts = reinterpret_cast<Part*>(static_cast<char*>(a->workspace) + n.dbytes);
    hipLaunchKernelGGL(fp4_prefill_kernel<kPrefillNT>, dim3(f.hkv, f.shares), dim3(256), 0, s, f);
  }
  const int decode = n.joined ? d.rows * d.hq : 0, prefill = n.shares > 1 ? (n.shares - 1) * f.hkv * 4 * kPrefillNT : 0;
  if (decode + prefill) hipLaunchKernelGGL(fp4_join_kernel, dim3(decode + prefill), dim3(256), 0, s, d, f, decode);
  return check_launch("paged_attention_fp4");
}
