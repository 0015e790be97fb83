// Eviction of cached tokens by accumulated attention weight (gfx950).
//
// A row of n > budget tokens keeps, for every kv head by itself, its newest
// `recent` tokens and the budget - recent heaviest of the others (ties: the
// lowest position), moved in position order to the row's first `budget`
// places.  Keys carry their rotary position, so attention over the moved
// tokens is the attention over the kept ones.  Two kernels: the choice, one
// workgroup per (layer, row, kv head), and the move.
#include "capi_internal.h"
#include "fp4.h"

namespace slo {
namespace {

constexpr int SELECT_NT = 512, RUN = 16;

struct EvictParams {
  float* scores;  // [layers, num_blocks, hkv, block_size]
  const int32_t* lens;
  const int32_t* tables;
  int table_stride, table_width, num_blocks, block_size, hkv, rows, budget, recent;
  float inv_block;    // 1 / block_size
  int32_t* new_lens;  // [rows]
  int32_t* kept;      // [layers, rows, hkv, budget]
};

__device__ __forceinline__ int length_of(const EvictParams& p, int r) {
  return min(max(p.lens[r], 0), p.table_width * p.block_size);
}

// token / block_size and the remainder, by the reciprocal and one correction
// (tokens are below 2^24, so the product is off by less than one).
__device__ __forceinline__ int block_of(const EvictParams& p, int token, int& off) {
  int b = (int)((float)token * p.inv_block);
  off = token - b * p.block_size;
  if (off < 0) {
    --b;
    off += p.block_size;
  } else if (off >= p.block_size) {
    ++b;
    off -= p.block_size;
  }
  return b;
}

__device__ __forceinline__ int page_at(const EvictParams& p, int r, int token, int& off) {
  const int b = p.tables[(int64_t)r * p.table_stride + block_of(p, token, off)];
  return b >= 0 && b < p.num_blocks ? b : -1;
}

// An unsigned key that orders like the weight: NaN, and tokens in no page,
// below every number; -0 equal to 0.
__device__ __forceinline__ uint32_t order_key(float w) {
  const uint32_t u = __float_as_uint(w + 0.0f);
  return w != w ? 0u : u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

// Exclusive sum over the workgroup's threads; `total` receives the whole.
__device__ __forceinline__ int block_scan(int x, int* sums, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int s = wave_scan(x);
  __syncthreads();
  if (lane == 63) sums[wave] = s;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < SELECT_NT / 64; ++w) {
    before += w < wave ? sums[w] : 0;
    all += sums[w];
  }
  total = all;
  return before + s - x;
}

// A thread's run of tokens t0 .. t0 + RUN - 1 (inside one page) as keys.
__device__ __forceinline__ void load_run(const EvictParams& p, const float* scores, int r, int head, int t0, int end,
                                         uint32_t (&k)[RUN]) {
  int b = -1, off = 0;
  if (t0 < end) b = page_at(p, r, t0, off);
#pragma unroll
  for (int i = 0; i < RUN; i += 4) {
    f32x4 x = {0, 0, 0, 0};
    if (b >= 0) x = *reinterpret_cast<const f32x4*>(scores + ((int64_t)b * p.hkv + head) * p.block_size + off + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) k[i + j] = b < 0 ? 0u : order_key(x[j]);
  }
}

// The choice.  The budget - recent heaviest of the first n - recent tokens are
// those above the key T of that rank and the first few equal to it.  T is
// found by its 11, 11 and 10 bits, most significant first, from a histogram of
// the keys that share the bits found so far; then one sum over the threads
// places every kept position.  A thread owns RUN consecutive tokens, so a row of
// up to SELECT_NT * RUN tokens is read once and stays in registers; a longer
// one is read again for each step.  One row of 1,500 tokens and 8 heads 11 us,
// a chain of round trips and barriers; 16 rows of 3,000-8,192 in 8 layers 33 us
// (148 with 8-bit digits and the weights read again for each).
__global__ void __launch_bounds__(SELECT_NT)
evict_select_kernel(EvictParams p) {
  __shared__ int hist[2048], sums[SELECT_NT / 64], found[2];
  const int head = blockIdx.x, r = blockIdx.y, layer = blockIdx.z;
  const int n = length_of(p, r), tid = threadIdx.x;
  int32_t* kept = p.kept + (((int64_t)layer * p.rows + r) * p.hkv + head) * p.budget;
  if (head == 0 && layer == 0 && tid == 0) p.new_lens[r] = min(n, p.budget);
  if (n <= p.budget) {
    for (int i = tid; i < p.budget; i += SELECT_NT) kept[i] = i < n ? i : -1;
    return;
  }
  const float* scores = p.scores + (int64_t)layer * p.num_blocks * p.hkv * p.block_size;
  const int old = n - p.recent;
  constexpr int SPAN = SELECT_NT * RUN;
  uint32_t k[RUN];
  load_run(p, scores, r, head, tid * RUN, old, k);
  int need = p.budget - p.recent;  // still to choose among the keys that match `prefix`
  uint32_t prefix = 0;
#pragma unroll 1  // three copies of this code take longer to fetch than to run
  for (int step = 0; step < 3; ++step) {
    const int shift = step == 0 ? 21 : step == 1 ? 10 : 0, bins = step == 2 ? 1024 : 2048;
    const uint32_t known = step == 0 ? 0u : step == 1 ? 0xffe00000u : 0xfffffc00u;
    if (need <= 0) break;
    for (int i = tid; i < 2048; i += SELECT_NT) hist[i] = 0;
    __syncthreads();
    for (int base = 0; base < old; base += SPAN) {
      const int t0 = base + tid * RUN;
      if (base) load_run(p, scores, r, head, t0, old, k);
#pragma unroll
      for (int i = 0; i < RUN; ++i)
        if (t0 + i < old && ((k[i] ^ prefix) & known) == 0) atomicAdd(&hist[(k[i] >> shift) & (bins - 1)], 1);
    }
    __syncthreads();
    // Thread t adds up the bins from the top: those above its own are before it.
    constexpr int PER = 2048 / SELECT_NT;
    int mine = 0, bin[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      bin[i] = hist[2047 - (tid * PER + i)];  // empty above `bins`
      mine += bin[i];
    }
    int total, above = block_scan(mine, sums, total);
    if (above < need && above + mine >= need) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (above < need && above + bin[i] >= need) {
          found[0] = 2047 - (tid * PER + i);
          found[1] = above;
        }
        above += bin[i];
      }
    }
    __syncthreads();
    prefix |= (uint32_t)found[0] << shift;
    need -= found[1];
    if (old > SPAN) load_run(p, scores, r, head, tid * RUN, old, k);
    __syncthreads();
  }
  // `need` of the keys equal to prefix are kept, the first ones; none where no
  // old token is kept.
  const bool any = p.budget > p.recent;
  int equal_before = 0, kept_before = 0;
  for (int base = 0; base < n; base += SPAN) {
    const int t0 = base + tid * RUN;
    if (base) load_run(p, scores, r, head, t0, old, k);
    int above = 0, equal = 0;
#pragma unroll
    for (int i = 0; i < RUN; ++i) {
      const int t = t0 + i;
      above += t < n && (t >= old || (any && k[i] > prefix));
      equal += t < old && any && k[i] == prefix;
    }
    int total;
    const int before = block_scan(above | equal << 16, sums, total);  // both are at most SPAN < 2^15
    int eq = equal_before + (before >> 16), at = kept_before + (before & 0xffff) + min(eq, need) - min(equal_before, need);
#pragma unroll
    for (int i = 0; i < RUN; ++i) {
      const int t = t0 + i;
      const bool is = t < old && any && k[i] == prefix;
      if ((t < n && (t >= old || (any && k[i] > prefix))) || (is && eq < need)) kept[at++] = t;
      eq += is;
    }
    kept_before += (total & 0xffff) + min(equal_before + (total >> 16), need) - min(equal_before, need);
    equal_before += total >> 16;
  }
}

// One array of the pool that moves with the tokens, or 64 bytes of each of its
// rows: `unit` bytes of a lane, `units` lanes a token.
struct Stream {
  uint8_t* base;
  int64_t layer_bytes, page_bytes, head_bytes;  // 2^24 tokens of 128 bytes are 2^31
  int token_bytes, unit, units;
};

constexpr int kMaxStreams = 20, kDepth = 8;

struct MoveParams {
  EvictParams e;
  Stream s[kMaxStreams];
};

// The move, in place: a workgroup takes one stream of one (layer, row, kv head)
// and fills its places in ascending order.  The token that comes to place i
// lies at i or later, so once the places up to some point have been read, what
// is stored there is not read again: a tile of 256 kDepth units is loaded whole,
// and stored after a barrier.  A row's order leaves no more workgroups than
// streams, so each keeps kDepth loads a lane in flight (a tile is 512 tokens of
// 64 bytes).  One row cut from 1,500 to 1,024 bf16 tokens: 8.8 us (10.6 with
// four in flight, 39 with four and whole rows); 16 rows to 2,048 tokens in 8
// layers of a 4-bit pool: 161 us for 0.57 GB, 3.5 TB/s.  What it moves is 0.81
// GB, 5.0 TB/s: 0.31 GB are written, but 0.50 GB read for 0.29, in lines of 128
// bytes, as the 64-byte rows that stay lie one or two to a line.  (When read
// backs were stored through the caches: 184, 213 with four in flight, 199 with
// four and twice the lanes, 6.7 there for the one row.)
template <typename U>
__device__ __forceinline__ void move_stream(const EvictParams& p, const Stream& s, int r, int head, int layer) {
  const int32_t* kept = p.kept + (((int64_t)layer * p.rows + r) * p.hkv + head) * p.budget;
  uint8_t* base = s.base + layer * s.layer_bytes + head * s.head_bytes;
  const int shift = s.units == 4 ? 2 : s.units == 2 ? 1 : 0;  // 1, 2 or 4 lanes a token
  const int part = (threadIdx.x & (s.units - 1)) * (int)sizeof(U), tile = (256 >> shift) * kDepth;
  for (int i0 = 0; i0 < p.budget; i0 += tile) {
    int src[kDepth];
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      const int i = i0 + ((256 * d + (int)threadIdx.x) >> shift);
      src[d] = i < p.budget ? kept[i] : -1;
      if (src[d] == i) src[d] = -1;  // already there
    }
    U x[kDepth];
    int64_t to[kDepth];
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      const int i = i0 + ((256 * d + (int)threadIdx.x) >> shift);
      to[d] = -1;
      if (src[d] < 0) continue;
      int soff, doff;
      const int sb = page_at(p, r, src[d], soff), db = page_at(p, r, i, doff);
      if (sb < 0 || db < 0) continue;
      x[d] = *reinterpret_cast<const U*>(base + (sb * s.page_bytes + (int64_t)soff * s.token_bytes + part));
      to[d] = db * s.page_bytes + (int64_t)doff * s.token_bytes + part;
    }
    // The barrier alone orders LDS accesses; the loads have to have come back.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int d = 0; d < kDepth; ++d)
      if (to[d] >= 0) *reinterpret_cast<U*>(base + to[d]) = x[d];
  }
}

__global__ void __launch_bounds__(256)
evict_move_kernel(MoveParams m) {
  const EvictParams& p = m.e;
  const int head = blockIdx.x % p.hkv, which = blockIdx.x / p.hkv, r = blockIdx.y, layer = blockIdx.z;
  const int n = length_of(p, r);
  if (n <= p.budget) return;
  const Stream& s = m.s[which];
  if (s.unit == 16) {
    move_stream<u32x4>(p, s, r, head, layer);
  } else if (s.unit == 4) {
    move_stream<uint32_t>(p, s, r, head, layer);
  } else {
    move_stream<uint16_t>(p, s, r, head, layer);
  }
  if (which) return;
  // Stream 0 is the scores: the places given up start again from zero.
  float* scores = p.scores + (int64_t)layer * p.num_blocks * p.hkv * p.block_size;
  for (int t = p.budget + threadIdx.x; t < n; t += 256) {
    int off;
    const int b = page_at(p, r, t, off);
    if (b >= 0) scores[((int64_t)b * p.hkv + head) * p.block_size + off] = 0.0f;
  }
}

}  // namespace
}  // namespace slo

using namespace slo;

extern "C" int slo_evict_kv(const slo_evict_kv_args* a, slo_stream_t stream) {
  if (!a) return fail(SLO_ERR_INVALID, "evict_kv: null args");
  if (a->num_layers <= 0 || a->num_rows < 0 || a->num_kv_heads <= 0 || a->num_blocks <= 0 || a->block_size <= 0)
    return fail(SLO_ERR_INVALID, "evict_kv: bad layer, row, head or block count");
  if (a->budget <= 0 || a->recent < 0 || a->recent > a->budget)
    return fail(SLO_ERR_INVALID, "evict_kv: budget must be positive and recent from 0 to budget");
  if (a->kv_dtype < KV_BF16 || a->kv_dtype > KV_FP4_E2M1) return fail(SLO_ERR_INVALID, "evict_kv: bad kv_dtype");
  if (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256)
    return fail(SLO_ERR_UNSUPPORTED, "evict_kv: head_dim must be 64, 128 or 256");
  if (a->num_rows > 65535 || a->num_layers > 65535 || a->num_kv_heads > 65535)
    return fail(SLO_ERR_UNSUPPORTED, "evict_kv: more than 65535 rows, layers or heads");
  if (a->num_rows == 0) return SLO_OK;
  if (!a->k_cache || !a->v_cache || !a->scores || !a->lens || !a->tables || !a->new_lens || !a->kept || a->table_width <= 0)
    return fail(SLO_ERR_INVALID, "evict_kv: null pointer");
  if (a->kv_dtype != KV_BF16 && (!a->k_scale || !a->v_scale)) return fail(SLO_ERR_INVALID, "evict_kv: a quantised pool needs its scales");
  if ((reinterpret_cast<uintptr_t>(a->k_cache) % 16) || (reinterpret_cast<uintptr_t>(a->v_cache) % 16) ||
      (reinterpret_cast<uintptr_t>(a->k_scale) % 4) || (reinterpret_cast<uintptr_t>(a->v_scale) % 4) ||
      (reinterpret_cast<uintptr_t>(a->scores) % 16))
    return fail(SLO_ERR_INVALID, "evict_kv: pools and scores must be 16-byte aligned");
  if (a->block_size % 64) return fail(SLO_ERR_UNSUPPORTED, "evict_kv: block_size must be a multiple of 64");
  if ((int64_t)a->table_width * a->block_size > (1 << 24) || a->budget > (1 << 24))
    return fail(SLO_ERR_UNSUPPORTED, "evict_kv: more than 2^24 tokens a row");
  MoveParams m = {};
  EvictParams& p = m.e;
  p.scores = a->scores;
  p.lens = a->lens;
  p.tables = a->tables;
  p.table_stride = a->table_stride;
  p.table_width = a->table_width;
  p.num_blocks = a->num_blocks;
  p.block_size = a->block_size;
  p.hkv = a->num_kv_heads;
  p.rows = a->num_rows;
  p.budget = a->budget;
  p.recent = a->recent;
  p.new_lens = a->new_lens;
  p.kept = a->kept;
  const bool fp4 = a->kv_dtype == KV_FP4_E2M1;
  p.inv_block = 1.0f / (float)a->block_size;
  // Rows of `row` bytes, pages head by head (4-bit pools and the scores) or
  // token by token, in streams of up to 64 bytes of each row.
  int streams = 0;
  auto add = [&](void* base, int row, bool by_head) {
    const int64_t page = (int64_t)a->block_size * a->num_kv_heads * row;
    const int unit = row % 16 == 0 ? 16 : row % 4 == 0 ? 4 : 2, most = 4 * unit;
    for (int at = 0; at < row; at += most) {
      const int bytes = row - at < most ? row - at : most;
      m.s[streams++] = Stream{static_cast<uint8_t*>(base) + at, page * a->num_blocks, page,
                              by_head ? (int64_t)a->block_size * row : row, by_head ? row : a->num_kv_heads * row, unit,
                              bytes / unit};
    }
  };
  const int row = a->kv_dtype == KV_BF16 ? 2 * a->head_dim : fp4 ? a->head_dim / 2 : a->head_dim;
  add(a->scores, 4, true);
  add(a->k_cache, row, fp4);
  add(a->v_cache, row, fp4);
  if (a->kv_dtype != KV_BF16) {
    const int scale = fp4 ? a->head_dim / kFp4Group : 4;
    add(a->k_scale, scale, fp4);
    add(a->v_scale, scale, fp4);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(evict_select_kernel, dim3(p.hkv, p.rows, a->num_layers), dim3(SELECT_NT), 0, s, p);
  hipLaunchKernelGGL(evict_move_kernel, dim3(p.hkv * streams, p.rows, a->num_layers), dim3(256), 0, s, m);
  return check_launch("evict_kv");
}
