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

constexpr int SELECT_NT = 1024;

struct EvictParams {
  float* scores;  // [layers, num_blocks, hkv, block_size]
  const int32_t* lens;
  const int32_t* tables;
  int table_stride, table_width, num_blocks, block_size, hkv, rows, budget, recent;
  int32_t* new_lens;  // [rows]
  int32_t* kept;      // [layers, rows, hkv, budget]
};

__device__ __forceinline__ int length_of(const EvictParams& p, int r) {
  return min(max(p.lens[r], 0), p.table_width * p.block_size);
}

__device__ __forceinline__ int page_at(const EvictParams& p, int r, int token, int& off) {
  const int page = token / p.block_size;
  off = token - page * p.block_size;
  const int b = p.tables[(int64_t)r * p.table_stride + page];
  return b >= 0 && b < p.num_blocks ? b : -1;
}

// An unsigned key that orders like the weight: NaN, and tokens in no page,
// below every number; -0 equal to 0.
__device__ __forceinline__ uint32_t order_key(float w) {
  const uint32_t u = __float_as_uint(w + 0.0f);
  return w != w ? 0u : u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ uint32_t key_at(const EvictParams& p, const float* scores, int r, int head, int token) {
  int off;
  const int b = page_at(p, r, token, off);
  return b < 0 ? 0u : order_key(scores[((int64_t)b * p.hkv + head) * p.block_size + off]);
}

// Exclusive sum over the workgroup's threads; `total` receives the whole.
__device__ __forceinline__ int block_scan(int x, int* sums, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  int s = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(s, d, 64);
    if (lane >= d) s += y;
  }
  __syncthreads();
  if (lane == 63) sums[wave] = s;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < waves; ++w) {
    before += w < wave ? sums[w] : 0;
    all += sums[w];
  }
  total = all;
  return before + s - x;
}

// The choice.  The budget - recent heaviest of the first n - recent tokens are
// those above the key T of that rank and the first few equal to it; T is found
// by its bytes, most significant first, from a histogram of the keys that
// share the bytes found so far.  Then one pass in position order writes the
// kept positions.
__global__ void __launch_bounds__(SELECT_NT)
evict_select_kernel(EvictParams p) {
  __shared__ int hist[256], sums[SELECT_NT / 64], found[2];
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
  int need = p.budget - p.recent;  // still to choose among the keys that match `prefix`
  uint32_t prefix = 0;
  for (int shift = 24; shift >= 0 && need > 0; shift -= 8) {
    for (int i = tid; i < 256; i += SELECT_NT) hist[i] = 0;
    __syncthreads();
    for (int t = tid; t < old; t += SELECT_NT) {
      const uint32_t k = key_at(p, scores, r, head, t);
      if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    // Thread b holds bin 255 - b: the keys above a bin are those before it.
    int total;
    const int mine = tid < 256 ? hist[255 - tid] : 0;
    const int above = block_scan(mine, sums, total);
    if (tid < 256 && above < need && above + mine >= need) {
      found[0] = 255 - tid;
      found[1] = above;
    }
    __syncthreads();
    prefix |= (uint32_t)found[0] << shift;
    need -= found[1];
    __syncthreads();
  }
  // need: how many of the keys equal to prefix are kept (none where no old token is).
  const bool any = p.budget > p.recent;
  int equal_before = 0, kept_before = 0;
  for (int t0 = 0; t0 < n; t0 += SELECT_NT) {
    const int t = t0 + tid;
    bool above = false, equal = false;
    if (t < n) {
      if (t >= old) {
        above = true;
      } else if (any) {
        const uint32_t k = key_at(p, scores, r, head, t);
        above = k > prefix;
        equal = k == prefix;
      }
    }
    int equals, keeps;
    const int e = equal_before + block_scan(equal, sums, equals);
    const bool keep = above || (equal && e < need);
    const int at = kept_before + block_scan(keep, sums, keeps);
    if (keep) kept[at] = t;
    equal_before += equals;
    kept_before += keeps;
  }
}

// One array of the pool that moves with the tokens: `unit` bytes of a token's
// `row` bytes per lane.
struct Stream {
  uint8_t* base;
  int64_t layer_bytes, page_bytes;
  int head_bytes, token_bytes, row;
};

struct MoveParams {
  EvictParams e;
  Stream s[5];
  int streams;
};

// The move, in place: a workgroup takes one array of one (layer, row, kv head)
// and fills its places in ascending order.  The token that comes to place i
// lies at i or later, so once the tiles up to some place have been read, what
// is stored there is not read again: each tile is loaded whole, and stored
// after a barrier.
template <typename U, int DEPTH>
__device__ void move_stream(const EvictParams& p, const Stream& s, int r, int head, int layer, int n) {
  const int per = s.row / (int)sizeof(U);  // units of a token
  const int32_t* kept = p.kept + (((int64_t)layer * p.rows + r) * p.hkv + head) * p.budget;
  uint8_t* base = s.base + layer * s.layer_bytes + (int64_t)head * s.head_bytes;
  const int units = p.budget * per;
  for (int u0 = 0; u0 < units; u0 += 256 * DEPTH) {
    U x[DEPTH];
    uint8_t* to[DEPTH];
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const int u = u0 + 256 * d + (int)threadIdx.x;
      to[d] = nullptr;
      if (u >= units) continue;
      const int i = u / per, part = (u - i * per) * (int)sizeof(U);
      const int src = kept[i];
      if (src == i || src < 0) continue;
      int soff, doff;
      const int sb = page_at(p, r, src, soff), db = page_at(p, r, i, doff);
      if (sb < 0 || db < 0) continue;
      x[d] = *reinterpret_cast<const U*>(base + sb * s.page_bytes + (int64_t)soff * s.token_bytes + part);
      to[d] = base + db * s.page_bytes + (int64_t)doff * s.token_bytes + part;
    }
    // The barrier alone orders LDS accesses; the loads have to have come back.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
      if (to[d]) *reinterpret_cast<U*>(to[d]) = x[d];
  }
}

__global__ void __launch_bounds__(256)
evict_move_kernel(MoveParams m) {
  const EvictParams& p = m.e;
  const int head = blockIdx.x % p.hkv, which = blockIdx.x / p.hkv, r = blockIdx.y, layer = blockIdx.z;
  const int n = length_of(p, r);
  if (n <= p.budget) return;
  const Stream& s = m.s[which];
  if (s.row % 16 == 0) {
    move_stream<u32x4, 4>(p, s, r, head, layer, n);
  } else if (s.row % 4 == 0) {
    move_stream<uint32_t, 4>(p, s, r, head, layer, n);
  } else {
    move_stream<uint16_t, 4>(p, s, r, head, layer, n);
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
      (reinterpret_cast<uintptr_t>(a->scores) % 4))
    return fail(SLO_ERR_INVALID, "evict_kv: pools must be 16-byte aligned");
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
  // Head by head pages (4-bit pools and the scores) or token by token.
  auto stream_of = [&](void* base, int row, bool by_head) {
    const int64_t page = (int64_t)a->block_size * a->num_kv_heads * row;
    return Stream{static_cast<uint8_t*>(base), page * a->num_blocks, page, by_head ? a->block_size * row : row,
                  by_head ? row : a->num_kv_heads * row, row};
  };
  const int row = a->kv_dtype == KV_BF16 ? 2 * a->head_dim : fp4 ? a->head_dim / 2 : a->head_dim;
  m.s[0] = stream_of(a->scores, 4, true);
  m.s[1] = stream_of(a->k_cache, row, fp4);
  m.s[2] = stream_of(a->v_cache, row, fp4);
  m.streams = 3;
  if (a->kv_dtype != KV_BF16) {
    const int scale = fp4 ? a->head_dim / kFp4Group : 4;
    m.s[3] = stream_of(a->k_scale, scale, fp4);
    m.s[4] = stream_of(a->v_scale, scale, fp4);
    m.streams = 5;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(evict_select_kernel, dim3(p.hkv, p.rows, a->num_layers), dim3(SELECT_NT), 0, s, p);
  hipLaunchKernelGGL(evict_move_kernel, dim3(p.hkv * m.streams, p.rows, a->num_layers), dim3(256), 0, s, m);
  return check_launch("evict_kv");
}
