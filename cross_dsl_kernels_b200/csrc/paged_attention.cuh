// What the attention reads of the paged caches share: the arguments, the even split of a batch's tiles over the CTAs, the
// matrix instructions.
#pragma once

#include <math.h>

#include "common.cuh"

namespace xdk {
namespace {

constexpr int kAttnWarps = 4;
constexpr int kAttnThreads = kAttnWarps * 32;
constexpr int kMaxSplits = 8;  // portable cluster size
__device__ __forceinline__ int warp_of(unsigned tid) { return static_cast<int>(tid >> 5); }

struct AttnArgs {
  const int64_t* positions;
  const int64_t* page_table;
  const int64_t* sequence_ids;
  int64_t max_pages, page_size;
  int q_heads, kv_heads;
  int hnd;
  int narrow;      // every position a page table row can hold fits 31 bits: 32-bit divisions
  float scale;
  int tokens;
  float* scratch;  // even split of the batch's tiles over the grid, partial results here; nullptr: grid = (splits, heads, tokens)
};

// Merges partial (m, l, acc) `b` into `a` (online softmax): both cover disjoint position sets.
__device__ __forceinline__ void merge_stats(float& m_a, float& l_a, float& scale_a, float& scale_b, float m_b, float l_b) {
  const float m = fmaxf(m_a, m_b);
  scale_a = m_a == -INFINITY ? 0.0f : __expf(m_a - m);
  scale_b = m_b == -INFINITY ? 0.0f : __expf(m_b - m);
  l_a = l_a * scale_a + l_b * scale_b;
  m_a = m;
}

// ---- even split of a batch ---------------------------------------------------------------------------------------
// Contexts differ from token to token, and only the device knows them.  The tiles of all (token, KV head) items stand
// one behind the other, token-major, and CTA b of B takes tiles [b W / B, (b + 1) W / B) of the W there are (B: the CTAs of the
// grid, or W, if there are fewer tiles than CTAs: the CTAs past W have no part in it).  An item
// that lies inside one CTA is finished there; the others leave one partial result (max, sum, accumulator per head) per
// CTA in scratch -- slot 2 b + 1 for the item that CTA b begins and does not end, slot 2 b for one begun before it --
// and a merge kernel adds them in CTA order.
constexpr int kMergeThreads = 256;
constexpr int kMaxTokensSplit = 16384;  // every CTA adds up the tiles of all tokens: longer batches have items enough
// Shorter contexts stay on the grid of splits: finding the share and the second launch cost 1 .. 4 us, which the even split
// only earns back on uneven or long ones.  (A caller that names no bound gets that of the page table's rows: one token, 2 heads x 64,
// 8.6 us on the grid of splits and 9.6 on the even one for a table of 1024; 16 tokens x 8 heads x 128, 9.8 / 11.2 for one of 256.)
// Short contexts under a long bound cost no more: one token, 8 heads x 128, 512 positions, bound 8192 8.8 / 10.9, 16 tokens 11.9 / 12.5 (one
// token of 2 heads x 64, 1024 positions 20.3 while CTAs without a share left zeros for the merge, which then had them all to add).
// us, contexts of every length up to the bound / all at the bound, even against
// splits: 16 tokens x 8 heads x 128, bound 512 13.8 / 13.3 against 12.3 / 14.9, 1024 15.9 / 19.4 against 15.9 / 18.1, 2048
// 20.0 / 33.2 against 24.1 / 32.9; one token, 8192 13.9 / 16.8 against 14.9 / 24.8; FP32, 64 tokens x 4 heads, 2048 63 / 102 against 123 / 131.
// Against the kernel before the even split, whose dead positions were read: 16 tokens, 8192 56 / 95 from 82 / 98; 64 tokens,
// 2048 58 / 96 from 103 / 122.
constexpr int kMinEvenContext = 1536;
// A larger bound on the contexts says no more than this one: it is far beyond any cache, and keeps tokens * heads * tiles, and the
// roundings up, inside 64 bits.
constexpr int64_t kMaxContextHint = 1LL << 38;

// 32-bit words of scratch per CTA: two accumulators, twice two statistics, a header
constexpr size_t partial_words(size_t g, size_t d) { return 2 * g * d + 2 * (2 * g) + 4; }

// Context length and sequence of the batch's first tokens, in shared memory: a step to the next item would otherwise cost two
// dependent trips to memory.
constexpr int kCachedTokens = 128;
struct TokenCache {
  int64_t ctx[kCachedTokens], seq[kCachedTokens];
};

struct ItemCursor {  // a tile of an item
  int token, kvh, tile, tiles;
  int64_t ctx;
  const int64_t* table;
  template <int U>  // positions per tile
  __device__ __forceinline__ void load(const AttnArgs& a, const TokenCache* cache) {
    const bool hit = cache != nullptr && token < kCachedTokens;
    ctx = hit ? cache->ctx[token] : a.positions[token] + 1;
    tiles = ctx > U ? static_cast<int>((ctx + U - 1) / U) : 1;  // an empty context is one dead tile
    table = a.page_table + (hit ? cache->seq[token] : a.sequence_ids[token]) * a.max_pages;
  }
  template <int U>
  __device__ __forceinline__ void advance(const AttnArgs& a, const TokenCache* cache) {  // not past the batch's last tile
    if (++tile < tiles) return;
    tile = 0;
    if (++kvh < a.kv_heads) return;
    kvh = 0, ++token;
    load<U>(a, cache);
  }
};

// CTAs that have a share of `total` tiles; each of them has at least one.
__device__ __forceinline__ int64_t share_ctas(int64_t total) { return total < gridDim.x ? total : gridDim.x; }

// Sets `at` to this CTA's first tile and returns how many tiles it has, 0 for a CTA without a share; `batch_tiles` (in shared memory): tiles of the batch.
// All threads call it.
template <int U>
__device__ __forceinline__ int64_t seek_share(const AttnArgs& a, ItemCursor& at, int64_t& batch_tiles, TokenCache& cache) {
  __shared__ int64_t warp_sums[kAttnWarps];
  __shared__ int64_t found[2];
  const int lane = threadIdx.x & 31, warp = warp_of(threadIdx.x);
  auto tiles_of = [&](int t) -> int64_t {
    if (t >= a.tokens) return 0;
    const int64_t ctx = a.positions[t] + 1;
    return (ctx > U ? (ctx + U - 1) / U : 1) * a.kv_heads;
  };
  static_assert(kCachedTokens == kAttnThreads, "one token per thread");
  if (static_cast<int>(threadIdx.x) < a.tokens) {
    cache.ctx[threadIdx.x] = a.positions[threadIdx.x] + 1;
    cache.seq[threadIdx.x] = a.sequence_ids[threadIdx.x];
  }
  const int64_t first = tiles_of(threadIdx.x);
  int64_t sum = first;
  for (int t = threadIdx.x + kAttnThreads; t < a.tokens; t += kAttnThreads) sum += tiles_of(t);
#pragma unroll
  for (int sh = 16; sh > 0; sh >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, sh);
  if (lane == 0) warp_sums[warp] = sum;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < kAttnWarps; ++w) total += warp_sums[w];
  if (threadIdx.x == 0) batch_tiles = total;
  const int64_t ctas = share_ctas(total);
  if (blockIdx.x >= ctas) return 0;
  const int64_t w0 = total * blockIdx.x / ctas, w1 = total * (blockIdx.x + 1) / ctas;
  int64_t before = 0;  // tiles of the tokens in front of the chunk
  for (int t0 = 0;; t0 += kAttnThreads) {
    const int64_t mine = t0 == 0 ? first : tiles_of(t0 + threadIdx.x);
    int64_t upto = mine;
#pragma unroll
    for (int sh = 1; sh < 32; sh <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, upto, sh);
      if (lane >= sh) upto += v;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = upto;
    __syncthreads();
    int64_t chunk = 0;
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) {
      if (w < warp) upto += warp_sums[w];
      chunk += warp_sums[w];
    }
    if (before + upto - mine <= w0 && w0 < before + upto) found[0] = t0 + threadIdx.x, found[1] = w0 - (before + upto - mine);
    before += chunk;
    if (w0 < before) break;  // same for all threads
  }
  __syncthreads();
  at.token = static_cast<int>(found[0]);
  at.load<U>(a, &cache);
  at.kvh = static_cast<int>(found[1] / at.tiles);
  at.tile = static_cast<int>(found[1] - static_cast<int64_t>(at.kvh) * at.tiles);
  return w1 - w0;
}

// ---- matrix instructions --------------------------------------------------------------------------------------------
template <typename T> struct Mma16816;
template <> struct Mma16816<__half> {
  __device__ static __forceinline__ void run(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  __device__ static __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <> struct Mma16816<__nv_bfloat16> {
  __device__ static __forceinline__ void run(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  __device__ static __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
// An 8 x 8 matrix of 16-bit elements spread over the warp as a fragment, transposed.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], const void* smem_row) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_u32(smem_row)));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], const void* smem_row) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_u32(smem_row)));
}

}  // namespace
}  // namespace xdk
