// Which pages of an 8-bit paged cache (kv8.cuh) a query reads: the ones whose mean key scores best.
//
//   codes of q, per head: qc = rint(q / unit), unit = max |q| * (1 / 127)         (q = qc * unit to half a unit)
//   score of a page in front of the token's last one: max over the heads of a group of (unit * (qc . mean)) * scale of the block
//   chosen: the top_pages - 1 best of them (the lowest page first among equals), and the last page always
// The dot products are sums of whole numbers below 2^24 and every other step is one correctly rounded FP32 operation, so the choice is
// the same whatever computes it.  One choice per token and KV head: the query heads that share it read its pages together.
//
// One CTA per (token, KV head).  Scores: mma.m16n8k32 on bytes, 16 pages as rows, the heads of the group as columns; a thread
// loads a quarter of two pages' means with 16-byte loads, four threads 64 bytes in a row (14.0 us for 16 tokens, 8 KV heads and 2048
// pages that L2 holds in part; a quarter of the dims in a row to each thread: 14.5), those of four blocks of 16 pages at a time (the next four
// loaded during these ones' products: 14.7), and the codes of q stand in registers in the same order of dims.  The scores stay in shared
// memory as sortable integers; up to three passes over 11, 11 and 10 bits of them find the value of the last one chosen (two, mostly:
// no other has its first 22 bits), one more writes the pages in order.
// Bound: 512 pages (7.0 us for one token) by the chain of loads and barriers; 2048 pages, whose means are 35 MB, from HBM (14.8 us) by
// the latency of their reads: 2.3 us in front of the scores, 10 for them, 3.3 for the choice.
#include <math.h>

#include "kv8.cuh"

namespace xdk {
namespace {

constexpr int kSelThreads = 512, kSelWarps = kSelThreads / 32;
constexpr int kBins = 2048, kBinsEach = kBins / kSelThreads;
constexpr int64_t kMaxCandidates = 51200;  // keys in shared memory

struct SelectArgs {
  const void* q;
  const int8_t* k_mean;
  const float* k_scale;
  const int64_t *positions, *page_table, *sequence_ids;
  int32_t* pages;
  int64_t max_pages;
  int q_heads, kv_heads, page_size, top_pages;
};

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Larger key: larger score; one that is not a number (a block with such a value) before all others.
__device__ __forceinline__ uint32_t key_of(float score) {
  if (score != score) return 0xffffffffu;
  const uint32_t b = __float_as_uint(score + 0.0f);  // -0 and 0 are equals
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <typename T, int D>
__global__ void __launch_bounds__(kSelThreads)
kv8_select_kernel(const __grid_constant__ SelectArgs a) {
  constexpr int kWords = D / 16;  // of four dims, per thread and page
  extern __shared__ uint32_t keys[];
  __shared__ __align__(16) uint32_t codes[8][D / 4];
  __shared__ float unit[8];
  __shared__ unsigned bins[kBins];
  __shared__ unsigned warp_sum[kSelWarps], chosen[3];
  __shared__ int warp_above[kSelWarps], warp_equal[kSelWarps];

  pdl_launch_dependents();
  pdl_wait();
  const int token = blockIdx.y, kvh = blockIdx.x;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int group = a.q_heads / a.kv_heads;
  int32_t* out = a.pages + (static_cast<int64_t>(token) * a.kv_heads + kvh) * a.top_pages;
  const int64_t pos = a.positions[token];
  if (pos < 0) {
    for (unsigned i = tid; i < static_cast<unsigned>(a.top_pages); i += kSelThreads) out[i] = -1;  // unsigned: the last step may pass 2^31
    return;
  }
  const int64_t at_page = pos / a.page_size;
  const int last = static_cast<int>(at_page < a.max_pages ? at_page : a.max_pages - 1);
  const int want = a.top_pages - 1;  // of the pages in front of the last one
  if (last <= want) {
    for (unsigned i = tid; i < static_cast<unsigned>(a.top_pages); i += kSelThreads) out[i] = i <= static_cast<unsigned>(last) ? static_cast<int>(i) : -1;
    return;
  }
  if (want == 0) {
    if (tid == 0) out[0] = last;
    return;
  }
  const int64_t* table = a.page_table + a.sequence_ids[token] * a.max_pages;

  if (warp < 8) {  // codes of head `warp` of the group, zeros for a head that is none
    constexpr int N = D / 32;
    float x[N], top = 0.0f;
    const T* q = static_cast<const T*>(a.q) + (static_cast<int64_t>(token) * a.q_heads + kvh * group + warp) * D + lane * N;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      x[e] = warp < group ? Elem<T>::to_f32(q[e]) : 0.0f;
      top = fmaxf(top, fabsf(x[e]));
    }
#pragma unroll
    for (int sh = 16; sh > 0; sh >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, sh));
    const float u = __fmul_rn(top, 1.0f / 127.0f);
    if (lane == 0) unit[warp] = u;
    int8_t* to = reinterpret_cast<int8_t*>(codes[warp]) + lane * N;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float c = u > 0.0f ? fminf(fmaxf(rintf(__fdiv_rn(x[e], u)), -127.0f), 127.0f) : 0.0f;
      to[e] = static_cast<int8_t>(static_cast<int>(c));
    }
  }
  __syncthreads();

  // ---- scores
  const int row = lane >> 2, quad = lane & 3;
  uint32_t b[kWords];  // head `row`, dims 64 i + 16 quad .. + 15
#pragma unroll
  for (int w = 0; w < kWords; ++w) b[w] = codes[row][w / 4 * 16 + quad * 4 + w % 4];
  const float unit0 = unit[2 * quad], unit1 = unit[2 * quad + 1];
  const bool live0 = 2 * quad < group, live1 = 2 * quad + 1 < group;
  constexpr int kAtOnce = D <= 128 ? 4 : 2;  // blocks of 16 pages whose loads are on their way together
  for (int base0 = warp * 16; base0 < last; base0 += kSelWarps * 16 * kAtOnce) {
    int64_t block[kAtOnce][2];
    uint32_t m[kAtOnce][2][kWords];
    float scale[kAtOnce][2];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int p = base0 + u * kSelWarps * 16 + row + r * 8;
        block[u][r] = table[p < last ? p : last - 1] * a.kv_heads + kvh;  // dead rows: one that is read anyway
      }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        if (base0 + u * kSelWarps * 16 >= last) continue;
#pragma unroll
        for (int w = 0; w < kWords; w += 4) {
          const U4 v = ld_ordered_stream16(a.k_mean + block[u][r] * D + w * 16 + quad * 16);
          m[u][r][w] = v.x, m[u][r][w + 1] = v.y, m[u][r][w + 2] = v.z, m[u][r][w + 3] = v.w;
        }
        scale[u][r] = a.k_scale[block[u][r]];
      }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int p0 = base0 + u * kSelWarps * 16 + row, p1 = p0 + 8;
      if (p0 - row >= last) break;  // the same for the warp
      int dot[4] = {};
#pragma unroll
      for (int w = 0; w < kWords; w += 2) mma_s8(dot, m[u][0][w], m[u][1][w], m[u][0][w + 1], m[u][1][w + 1], b[w], b[w + 1]);
      float s[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float x = live0 ? __fmul_rn(static_cast<float>(dot[2 * e]), unit0) : -INFINITY;
        const float y = live1 ? __fmul_rn(static_cast<float>(dot[2 * e + 1]), unit1) : -INFINITY;
        s[e] = fmaxf(x, y);
#pragma unroll
        for (int sh = 1; sh < 4; sh <<= 1) s[e] = fmaxf(s[e], __shfl_xor_sync(0xffffffffu, s[e], sh));
      }
      if (quad == 0 && p0 < last) keys[p0] = key_of(__fmul_rn(s[0], scale[u][0]));
      if (quad == 1 && p1 < last) keys[p1] = key_of(__fmul_rn(s[1], scale[u][1]));
    }
  }

  // ---- the key of the last one chosen, from its high bits down; `left`: how many of the keys that agree so far are wanted
  uint32_t prefix = 0;
  unsigned left = static_cast<unsigned>(want);
  bool exact = false;  // all bits of prefix are known; else all keys that agree with the known ones are wanted
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bits = pass == 2 ? 10 : 11;
#pragma unroll
    for (int i = 0; i < kBinsEach; ++i) bins[i * kSelThreads + tid] = 0;
    __syncthreads();
    const uint32_t mask = pass == 0 ? 0u : 0xffffffffu << (shift + bits);
    for (int i = tid; i < last; i += kSelThreads)
      if ((keys[i] & mask) == prefix) atomicAdd(&bins[keys[i] >> shift & ((1u << bits) - 1u)], 1u);
    __syncthreads();
    // thread t: kBinsEach bins from the top down; keys in them and in those above
    unsigned mine[kBinsEach], upto = 0;
#pragma unroll
    for (int i = 0; i < kBinsEach; ++i) upto += mine[i] = bins[kBins - 1 - (tid * kBinsEach + i)];
    const unsigned own = upto;
#pragma unroll
    for (int sh = 1; sh < 32; sh <<= 1) {
      const unsigned v = __shfl_up_sync(0xffffffffu, upto, sh);
      if (lane >= sh) upto += v;
    }
    if (lane == 31) warp_sum[warp] = upto;
    __syncthreads();
    for (int w = 0; w < warp; ++w) upto += warp_sum[w];
    unsigned above = upto - own;
    if (above < left && left <= upto) {
#pragma unroll
      for (int i = 0; i < kBinsEach; ++i) {
        if (above < left && left <= above + mine[i]) chosen[0] = kBins - 1 - (tid * kBinsEach + i), chosen[1] = left - above, chosen[2] = mine[i];
        above += mine[i];
      }
    }
    __syncthreads();
    prefix |= chosen[0] << shift, left = chosen[1];
    exact = pass == 2;
    if (chosen[2] == left) break;  // the same for all threads
  }

  // ---- pages whose key is above, and the first `left` of the equals, in order: a thread has some consecutive ones
  const int each = (last + kSelThreads - 1) / kSelThreads, begin = tid * each < last ? tid * each : last;
  const int end = begin + each < last ? begin + each : last, limit = static_cast<int>(left);
  auto is_above = [&](uint32_t key) { return exact ? key > prefix : key >= prefix; };
  auto is_equal = [&](uint32_t key) { return exact && key == prefix; };
  int above = 0, equal = 0;
  for (int p = begin; p < end; ++p) above += is_above(keys[p]), equal += is_equal(keys[p]);
  int above_upto = above, equal_upto = equal;
#pragma unroll
  for (int sh = 1; sh < 32; sh <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, above_upto, sh), w = __shfl_up_sync(0xffffffffu, equal_upto, sh);
    if (lane >= sh) above_upto += v, equal_upto += w;
  }
  if (lane == 31) warp_above[warp] = above_upto, warp_equal[warp] = equal_upto;
  __syncthreads();
  above = above_upto - above, equal = equal_upto - equal;  // in front of this thread's pages
  for (int w = 0; w < warp; ++w) above += warp_above[w], equal += warp_equal[w];
  for (int p = begin; p < end; ++p) {
    const uint32_t key = keys[p];
    if (is_above(key) || (is_equal(key) && equal < limit)) out[above + (equal < limit ? equal : limit)] = p;
    above += is_above(key), equal += is_equal(key);
  }
  if (tid == 0) out[want] = last;
}

template <typename T>
int dispatch_select(int64_t d, const SelectArgs& a, dim3 grid, size_t smem, cudaStream_t s) {
  auto run = [&](auto kernel) {
    if (smem > 32 * 1024) {  // with the 9 KB that it has statically, beyond what a launch gets unasked
      if (int st = allow_smem(reinterpret_cast<const void*>(kernel), smem)) return st;
    }
    return launch_dependent(kernel, grid, dim3(kSelThreads), smem, s, a);
  };
  switch (d) {
    case 64: return run(kv8_select_kernel<T, 64>);
    case 128: return run(kv8_select_kernel<T, 128>);
    case 256: return run(kv8_select_kernel<T, 256>);
    default: return XDK_ERR_LIMIT;
  }
}

}  // namespace
}  // namespace xdk

extern "C" int xdk_kv8_select_pages(const void* q, const int8_t* k_mean, const float* k_scale, const int64_t* positions,
                                    const int64_t* page_table, const int64_t* sequence_ids, int32_t* pages, int64_t tokens, int64_t q_heads,
                                    int64_t kv_heads, int64_t head_dim, int64_t max_pages_per_seq, int64_t page_size, int64_t top_pages,
                                    int dtype, unsigned flags, void* stream) {
  using namespace xdk;
  if (flags & ~XDK_DEPENDENT_LAUNCH) return XDK_ERR_ARG;
  CallFlagsScope scope(flags);
  if (!q || !k_mean || !k_scale || !positions || !page_table || !sequence_ids || !pages) return XDK_ERR_ARG;
  if (tokens < 1 || q_heads < 1 || kv_heads < 1 || head_dim < 1 || page_size < 1 || max_pages_per_seq < 1 || top_pages < 1) return XDK_ERR_ARG;
  if (q_heads % kv_heads != 0 || !aligned16(k_mean)) return XDK_ERR_ARG;
  if (dtype != XDK_F32 && dtype != XDK_BF16 && dtype != XDK_F16) return XDK_ERR_ARG;
  if (!kv8_head_dim(head_dim) || q_heads / kv_heads > 8 || tokens > 65535 || top_pages > 2147483647LL || max_pages_per_seq > kMaxCandidates)
    return XDK_ERR_LIMIT;
  if (int st = kv8_limits(tokens, kv_heads, max_pages_per_seq, page_size)) return st;
  if (int st = require_sm100()) return st;
  SelectArgs a;
  a.q = q, a.k_mean = k_mean, a.k_scale = k_scale, a.positions = positions, a.page_table = page_table, a.sequence_ids = sequence_ids;
  a.pages = pages, a.max_pages = max_pages_per_seq;
  a.q_heads = static_cast<int>(q_heads), a.kv_heads = static_cast<int>(kv_heads), a.page_size = static_cast<int>(page_size);
  a.top_pages = static_cast<int>(top_pages);
  const dim3 grid(static_cast<unsigned>(kv_heads), static_cast<unsigned>(tokens));
  const size_t smem = static_cast<size_t>(max_pages_per_seq) * 4;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case XDK_F32: return dispatch_select<float>(head_dim, a, grid, smem, s);
    case XDK_BF16: return dispatch_select<__nv_bfloat16>(head_dim, a, grid, smem, s);
    case XDK_F16: return dispatch_select<__half>(head_dim, a, grid, smem, s);
    default: return XDK_ERR_ARG;
  }
}
