// Rotation and append into the 8-bit paged K/V cache (kv8.cuh).
//
//   Q and K are rotated in FP32 as by the 16-bit append (separately rounded products and sums); rotated Q is rounded to its type, K
//   and V go to their slots as codes.  A block is a page of one KV head, W its rows that the call writes (of several tokens for one
//   slot the last), A the largest |x| in them:
//     before = 0 if row 0 is in W, else the block's scale       (a page that is used again begins anew)
//     scale  = max(before, A * (1 / top))                       (NaN once a value that is not finite was written)
//     rows in W:  code = round(x / scale);   the others, where the scale grew:  code = round(code * (before / scale))
//     mean of the keys, once the last row is in W:  rint(sum of the codes * c) as int8, in units of scale (int8 codes) or of
//     scale * 448 / 127 (e4m3)
//   Every step is a correctly rounded FP32 operation or a sum of whole numbers: the bytes are defined, whatever the order.
//
// One CTA owns a block of K and V: it finds the rows from the batch's index vectors, so tokens may come in any order, several for
// a page or for a slot.  Up to kSmallBatch tokens every CTA looks all of them up (one launch; the first token of a page does its
// work); longer batches are grouped by page in a table in scratch while Q is rotated, and a second launch walks the groups.
//
// Bound: a decode batch by its chain of dependent loads (position, sequence, page, then the block's scale), a prefill chunk by
// HBM (values read once, codes written once).
#include <math.h>

#include "kv8.cuh"

namespace xdk {
namespace {

constexpr int kThreads = 128;
constexpr int kSmallBatch = 128;

struct AppendArgs {
  const void *q, *k, *v;
  const float *cos, *sin;
  const int64_t *positions, *page_table, *sequence_ids;
  void* q_out;
  uint8_t *k_cache, *v_cache;
  float *k_scale, *v_scale;
  int8_t* k_mean;
  int64_t max_pages, q_stride, k_stride, v_stride;
  int tokens, q_heads, kv_heads, page_size, rope_dim, cos_width;
  int interleaved, hnd;
  float mean_unit;
};

// Where the tokens of a long batch go, by physical page: an open hash table of `slots` entries, all bytes 0xff before the call.
struct Groups {
  unsigned long long* page;  // [slots], ~0: free
  unsigned* first;           // [slots] first and last token of the page
  int* last;
  int* list;                 // [slots] the entries in use, in any order
  int* slot_of;              // [tokens] entry of a token's page, -1: no page
  int* count;                // entries in use - 1
  unsigned mask;             // slots - 1
};
inline int64_t group_slots(int64_t tokens) {
  int64_t s = 1;
  while (s < 2 * tokens) s <<= 1;
  return s;
}
inline size_t group_bytes(int64_t tokens) { return static_cast<size_t>(group_slots(tokens)) * 20 + static_cast<size_t>(tokens + 1) * 4; }
inline Groups groups_at(void* scratch, int64_t tokens) {
  const int64_t s = group_slots(tokens);
  Groups g;
  g.page = static_cast<unsigned long long*>(scratch);
  g.first = reinterpret_cast<unsigned*>(g.page + s);
  g.last = reinterpret_cast<int*>(g.first + s);
  g.list = g.last + s;
  g.slot_of = g.list + s;
  g.count = g.slot_of + tokens;
  g.mask = static_cast<unsigned>(s - 1);
  return g;
}

template <typename T, bool VEC> __device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  if constexpr (VEC) {
    constexpr int E = Elem<T>::kPerVec;
#pragma unroll
    for (int i = 0; i < 8 / E; ++i) {
      float f[E];
      unpack16<T>(ld_ordered16(p + i * E), f);
#pragma unroll
      for (int e = 0; e < E; ++e) x[i * E + e] = f[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = Elem<T>::to_f32(p[e]);
  }
}
template <bool VEC> __device__ __forceinline__ void load_angles(const float* p, float* x, int n) {  // n: 4 or 8, 16-byte aligned if VEC
#pragma unroll
  for (int i = 0; i < 8; i += 4) {
    if (i >= n) break;
    if constexpr (VEC) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(p + i));
      x[i] = f.x, x[i + 1] = f.y, x[i + 2] = f.z, x[i + 3] = f.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[i + e] = __ldg(p + i + e);
    }
  }
}

// Dims d0 .. d0 + 7 of a head, rotated.  VEC: whole vectors are rotated or not, and partners and angles are 16-byte vectors too.
template <typename T, bool VEC>
__device__ __forceinline__ void rotated8(const AppendArgs& a, const T* head, int d0, int64_t pos, float (&x)[8]) {
  load8<T, VEC>(head + d0, x);
  const float *crow = a.cos + pos * a.cos_width, *srow = a.sin + pos * a.cos_width;
  const int half = a.rope_dim / 2;
  if constexpr (VEC) {
    if (d0 >= a.rope_dim) return;
    float c[8], s[8];
    if (a.interleaved) {
      load_angles<true>(crow + d0 / 2, c, 4), load_angles<true>(srow + d0 / 2, s, 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float lo = x[2 * e], hi = x[2 * e + 1];
        x[2 * e] = __fsub_rn(__fmul_rn(lo, c[e]), __fmul_rn(hi, s[e]));
        x[2 * e + 1] = __fadd_rn(__fmul_rn(lo, s[e]), __fmul_rn(hi, c[e]));
      }
      return;
    }
    const bool upper = d0 >= half;
    const int at = upper ? d0 - half : d0;
    float p[8];
    load8<T, true>(head + (upper ? at : d0 + half), p);
    load_angles<true>(crow + at, c, 8), load_angles<true>(srow + at, s, 8);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      x[e] = upper ? __fadd_rn(__fmul_rn(p[e], s[e]), __fmul_rn(x[e], c[e])) : __fsub_rn(__fmul_rn(x[e], c[e]), __fmul_rn(p[e], s[e]));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = d0 + e;
      if (d >= a.rope_dim) break;
      const bool upper = a.interleaved ? (d & 1) != 0 : d >= half;
      const int at = a.interleaved ? d >> 1 : (upper ? d - half : d);
      const float p = Elem<T>::to_f32(head[a.interleaved ? d ^ 1 : (upper ? at : d + half)]);
      const float c = __ldg(crow + at), s = __ldg(srow + at);
      x[e] = upper ? __fadd_rn(__fmul_rn(p, s), __fmul_rn(x[e], c)) : __fsub_rn(__fmul_rn(x[e], c), __fmul_rn(p, s));
    }
  }
}

// Eight dims of one Q head per thread; unit: of the token's q_heads * D / 8.  A token without a position gets zeros.
template <typename T, int D, bool VEC>
__device__ __forceinline__ void rotate_q(const AppendArgs& a, int token, int unit) {
  if (unit >= a.q_heads * (D / 8)) return;
  const int head = unit / (D / 8), d0 = (unit - head * (D / 8)) * 8;
  const int64_t pos = a.positions[token];
  float x[8] = {};
  if (pos >= 0) rotated8<T, VEC>(a, static_cast<const T*>(a.q) + token * a.q_stride + head * D, d0, pos, x);
  T* dst = static_cast<T*>(a.q_out) + (static_cast<int64_t>(token) * a.q_heads + head) * D + d0;  // torch's own, or 16-byte aligned
  constexpr int E = Elem<T>::kPerVec;
#pragma unroll
  for (int i = 0; i < 8 / E; ++i) {
    float f[E];
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = x[i * E + e];
    *reinterpret_cast<U4*>(dst + i * E) = pack16<T>(f);
  }
}

struct BlockShared {
  int token_of[kKV8MaxPage];  // row -> token, -1: not written by this call
  unsigned top_k[kThreads / 32], top_v[kThreads / 32];
  int sums[256];
};

__device__ __forceinline__ unsigned largest8(unsigned top, const float (&x)[8]) {  // of the bits of |x|: NaN over infinity over numbers
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
  return top;
}
// The scale behind the call from the one before and the largest value: NaN for anything that is not a finite number.
__device__ __forceinline__ float grown(float before, unsigned top_bits, float per_top) {
  if (!isfinite(before) || top_bits >= 0x7f800000u) return __uint_as_float(0x7fffffffu);
  return fmaxf(before, __fmul_rn(__uint_as_float(top_bits), per_top));
}
template <typename C> __device__ __forceinline__ uint2 encode8(const float (&x)[8], float scale) {
  float y[8];
  const bool some = scale > 0.0f;  // not of a block of zeros, nor of one with a NaN
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = some ? __fdiv_rn(x[e], scale) : 0.0f;
  return make_uint2(Codec<C>::pack4(y), Codec<C>::pack4(y + 4));
}

// Block (page, kvh) of K and V; s.token_of is filled and visible.  All threads call it.
template <typename T, typename C, int D, bool VEC>
__device__ __forceinline__ void write_block(const AppendArgs& a, BlockShared& s, int64_t page, int kvh) {
  constexpr int kPerRow = D / 8, kRows = kThreads / kPerRow;  // threads of a row, rows at a time
  constexpr int kKept = 2;                                    // passes whose values stay in registers
  const int group = threadIdx.x / kPerRow, d0 = (threadIdx.x - group * kPerRow) * 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T *k = static_cast<const T*>(a.k) + kvh * D, *v = static_cast<const T*>(a.v) + kvh * D;
  const int64_t at_scale = page * a.kv_heads + kvh;
  const float was_k = a.k_scale[at_scale], was_v = a.v_scale[at_scale];
  auto values = [&](int token, float (&kx)[8], float (&vx)[8]) {
    rotated8<T, VEC>(a, k + token * a.k_stride, d0, a.positions[token], kx);
    load8<T, VEC>(v + token * a.v_stride + d0, vx);
  };
  float kk[kKept][8], vv[kKept][8];
  unsigned top_k = 0, top_v = 0;
#pragma unroll
  for (int i = 0; i < kKept; ++i) {
    const int row = group + i * kRows;
    if (row < a.page_size && s.token_of[row] >= 0) {
      values(s.token_of[row], kk[i], vv[i]);
      top_k = largest8(top_k, kk[i]), top_v = largest8(top_v, vv[i]);
    }
  }
  for (int row = group + kKept * kRows; row < a.page_size; row += kRows) {
    if (s.token_of[row] < 0) continue;
    float kx[8], vx[8];
    values(s.token_of[row], kx, vx);
    top_k = largest8(top_k, kx), top_v = largest8(top_v, vx);
  }
  top_k = __reduce_max_sync(0xffffffffu, top_k), top_v = __reduce_max_sync(0xffffffffu, top_v);
  if (lane == 0) s.top_k[warp] = top_k, s.top_v[warp] = top_v;
  const bool means = a.k_mean != nullptr && s.token_of[a.page_size - 1] >= 0;
  const bool begins = s.token_of[0] >= 0;
  for (int i = threadIdx.x; i < D; i += kThreads) s.sums[i] = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) top_k = max(top_k, s.top_k[w]), top_v = max(top_v, s.top_v[w]);
  const float before_k = begins ? 0.0f : was_k, before_v = begins ? 0.0f : was_v;
  const float scale_k = grown(before_k, top_k, 1.0f / Codec<C>::kTop), scale_v = grown(before_v, top_v, 1.0f / Codec<C>::kTop);
  if (threadIdx.x == 0) a.k_scale[at_scale] = scale_k, a.v_scale[at_scale] = scale_v;
  const bool move_k = !begins && scale_k > before_k, move_v = !begins && scale_v > before_v;
  const float ratio_k = __fdiv_rn(before_k, scale_k), ratio_v = __fdiv_rn(before_v, scale_v);

  int sums[8] = {};
  auto moved = [](uint2 old, float ratio) {
    float f[8];
    Codec<C>::unpack4(old.x, f), Codec<C>::unpack4(old.y, f + 4);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = __fmul_rn(f[e], ratio);
    return make_uint2(Codec<C>::pack4(f), Codec<C>::pack4(f + 4));
  };
  auto finish_row = [&](int row, const float (&kx)[8], const float (&vx)[8]) {
    const bool fresh = s.token_of[row] >= 0;
    const int64_t at = (a.hnd ? (page * a.kv_heads + kvh) * a.page_size + row : (page * a.page_size + row) * a.kv_heads + kvh) * D + d0;
    uint2 *kc = reinterpret_cast<uint2*>(a.k_cache + at), *vc = reinterpret_cast<uint2*>(a.v_cache + at);
    uint2 code = {};
    if (fresh) {
      *kc = code = encode8<C>(kx, scale_k);
      *vc = encode8<C>(vx, scale_v);
    } else {
      if (move_k || means) code = *kc;
      if (move_k) *kc = code = moved(code, ratio_k);
      if (move_v) *vc = moved(*vc, ratio_v);
    }
    if (means) {
      float f[8];
      Codec<C>::unpack4(code.x, f), Codec<C>::unpack4(code.y, f + 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) sums[e] += static_cast<int>(f[e] * Codec<C>::kUnits);
    }
  };
#pragma unroll
  for (int i = 0; i < kKept; ++i)
    if (group + i * kRows < a.page_size) finish_row(group + i * kRows, kk[i], vv[i]);
  for (int row = group + kKept * kRows; row < a.page_size; row += kRows) {
    float kx[8], vx[8];
    if (s.token_of[row] >= 0) values(s.token_of[row], kx, vx);
    finish_row(row, kx, vx);
  }
  if (!means) return;  // the same for all threads
#pragma unroll
  for (int e = 0; e < 8; ++e) {
#pragma unroll
    for (int sh = kPerRow; sh < 32; sh <<= 1) sums[e] += __shfl_xor_sync(0xffffffffu, sums[e], sh);
    if (lane < kPerRow || kPerRow == 32) atomicAdd(&s.sums[d0 + e], sums[e]);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += kThreads) {
    const float m = rintf(__fmul_rn(static_cast<float>(s.sums[d]), a.mean_unit));
    a.k_mean[at_scale * D + d] = static_cast<int8_t>(static_cast<int>(fminf(fmaxf(m, -127.0f), 127.0f)));
  }
}

// Batches of up to kSmallBatch tokens: y < kv_heads: the block of the token's page, if no token before it has the same page; the
// other y rotate Q.
template <typename T, typename C, int D, bool VEC>
__global__ void __launch_bounds__(kThreads)
kv8_append_kernel(const __grid_constant__ AppendArgs a) {
  __shared__ BlockShared s;
  __shared__ int64_t pages[kSmallBatch];
  pdl_launch_dependents();
  pdl_wait();  // q, k, v may be the preceding kernel's output; the caches may still be read by it
  const int token = blockIdx.x, kvh = blockIdx.y;
  if (kvh >= a.kv_heads) {
    rotate_q<T, D, VEC>(a, token, (kvh - a.kv_heads) * kThreads + threadIdx.x);
    return;
  }
  const int other = threadIdx.x;
  int64_t page = -1;
  int row = 0;
  if (other < a.tokens) {
    const int64_t pos = a.positions[other];
    if (pos >= 0) {
      const int64_t logical = pos / a.page_size;
      row = static_cast<int>(pos - logical * a.page_size);
      page = a.page_table[a.sequence_ids[other] * a.max_pages + logical];
    }
    pages[other] = page;
  }
  for (int i = threadIdx.x; i < a.page_size; i += kThreads) s.token_of[i] = -1;
  __syncthreads();
  const int64_t mine = pages[token];
  if (__syncthreads_or(mine < 0 || (other < token && page == mine))) return;
  if (other < a.tokens && page == mine) atomicMax(&s.token_of[row], other);
  __syncthreads();
  write_block<T, C, D, VEC>(a, s, mine, kvh);
}

// Longer batches, first launch: rotates Q, and enters every token's page into the table.
template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(kThreads)
kv8_group_kernel(const __grid_constant__ AppendArgs a, const __grid_constant__ Groups g) {
  pdl_launch_dependents();
  pdl_wait();
  const int token = blockIdx.x;
  if (blockIdx.y == 0 && threadIdx.x == 0) {
    const int64_t pos = a.positions[token];
    const int64_t physical = pos >= 0 ? a.page_table[a.sequence_ids[token] * a.max_pages + pos / a.page_size] : -1;
    int slot = -1;
    if (physical >= 0) {
      const unsigned long long page = static_cast<unsigned long long>(physical);
      unsigned at = static_cast<unsigned>((page * 0x9e3779b97f4a7c15ull) >> 32) & g.mask;
      for (unsigned tries = 0; tries <= g.mask; ++tries, at = (at + 1) & g.mask) {  // half of the entries stay free
        const unsigned long long found = atomicCAS(&g.page[at], ~0ull, page);
        if (found == ~0ull) g.list[atomicAdd(g.count, 1) + 1] = static_cast<int>(at);
        if (found == ~0ull || found == page) {
          slot = static_cast<int>(at);
          break;
        }
      }
      if (slot >= 0) {
        atomicMin(&g.first[slot], static_cast<unsigned>(token));
        atomicMax(&g.last[slot], token);
      }
    }
    g.slot_of[token] = slot;
  }
  rotate_q<T, D, VEC>(a, token, blockIdx.y * kThreads + threadIdx.x);
}

// Second launch: the blocks of the pages in the table, in turn.
template <typename T, typename C, int D, bool VEC>
__global__ void __launch_bounds__(kThreads)
kv8_blocks_kernel(const __grid_constant__ AppendArgs a, const __grid_constant__ Groups g) {
  __shared__ BlockShared s;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t items = static_cast<int64_t>(*g.count + 1) * a.kv_heads;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int entry = static_cast<int>(item / a.kv_heads), kvh = static_cast<int>(item - static_cast<int64_t>(entry) * a.kv_heads);
    const int slot = g.list[entry];
    for (int i = threadIdx.x; i < a.page_size; i += kThreads) s.token_of[i] = -1;
    __syncthreads();
    const int last = g.last[slot];
    for (int t = static_cast<int>(g.first[slot]) + threadIdx.x; t <= last; t += kThreads)
      if (g.slot_of[t] == slot) atomicMax(&s.token_of[static_cast<int>(a.positions[t] % a.page_size)], t);
    __syncthreads();
    write_block<T, C, D, VEC>(a, s, static_cast<int64_t>(g.page[slot]), kvh);
    __syncthreads();  // its shared memory is free again
  }
}

template <typename T, typename C, int D, bool VEC>
int launch_append(const AppendArgs& a, void* scratch, cudaStream_t stream) {
  const int64_t q_blocks = (static_cast<int64_t>(a.q_heads) * (D / 8) + kThreads - 1) / kThreads;
  if (q_blocks + a.kv_heads > 65535) return XDK_ERR_LIMIT;
  if (a.tokens <= kSmallBatch)
    return launch_dependent(kv8_append_kernel<T, C, D, VEC>, dim3(static_cast<unsigned>(a.tokens), static_cast<unsigned>(a.kv_heads + q_blocks)),
                            dim3(kThreads), 0, stream, a);
  const Groups g = groups_at(scratch, a.tokens);
  if (int st = note_launch(cudaMemsetAsync(scratch, 0xff, group_bytes(a.tokens), stream))) return st;
  if (int st = launch_opts(kv8_group_kernel<T, D, VEC>, dim3(static_cast<unsigned>(a.tokens), static_cast<unsigned>(q_blocks)), dim3(kThreads), 0,
                           stream, 1u, false, a, g))
    return st;
  const int64_t most = static_cast<int64_t>(a.tokens) * a.kv_heads, wave = static_cast<int64_t>(sm_count()) * 8;
  return launch_opts(kv8_blocks_kernel<T, C, D, VEC>, dim3(static_cast<unsigned>(most < wave ? most : wave)), dim3(kThreads), 0, stream, 1u, true,
                     a, g);
}

template <typename T, typename C>
int dispatch_append(int64_t d, const AppendArgs& a, void* scratch, cudaStream_t s) {
  constexpr int E = Elem<T>::kPerVec;
  // whole 16-byte vectors, whose rotation partners and angles are whole vectors too
  const bool vec = aligned16(a.q) && aligned16(a.k) && aligned16(a.v) && aligned16(a.cos) && aligned16(a.sin) && a.q_stride % E == 0 &&
                   a.k_stride % E == 0 && a.v_stride % E == 0 && a.cos_width % 4 == 0 && a.rope_dim % (a.interleaved ? 8 : 16) == 0;
#define XDK_APPEND(DD) return vec ? launch_append<T, C, DD, true>(a, scratch, s) : launch_append<T, C, DD, false>(a, scratch, s)
  switch (d) {
    case 64: XDK_APPEND(64);
    case 128: XDK_APPEND(128);
    case 256: XDK_APPEND(256);
    default: return XDK_ERR_LIMIT;
  }
#undef XDK_APPEND
}

}  // namespace
}  // namespace xdk

extern "C" size_t xdk_kv8_append_scratch_bytes(int64_t tokens) {
  return tokens <= xdk::kSmallBatch || tokens > (1LL << 26) ? 0 : xdk::group_bytes(tokens);
}

extern "C" int xdk_kv8_append(const void* q, const void* k, const void* v, const float* cos, const float* sin, const int64_t* positions,
                              const int64_t* page_table, const int64_t* sequence_ids, void* q_out, void* k_cache, void* v_cache,
                              float* k_scale, float* v_scale, int8_t* k_mean, int64_t tokens, int64_t q_heads, int64_t kv_heads,
                              int64_t head_dim, int64_t cos_width, int64_t max_pages_per_seq, int64_t page_size, int64_t rope_dim,
                              int64_t q_token_stride, int64_t k_token_stride, int64_t v_token_stride, int interleaved, int cache_is_hnd,
                              int dtype, int codes, void* scratch, size_t scratch_bytes, unsigned flags, void* stream) {
  using namespace xdk;
  if (flags & ~XDK_DEPENDENT_LAUNCH) return XDK_ERR_ARG;
  CallFlagsScope scope(flags);
  if (!q || !k || !v || !cos || !sin || !positions || !page_table || !sequence_ids || !q_out || !k_cache || !v_cache || !k_scale || !v_scale)
    return XDK_ERR_ARG;
  if (tokens < 1 || q_heads < 1 || kv_heads < 1 || head_dim < 1 || page_size < 1 || max_pages_per_seq < 1) return XDK_ERR_ARG;
  if (q_heads % kv_heads != 0 || rope_dim < 2 || rope_dim % 2 != 0 || rope_dim > head_dim || cos_width < rope_dim / 2) return XDK_ERR_ARG;
  if (q_token_stride < q_heads * head_dim || k_token_stride < kv_heads * head_dim || v_token_stride < kv_heads * head_dim) return XDK_ERR_ARG;
  if (!aligned16(q_out) || !aligned16(k_cache) || !aligned16(v_cache)) return XDK_ERR_ARG;
  if (!kv8_head_dim(head_dim) || q_heads > 65535 || cos_width > 2147483647LL) return XDK_ERR_LIMIT;
  if (int st = kv8_limits(tokens, kv_heads, max_pages_per_seq, page_size)) return st;
  const size_t need = xdk_kv8_append_scratch_bytes(tokens);
  if (need > 0 && (!scratch || scratch_bytes < need || !aligned16(scratch))) return XDK_ERR_ARG;
  if (codes != XDK_KV8_INT8 && codes != XDK_KV8_E4M3) return XDK_ERR_ARG;
  if (dtype != XDK_F32 && dtype != XDK_BF16 && dtype != XDK_F16) return XDK_ERR_ARG;
  if (int st = require_sm100()) return st;
  AppendArgs a;
  a.q = q, a.k = k, a.v = v, a.cos = cos, a.sin = sin;
  a.positions = positions, a.page_table = page_table, a.sequence_ids = sequence_ids, a.q_out = q_out;
  a.k_cache = static_cast<uint8_t*>(k_cache), a.v_cache = static_cast<uint8_t*>(v_cache);
  a.k_scale = k_scale, a.v_scale = v_scale, a.k_mean = k_mean;
  a.max_pages = max_pages_per_seq, a.q_stride = q_token_stride, a.k_stride = k_token_stride, a.v_stride = v_token_stride;
  a.tokens = static_cast<int>(tokens), a.q_heads = static_cast<int>(q_heads), a.kv_heads = static_cast<int>(kv_heads);
  a.page_size = static_cast<int>(page_size), a.rope_dim = static_cast<int>(rope_dim), a.cos_width = static_cast<int>(cos_width);
  a.interleaved = interleaved != 0, a.hnd = cache_is_hnd != 0;
  // the mean of int8 codes in units of the scale; of e4m3 codes, summed in units of 2^-9, in units of scale * 448 / 127
  a.mean_unit = static_cast<float>(codes == XDK_KV8_INT8 ? 1.0 / static_cast<double>(page_size)
                                                          : 127.0 / (448.0 * 512.0 * static_cast<double>(page_size)));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define XDK_APPEND(T) \
  return codes == XDK_KV8_INT8 ? dispatch_append<T, Int8Codes>(head_dim, a, scratch, s) : dispatch_append<T, E4m3Codes>(head_dim, a, scratch, s)
  switch (dtype) {
    case XDK_F32: XDK_APPEND(float);
    case XDK_BF16: XDK_APPEND(__nv_bfloat16);
    case XDK_F16: XDK_APPEND(__half);
    default: return XDK_ERR_ARG;
  }
#undef XDK_APPEND
}
