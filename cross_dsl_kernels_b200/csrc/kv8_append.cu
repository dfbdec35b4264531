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
// A block's rows come from the batch's index vectors, so tokens may come in any order, several for a page or for a slot.  Up to
// kSmallBatch tokens: one launch, every CTA looks all of them up, and the first token of a page does its work, a warp to a block.  Longer
// batches: the first launch enters the tokens by page into a table in scratch and leaves the largest value of every row of K and V; the
// second one walks the table, and can write a row at once, while other CTAs of it rotate Q.  (Blocks that first read their rows for the
// largest value and then write them, in one kernel: a CTA to a block 46 us for 4096 tokens with 32 + 2 * 8 heads of 128, a warp to a block
// 49; Q in the first launch 36.)  A CTA of the second launch has some 64 rows: four blocks of 16, or one of a page of 64 (four of those: 43
// us), whose mean its threads sum in slices (by one warp: 50).
// A lane holds two vectors of eight dims of a row, rotation partners where there are some, and so reads every value and angle once.
//
// Bound: a decode batch by its chain of dependent loads: position, sequence, page, then the block's scale (3.5 us where no scale grows), and then the
// rows that a grown scale moves, a few at a time by the block's warp: row 8 of pages of 16 4.1 -> 5.0 us, row 33 of 64 5.0 -> 9.2.  4096 tokens: 30 us,
// where HBM takes 14 (values read once, codes written once; the second launch finds K and V in L2): 2 us for the memset, 6 for the first launch,
// 5 for the second one's chain of loads, then the rows, by latency first (57 % of the cycles issue), then by rotation and exact division.
// A page's tokens are looked for between its first and last one: in random order 65536 tokens of 2 KV heads of 64 take 168 us for 73, 262144 1839 for 305.
#include <math.h>

#include "kv8.cuh"

namespace xdk {
namespace {

constexpr int kThreads = 128;
constexpr int kSmallBatch = 128;
constexpr int kBlocksOf = kThreads / 32;

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

// Where the tokens of a long batch go, by physical page: an open hash table of `slots` entries; what stands up to `count` is
// filled with 0xff before the first launch.
struct Groups {
  unsigned long long* page;  // [slots], ~0: free
  unsigned* first;           // [slots] first and last token of the page
  int* last;
  int* list;                 // [slots] the entries in use, in any order
  int* slot_of;              // [tokens] entry of a token's page, -1: no page
  int* count;                // entries in use - 1
  unsigned* tops;            // [tokens, 2 * kv_heads] the bits of the largest |value| of a row of K, then of V
  uint16_t* row_of;          // [tokens] row in the page
  unsigned mask;             // slots - 1
  int each;                  // blocks of a page that a CTA writes, at most kBlocksOf
};
inline int64_t group_slots(int64_t tokens) {
  int64_t s = 1;
  while (s < 2 * tokens) s <<= 1;
  return s;
}
inline size_t cleared_bytes(int64_t tokens) { return static_cast<size_t>(group_slots(tokens)) * 20 + 4; }
inline size_t group_bytes(int64_t tokens, int64_t kv_heads) {
  return cleared_bytes(tokens) + static_cast<size_t>(tokens) * static_cast<size_t>(4 + 2 + 8 * kv_heads);
}
inline Groups groups_at(void* scratch, int64_t tokens, int64_t kv_heads) {
  const int64_t s = group_slots(tokens);
  Groups g;
  g.page = static_cast<unsigned long long*>(scratch);
  g.first = reinterpret_cast<unsigned*>(g.page + s);
  g.last = reinterpret_cast<int*>(g.first + s);
  g.list = g.last + s;
  g.count = g.list + s;
  g.slot_of = g.count + 1;
  g.tops = reinterpret_cast<unsigned*>(g.slot_of + tokens);
  g.row_of = reinterpret_cast<uint16_t*>(g.tops + tokens * 2 * kv_heads);
  g.mask = static_cast<unsigned>(s - 1);
  return g;
}

template <typename T, bool VEC> __device__ __forceinline__ void load8(const T* p, float* x) {
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
// The two vectors of eight dims that thread t of a row's D / 16 holds: rotation partners, where these are whole vectors, or two next
// to each other.
template <bool VEC> __device__ __forceinline__ void dims_of(const AppendArgs& a, int t, int& d0, int& d1) {
  const int pairs = !VEC || a.interleaved ? 0 : a.rope_dim / 16;
  if (t < pairs) d0 = t * 8, d1 = d0 + a.rope_dim / 2;
  else d0 = pairs * 16 + (t - pairs) * 16, d1 = d0 + 8;
}
// Angles of the pairs in vectors d0, d1: eight of a non-interleaved pair of vectors, four of each of interleaved ones.
__device__ __forceinline__ void angles_of(const AppendArgs& a, int d0, int d1, int64_t pos, float (&c)[8], float (&s)[8]) {
  const float *crow = a.cos + pos * a.cos_width, *srow = a.sin + pos * a.cos_width;
  auto load = [](const float* p, float* x) {
    const float4 f = __ldg(reinterpret_cast<const float4*>(p));
    x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
  };
  const bool first = d0 < a.rope_dim, second = d1 < a.rope_dim;
  const int at0 = a.interleaved ? d0 / 2 : d0, at1 = a.interleaved ? d1 / 2 : d0 + 4;
  if (first) load(crow + at0, c), load(srow + at0, s);
  if (second) load(crow + at1, c + 4), load(srow + at1, s + 4);
}
// Turns x (at dims d0 .. and d1 ..) by the angles; separately rounded products and sums.
__device__ __forceinline__ void turn(const AppendArgs& a, int d0, int d1, const float (&c)[8], const float (&s)[8], float (&x)[16]) {
  auto pair = [](float& lo, float& hi, float cv, float sv) {
    const float l = lo, h = hi;
    lo = __fsub_rn(__fmul_rn(l, cv), __fmul_rn(h, sv));
    hi = __fadd_rn(__fmul_rn(l, sv), __fmul_rn(h, cv));
  };
  if (a.interleaved) {
    if (d0 < a.rope_dim)
#pragma unroll
      for (int e = 0; e < 4; ++e) pair(x[2 * e], x[2 * e + 1], c[e], s[e]);
    if (d1 < a.rope_dim)
#pragma unroll
      for (int e = 0; e < 4; ++e) pair(x[8 + 2 * e], x[9 + 2 * e], c[4 + e], s[4 + e]);
  } else if (d0 < a.rope_dim) {
#pragma unroll
    for (int e = 0; e < 8; ++e) pair(x[e], x[8 + e], c[e], s[e]);
  }
}
// Any rotation width and any alignment: dim by dim.
template <typename T>
__device__ __forceinline__ void rotated_scalar(const AppendArgs& a, const T* head, int d0, int64_t pos, float* x) {
  const float *crow = a.cos + pos * a.cos_width, *srow = a.sin + pos * a.cos_width;
  const int half = a.rope_dim / 2;
  load8<T, false>(head + d0, x);
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
template <typename T, bool VEC>
__device__ __forceinline__ void rotated16(const AppendArgs& a, const T* head, int d0, int d1, int64_t pos, float (&x)[16]) {
  if constexpr (VEC) {
    float c[8], s[8];
    load8<T, true>(head + d0, x), load8<T, true>(head + d1, x + 8);
    angles_of(a, d0, d1, pos, c, s);
    turn(a, d0, d1, c, s, x);
  } else {
    rotated_scalar(a, head, d0, pos, x), rotated_scalar(a, head, d1, pos, x + 8);
  }
}

// A unit: a thread has the same 16 dims of a few heads of a token, of Q, of K or of V, so the angles are loaded once for them.  Q is
// rotated and written (a token without a position gets zeros); of K, rotated, and of V the largest values of the rows are left in `tops`.
template <typename T> constexpr int kHeadsOf = sizeof(T) == 4 ? 2 : 4;     // heads of a unit of Q
template <typename T> constexpr int kTopHeadsOf = sizeof(T) == 4 ? 1 : 2;  // and of K and V
template <int D> __host__ __device__ constexpr int units_of(int heads, int each) { return (heads + each - 1) / each * (D / 16); }  // threads of a token
__device__ __forceinline__ unsigned largest(const float (&x)[16]) {  // the bits of the largest |value|: NaN over infinity over numbers
  unsigned top = 0;
#pragma unroll
  for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
  return top;
}
template <int D> __device__ __forceinline__ unsigned row_max(unsigned top) {  // over the D / 16 lanes of a row
#pragma unroll
  for (int sh = 1; sh < D / 16; sh <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, sh));
  return top;
}
template <typename T, int D, bool VEC>
__device__ __forceinline__ void rotate_q(const AppendArgs& a, int token, int rest) {  // rest: unit of the token's heads of Q
  constexpr int kHeads = kHeadsOf<T>, E = Elem<T>::kPerVec;
  const int head0 = rest / (D / 16) * kHeads, heads = a.q_heads - head0 < kHeads ? a.q_heads - head0 : kHeads;
  int d0, d1;
  dims_of<VEC>(a, rest % (D / 16), d0, d1);
  const int64_t pos = a.positions[token];
  const T* src = static_cast<const T*>(a.q) + token * a.q_stride + head0 * D;
  T* dst = static_cast<T*>(a.q_out) + (static_cast<int64_t>(token) * a.q_heads + head0) * D;  // 16-byte aligned
  float c[8], s[8];
  if (VEC && pos >= 0) angles_of(a, d0, d1, pos, c, s);
#pragma unroll 2
  for (int h = 0; h < heads; ++h) {
    float x[16] = {};
    if (pos >= 0) {
      if constexpr (VEC) {
        load8<T, true>(src + h * D + d0, x), load8<T, true>(src + h * D + d1, x + 8);
        turn(a, d0, d1, c, s, x);
      } else {
        rotated16<T, false>(a, src + h * D, d0, d1, pos, x);
      }
    }
#pragma unroll
    for (int i = 0; i < 16 / E; ++i) {
      float f[E];
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = x[i * E + e];
      *reinterpret_cast<U4*>(dst + h * D + (i < 8 / E ? d0 + i * E : d1 + i * E - 8)) = pack16<T>(f);
    }
  }
}
// rest: unit of the token's heads of K, then of V; `live`: there is such a unit.  Whole warps call it.  The values are on their way
// before the position is known, which only says by which angles K turns and whether they count.
template <typename T, int D, bool VEC>
__device__ __forceinline__ void find_tops(const AppendArgs& a, unsigned* tops, int token, int rest, bool live) {
  constexpr int kHeads = kTopHeadsOf<T>, E = Elem<T>::kPerVec, kVecs = 16 / E;
  const int per_kind = units_of<D>(a.kv_heads, kHeads);
  const bool is_v = rest >= per_kind;
  if (is_v) rest -= per_kind;
  const int head0 = rest / (D / 16) * kHeads, heads = !live ? 0 : (a.kv_heads - head0 < kHeads ? a.kv_heads - head0 : kHeads);
  int d0, d1;
  dims_of<VEC>(a, rest % (D / 16), d0, d1);
  const T* src = static_cast<const T*>(is_v ? a.v : a.k) + token * (is_v ? a.v_stride : a.k_stride) + head0 * D;
  U4 raw[kHeads][kVecs];
  if constexpr (VEC) {
#pragma unroll
    for (int h = 0; h < kHeads; ++h)
#pragma unroll
      for (int w = 0; w < kVecs; ++w)
        if (h < heads) raw[h][w] = ld_ordered16(src + h * D + (w < kVecs / 2 ? d0 + w * E : d1 + (w - kVecs / 2) * E));
  }
  const int64_t pos = live ? a.positions[token] : -1;
  float c[8], s[8];
  if (VEC && pos >= 0 && !is_v) angles_of(a, d0, d1, pos, c, s);
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    unsigned top = 0;
    const bool some = pos >= 0 && h < heads;
    if (some) {
      float x[16];
      if constexpr (VEC) {
#pragma unroll
        for (int w = 0; w < kVecs; ++w) {
          float f[E];
          unpack16<T>(raw[h][w], f);
#pragma unroll
          for (int e = 0; e < E; ++e) x[w * E + e] = f[e];
        }
        if (!is_v) turn(a, d0, d1, c, s, x);
      } else if (is_v) {
        load8<T, false>(src + h * D + d0, x), load8<T, false>(src + h * D + d1, x + 8);
      } else {
        rotated16<T, false>(a, src + h * D, d0, d1, pos, x);
      }
      top = largest(x);
    }
    top = row_max<D>(top);
    if (some && rest % (D / 16) == 0) tops[(static_cast<int64_t>(token) * 2 + (is_v ? 1 : 0)) * a.kv_heads + head0 + h] = top;
  }
}

// The scale behind the call from the one before and the bits of the largest |value|: NaN for anything that is not a finite number.
__device__ __forceinline__ float grown(float before, unsigned top_bits, float per_top) {
  if (!isfinite(before) || top_bits >= 0x7f800000u) return __uint_as_float(0x7fffffffu);
  return fmaxf(before, __fmul_rn(__uint_as_float(top_bits), per_top));
}
// x / scale, correctly rounded, by Markstein's theorem: from the correctly rounded reciprocal r and a quotient q that is off by less than
// a unit in the last place, q + r * (x - q * scale) is the rounded quotient, where nothing underflows.  x * r may be off by two, so it is
// corrected twice.  x and a scale far from 1 are multiplied by a power of two first, which changes neither the quotient nor, for what can
// become another code than 0, a bit of x.
struct Divider {
  float scale, r, lift;
  bool some;  // not the scale of a block of zeros, nor NaN: all codes are 0
};
__device__ __forceinline__ Divider divider(float s) {
  Divider d;
  d.some = s > 0.0f;
  d.lift = s > 1.2089258e24f ? 8.6736174e-19f : (s >= 8.2718061e-25f ? 1.0f : 1.2676506e30f);  // above 2^80: 2^-60, below 2^-80: 2^100
  d.scale = d.some ? s * d.lift : 1.0f, d.r = __fdiv_rn(1.0f, d.scale);
  return d;
}
template <typename C> __device__ __forceinline__ void divide16(const Divider& d, float (&x)[16]) {
  if (d.lift != 1.0f) {  // also of a scale of 0 and of NaN
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = d.some ? __fmul_rn(x[e], d.lift) : 0.0f;
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    float q = __fmul_rn(x[e], d.r);
    q = __fmaf_rn(__fmaf_rn(-q, d.scale, x[e]), d.r, q);
    x[e] = copysignf(__fmaf_rn(__fmaf_rn(-q, d.scale, x[e]), d.r, q), x[e]);  // -0 too, which e4m3 has
  }
  if (d.lift != 1.0f) {  // a quotient passes the largest code where the scale is subnormal
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = fminf(fmaxf(x[e], -Codec<C>::kTop), Codec<C>::kTop);
  }
}

// A block of one call: where it is, and its scale before and behind the call.
struct Block {
  int64_t page;
  int kvh;
  bool is_v, move;  // move: rows that are not written anew are rounded to the grown scale
  float ratio;
  Divider by_scale;
};
__device__ __forceinline__ float* scale_of(const AppendArgs& a, const Block& b) { return (b.is_v ? a.v_scale : a.k_scale) + b.page * a.kv_heads + b.kvh; }
__device__ __forceinline__ uint8_t* row_of(const AppendArgs& a, const Block& b, int row, int dim) {
  return (b.is_v ? a.v_cache : a.k_cache) +
         (a.hnd ? (b.page * a.kv_heads + b.kvh) * a.page_size + row : (b.page * a.page_size + row) * a.kv_heads + b.kvh) * dim;
}
template <typename C> __device__ __forceinline__ float rescale(Block& b, float was, bool begins, unsigned top) {
  const float before = begins ? 0.0f : was, scale = grown(before, top, 1.0f / Codec<C>::kTop);
  b.move = !begins && scale > before;
  b.ratio = __fdiv_rn(before, scale);
  b.by_scale = divider(scale);
  return scale;
}
// Sixteen dims of row `row`: those of `token`, or of the codes that stand there.
template <typename T, int D, bool VEC>
__device__ __forceinline__ void row_values(const AppendArgs& a, bool is_v, int kvh, int token, int d0, int d1, float (&x)[16]) {
  if (!is_v) rotated16<T, VEC>(a, static_cast<const T*>(a.k) + token * a.k_stride + kvh * D, d0, d1, a.positions[token], x);
  else {
    const T* head = static_cast<const T*>(a.v) + token * a.v_stride + kvh * D;
    load8<T, VEC>(head + d0, x), load8<T, VEC>(head + d1, x + 8);
  }
}
template <typename T, typename C, int D, bool VEC>
__device__ __forceinline__ void write_row(const AppendArgs& a, const Block& b, int row, int token, int d0, int d1) {
  if (token < 0 && !b.move) return;
  uint8_t* to = row_of(a, b, row, D);
  uint2 *at0 = reinterpret_cast<uint2*>(to + d0), *at1 = reinterpret_cast<uint2*>(to + d1);
  float x[16];
  if (token >= 0) {
    row_values<T, D, VEC>(a, b.is_v, b.kvh, token, d0, d1, x);
    divide16<C>(b.by_scale, x);
  } else {
    const uint2 c0 = *at0, c1 = *at1;
    Codec<C>::unpack4(c0.x, x), Codec<C>::unpack4(c0.y, x + 4), Codec<C>::unpack4(c1.x, x + 8), Codec<C>::unpack4(c1.y, x + 12);
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = fmaxf(__fmul_rn(x[e], b.ratio), -Codec<C>::kTop);  // an int8 code may be -128
  }
  *at0 = make_uint2(Codec<C>::pack4(x), Codec<C>::pack4(x + 4));
  *at1 = make_uint2(Codec<C>::pack4(x + 8), Codec<C>::pack4(x + 12));
}
// The mean of four dims of a block of K, whose codes are all written: sums of every so many rows, and what they come to.
template <typename C, int D> __device__ __forceinline__ void sum_rows(const AppendArgs& a, const Block& b, int d, int first, int step, int (&sums)[4]) {
#pragma unroll 8
  for (int row = first; row < a.page_size; row += step) {
    float f[4];
    Codec<C>::unpack4(__ldcg(reinterpret_cast<const uint32_t*>(row_of(a, b, row, D) + d)), f);
#pragma unroll
    for (int e = 0; e < 4; ++e) sums[e] += static_cast<int>(f[e] * Codec<C>::kUnits);
  }
}
template <int D> __device__ __forceinline__ void write_mean(const AppendArgs& a, const Block& b, int d, const int (&sums)[4]) {
  uint32_t packed = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float m = rintf(__fmul_rn(static_cast<float>(sums[e]), a.mean_unit));
    packed |= (static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(m, -127.0f), 127.0f))) & 0xffu) << (8 * e);
  }
  *reinterpret_cast<uint32_t*>(a.k_mean + (b.page * a.kv_heads + b.kvh) * D + d) = packed;
}

// Batches of up to kSmallBatch tokens: a CTA has four of the 2 * kv_heads blocks of K and V of the token's page, if no token before it has
// the same page; the CTAs behind those (`block_rows` of them) rotate Q.
template <typename T, typename C, int D, bool VEC>
__global__ void __launch_bounds__(kThreads)
kv8_append_kernel(const __grid_constant__ AppendArgs a, int block_rows) {
  extern __shared__ int token_of[];  // [page_size]
  __shared__ int64_t pages[kSmallBatch];
  pdl_launch_dependents();
  pdl_wait();  // q, k, v may be the preceding kernel's output; the caches may still be read by it
  const int token = blockIdx.x, part = blockIdx.y;
  if (part >= block_rows) {
    const int unit = (part - block_rows) * kThreads + threadIdx.x;
    if (unit < units_of<D>(a.q_heads, kHeadsOf<T>)) rotate_q<T, D, VEC>(a, token, unit);
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
  for (int i = threadIdx.x; i < a.page_size; i += kThreads) token_of[i] = -1;
  __syncthreads();
  const int64_t mine = pages[token];
  if (__syncthreads_or(mine < 0 || (other < token && page == mine))) return;
  if (other < a.tokens && page == mine) atomicMax(&token_of[row], other);
  __syncthreads();
  const int head = part * (kThreads / 32) + (threadIdx.x >> 5);  // of K, then of V
  if (head >= 2 * a.kv_heads) return;
  Block b;
  b.page = mine, b.is_v = head >= a.kv_heads, b.kvh = b.is_v ? head - a.kv_heads : head;
  constexpr int kPerRow = D / 16, kRows = 32 / kPerRow;  // lanes of a row, rows at a time
  const int lane = threadIdx.x & 31, group = lane / kPerRow;
  int d0, d1;
  dims_of<VEC>(a, lane - group * kPerRow, d0, d1);
  float* scale_at = scale_of(a, b);
  const float was = *scale_at;
  unsigned top = 0;
#pragma unroll 1
  for (int r = group; r < a.page_size; r += kRows)
    if (token_of[r] >= 0) {
      float x[16];
      row_values<T, D, VEC>(a, b.is_v, b.kvh, token_of[r], d0, d1, x);
      top = max(top, largest(x));
    }
  top = __reduce_max_sync(0xffffffffu, top);
  const float scale = rescale<C>(b, was, token_of[0] >= 0, top);
  if (lane == 0) *scale_at = scale;  // every lane has read it: the reduction stands between
#pragma unroll 1
  for (int r = group; r < a.page_size; r += kRows) write_row<T, C, D, VEC>(a, b, r, token_of[r], d0, d1);  // values again, from L1
  if (b.is_v || a.k_mean == nullptr || token_of[a.page_size - 1] < 0) return;  // the same for all lanes
  __syncwarp();
  for (int d = lane * 4; d < D; d += 32 * 4) {
    int sums[4] = {};
    sum_rows<C, D>(a, b, d, 0, 1, sums);
    write_mean<D>(a, b, d, sums);
  }
}

// The token and the unit in it of thread t of CTA `cta`, `per_token` units to a token.
__device__ __forceinline__ int2 token_and_unit(int64_t cta, int per_token) {
  const int64_t first = cta * kThreads;
  int token = static_cast<int>(first / per_token), unit = static_cast<int>(first - static_cast<int64_t>(token) * per_token) + threadIdx.x;
  const int further = unit / per_token;
  return make_int2(token + further, unit - further * per_token);
}
// Longer batches, first launch: the first `entries` CTAs enter every token's page into the table, the others find the largest values of K
// and V.
template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(kThreads)
kv8_group_kernel(const __grid_constant__ AppendArgs a, const __grid_constant__ Groups g, unsigned entries) {
  pdl_launch_dependents();
  pdl_wait();
  if (blockIdx.x >= entries) {
    const int2 at = token_and_unit(blockIdx.x - entries, 2 * units_of<D>(a.kv_heads, kTopHeadsOf<T>));
    find_tops<T, D, VEC>(a, g.tops, at.x < a.tokens ? at.x : 0, at.y, at.x < a.tokens);
    return;
  }
  const int token = blockIdx.x * kThreads + threadIdx.x;
  if (token >= a.tokens) return;
  const int64_t pos = a.positions[token];
  const int64_t logical = pos / a.page_size;
  const int64_t physical = pos >= 0 ? a.page_table[a.sequence_ids[token] * a.max_pages + logical] : -1;
  g.row_of[token] = static_cast<uint16_t>(pos - logical * a.page_size);
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

// Second launch: `block_ctas` CTAs take some blocks of a page in the table in turn.  A warp finds the scale of one, then all threads write
// the rows of all.  The others rotate Q, `q_first` of them in front, which keeps HBM busy while those wait for their chains of loads.
template <typename T, typename C, int D, bool VEC>
__global__ void __launch_bounds__(kThreads)
kv8_blocks_kernel(const __grid_constant__ AppendArgs a, const __grid_constant__ Groups g, unsigned parts, unsigned block_ctas, unsigned q_first) {
  constexpr int kPerRow = D / 16;
  extern __shared__ int token_of[];  // [page_size]
  __shared__ Block blocks[kBlocksOf];
  __shared__ int part_sums[kThreads][5];
  pdl_launch_dependents();
  const bool is_q = blockIdx.x < q_first || blockIdx.x >= q_first + block_ctas;
  const unsigned cta = blockIdx.x < q_first ? blockIdx.x : blockIdx.x - (is_q ? block_ctas : q_first);
  if (is_q) {  // no wait: nothing of the first launch is read, which began when all work before it had ended
    const int2 at = token_and_unit(cta, units_of<D>(a.q_heads, kHeadsOf<T>));
    if (at.x < a.tokens) rotate_q<T, D, VEC>(a, at.x, at.y);
    return;
  }
  pdl_wait();
  const unsigned part = cta % parts;  // of a page's blocks; block_ctas is a multiple of them
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, heads = 2 * a.kv_heads;
  const int head0 = part * g.each, head = head0 + warp, some = heads - head0 < g.each ? heads - head0 : g.each;  // K, then V
  int d0, d1;
  dims_of<VEC>(a, threadIdx.x % kPerRow, d0, d1);
  for (unsigned entry = cta / parts; entry <= g.mask; entry += block_ctas / parts) {
    const int slot = g.list[entry];
    if (slot < 0) return;  // behind the last one; the same for all threads
    for (int i = threadIdx.x; i < a.page_size; i += kThreads) token_of[i] = -1;
    const int first = static_cast<int>(g.first[slot]), last = g.last[slot];
    Block b;
    b.page = static_cast<int64_t>(g.page[slot]), b.is_v = head >= a.kv_heads, b.kvh = b.is_v ? head - a.kv_heads : head;
    const float was = warp < some ? *scale_of(a, b) : 0.0f;
    __syncthreads();
    for (int t = first + threadIdx.x; t <= last; t += kThreads) {
      const int row = g.row_of[t];
      if (g.slot_of[t] == slot) atomicMax(&token_of[row], t);
    }
    __syncthreads();
    if (warp < some) {
      unsigned top = 0;
      for (int r = lane; r < a.page_size; r += 32)
        if (token_of[r] >= 0) top = max(top, g.tops[static_cast<int64_t>(token_of[r]) * heads + head]);
      top = __reduce_max_sync(0xffffffffu, top);
      const float scale = rescale<C>(b, was, token_of[0] >= 0, top);
      if (lane == 0) {
        *scale_of(a, b) = scale;
        blocks[warp] = b;
      }
    }
    __syncthreads();
    // rows of one block after the other: neighbours in HND; in NHD the blocks' rows stand side by side
    for (int i = threadIdx.x / kPerRow; i < a.page_size * some; i += kThreads / kPerRow) {
      const int of = i / a.page_size, row = i - of * a.page_size;
      write_row<T, C, D, VEC>(a, blocks[of], row, token_of[row], d0, d1);
    }
    const bool means = a.k_mean != nullptr && token_of[a.page_size - 1] >= 0 && head0 < a.kv_heads;
    __syncthreads();  // the codes are written
    const int lanes = some * (D / 4);
    if (means && g.each > 1) {
      for (int i = threadIdx.x; i < lanes; i += kThreads) {
        const Block& of = blocks[i / (D / 4)];
        if (of.is_v) continue;
        int sums[4] = {};
        sum_rows<C, D>(a, of, i % (D / 4) * 4, 0, 1, sums);
        write_mean<D>(a, of, i % (D / 4) * 4, sums);
      }
    } else if (means) {  // one block, of many rows: D / 4 threads at a slice of them
      constexpr int kSlices = kThreads / (D / 4);
      const int d = threadIdx.x % (D / 4) * 4;
      int sums[4] = {};
      sum_rows<C, D>(a, blocks[0], d, threadIdx.x / (D / 4), kSlices, sums);
#pragma unroll
      for (int e = 0; e < 4; ++e) part_sums[threadIdx.x][e] = sums[e];
      __syncthreads();
      if (threadIdx.x < D / 4) {
#pragma unroll
        for (int i = 1; i < kSlices; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) sums[e] += part_sums[i * (D / 4) + threadIdx.x][e];
        write_mean<D>(a, blocks[0], d, sums);
      }
    }
    __syncthreads();  // shared memory is free again
  }
}

template <typename T, typename C, int D, bool VEC>
int launch_append(const AppendArgs& a, void* scratch, cudaStream_t stream) {
  const int64_t q_units = units_of<D>(a.q_heads, kHeadsOf<T>), heads = 2 * static_cast<int64_t>(a.kv_heads), warps = kThreads / 32;
  const size_t map = static_cast<size_t>(a.page_size) * 4;
  if (a.tokens <= kSmallBatch) {
    const int64_t parts = (heads + warps - 1) / warps;
    const int64_t rows = parts + (q_units + kThreads - 1) / kThreads;
    if (rows > 65535) return XDK_ERR_LIMIT;
    return launch_dependent(kv8_append_kernel<T, C, D, VEC>, dim3(static_cast<unsigned>(a.tokens), static_cast<unsigned>(rows)), dim3(kThreads), map,
                            stream, a, static_cast<int>(parts));
  }
  Groups g = groups_at(scratch, a.tokens, a.kv_heads);
  g.each = a.page_size <= 16 ? kBlocksOf : (a.page_size <= 32 ? 2 : 1);  // some 64 rows to a CTA
  const int64_t parts = (heads + g.each - 1) / g.each;
  const int64_t entries = (a.tokens + kThreads - 1) / kThreads, q_ctas = (a.tokens * q_units + kThreads - 1) / kThreads;
  const int64_t kv_ctas = (a.tokens * 2 * units_of<D>(a.kv_heads, kTopHeadsOf<T>) + kThreads - 1) / kThreads;
  // as many CTAs as there can be work for, or the SMs hold
  const int64_t wave = (static_cast<int64_t>(sm_count()) * 8 + parts - 1) / parts, block_ctas = (a.tokens < wave ? a.tokens : wave) * parts;
  // Q's CTAs in front of the blocks': they start while the first launch ends.  Five to an SM: 29.4 us for 4096 tokens; none 31.6, all 33.0, in
  // turn with the blocks' 30.7
  const int64_t in_front = static_cast<int64_t>(sm_count()) * 5, q_first = q_ctas < in_front ? q_ctas : in_front;
  if (entries + kv_ctas > 2147483647LL || block_ctas + q_ctas > 2147483647LL) return XDK_ERR_LIMIT;
  if (int st = note_launch(cudaMemsetAsync(scratch, 0xff, cleared_bytes(a.tokens), stream))) return st;
  if (int st = launch_opts(kv8_group_kernel<T, D, VEC>, dim3(static_cast<unsigned>(entries + kv_ctas)), dim3(kThreads), 0, stream, 1u, false, a, g,
                           static_cast<unsigned>(entries)))
    return st;
  return launch_opts(kv8_blocks_kernel<T, C, D, VEC>, dim3(static_cast<unsigned>(block_ctas + q_ctas)), dim3(kThreads), map, stream, 1u, true, a, g,
                     static_cast<unsigned>(parts), static_cast<unsigned>(block_ctas), static_cast<unsigned>(q_first));
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

extern "C" size_t xdk_kv8_append_scratch_bytes(int64_t tokens, int64_t kv_heads) {
  if (tokens <= xdk::kSmallBatch || tokens > (1LL << 26) || kv_heads < 1 || kv_heads > 65535) return 0;
  return xdk::group_bytes(tokens, kv_heads);
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
  if (!aligned16(q_out) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(k_mean)) return XDK_ERR_ARG;
  if (!kv8_head_dim(head_dim) || q_heads > 65535 || cos_width > 2147483647LL) return XDK_ERR_LIMIT;
  if (int st = kv8_limits(tokens, kv_heads, max_pages_per_seq, page_size)) return st;
  const size_t need = xdk_kv8_append_scratch_bytes(tokens, kv_heads);
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
