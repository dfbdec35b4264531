// Attention of one query token per sequence over the 8-bit paged cache (kv8.cuh), over all of its context or over listed pages.
//
//   s_j = scale * ks[page of j] * (q . kc_j),   out = sum_j softmax(s)_j * vs[page of j] * vc_j
// with codes kc, vc and a scale per page and KV head; j runs over 0 .. position, or over those of them that lie in the pages of
// the token's list.  Nothing to attend to: zeros.
//
// A code is exact in FP16, so both contractions are mma.m16n8k16 on FP16 with positions (scores) and dims (values) as the 16 rows and the
// heads of the group as the 8 columns:
//   * q is scaled by a power of two, so that its largest value is near 2^14, and rounded to FP16 (FP16 and BF16 values pass whole unless
//     they are 2^-27 of the largest); an FP32 q is the sum of two such numbers, and each product two products.
//   * the weights are the softmax weights times the block scales of V, w = p * vs = 2^(s + log2 vs): one running maximum, of the whole exponent,
//     and one exponential; the softmax sum takes vs out again.  That holds while the scales of V are within 2^30 of the first tile's.  From a tile
//     on that has one farther away, or 0, the sum has a maximum and an exponential of its own, and the weights are 2^(s - max s + log2 vs), which
//     large scores do not take the scale from (this for every tile: 2 - 3 % more time).  The largest weight of a head is 2^14, which FP16 has, so that
//     what rounds away is below 2^-38 of it; the others are rounded to FP16 (half a step: 2^-11).
//     For FP32 results a weight is the sum of two FP16 numbers, and the logarithm of a far vs would be off by too much: its exponent goes with s, its
//     significand is a factor.
//   * int8 codes enter as the subnormal halves (code + 128) * 2^-24, which a byte permute makes; the sums begin with -128 times the sum of
//     the other operand.  FP32 results would see the few 2^-23 of 128 that this rounds away: for them the codes are centred first.
//   * a tile's sum is added to the accumulators by FP32 FMAs, with rounding; the tensor core truncates.
// Bytes of a row come as 16-bit pairs through ldmatrix: for K four dims of a position (q in the same order), for V, transposed, two dims of
// two positions, which byte permutes sort while they widen the codes.
//
// HBM-bound in the long run.  The tiles of 32 positions of all (token, KV head) items stand in one line, and every warp -- a CTA of its own, as
// many as the SMs hold -- takes an equal range: no barrier but the warp's, and its ring of cp.async stages never runs dry, not at
// the end of an item either.  Of an item that several warps share each leaves the result over its positions in scratch, with its share of the
// weights, and a second launch adds them in their order.  (Chunks that the hardware hands out as warps finish, by CTAs or by cancelled launches, measured slower: 70 us for 16
// contexts of 8192, where equal ranges took 61 with the same tiles; a chunk's start costs its warp 6 us without loads.)
//
// 32 / 8 heads of 128, us: 16 contexts of 32768 176 (6.1 TB/s), of 8192 57 (4.7), 64 of 1 .. 2048 38, one of 8192 14.  Of short work it is bound by
// its two launches and the chain position -> page table -> rows (8 us), of long work by HBM.
#include <math.h>

#include <type_traits>

#include "kv8.cuh"
#include "mma_f16.cuh"

namespace xdk {
namespace {

struct Kv8Args {
  const void* q;
  const uint8_t *k_cache, *v_cache;
  const float *k_scale, *v_scale;
  const int64_t *positions, *page_table, *sequence_ids;
  const int32_t* pages;  // [tokens, kv_heads, n_pages], sparse only
  float* scratch;
  int64_t max_pages, page_size;
  int tokens, q_heads, kv_heads, group;  // group: query heads of a KV head
  int n_pages, dtype;                    // dtype: of q and out
  int tile;                              // positions of a tile
  int hnd, narrow;                       // narrow: every position that a page table row can hold fits 31 bits
  int by_warp;                           // see Partials
  int paired;                            // two dims of the output are one store
  float scale;
};

constexpr int kMaxGroup = 8;                 // heads of a group: columns of a matrix instruction
template <int D> constexpr int kTileOf = D == 64 ? 64 : 32;  // positions of a tile: of 8 KB or more
inline int tile_of(int64_t dim) { return dim == 64 ? kTileOf<64> : kTileOf<128>; }
constexpr int kEntry = 2;                    // what the change to another item costs a warp, in tiles
constexpr int64_t kMaxContextHint = 1LL << 38;
// A maximum of nothing: finite, so that differences of two are numbers, and a score of -infinity is infinitely far below it.
constexpr float kNone = -3.0e38f;
constexpr float kNear = 1073741824.0f;  // 2^30: scales of V within that of their unit are near it
constexpr float kLeastWeight = -256.0f; // log2 of weights below which no result comes; no maximum of theirs is lower, which keeps its bits
constexpr float kWeightLog2 = 14.0f;  // the largest weight of a head in FP16 is 2^14 (SPLIT: up to 2^15)

// A stage: K rows, V rows (16-byte pieces xor-swizzled, so that eight rows of an ldmatrix lie on eight bank groups).
template <int D>
struct Stage {
  static constexpr int kStages = D == 256 ? 1 : 2;
  static constexpr int kRows = kTileOf<D> * D;
  static constexpr int kBytes = 2 * kRows;
  __device__ static __forceinline__ int at(int row, int piece) {
    if constexpr (D == 64) return row * D + ((piece ^ (row >> 1 & 3)) << 4);
    return row * D + ((piece ^ (row & 7)) << 4);
  }
};
template <int D> constexpr int ring_bytes() { return Stage<D>::kStages * Stage<D>::kBytes; }

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void prefetch_l1(const void* p) {  // a load that nobody waits for
  uint16_t unused;
  asm volatile("ld.global.u16 %0, [%1];" : "=h"(unused) : "l"(p));
}
__device__ __forceinline__ float log2_fast(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The matrix instructions without `volatile`, so that loads and products of a tile may pass each other; the caller keeps them
// between its barriers with pin().
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
template <bool TRANS> __device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t smem_row) {
  if constexpr (TRANS)
    asm("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_row));
  else
    asm("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_row));
}
__device__ __forceinline__ void pin(uint32_t& x) { asm volatile("" : "+r"(x)::"memory"); }
__device__ __forceinline__ void pin(float& x) { asm volatile("" : "+f"(x)); }
// Dims 4 quad .. + 3 of each of N pieces of 16, from `at` on.  One type and one branch for all of them, so that the loads go out together.
template <typename T, int N> __device__ __forceinline__ void load_quads(const T* at, bool vectors, float (&x)[N][4]) {
  if (vectors) {
#pragma unroll
    for (int c = 0; c < N; ++c) {
      if constexpr (sizeof(T) == 4) {
        const float4 v = *reinterpret_cast<const float4*>(at + c * 16);
        x[c][0] = v.x, x[c][1] = v.y, x[c][2] = v.z, x[c][3] = v.w;
      } else {
        const uint2 v = *reinterpret_cast<const uint2*>(at + c * 16);
        const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[c][i] = Elem<T>::to_f32(e[i]);
      }
    }
  } else {
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[c][i] = Elem<T>::to_f32(at[c * 16 + i]);
  }
}
__device__ __forceinline__ void store_from_f32(const PeerOut& out, int64_t row, int64_t col, float v, int dtype) {
  if (dtype == XDK_F32) peer_store(out, row, col, v);
  else if (dtype == XDK_BF16) peer_store(out, row, col, __float2bfloat16_rn(v));
  else peer_store(out, row, col, __float2half_rn(v));
}
// Dims 16 c and 16 c + 1 behind `col` of one row, c < N: value(c, 0) and value(c, 1).  `paired`: both in one store, everywhere.
template <bool WIDE, typename Value, typename N>
__device__ __forceinline__ void store_dims(const PeerOut& out, int64_t row, int64_t col, int dtype, bool paired, Value value, N) {
  const int64_t at = row * out.ld + out.col0 + col;
#pragma unroll 1
  for (int p = 0; p < out.world; ++p) {
    if constexpr (WIDE) {
      float* to = static_cast<float*>(out.ptr[p]) + at;
#pragma unroll
      for (int c = 0; c < N::value; ++c) {
        if (paired) *reinterpret_cast<float2*>(to + c * 16) = make_float2(value(c, 0), value(c, 1));
        else to[c * 16] = value(c, 0), to[c * 16 + 1] = value(c, 1);
      }
    } else {
      uint16_t* to = static_cast<uint16_t*>(out.ptr[p]) + at;
#pragma unroll
      for (int c = 0; c < N::value; ++c) {
        const uint32_t both = dtype == XDK_BF16 ? Mma16816<__nv_bfloat16>::pack(value(c, 0), value(c, 1)) : Mma16816<__half>::pack(value(c, 0), value(c, 1));
        if (paired) *reinterpret_cast<uint32_t*>(to + c * 16) = both;
        else to[c * 16] = static_cast<uint16_t>(both), to[c * 16 + 1] = static_cast<uint16_t>(both >> 16);
      }
    }
  }
}
// What the exponents of the weights are taken from for a maximum of `most`: kWeightLog2 below it, as far as a large one shows that; at most 15,
// so that no weight passes FP16.
__device__ __forceinline__ float weights_from(float most) {
  const float from = most - kWeightLog2;
  return most - from <= 15.0f ? from : most;
}
// The e of a scale that is not below 0 as 2^e * f, f in [1, 2), which takes its place; 0: 2^-infinity times 0, what is not finite: 2^0 times that.
__device__ __forceinline__ float split_scale(float& scale) {
  if (scale == 0.0f) return -INFINITY;
  if (!(scale < INFINITY)) return 0.0f;
  const bool small = scale < 7.8886091e-31f;  // 2^-100; below 2^-126 the exponent's bits do not tell it
  const uint32_t bits = __float_as_uint(small ? scale * 1.2676506e30f : scale);
  scale = __uint_as_float((bits & 0x7fffffu) | 0x3f800000u);
  return static_cast<float>(static_cast<int>(bits >> 23) - (small ? 227 : 127));
}

// ---- the line of tiles ---------------------------------------------------------------------------------------------------
// Token by token, its KV heads; to each kEntry units and one for every tile of the context (one dead tile for an empty one).  Only the
// device knows the contexts: each warp adds them up.  Warp b of B has the tiles among units [b U / B, (b + 1) U / B) of the U there are, B:
// the warps of the grid, or U if that is less.  (Without the entries a warp among contexts of a tile or two has nine of them to begin and
// to end: 64 contexts of 1 .. 2048 took 72 us then, 44 with them.  One unit to an
// entry: 37.6 against 38.0 there, but 88 against 76 for 16 contexts of 8192 with head_dim 64.)
struct Cursor {
  int token, kvh, tile, tiles;
  int64_t left;  // units of the warp from this tile on
};
template <bool SPARSE> __device__ __forceinline__ int tiles_of(const Kv8Args& a, int64_t context) {
  if (context <= 0) return 1;
  return static_cast<int>(((SPARSE ? a.n_pages * a.page_size : context) + a.tile - 1) / a.tile);
}
template <bool SPARSE> __device__ __forceinline__ int units_of(const Kv8Args& a, int token) {  // of one of its heads
  return token < a.tokens ? tiles_of<SPARSE>(a, a.positions[token] + 1) + kEntry : 0;
}
__device__ __forceinline__ int64_t divide(int64_t x, int64_t y) {  // of what is not below 0; in 32 bits where they do
  return ((x | y) >> 31) == 0 ? static_cast<uint32_t>(x) / static_cast<uint32_t>(y) : x / y;
}
// Whole warps call these.
__device__ __forceinline__ int64_t sum_upto(int64_t x) {  // over the lanes up to this one
#pragma unroll
  for (int sh = 1; sh < 32; sh <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, x, sh);
    if (static_cast<int>(threadIdx.x) >= sh) x += v;
  }
  return x;
}
// The units of the line; of the first 32 tokens lane t knows those of a head of token t, and of all heads of the tokens up to it.
struct Line {
  int units;
  int64_t upto, total;
};
template <bool SPARSE> __device__ __forceinline__ Line count_units(const Kv8Args& a) {
  Line l;
  l.units = units_of<SPARSE>(a, threadIdx.x);
  l.upto = sum_upto(static_cast<int64_t>(l.units) * a.kv_heads);
  l.total = __shfl_sync(0xffffffffu, l.upto, 31);
  if (a.tokens > 32) {
    int64_t further = 0;
#pragma unroll 4
    for (int t = threadIdx.x + 32; t < a.tokens; t += 32) further += units_of<SPARSE>(a, t);
#pragma unroll
    for (int sh = 16; sh > 0; sh >>= 1) further += __shfl_xor_sync(0xffffffffu, further, sh);
    l.total += further * a.kv_heads;
  }
  return l;
}
// The first tile among units [from, to), whose `left` is 0 if there is none.
template <bool SPARSE> __device__ __forceinline__ Cursor find_unit(const Kv8Args& a, const Line& line, int64_t from, int64_t to) {
  constexpr int kEach = 4;  // tokens of a lane at a time, behind the first 32 (one: 4096 tokens of 32 positions 19 us more)
  const int lane = threadIdx.x;
  Cursor c = {};
  int64_t at = from;  // of the units from token c.token on
  int each = 0;       // units of a head of that
  unsigned who = __ballot_sync(0xffffffffu, from < line.upto);
  if (who != 0) {
    c.token = __ffs(who) - 1;
    each = __shfl_sync(0xffffffffu, line.units, c.token);
    at -= __shfl_sync(0xffffffffu, line.upto, c.token) - static_cast<int64_t>(each) * a.kv_heads;
  } else {
    at -= __shfl_sync(0xffffffffu, line.upto, 31);
    for (int t0 = 32; t0 < a.tokens; t0 += 32 * kEach) {
      int units[kEach];
      int64_t mine = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) units[i] = units_of<SPARSE>(a, t0 + lane * kEach + i), mine += units[i];
      mine *= a.kv_heads;
      const int64_t upto = sum_upto(mine);
      who = __ballot_sync(0xffffffffu, at < upto);
      if (who == 0) {
        at -= __shfl_sync(0xffffffffu, upto, 31);
        continue;
      }
      const int src = __ffs(who) - 1, first = t0 + src * kEach;
      at -= __shfl_sync(0xffffffffu, upto - mine, src);
      c.token = first, each = __shfl_sync(0xffffffffu, units[0], src);
#pragma unroll
      for (int i = 1; i < kEach; ++i) {
        const int further = __shfl_sync(0xffffffffu, units[i], src);
        const int64_t of = static_cast<int64_t>(each) * a.kv_heads;
        if (c.token == first + i - 1 && at >= of) at -= of, each = further, ++c.token;
      }
      break;
    }
  }
  if (each == 0) return c;
  c.tiles = each - kEntry;
  c.kvh = static_cast<int>(divide(at, each));
  const int in = static_cast<int>(at - static_cast<int64_t>(c.kvh) * each) - kEntry;
  c.tile = in > 0 ? in : 0;
  c.left = to - from + (in < 0 ? in : 0);
  if (c.left < 0) c.left = 0;
  return c;
}
// On to the warp's next tile; `context(token)`: what a change of tokens takes.  0: there is none (left is 0), 1: of the same item, 2: of another.
template <bool SPARSE, typename Context> __device__ __forceinline__ int advance(const Kv8Args& a, Cursor& c, Context context) {
  ++c.tile, --c.left;
  if (c.left > 0 && c.tile < c.tiles) return 1;
  c.left -= kEntry;
  if (c.left <= 0) {
    c.left = 0;
    return 0;
  }
  c.tile = 0;
  if (++c.kvh == a.kv_heads) c.kvh = 0, c.tiles = tiles_of<SPARSE>(a, context(++c.token));
  return 2;
}

// Scratch of a grid of `warps`: slot 2 b + 1 is for the item that warp b begins and does not end, slot 2 b for one begun before
// it.  Results over the warp's positions [slots][group * dim], running maxima and sums [slots][8] of each; and `shares`, which the warp that begins an item
// writes.  By item: that warp and how many warps have a part of it.  By warp, where there are more items than warps: the item that it begins and
// does not end (there is one at most), and how many have a part of it, 1 if there is none.
struct Partials {
  float *acc, *m, *l;
  int2* shares;
  __device__ Partials(float* scratch, int warps, int values) {
    acc = scratch;
    m = acc + static_cast<size_t>(2 * warps) * values;
    l = m + static_cast<size_t>(2 * warps) * kMaxGroup;
    shares = reinterpret_cast<int2*>(l + static_cast<size_t>(2 * warps) * kMaxGroup);
  }
};
constexpr size_t partial_bytes(size_t warps, size_t items, size_t values) { return 2 * warps * (values + 2 * kMaxGroup) * 4 + items * 8; }

template <typename C, int D, bool SPLIT, bool SPARSE>
__global__ void __launch_bounds__(32, D == 256 ? 8 : 12)
kv8_attention_kernel(const __grid_constant__ Kv8Args a, const __grid_constant__ PeerOut out) {
  using St = Stage<D>;
  constexpr int TP = kTileOf<D>, R = TP / 32;  // R: rows that a lane looks up
  constexpr int PB = TP / 16, NC = D / 16, NST = St::kStages;  // PB: blocks of 16 positions, NC: pieces of 16 dims
  constexpr int NQ = SPLIT ? 2 : 1;  // FP16 numbers to a value of q (SPLIT: FP32) or weight
  constexpr bool CENTRED = SPLIT;    // FP32 results would see what an offset of the codes cancels
  extern __shared__ __align__(128) unsigned char ring[];
  __shared__ int64_t rows[TP];     // byte offsets of the rows that are fetched
  __shared__ float4 per_row[TP];   // of a tile's positions: scale of K; of V as `far` takes it
  __shared__ float s_max[kMaxGroup];  // see `far`

  pdl_launch_dependents();
  pdl_wait();  // q and the caches are the preceding kernels' output
  const int lane = threadIdx.x;
  const int grow = lane >> 2, quad = lane & 3;
  const int G = a.group;
  if (lane < a.tokens) prefetch_l1(a.sequence_ids + lane);  // needed once the token is known
  if (a.by_warp && lane == 0) Partials(a.scratch, gridDim.x, G * D).shares[blockIdx.x] = make_int2(0, 1);
  const Line line = count_units<SPARSE>(a);
  const int64_t total = line.total, warps = total < gridDim.x ? total : gridDim.x;
  if (blockIdx.x >= warps) return;
  const int64_t end_unit = divide(total * (blockIdx.x + 1), warps);
  Cursor cur = find_unit<SPARSE>(a, line, divide(total * blockIdx.x, warps), end_unit);  // the tile that is computed next
  if (cur.left == 0) return;
  Cursor next = cur;  // the tile that is fetched next, and what its rows are found by
  int64_t ctx = 0, coming_ctx = 0, coming_seq = 0;  // of the token, and of the one behind it
  const int64_t* table = nullptr;
  const int32_t* list = nullptr;
  auto glance = [&]() {  // at the token behind
    if (next.token + 1 < a.tokens) coming_ctx = a.positions[next.token + 1] + 1, coming_seq = a.sequence_ids[next.token + 1];
  };
  auto enter = [&](bool other_token) {
    if (other_token) {
      ctx = coming_ctx, table = a.page_table + coming_seq * a.max_pages;
      glance();
    }
    if constexpr (SPARSE) list = a.pages + (static_cast<int64_t>(next.token) * a.kv_heads + next.kvh) * a.n_pages;
    // q of the item, which is loaded when its first tile is computed, on its way to L1
    const int bytes = G * D * (SPLIT ? 4 : 2);
    const unsigned char* at = static_cast<const unsigned char*>(a.q) + (static_cast<int64_t>(next.token) * a.q_heads + next.kvh * G) * (D * (SPLIT ? 4 : 2));
    for (int i = lane * 128; i < bytes; i += 32 * 128) prefetch_l1(at + i);
  };
  int64_t page[R];  // of this lane's rows of it, -1: dead
  int off[R];
  auto look_up = [&]() {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      page[r] = -1, off[r] = 0;
      if constexpr (!SPARSE) {
        const int64_t i = static_cast<int64_t>(next.tile) * TP + r * 32 + lane;
        if (i < ctx) {
          const int64_t logical = a.narrow ? static_cast<uint32_t>(i) / static_cast<uint32_t>(a.page_size) : i / a.page_size;
          off[r] = static_cast<int>(i - logical * a.page_size);
          page[r] = table[logical];
        }
      } else {
        const uint32_t i = static_cast<uint32_t>(next.tile) * TP + r * 32 + lane;  // of at most 2^31 positions
        const int entry = static_cast<int>(i / static_cast<uint32_t>(a.page_size));
        if (entry < a.n_pages && ctx > 0) {
          const int64_t logical = list[entry];
          off[r] = static_cast<int>(i) - entry * static_cast<int>(a.page_size);
          // the list ascends: an entry that does not (a second one of a page) is not read
          if (logical >= 0 && (entry == 0 || list[entry - 1] < logical) && logical * a.page_size + off[r] < ctx) page[r] = table[logical];
        }
      }
    }
  };
  const uint8_t *k_lane = a.k_cache + lane % NC * 16, *v_lane = a.v_cache + lane % NC * 16;
  float ks[NST][R], vs[NST][R];  // scales of this lane's positions in the tiles on their way, oldest first; -1: dead
  auto fetch = [&](int stage, float (&k_scale)[R], float (&v_scale)[R]) {  // tile `next` into a stage
    unsigned char* st = ring + stage * St::kBytes;
    const int kvh = next.kvh;
    bool all_live = true;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool live = page[r] >= 0;
      all_live = all_live && live;
      const int64_t block = live ? page[r] * a.kv_heads + kvh : 0;
      rows[r * 32 + lane] = live ? (a.hnd ? block * a.page_size + off[r] : (page[r] * a.page_size + off[r]) * a.kv_heads + kvh) * D : -1;
      k_scale[r] = live ? a.k_scale[block] : 0.0f;
      v_scale[r] = live ? a.v_scale[block] : -1.0f;
    }
    constexpr int kAtOnce = 32 / NC;  // rows of NC pieces
    if (__all_sync(0xffffffffu, all_live)) {
      __syncwarp();
#pragma unroll
      for (int i = 0; i < TP / kAtOnce; ++i) {
        const int r = i * kAtOnce + lane / NC;
        const int64_t from = rows[r];
        cp_async16(st + St::at(r, lane % NC), k_lane + from);
        cp_async16(st + St::kRows + St::at(r, lane % NC), v_lane + from);
      }
    } else {
      __syncwarp();
#pragma unroll
      for (int i = 0; i < TP / kAtOnce; ++i) {
        const int r = i * kAtOnce + lane / NC;
        const int64_t from = rows[r];
        const bool there = from >= 0;
        cp_async16_or_zero(st + St::at(r, lane % NC), k_lane + (there ? from : 0), there);
        cp_async16_or_zero(st + St::kRows + St::at(r, lane % NC), v_lane + (there ? from : 0), there);
      }
    }
    __syncwarp();  // rows is free again
  };
  auto fetch_next = [&](int stage, float (&k_scale)[R], float (&v_scale)[R]) {  // one group per call, whether or not there is a tile left
    if (next.left > 0) {
      fetch(stage, k_scale, v_scale);
      const int step = advance<SPARSE>(a, next, [&](int) { return coming_ctx; });
      if (step == 2) enter(next.kvh == 0);
      if (step != 0) look_up();  // the page of the row after that is on its way meanwhile
    }
    cp_async_commit();
  };
  coming_ctx = a.positions[next.token] + 1, coming_seq = a.sequence_ids[next.token];
  enter(true);
  look_up();
#pragma unroll
  for (int s = 0; s < NST - 1; ++s) fetch_next(s, ks[s], vs[s]);
  const uint32_t ring_at = smem_u32(ring);
  int stage = 0;

  for (;;) {  // the warp's part of one item after the other
  const int token = cur.token, kvh = cur.kvh, first = cur.tile;
  const int end = cur.tiles - first < cur.left ? cur.tiles : first + static_cast<int>(cur.left);
  float x[NC][4];  // q: dims 16 c + 4 quad .. of head grow
  const bool head_live = grow < G;
  {
    const int64_t qrow = (static_cast<int64_t>(token) * a.q_heads + kvh * G + (head_live ? grow : 0)) * D + quad * 4;
    const bool vectors = (reinterpret_cast<uintptr_t>(a.q) & 15) == 0;
    if constexpr (SPLIT) load_quads(static_cast<const float*>(a.q) + qrow, vectors, x);
    else if (a.dtype == XDK_BF16) load_quads(static_cast<const __nv_bfloat16*>(a.q) + qrow, vectors, x);
    else load_quads(static_cast<const __half*>(a.q) + qrow, vectors, x);
  }
  uint32_t qb[NQ][NC][2];  // q^T as B fragments: dims 16 c + 4 quad + {0,1}, {2,3} of head grow
  float unit[2];           // of the scores of heads 2 quad + {0, 1}: scale * log2(e) * the power of two that q was divided by
  // Codes that are not centred are multiples of kUnit, by which the units of the scores are divided, or, beside a q above 2^37, the scales of
  // K are multiplied: the quotient of either would not always be finite, and beside such a q a scale of K above 2^104 gives no finite score.
  constexpr float kPerUnit = CENTRED ? 1.0f : 1.0f / Codec<C>::kUnit;
  float k_lift = 1.0f;
  {
    float top = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (!head_live) x[c][e] = 0.0f;
        top = fmaxf(top, fabsf(x[c][e]));
      }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int exponent = static_cast<int>(__float_as_uint(top) >> 23) - 127;
    int up = 13 - exponent;  // largest value in [2^13, 2^14)
    up = up > 126 ? 126 : up;
    const float by = __int_as_float((up + 127) << 23), back = __int_as_float((127 - up) << 23);
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float x0 = x[c][2 * h] * by, x1 = x[c][2 * h + 1] * by;
        const __half2 hi = __floats2half2_rn(x0, x1);
        qb[0][c][h] = *reinterpret_cast<const uint32_t*>(&hi);
        if constexpr (SPLIT) {
          const float2 f = __half22float2(hi);
          qb[NQ - 1][c][h] = Mma16816<__half>::pack(x0 - f.x, x1 - f.y);
        }
      }
    float per_unit = a.scale * 1.4426950408889634f;
    if constexpr (kPerUnit != 1.0f) {
      if (__any_sync(0xffffffffu, exponent > 36)) k_lift = kPerUnit;
      else per_unit *= kPerUnit;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) unit[e] = __shfl_sync(0xffffffffu, back, (2 * quad + e) * 4) * per_unit;
  }
  float s_zero[2] = {0.0f, 0.0f};  // what a score begins with: codes that are not centred add kOffset * q
  if constexpr (!CENTRED && Codec<C>::kOffset != 0.0f) {
    float sum = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&qb[0][c][h]));
        sum += f.x + f.y;
      }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
    for (int e = 0; e < 2; ++e) s_zero[e] = -Codec<C>::kOffset * Codec<C>::kUnit * __shfl_sync(0xffffffffu, sum, (2 * quad + e) * 4);
  }
  // Scales of V are taken in units of v_unit, the power of two of the largest in the first tile, as long as all of them are near it.  Of heads
  // 2 quad + {0, 1}: w_run, the running maximum of s + log2(vs / v_unit), in units of log2, which makes the largest weight 2^kWeightLog2, and this
  // thread's share of the sum of the softmax weights, l_run: the weights with vs / v_unit taken out again.
  // far (v_unit is 0): from the first tile on that has a scale that is not near it, 0 among them, the sum is that of 2^(s - s_max), s_max the
  // running maximum of s, and w_run that of (s - s_max) + log2 vs (SPLIT: the exponent of vs, whose significand is a factor then).
  float w_run[2], l_run[2], v_unit = 1.0f;
  float o[NC][4];  // O^T: dims 16 c + 2 grow (+ 1 in the upper two), the same heads
#pragma unroll
  for (int e = 0; e < 2; ++e) w_run[e] = kNone, l_run[e] = 0.0f;
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[c][e] = 0.0f;

  // rows pb * 16 + lane % 16, pieces c + lane / 16 of an even c: offsets that the stage and pb are added to
  uint32_t at_piece[NC / 2];
#pragma unroll
  for (int c = 0; c < NC; c += 2) at_piece[c / 2] = St::at(lane & 15, c + (lane >> 4));

  for (int u = first; u < end; ++u) {
    fetch_next(stage == 0 ? NST - 1 : stage - 1, ks[NST - 1], vs[NST - 1]);
    if (u == first) {
      float most = vs[0][0];
#pragma unroll
      for (int r = 1; r < R; ++r) most = fmaxf(most, vs[0][r]);
#pragma unroll
      for (int sh = 16; sh > 0; sh >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, sh));
      if (most > 1e-37f && most < 8e37f) v_unit = __uint_as_float(__float_as_uint(most) & 0x7f800000u);  // 2^-123 .. 2^125
    }
    const float to_unit = __uint_as_float(0x7f000000u - __float_as_uint(v_unit));  // one over it
    bool leaves = false;
#pragma unroll
    for (int r = 0; r < R; ++r) {  // not NaN, which shows either way
      const float rel = vs[0][r] * to_unit;
      leaves = leaves || (rel >= 0.0f && !(rel >= 1.0f / kNear && rel <= kNear));
    }
    if (v_unit != 0.0f && __any_sync(0xffffffffu, leaves)) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {  // l_run is a sum of 2^(s - weights_from(w_run)) so far
        const bool none = w_run[e] == kNone;
        if (grow == 0) s_max[2 * quad + e] = none ? kNone : weights_from(w_run[e]);
        w_run[e] = none ? kLeastWeight : static_cast<float>(static_cast<int>(__float_as_uint(v_unit) >> 23) - 127) + kWeightLog2;
      }
      v_unit = 0.0f;
    }
    const bool far = v_unit == 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool live = !(vs[0][r] < 0.0f);  // NaN is alive
      float4& of = per_row[r * 32 + lane];
      if (!far) {  // log2 (-infinity: dead) and one over it
        const float in_exponent = log2_fast(vs[0][r] * to_unit);
        of = make_float4(ks[0][r] * k_lift, live ? in_exponent : -INFINITY, live ? exp2_fast(-in_exponent) : 0.0f, 0.0f);
      } else {  // 0 (-infinity: dead), significand, and logarithm (SPLIT: exponent)
        float significand = live ? vs[0][r] : 0.0f, exponent = split_scale(significand);
        if constexpr (!SPLIT) exponent += live ? log2_fast(significand) : 0.0f;
        of = make_float4(ks[0][r] * k_lift, live ? 0.0f : -INFINITY, significand, exponent);
      }
#pragma unroll
      for (int s = 0; s < NST - 1; ++s) ks[s][r] = ks[s + 1][r], vs[s][r] = vs[s + 1][r];
    }
    cp_async_wait<NST - 1>();
    __syncwarp();
    uint32_t kt = ring_at + stage * St::kBytes;
    pin(kt);
    const uint32_t vt = kt + St::kRows;

    // ---- S^T = K q^T: per load, rows 0-7 and 8-15 of a block and two pieces
    float sc[PB][4];  // positions 16 pb + grow (+ 8 in the upper two), heads 2 quad + {0, 1}
#pragma unroll
    for (int pb = 0; pb < PB; ++pb)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[pb][e] = s_zero[e & 1];
#pragma unroll
    for (int c = 0; c < NC; c += 2)
#pragma unroll
      for (int pb = 0; pb < PB; ++pb) {
        uint32_t raw[4];
        load_matrices<false>(raw, kt + at_piece[c / 2] + pb * 16 * D);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t k[4];
          Codec<C>::template neighbours<CENTRED>(raw[2 * h], k[0], k[2]);
          Codec<C>::template neighbours<CENTRED>(raw[2 * h + 1], k[1], k[3]);
#pragma unroll
          for (int n = 0; n < NQ; ++n) mma(sc[pb], k, qb[n][c + h]);
        }
      }
    // ---- online softmax of the two heads
    uint32_t wb[NQ][PB][2];  // w^T as B fragments: positions 16 pb + 2 quad + {0,1} (+ 8 in [1]), head grow
    float corr[2], t_zero[2] = {0.0f, 0.0f};  // what o takes for the new maximum; as s_zero: kOffset * the tile's weights
    auto over_lanes = [&](float most) {
#pragma unroll
      for (int sh = 4; sh < 32; sh <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, sh));
      return most;
    };
    auto put_weights = [&](int pb, int r, float x0, float x1) {
      const __half2 hi = __floats2half2_rn(x0, x1);
      wb[0][pb][r] = transpose8x8(*reinterpret_cast<const uint32_t*>(&hi));
      if constexpr (SPLIT || Codec<C>::kOffset != 0.0f) {
        const float2 h = __half22float2(hi);
        if constexpr (SPLIT) wb[NQ - 1][pb][r] = transpose8x8(Mma16816<__half>::pack(x0 - h.x, x1 - h.y));
        else t_zero[0] += h.x, t_zero[1] += h.y;
      }
    };
    if (!far) {
      float mw[2] = {w_run[0], w_run[1]}, take_out[PB][2];
#pragma unroll
      for (int pb = 0; pb < PB; ++pb)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float4 f = per_row[pb * 16 + grow + r * 8];
          take_out[pb][r] = f.z;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& s = sc[pb][2 * r + e];
            s = fmaf(s, f.x * unit[e], f.y);
            mw[e] = fmaxf(mw[e], s);
          }
        }
      float from[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mw[e] = over_lanes(mw[e]);
        from[e] = weights_from(mw[e]);
        corr[e] = exp2_fast(weights_from(w_run[e]) - from[e]);
        w_run[e] = mw[e];
        l_run[e] *= corr[e];
      }
#pragma unroll
      for (int pb = 0; pb < PB; ++pb)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float x0 = exp2_fast(sc[pb][2 * r] - from[0]), x1 = exp2_fast(sc[pb][2 * r + 1] - from[1]);
          l_run[0] = fmaf(x0, take_out[pb][r], l_run[0]), l_run[1] = fmaf(x1, take_out[pb][r], l_run[1]);
          put_weights(pb, r, x0, x1);
        }
    } else {
      float ms[2] = {s_max[2 * quad], s_max[2 * quad + 1]}, mw[2];
      const float before[2] = {ms[0], ms[1]};
#pragma unroll
      for (int pb = 0; pb < PB; ++pb)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float4 f = per_row[pb * 16 + grow + r * 8];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& s = sc[pb][2 * r + e];
            s = fmaf(s, f.x * unit[e], f.y);
            ms[e] = fmaxf(ms[e], s);
          }
        }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        ms[e] = over_lanes(ms[e]);
        if (grow == 0) s_max[2 * quad + e] = ms[e];  // all lanes have read it: the shuffles stand between
        const float back = before[e] - ms[e];
        l_run[e] *= exp2_fast(back);
        corr[e] = back + w_run[e];
        mw[e] = fmaxf(corr[e], kLeastWeight);
      }
#pragma unroll
      for (int pb = 0; pb < PB; ++pb)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float in_exponent = per_row[pb * 16 + grow + r * 8].w;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& s = sc[pb][2 * r + e];
            s -= ms[e];
            l_run[e] += exp2_fast(s);
            s += in_exponent;
            mw[e] = fmaxf(mw[e], s);
          }
        }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        w_run[e] = over_lanes(mw[e]);
        corr[e] = exp2_fast(corr[e] - w_run[e]);
      }
#pragma unroll
      for (int pb = 0; pb < PB; ++pb)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float factor = SPLIT ? per_row[pb * 16 + grow + r * 8].z : 1.0f;
          put_weights(pb, r, exp2_fast(sc[pb][2 * r] - (w_run[0] - kWeightLog2)) * factor, exp2_fast(sc[pb][2 * r + 1] - (w_run[1] - kWeightLog2)) * factor);
        }
    }
    if constexpr (!CENTRED && Codec<C>::kOffset != 0.0f) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int sh = 4; sh < 32; sh <<= 1) t_zero[e] += __shfl_xor_sync(0xffffffffu, t_zero[e], sh);
        t_zero[e] *= -Codec<C>::kOffset * Codec<C>::kUnit;
      }
    }
    // ---- O^T += V^T w^T: per load, position halves of a block and two pieces
#pragma unroll
    for (int c = 0; c < NC; c += 2) {
      float t[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) t[h][e] = t_zero[e & 1];
#pragma unroll
      for (int pb = 0; pb < PB; ++pb) {
        uint32_t raw[4];
        load_matrices<true>(raw, vt + at_piece[c / 2] + pb * 16 * D);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t v[4];
          Codec<C>::template alternate<CENTRED>(raw[2 * h], v[0], v[1]);
          Codec<C>::template alternate<CENTRED>(raw[2 * h + 1], v[2], v[3]);
#pragma unroll
          for (int n = 0; n < NQ; ++n) mma(t[h], v, wb[n][pb]);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          o[c + h][e] = fmaf(o[c + h][e], corr[e & 1], t[h][e]);
          pin(o[c + h][e]);
        }
    }
    __syncwarp();  // every lane has read the tile
    stage = stage + 1 == NST ? 0 : stage + 1;
  }

  // ---- the result, or this warp's share of it
  const bool whole = first == 0 && end == cur.tiles;
  constexpr float kValueUnit = CENTRED ? 1.0f : 1.0f / Codec<C>::kUnit;
  const Partials part(a.scratch, gridDim.x, G * D);
  const size_t slot = 2 * static_cast<size_t>(blockIdx.x) + (first == 0 ? 1 : 0);
  if (first == 0 && lane == 0) {  // an item that others go on with ends cur.tiles - end units behind this warp's share
    const int last = whole ? blockIdx.x : static_cast<int>(((end_unit + cur.tiles - end) * warps - 1) / total);
    const int item = token * a.kv_heads + kvh, count = last - blockIdx.x + 1;
    if (!a.by_warp) part.shares[item] = make_int2(blockIdx.x, count);
    else if (!whole) part.shares[blockIdx.x] = make_int2(item, count);
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
#pragma unroll
    for (int sh = 4; sh < 32; sh <<= 1) l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], sh);
    const int head = quad * 2 + e;
    if (head >= G) continue;
    // o / l, then the unit of V; far: 2^(w_run - kWeightLog2), in two halves.  In turn, which keeps what is on the way in range.
    const float each = l_run[e] == 0.0f ? 0.0f : 1.0f / l_run[e] * kValueUnit;
    float value_unit = v_unit, m = weights_from(w_run[e]);
    if (v_unit == 0.0f) {
      value_unit = exp2_fast(0.5f * (w_run[e] - kWeightLog2)), m = s_max[head];
#pragma unroll
      for (int c = 0; c < NC; ++c) o[c][e] *= value_unit, o[c][e + 2] *= value_unit;
    }
    auto value = [&](int c, int i) { return o[c][e + 2 * i] * each * value_unit; };
    if (whole) {
      store_dims<SPLIT>(out, token, static_cast<int64_t>(kvh * G + head) * D + 2 * grow, a.dtype, a.paired, value, std::integral_constant<int, NC>());
    } else {
      float* to = part.acc + (slot * G + head) * D + 2 * grow;
#pragma unroll
      for (int c = 0; c < NC; ++c) *reinterpret_cast<float2*>(to + c * 16) = make_float2(value(c, 0), value(c, 1));
      if (grow == 0) {
        part.m[slot * kMaxGroup + head] = m;
        part.l[slot * kMaxGroup + head] = l_run[e];
      }
    }
  }
  cur.left -= end - 1 - first, cur.tile = end - 1;
  if (advance<SPARSE>(a, cur, [&](int t) { return a.positions[t] + 1; }) == 0) return;
  }
}

// Of one head: the result of some positions, and the sum of their softmax weights, l, in units of 2^m.
struct Part {
  float4 value;
  float m, l;
};
// Adds N parts to a sum of parts.  The values enter with their shares of all weights, so that they pass no range that the result does not; a
// share has its power of two in two halves, as a large value counts with one below 2^-126 where all others are as small.
template <int N> __device__ __forceinline__ void add_parts(Part& sum, const Part (&p)[N]) {
  float m = sum.m;
#pragma unroll
  for (int i = 0; i < N; ++i) m = fmaxf(m, p[i].m);
  const float had = exp2_fast(0.5f * (sum.m - m));
  float half[N], l = sum.l * had * had;
#pragma unroll
  for (int i = 0; i < N; ++i) half[i] = exp2_fast(0.5f * (p[i].m - m)), l += p[i].l * half[i] * half[i];
  const float per = l == 0.0f ? 0.0f : 1.0f / l;
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  auto add = [&](const Part& part, float h) {
    const float share = part.l * per * h;
    v.x = fmaf(part.value.x * h, share, v.x), v.y = fmaf(part.value.y * h, share, v.y);
    v.z = fmaf(part.value.z * h, share, v.z), v.w = fmaf(part.value.w * h, share, v.w);
  };
  add(sum, had);
#pragma unroll
  for (int i = 0; i < N; ++i) add(p[i], half[i]);
  sum = {v, m, l};
}

// Adds the parts of an item, one for each entry of `shares`: L lanes of four values each to a CTA, the THREADS / L groups of them every so
// many parts, two at a time; the groups' sums meet in shared memory.  Always in the same order.  L: a warp where there are few items, so that many CTAs
// share an item; else what the group * dim values take, at most all threads.
template <int L, int THREADS>
__global__ void __launch_bounds__(THREADS)
kv8_attention_merge_kernel(const __grid_constant__ Kv8Args a, const __grid_constant__ PeerOut out, int dim, int grid) {
  constexpr int kGroups = THREADS / L, N = 2;
  __shared__ float4 accs[kGroups][L];
  __shared__ float ms[kGroups][L], ls[kGroups][L];
  pdl_launch_dependents();
  pdl_wait();
  const int group = threadIdx.x / L, lane = threadIdx.x - group * L;
  const int all = a.group * dim, at = (blockIdx.y * L + lane) * 4;  // dim is a multiple of 64: four values of one head
  const Partials part(a.scratch, grid, all);
  const int2 share = __ldcg(part.shares + blockIdx.x);
  if (share.y == 1) return;  // the same for all threads
  const int item = a.by_warp ? share.x : blockIdx.x, begins = a.by_warp ? blockIdx.x : share.x;
  const bool some = at < all;
  const int head = some ? at / dim : 0;
  const Part none = {make_float4(0.0f, 0.0f, 0.0f, 0.0f), kNone, 0.0f};
  Part sum = none, p[N];
#pragma unroll 1
  for (int first = group; first < share.y; first += kGroups * N) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int i = first + k * kGroups;
      const size_t slot = 2 * static_cast<size_t>(begins + i) + (i == 0 ? 1 : 0);
      p[k] = none;
      if (some && i < share.y) {
        p[k].value = __ldcg(reinterpret_cast<const float4*>(part.acc + slot * all + at));
        p[k].m = __ldcg(part.m + slot * kMaxGroup + head), p[k].l = __ldcg(part.l + slot * kMaxGroup + head);
      }
    }
    add_parts(sum, p);
  }
  if constexpr (kGroups > 1) {
    accs[group][lane] = sum.value, ms[group][lane] = sum.m, ls[group][lane] = sum.l;
    __syncthreads();
    if (group != 0) return;
    constexpr int kRest = kGroups < 8 ? kGroups : 8;
    sum = none;
#pragma unroll
    for (int first = 0; first < kGroups; first += kRest) {
      Part q[kRest];
#pragma unroll
      for (int k = 0; k < kRest; ++k) q[k] = {accs[first + k][lane], ms[first + k][lane], ls[first + k][lane]};
      add_parts(sum, q);
    }
  }
  if (!some) return;
  const int token = item / a.kv_heads, kvh = item - token * a.kv_heads;
  const int64_t col = static_cast<int64_t>(kvh) * all + at;
  store_from_f32(out, token, col, sum.value.x, a.dtype);
  store_from_f32(out, token, col + 1, sum.value.y, a.dtype);
  store_from_f32(out, token, col + 2, sum.value.z, a.dtype);
  store_from_f32(out, token, col + 3, sum.value.w, a.dtype);
}

// ---- host --------------------------------------------------------------------------------------------------------------

// Warps of a launch: what the SMs hold at once, by the shared memory of a CTA (and 1 KB reserved) and the launch bounds, and no more than
// leaves every one as many tiles as the busiest has anyway, if no context has more than `tiles`.
int grid_for(int64_t items, int64_t dim, int64_t tiles) {
  const int ring = (dim == 64 ? ring_bytes<64>() : (dim == 128 ? ring_bytes<128>() : ring_bytes<256>())) + tile_of(dim) * 24 + 1024;
  const int by_smem = 228 * 1024 / ring, by_regs = dim == 256 ? 8 : 12;
  const int64_t most = static_cast<int64_t>(by_smem < by_regs ? by_smem : by_regs) * sm_count();
  if (tiles > most) return static_cast<int>(most);
  const int64_t all = items * ((tiles < 1 ? 1 : tiles) + kEntry), warps = all < most ? all : most, each = (all + warps - 1) / warps;
  return static_cast<int>((all + each - 1) / each);
}
int64_t hint_tiles(int64_t context, int64_t dim) {
  return ((context < 1 || context > kMaxContextHint ? kMaxContextHint : context) + tile_of(dim) - 1) / tile_of(dim);
}

template <typename C, int D, bool SPLIT, bool SPARSE>
int launch_kv8(Kv8Args a, const PeerOut& out, int warps, cudaStream_t s) {
  const int items = a.tokens * a.kv_heads, lanes = a.group * D / 4;
  a.by_warp = items > warps;
  if (int st = launch_dependent(kv8_attention_kernel<C, D, SPLIT, SPARSE>, dim3(static_cast<unsigned>(warps)), dim3(32), ring_bytes<D>(), s, a, out))
    return st;
  const int entries = a.by_warp ? warps : items;
  auto merge = [&](auto kernel, int l, int threads) {
    return launch_opts(kernel, dim3(static_cast<unsigned>(entries), static_cast<unsigned>((lanes + l - 1) / l)), dim3(threads), 0, s, 1u, true, a, out, D,
                       warps);
  };
  // at most one CTA to an SM: of 512 threads, sixteen groups (one context of 8192, 130 parts a head: 15.9 -> 13.9 us when both had one part at a
  // time; in more CTAs than that 256 threads are faster, 57.5 against 58.9 for 16 of them)
  if (entries * ((lanes + 31) / 32) <= sm_count()) return merge(kv8_attention_merge_kernel<32, 512>, 32, 512);
  if (entries <= sm_count() || lanes <= 32) return merge(kv8_attention_merge_kernel<32, 256>, 32, 256);
  return lanes <= 128 ? merge(kv8_attention_merge_kernel<128, 256>, 128, 256) : merge(kv8_attention_merge_kernel<256, 256>, 256, 256);
}

template <typename C, bool SPARSE>
int dispatch_kv8(int64_t d, const Kv8Args& a, const PeerOut& out, int warps, cudaStream_t s) {
  const bool split = a.dtype == XDK_F32;
  switch (d) {
    case 64: return split ? launch_kv8<C, 64, true, SPARSE>(a, out, warps, s) : launch_kv8<C, 64, false, SPARSE>(a, out, warps, s);
    case 128: return split ? launch_kv8<C, 128, true, SPARSE>(a, out, warps, s) : launch_kv8<C, 128, false, SPARSE>(a, out, warps, s);
    case 256: return split ? launch_kv8<C, 256, true, SPARSE>(a, out, warps, s) : launch_kv8<C, 256, false, SPARSE>(a, out, warps, s);
    default: return XDK_ERR_LIMIT;
  }
}

// The checks and the arguments that both entry points share.
int kv8_arguments(const void* q, const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                  const int64_t* positions, const int64_t* page_table, const int64_t* sequence_ids, const xdk_peer_out* out_dst,
                  int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t max_pages, int64_t page_size, int hnd,
                  float scale, int dtype, int codes, unsigned flags, Kv8Args* a, PeerOut* out) {
  if (int st = make_out(out_dst, nullptr, 1, out)) return st;
  if (flags & ~XDK_DEPENDENT_LAUNCH) return XDK_ERR_ARG;
  if (!q || !k_cache || !v_cache || !k_scale || !v_scale || !positions || !page_table || !sequence_ids) return XDK_ERR_ARG;
  if (tokens < 1 || q_heads < 1 || kv_heads < 1 || head_dim < 1 || max_pages < 1 || page_size < 1) return XDK_ERR_ARG;
  if (q_heads % kv_heads != 0 || !isfinite(scale) || out->ld < out->col0 + q_heads * head_dim) return XDK_ERR_ARG;
  if (!aligned16(k_cache) || !aligned16(v_cache)) return XDK_ERR_ARG;
  if (dtype != XDK_F32 && dtype != XDK_BF16 && dtype != XDK_F16) return XDK_ERR_ARG;
  if (codes != XDK_KV8_INT8 && codes != XDK_KV8_E4M3) return XDK_ERR_ARG;
  if (!kv8_head_dim(head_dim) || q_heads / kv_heads > kMaxGroup || tokens > 65535 || tokens * kv_heads > (1 << 26)) return XDK_ERR_LIMIT;
  if (int st = kv8_limits(tokens, kv_heads, max_pages, page_size)) return st;
  *a = {};
  a->q = q, a->k_cache = static_cast<const uint8_t*>(k_cache), a->v_cache = static_cast<const uint8_t*>(v_cache);
  a->k_scale = k_scale, a->v_scale = v_scale;
  a->positions = positions, a->page_table = page_table, a->sequence_ids = sequence_ids;
  a->max_pages = max_pages, a->page_size = page_size;
  a->tokens = static_cast<int>(tokens), a->q_heads = static_cast<int>(q_heads), a->kv_heads = static_cast<int>(kv_heads);
  a->group = static_cast<int>(q_heads / kv_heads), a->dtype = dtype;
  a->hnd = hnd ? 1 : 0;
  a->narrow = page_size * max_pages < (1LL << 31) ? 1 : 0;
  a->scale = scale;
  a->paired = out->ld % 2 == 0 && out->col0 % 2 == 0;
  for (int p = 0; p < out->world; ++p) a->paired &= reinterpret_cast<uintptr_t>(out->ptr[p]) % (dtype == XDK_F32 ? 8 : 4) == 0;
  a->tile = tile_of(head_dim);
  return XDK_OK;
}
size_t scratch_for(int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t tiles) {
  if (tokens < 1 || tokens > 65535 || kv_heads < 1 || kv_heads > 65535 || q_heads < kv_heads || q_heads % kv_heads != 0) return 0;
  if (q_heads / kv_heads > kMaxGroup || !kv8_head_dim(head_dim) || tokens * kv_heads > (1 << 26)) return 0;
  return partial_bytes(static_cast<size_t>(grid_for(tokens * kv_heads, head_dim, tiles)), static_cast<size_t>(tokens * kv_heads),
                       static_cast<size_t>(q_heads / kv_heads * head_dim));
}

}  // namespace

}  // namespace xdk

extern "C" size_t xdk_kv8_decode_attention_scratch_bytes(int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                                         int64_t context_hint) {
  return xdk::scratch_for(tokens, q_heads, kv_heads, head_dim, xdk::hint_tiles(context_hint, head_dim));
}
extern "C" size_t xdk_kv8_sparse_attention_scratch_bytes(int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                                         int64_t page_size, int64_t n_pages) {
  if (page_size < 1 || n_pages < 1 || page_size > xdk::kKV8MaxPage || n_pages > 2147483647LL / xdk::kKV8MaxPage) return 0;
  return xdk::scratch_for(tokens, q_heads, kv_heads, head_dim, xdk::hint_tiles(n_pages * page_size, head_dim));
}

extern "C" int xdk_kv8_decode_attention(const void* q, const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                                        const int64_t* positions, const int64_t* page_table, const int64_t* sequence_ids,
                                        const xdk_peer_out* out_dst, int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                        int64_t max_pages_per_seq, int64_t page_size, int cache_is_hnd, float scale, int64_t context_hint,
                                        int dtype, int codes, void* scratch, size_t scratch_bytes, unsigned flags, void* stream) {
  using namespace xdk;
  Kv8Args a;
  PeerOut out;
  if (int st = kv8_arguments(q, k_cache, v_cache, k_scale, v_scale, positions, page_table, sequence_ids, out_dst, tokens, q_heads, kv_heads,
                             head_dim, max_pages_per_seq, page_size, cache_is_hnd, scale, dtype, codes, flags, &a, &out))
    return st;
  if (!scratch || !aligned16(scratch) ||
      scratch_bytes < xdk_kv8_decode_attention_scratch_bytes(tokens, q_heads, kv_heads, head_dim, context_hint))
    return XDK_ERR_ARG;
  if (int st = require_sm100()) return st;
  CallFlagsScope scope(flags);
  a.scratch = static_cast<float*>(scratch);
  const int warps = grid_for(tokens * kv_heads, head_dim, hint_tiles(context_hint, head_dim));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return codes == XDK_KV8_INT8 ? dispatch_kv8<Int8Codes, false>(head_dim, a, out, warps, s) : dispatch_kv8<E4m3Codes, false>(head_dim, a, out, warps, s);
}

extern "C" int xdk_kv8_sparse_attention(const void* q, const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                                        const int32_t* pages, const int64_t* positions, const int64_t* page_table,
                                        const int64_t* sequence_ids, const xdk_peer_out* out_dst, int64_t tokens, int64_t q_heads,
                                        int64_t kv_heads, int64_t head_dim, int64_t max_pages_per_seq, int64_t page_size, int64_t n_pages,
                                        int cache_is_hnd, float scale, int dtype, int codes, void* scratch, size_t scratch_bytes,
                                        unsigned flags, void* stream) {
  using namespace xdk;
  Kv8Args a;
  PeerOut out;
  if (!pages || n_pages < 1) return XDK_ERR_ARG;
  if (n_pages > 2147483647LL / kKV8MaxPage) return XDK_ERR_LIMIT;
  if (int st = kv8_arguments(q, k_cache, v_cache, k_scale, v_scale, positions, page_table, sequence_ids, out_dst, tokens, q_heads, kv_heads,
                             head_dim, max_pages_per_seq, page_size, cache_is_hnd, scale, dtype, codes, flags, &a, &out))
    return st;
  if (!scratch || !aligned16(scratch) ||
      scratch_bytes < xdk_kv8_sparse_attention_scratch_bytes(tokens, q_heads, kv_heads, head_dim, page_size, n_pages))
    return XDK_ERR_ARG;
  if (int st = require_sm100()) return st;
  CallFlagsScope scope(flags);
  a.pages = pages, a.n_pages = static_cast<int>(n_pages);
  a.scratch = static_cast<float*>(scratch);
  const int warps = grid_for(tokens * kv_heads, head_dim, hint_tiles(n_pages * page_size, head_dim));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return codes == XDK_KV8_INT8 ? dispatch_kv8<Int8Codes, true>(head_dim, a, out, warps, s) : dispatch_kv8<E4m3Codes, true>(head_dim, a, out, warps, s);
}
