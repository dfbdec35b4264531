// Attention of one query token per sequence over the 8-bit paged cache (kv8.cuh), over all of its context or over listed pages.
//
//   s_j = scale * ks[page of j] * (q . kc_j),   out = sum_j softmax(s)_j * vs[page of j] * vc_j
// with codes kc, vc and a scale per page and KV head; j runs over 0 .. position, or over those of them that lie in the pages of
// the token's list.  Nothing to attend to: zeros.
//
// Work is dealt out as in the 16-bit read (paged_attention.cuh): CTAs of four warps, a warp takes 32 positions of a tile of 128,
// K and V rows staged together with cp.async.  A code is exact in FP16, so both contractions are mma.m16n8k16 on FP16 with positions
// (scores) and dims (values) as the 16 rows and the heads of the group as the 8 columns:
//   * q is scaled by a power of two, so that its largest value is near 2^14, and rounded to FP16 (FP16 and BF16 values pass whole unless
//     they are 2^-27 of the largest); an FP32 q is the sum of two such numbers, and each product two products.
//   * the softmax weights times the block scales, w = p * vs, span any range.  They are taken relative to the running largest of each
//     head (times 2^14: what rounds away is then below 2^-38 of it), rounded to FP16 (half a step: 2^-12, below the output's 2^-12 or 2^-9), for FP32
//     again as the sum of two.  The accumulators follow the running largest like the running maximum of the scores.
//   * a tile's sum is added to the accumulators by FP32 FMAs, with rounding; the tensor core truncates.
// Bytes of a row come as 16-bit pairs through ldmatrix: for K four dims of a position (q in the same order), for V, transposed, two dims of
// two positions, which byte permutes sort while they widen the codes.
#include <cooperative_groups.h>
#include <math.h>

#include "kv8.cuh"
#include "paged_attention.cuh"

namespace cg = cooperative_groups;

namespace xdk {
namespace {

struct Kv8Args {
  AttnArgs at;
  const void* q;
  const uint8_t *k_cache, *v_cache;
  const float *k_scale, *v_scale;
  const int32_t* pages;  // [tokens, kv_heads, n_pages], sparse only
  int n_pages;
  int group;  // query heads of a KV head
  int dtype;  // of q and out
};

constexpr int kMaxGroup = 8;             // heads of a group: columns of a matrix instruction
constexpr float kWeightTop = 16384.0f;     // 2^14: the largest weight of a head in FP16
constexpr float kLeastTop = 7.8886091e-31f;  // 2^-100: weights are not taken relative to less

// A warp's stage: K rows, V rows (16-byte pieces xor-swizzled, so that eight rows of an ldmatrix lie on eight bank groups), the
// scales of the positions, and which of them are alive.
template <int D>
struct Stage {
  static constexpr int kPositions = 32, kStages = D == 256 ? 1 : 2;
  static constexpr int kRows = kPositions * D;
  static constexpr int kBytes = 2 * kRows + 2 * kPositions * 4 + 16;
  static_assert(kMaxGroup * D * 4 <= 2 * kRows, "a warp's accumulators fit the stage that it is done with");
  __device__ static __forceinline__ int at(int row, int piece) {
    if constexpr (D == 64) return row * D + ((piece ^ (row >> 1 & 3)) << 4);
    return row * D + ((piece ^ (row & 7)) << 4);
  }
};
template <int D> constexpr size_t ring_bytes() { return static_cast<size_t>(kAttnWarps) * Stage<D>::kStages * Stage<D>::kBytes; }

__device__ __forceinline__ void cp_async4_or_zero(void* dst_smem, const void* src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst_smem)), "l"(src), "r"(live ? 4 : 0) : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float load_as_f32(const void* p, int64_t at, int dtype) {
  if (dtype == XDK_F32) return static_cast<const float*>(p)[at];
  if (dtype == XDK_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]);
  return __half2float(static_cast<const __half*>(p)[at]);
}
__device__ __forceinline__ void store_from_f32(const PeerOut& out, int64_t row, int64_t col, float v, int dtype) {
  if (dtype == XDK_F32) peer_store(out, row, col, v);
  else if (dtype == XDK_BF16) peer_store(out, row, col, __float2bfloat16_rn(v));
  else peer_store(out, row, col, __float2half_rn(v));
}
// Statistics in units of log2: merges (m, l) of b into a.
__device__ __forceinline__ void merge_stats2(float& m_a, float& l_a, float& scale_a, float& scale_b, float m_b, float l_b) {
  const float m = fmaxf(m_a, m_b);
  scale_a = m_a == -INFINITY ? 0.0f : exp2_fast(m_a - m);
  scale_b = m_b == -INFINITY ? 0.0f : exp2_fast(m_b - m);
  l_a = l_a * scale_a + l_b * scale_b;
  m_a = m;
}
// What the sum of the weights divides: nothing was attended to where it is 0.
__device__ __forceinline__ float normalised(float acc, float l) { return l == 0.0f ? 0.0f : acc / l; }

// Scratch of a grid of `ctas` that split the batch evenly, as in the 16-bit read, for a group of any size.
struct Kv8Partials {
  float *acc, *m, *l;  // [2 ctas][group * dim], [2 ctas][group], [2 ctas][group]
  int* header;         // [ctas][4]
  __device__ Kv8Partials(float* base, int ctas, int group, int dim) {
    acc = base;
    m = acc + static_cast<size_t>(2) * group * dim * ctas;
    l = m + static_cast<size_t>(2) * group * ctas;
    header = reinterpret_cast<int*>(l + static_cast<size_t>(2) * group * ctas);
  }
};

template <typename C, int D, bool SPLIT, bool SPARSE>
__global__ void __launch_bounds__(kAttnThreads, D <= 128 ? 3 : 2)
kv8_attention_kernel(const __grid_constant__ Kv8Args p, const __grid_constant__ PeerOut out, int splits) {
  using St = Stage<D>;
  constexpr int TP = St::kPositions, PB = TP / 16, NC = D / 16;  // blocks of 16 positions, pieces of 16 dims
  constexpr int NST = St::kStages, kUnit = kAttnWarps * TP;
  constexpr int NQ = SPLIT ? 2 : 1;  // FP16 numbers to a value of q or weight
  extern __shared__ __align__(128) unsigned char smem[];
  unsigned char* ring = smem + warp_of(threadIdx.x) * NST * St::kBytes;
  __shared__ float part_m[kAttnWarps][kMaxGroup], part_l[kAttnWarps][kMaxGroup];
  __shared__ float cta_m[kMaxGroup], cta_l[kMaxGroup];
  __shared__ int64_t batch_tiles;
  __shared__ TokenCache cache;
  const AttnArgs& a = p.at;

  pdl_launch_dependents();
  pdl_wait();  // q and the caches are the preceding kernels' output
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int grow = lane >> 2, quad = lane & 3;
  const int G = p.group;
  const bool even = !SPARSE && a.scratch != nullptr;
  const int split = even ? 0 : blockIdx.x;
  ItemCursor cur;  // the tile that is computed next
  int n_tiles;
  if (even) {
    if (threadIdx.x == 0) Kv8Partials(a.scratch, gridDim.x, G, D).header[4 * blockIdx.x] = -1;
    n_tiles = static_cast<int>(seek_share<kUnit>(a, cur, batch_tiles, cache));
    if (n_tiles == 0) return;
  } else {
    cur.kvh = blockIdx.y, cur.token = blockIdx.z, cur.load<kUnit>(a, nullptr);
    if constexpr (SPARSE) cur.tiles = cur.ctx > 0 ? static_cast<int>((static_cast<int64_t>(p.n_pages) * a.page_size + kUnit - 1) / kUnit) : 1;
    cur.tile = static_cast<int>(static_cast<int64_t>(cur.tiles) * split / splits);
    n_tiles = static_cast<int>(static_cast<int64_t>(cur.tiles) * (split + 1) / splits) - cur.tile;
  }
  ItemCursor next = cur;  // the tile whose rows are fetched next
  const int32_t* list = nullptr;
  if constexpr (SPARSE) list = p.pages + (static_cast<int64_t>(cur.token) * a.kv_heads + cur.kvh) * p.n_pages;

  struct {
    int64_t page;  // -1: dead
    int off;
  } at;  // this lane's row of tile `next`
  auto look_up = [&]() {
    const int64_t i = static_cast<int64_t>(next.tile) * kUnit + warp * TP + lane;
    at.page = -1, at.off = 0;
    if constexpr (!SPARSE) {
      if (i >= next.ctx) return;
      const int64_t logical = a.narrow ? static_cast<uint32_t>(i) / static_cast<uint32_t>(a.page_size) : i / a.page_size;
      at.off = static_cast<int>(i - logical * a.page_size);
      at.page = next.table[logical];
    } else {
      const int entry = static_cast<int>(static_cast<uint32_t>(i) / static_cast<uint32_t>(a.page_size));  // of at most 2^31 positions
      if (entry >= p.n_pages) return;
      const int64_t logical = list[entry];
      // the list ascends: an entry that does not (a second one of a page) is not read
      if (logical < 0 || (entry > 0 && list[entry - 1] >= logical)) return;
      at.off = static_cast<int>(i) - entry * static_cast<int>(a.page_size);
      if (logical * a.page_size + at.off < next.ctx) at.page = next.table[logical];
    }
  };
  auto fetch = [&](int stage) {  // tile `next` into a stage, and on to the next one
    unsigned char* st = ring + stage * St::kBytes;
    float* scales = reinterpret_cast<float*>(st + 2 * St::kRows);
    const bool live = at.page >= 0;
    const unsigned alive = __ballot_sync(0xffffffffu, live);
    const int64_t row = live ? (a.hnd ? (at.page * a.kv_heads + next.kvh) * a.page_size + at.off
                                      : (at.page * a.page_size + at.off) * a.kv_heads + next.kvh) * D
                             : 0;
    const int64_t block = live ? at.page * a.kv_heads + next.kvh : 0;
    cp_async4_or_zero(scales + lane, p.k_scale + block, live);
    cp_async4_or_zero(scales + TP + lane, p.v_scale + block, live);
    if (lane == 0) *reinterpret_cast<unsigned*>(scales + 2 * TP) = alive;
#pragma unroll
    for (int i = 0; i < NC; ++i) {  // NC pieces to a row
      const int c = i * 32 + lane, r = c / NC, piece = c - r * NC;
      const int64_t from = __shfl_sync(0xffffffffu, row, r) + piece * 16;
      const bool there = alive >> r & 1u;
      cp_async16_or_zero(st + St::at(r, piece), p.k_cache + from, there);
      cp_async16_or_zero(st + St::kRows + St::at(r, piece), p.v_cache + from, there);
    }
  };
  auto step = [&](ItemCursor& c) {
    if (even) c.advance<kUnit>(a, &cache);
    else ++c.tile;
  };

  uint32_t qb[NQ][NC][2];    // q^T as B fragments: dims 16 c + 4 quad + {0,1}, {2,3} of head grow
  float unit[2];             // of the scores of heads 2 quad + {0, 1}: scale * log2(e) * the power of two that q was divided by
  float m_run[2], l_run[2];  // of these heads; l_run is this thread's share of the sum
  float w_top[2];            // the largest weight of these heads so far, as of m_run
  float o[NC][4];            // O^T: dims 16 c + 2 grow (+ 1 in the upper two), heads 2 quad + {0, 1}; in units of w_top / kWeightTop
  auto begin_segment = [&](int token, int kvh) {
#pragma unroll
    for (int e = 0; e < 2; ++e) m_run[e] = -INFINITY, l_run[e] = 0.0f, w_top[e] = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[c][e] = 0.0f;
    const bool head_live = grow < G;
    const int64_t qrow = (static_cast<int64_t>(token) * a.q_heads + kvh * G + (head_live ? grow : 0)) * D + quad * 4;
    float top = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) top = fmaxf(top, head_live ? fabsf(load_as_f32(p.q, qrow + c * 16 + e, p.dtype)) : 0.0f);
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
        float x[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) x[e] = head_live ? load_as_f32(p.q, qrow + c * 16 + 2 * h + e, p.dtype) * by : 0.0f;
        const __half2 hi = __floats2half2_rn(x[0], x[1]);
        qb[0][c][h] = *reinterpret_cast<const uint32_t*>(&hi);
        if constexpr (SPLIT) {
          const float2 f = __half22float2(hi);
          qb[NQ - 1][c][h] = Mma16816<__half>::pack(x[0] - f.x, x[1] - f.y);
        }
      }
#pragma unroll
    for (int e = 0; e < 2; ++e) unit[e] = __shfl_sync(0xffffffffu, back, (2 * quad + e) * 4) * (a.scale * 1.4426950408889634f);
  };
  // a warp's accumulators [group * D], in a stage that it is done with
  auto acc_of = [&](int w, int done) { return reinterpret_cast<float*>(smem + (w * NST + done) * St::kBytes); };
  auto write_partials = [&](int done) {  // of this warp
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int sh = 4; sh < 32; sh <<= 1) l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], sh);
      const int head = quad * 2 + e;
      if (head < G) {
        if (grow == 0) part_m[warp][head] = m_run[e], part_l[warp][head] = l_run[e];
        const float back = w_top[e] * (1.0f / kWeightTop);
        float* to = acc_of(warp, done) + head * D + 2 * grow;
#pragma unroll
        for (int c = 0; c < NC; ++c) *reinterpret_cast<float2*>(to + c * 16) = make_float2(o[c][e] * back, o[c][e + 2] * back);
      }
    }
  };
  // The four warps' partial results -> the output, when the CTA has the whole item, or this CTA's slot of scratch.
  auto finish_segment = [&](int done, int token, int kvh, int tiles_left, bool begins) {
    __syncthreads();
    const Kv8Partials part(a.scratch, gridDim.x, G, D);
    const int slot = 2 * blockIdx.x + (begins ? 1 : 0);
    const bool ends = tiles_left == 0;  // of the item, behind this segment
    if (begins && !ends && threadIdx.x == 0) {
      // the CTA that holds the item's last tile: the tile's number in the batch is this CTA's last one + what is left
      const int64_t ctas = share_ctas(batch_tiles), last = batch_tiles * (blockIdx.x + 1) / ctas + tiles_left - 1;
      int* h = part.header + 4 * blockIdx.x;
      h[0] = token, h[1] = kvh, h[2] = static_cast<int>(((last + 1) * ctas - 1) / batch_tiles);
    }
    for (int i = threadIdx.x; i < G * D; i += kAttnThreads) {
      const int g = i / D, d = i - g * D;
      float mm = part_m[0][g], ll = part_l[0][g], aa = acc_of(0, done)[i];
      for (int w = 1; w < kAttnWarps; ++w) {
        float sa, sb;
        merge_stats2(mm, ll, sa, sb, part_m[w][g], part_l[w][g]);
        aa = aa * sa + acc_of(w, done)[i] * sb;
      }
      if (begins && ends) {
        store_from_f32(out, token, (kvh * G + g) * D + d, normalised(aa, ll), p.dtype);
      } else {
        part.acc[static_cast<size_t>(slot) * G * D + i] = aa;
        if (d == 0) part.m[slot * G + g] = mm, part.l[slot * G + g] = ll;
      }
    }
    __syncthreads();
  };

  int fetched = 0;
  if (n_tiles > 0) look_up();
  auto fetch_next = [&](int stage) {  // one group per call, whether or not there is a tile left
    if (fetched < n_tiles) {
      fetch(stage);
      if (++fetched < n_tiles) {  // the page of the row after that is on its way meanwhile
        step(next);
        look_up();
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < NST - 1; ++s) fetch_next(s);
  bool fresh = true;    // the tile begins a segment
  bool begins = false;  // the segment begins at its item's first tile
  if (n_tiles == 0) begin_segment(cur.token, cur.kvh);  // a split without tiles contributes nothing

  int stage = 0;
  for (int u = 0; u < n_tiles; ++u) {
    fetch_next(stage == 0 ? NST - 1 : stage - 1);
    if (fresh) {
      begin_segment(cur.token, cur.kvh);
      begins = cur.tile == 0;
    }
    cp_async_wait<NST - 1>();
    __syncwarp();
    const unsigned char* ktile = ring + stage * St::kBytes;
    const unsigned char* vtile = ktile + St::kRows;
    const float* scales = reinterpret_cast<const float*>(ktile + 2 * St::kRows);
    const unsigned alive = *reinterpret_cast<const unsigned*>(scales + 2 * TP);

    // ---- S^T = K q^T: per load, rows 0-7 and 8-15 of a block and two pieces
    float sc[PB][4];  // positions 16 pb + grow (+ 8 in the upper two), heads 2 quad + {0, 1}
#pragma unroll
    for (int pb = 0; pb < PB; ++pb)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[pb][e] = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; c += 2)
#pragma unroll
      for (int pb = 0; pb < PB; ++pb) {
        uint32_t raw[4];
        ldmatrix_x4(raw, ktile + St::at(pb * 16 + (lane & 15), c + (lane >> 4)));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t k[4];
          Codec<C>::neighbours(raw[2 * h], k[0], k[2]);
          Codec<C>::neighbours(raw[2 * h + 1], k[1], k[3]);
#pragma unroll
          for (int n = 0; n < NQ; ++n) Mma16816<__half>::run(sc[pb], k, qb[n][c + h][0], qb[n][c + h][1]);
        }
      }
    // ---- online softmax of the two heads, in units of log2; weights relative to the largest
    float mx[2] = {-INFINITY, -INFINITY}, vs[PB][2];
#pragma unroll
    for (int pb = 0; pb < PB; ++pb)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int j = pb * 16 + grow + r * 8;
        const float ks = scales[j];
        vs[pb][r] = scales[TP + j];
        const bool live = alive >> j & 1u;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float& s = sc[pb][2 * r + e];
          s = live ? s * (ks * unit[e]) : -INFINITY;
          mx[e] = fmaxf(mx[e], s);
        }
      }
    float corr[2], wt[2] = {0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int sh = 4; sh < 32; sh <<= 1) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], sh));
      const float m_new = fmaxf(m_run[e], mx[e]);
      corr[e] = m_run[e] == -INFINITY ? 0.0f : exp2_fast(m_run[e] - m_new);
      m_run[e] = m_new;
      l_run[e] *= corr[e];
    }
#pragma unroll
    for (int pb = 0; pb < PB; ++pb)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float pr = sc[pb][e] == -INFINITY ? 0.0f : exp2_fast(sc[pb][e] - m_run[e & 1]);
        l_run[e & 1] += pr;
        sc[pb][e] = pr * vs[pb][e >> 1];
        wt[e & 1] = fmaxf(wt[e & 1], fabsf(sc[pb][e]));
      }
    float rel[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int sh = 4; sh < 32; sh <<= 1) wt[e] = fmaxf(wt[e], __shfl_xor_sync(0xffffffffu, wt[e], sh));
      const float was = w_top[e] * corr[e];
      w_top[e] = fmaxf(fmaxf(was, wt[e]), kLeastTop);
      rel[e] = __fdividef(kWeightTop, w_top[e]);
      corr[e] = was * (rel[e] * (1.0f / kWeightTop));
    }
    uint32_t wb[NQ][PB][2];  // w^T as B fragments: positions 16 pb + 2 quad + {0,1} (+ 8 in [1]), head grow
#pragma unroll
    for (int pb = 0; pb < PB; ++pb)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float x0 = sc[pb][2 * r] * rel[0], x1 = sc[pb][2 * r + 1] * rel[1];
        const __half2 hi = __floats2half2_rn(x0, x1);
        wb[0][pb][r] = transpose8x8(*reinterpret_cast<const uint32_t*>(&hi));
        if constexpr (SPLIT) {
          const float2 f = __half22float2(hi);
          wb[NQ - 1][pb][r] = transpose8x8(Mma16816<__half>::pack(x0 - f.x, x1 - f.y));
        }
      }
    // ---- O^T += V^T w^T: per load, position halves of a block and two pieces
#pragma unroll
    for (int c = 0; c < NC; c += 2) {
      float t[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) t[h][e] = 0.0f;
#pragma unroll
      for (int pb = 0; pb < PB; ++pb) {
        uint32_t raw[4];
        ldmatrix_x4_trans(raw, vtile + St::at(pb * 16 + (lane & 15), c + (lane >> 4)));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t v[4];
          Codec<C>::alternate(raw[2 * h], v[0], v[1]);
          Codec<C>::alternate(raw[2 * h + 1], v[2], v[3]);
#pragma unroll
          for (int n = 0; n < NQ; ++n) Mma16816<__half>::run(t[h], v, wb[n][pb][0], wb[n][pb][1]);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[c + h][e] = fmaf(o[c + h][e], corr[e & 1], t[h][e]);
    }
    __syncwarp();  // every lane has read the tile
    const int done = stage;
    stage = stage + 1 == NST ? 0 : stage + 1;

    const int tiles_left = cur.tiles - 1 - cur.tile;
    fresh = even && (tiles_left == 0 || u + 1 == n_tiles);
    if (fresh) {
      write_partials(done);
      finish_segment(done, cur.token, cur.kvh, tiles_left, begins);
    }
    if (u + 1 < n_tiles) step(cur);
  }
  if (even) return;

  // ---- grid of splits: warp totals, then the four warps of the CTA (fixed order), then the cluster
  const int token = cur.token, kvh = cur.kvh;
  write_partials(0);
  float* accs = acc_of(0, 0);
  __syncthreads();
  for (int i = threadIdx.x; i < G * D; i += kAttnThreads) {
    const int g = i / D, d = i - g * D;
    float mm = part_m[0][g], ll = part_l[0][g], aa = accs[i];
    for (int w = 1; w < kAttnWarps; ++w) {
      float sa, sb;
      merge_stats2(mm, ll, sa, sb, part_m[w][g], part_l[w][g]);
      aa = aa * sa + acc_of(w, 0)[i] * sb;
    }
    accs[i] = aa;
    if (d == 0) cta_m[g] = mm, cta_l[g] = ll;
  }
  __syncthreads();
  if (splits > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();  // every slice's partial is in its CTA's shared memory
    if (split == 0) {
      for (int i = threadIdx.x; i < G * D; i += kAttnThreads) {
        const int g = i / D, d = i - g * D;
        float mm = cta_m[g], ll = cta_l[g], aa = accs[i];
        for (int r = 1; r < splits; ++r) {  // rank order
          const float mr = *cluster.map_shared_rank(&cta_m[g], r), lr = *cluster.map_shared_rank(&cta_l[g], r);
          const float ar = *cluster.map_shared_rank(&accs[i], r);
          float sa, sb;
          merge_stats2(mm, ll, sa, sb, mr, lr);
          aa = aa * sa + ar * sb;
        }
        store_from_f32(out, token, (kvh * G + g) * D + d, normalised(aa, ll), p.dtype);
      }
    }
    cluster.sync();  // nobody leaves while rank 0 may still read its shared memory
  } else {
    for (int i = threadIdx.x; i < G * D; i += kAttnThreads) {
      const int g = i / D, d = i - g * D;
      store_from_f32(out, token, (kvh * G + g) * D + d, normalised(accs[i], cta_l[g]), p.dtype);
    }
  }
}

// Block b adds the partial results of the item that CTA b began and others went on with, a thread four head dims, in CTA order.
__global__ void __launch_bounds__(kMergeThreads)
kv8_attention_merge_kernel(const __grid_constant__ PeerOut out, float* scratch, int group, int dim, int dtype) {
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.x;
  const Kv8Partials p(scratch, gridDim.x, group, dim);
  const int4 h = __ldcg(reinterpret_cast<const int4*>(p.header + 4 * b));
  if (h.x < 0) return;
  const int count = h.z - b + 1, all = group * dim / 4;
  for (int l4 = threadIdx.x; l4 < all; l4 += kMergeThreads) {
    const int g = l4 * 4 / dim;
    float m = -INFINITY, l = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int i = 0; i < count; ++i) {
      const int slot = i == 0 ? 2 * b + 1 : 2 * (b + i);
      const float4 v = __ldcg(reinterpret_cast<const float4*>(p.acc) + static_cast<size_t>(slot) * all + l4);
      float sa, sb;
      merge_stats2(m, l, sa, sb, __ldcg(p.m + slot * group + g), __ldcg(p.l + slot * group + g));
      acc.x = acc.x * sa + v.x * sb, acc.y = acc.y * sa + v.y * sb;
      acc.z = acc.z * sa + v.z * sb, acc.w = acc.w * sa + v.w * sb;
    }
    const int col = h.y * group * dim + l4 * 4;
    store_from_f32(out, h.x, col, normalised(acc.x, l), dtype);
    store_from_f32(out, h.x, col + 1, normalised(acc.y, l), dtype);
    store_from_f32(out, h.x, col + 2, normalised(acc.z, l), dtype);
    store_from_f32(out, h.x, col + 3, normalised(acc.w, l), dtype);
  }
}

inline size_t cta_smem(int64_t dim) { return dim == 64 ? ring_bytes<64>() : (dim == 128 ? ring_bytes<128>() : ring_bytes<256>()); }
// CTAs that an SM holds: by the shared memory (with what they have statically and what is reserved) and by the kernel's launch bounds
inline int64_t resident(int64_t dim) {
  const int64_t by_smem = static_cast<int64_t>((227 * 1024) / (cta_smem(dim) + 4096)), by_regs = dim <= 128 ? 3 : 2;
  return by_smem < 1 ? 1 : (by_smem < by_regs ? by_smem : by_regs);
}
// CTAs of a launch that splits the batch evenly (0: the batch stays on the grid of splits), as in the 16-bit read.
inline int kv8_even_grid(int64_t tokens, int64_t kv_heads, int64_t dim, int64_t hint) {
  if (tokens > kMaxTokensSplit || hint < kMinEvenContext) return 0;
  int64_t ctas = resident(dim) * sm_count();
  const int64_t most = tokens * kv_heads * ((hint + kAttnThreads - 1) / kAttnThreads);  // tiles
  if (most < ctas) ctas = most;
  const int64_t each = (most + ctas - 1) / ctas;
  return static_cast<int>((most + each - 1) / each);
}

template <typename C, int D, bool SPLIT, bool SPARSE>
int launch_kv8(const Kv8Args& p, const PeerOut& out, int splits, cudaStream_t s) {
  const AttnArgs& a = p.at;
  auto kernel = kv8_attention_kernel<C, D, SPLIT, SPARSE>;
  const size_t smem = cta_smem(D);
  if (smem > 40 * 1024) {
    const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (err != cudaSuccess) return note_launch(err);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = a.scratch ? dim3(static_cast<unsigned>(splits))
                          : dim3(static_cast<unsigned>(splits), static_cast<unsigned>(a.kv_heads), static_cast<unsigned>(a.tokens));
  cfg.blockDim = dim3(kAttnThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  unsigned n = 0;
  if (splits > 1 && !a.scratch) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = static_cast<unsigned>(splits);
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (call_flags() & XDK_DEPENDENT_LAUNCH) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  const int st = note_launch(cudaLaunchKernelEx(&cfg, kernel, p, out, splits));
  if (st != XDK_OK || !a.scratch) return st;
  return launch_opts(kv8_attention_merge_kernel, dim3(static_cast<unsigned>(splits)), dim3(kMergeThreads), 0, s, 1u, true, out, a.scratch,
                     p.group, D, p.dtype);
}

template <typename C, bool SPARSE>
int dispatch_kv8(int64_t d, const Kv8Args& p, const PeerOut& out, int splits, cudaStream_t s) {
  const bool split = p.dtype == XDK_F32;
  switch (d) {
    case 64: return split ? launch_kv8<C, 64, true, SPARSE>(p, out, splits, s) : launch_kv8<C, 64, false, SPARSE>(p, out, splits, s);
    case 128: return split ? launch_kv8<C, 128, true, SPARSE>(p, out, splits, s) : launch_kv8<C, 128, false, SPARSE>(p, out, splits, s);
    case 256: return split ? launch_kv8<C, 256, true, SPARSE>(p, out, splits, s) : launch_kv8<C, 256, false, SPARSE>(p, out, splits, s);
    default: return XDK_ERR_LIMIT;
  }
}

// The checks and the arguments that both entry points share.
int kv8_arguments(const void* q, const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                  const int64_t* positions, const int64_t* page_table, const int64_t* sequence_ids, const xdk_peer_out* out_dst,
                  int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t max_pages, int64_t page_size, int hnd,
                  float scale, int dtype, int codes, unsigned flags, Kv8Args* p, PeerOut* out) {
  if (int st = make_out(out_dst, nullptr, 1, out)) return st;
  if (flags & ~XDK_DEPENDENT_LAUNCH) return XDK_ERR_ARG;
  if (!q || !k_cache || !v_cache || !k_scale || !v_scale || !positions || !page_table || !sequence_ids) return XDK_ERR_ARG;
  if (tokens < 1 || q_heads < 1 || kv_heads < 1 || head_dim < 1 || max_pages < 1 || page_size < 1) return XDK_ERR_ARG;
  if (q_heads % kv_heads != 0 || !isfinite(scale) || out->ld < out->col0 + q_heads * head_dim) return XDK_ERR_ARG;
  if (!aligned16(k_cache) || !aligned16(v_cache)) return XDK_ERR_ARG;
  if (dtype != XDK_F32 && dtype != XDK_BF16 && dtype != XDK_F16) return XDK_ERR_ARG;
  if (codes != XDK_KV8_INT8 && codes != XDK_KV8_E4M3) return XDK_ERR_ARG;
  if (!kv8_head_dim(head_dim) || q_heads / kv_heads > kMaxGroup || tokens > 65535) return XDK_ERR_LIMIT;
  if (int st = kv8_limits(tokens, kv_heads, max_pages, page_size)) return st;
  if (int st = require_sm100()) return st;
  *p = {};
  AttnArgs& a = p->at;
  a.positions = positions, a.page_table = page_table, a.sequence_ids = sequence_ids;
  a.max_pages = max_pages, a.page_size = page_size;
  a.q_heads = static_cast<int>(q_heads), a.kv_heads = static_cast<int>(kv_heads);
  a.hnd = hnd ? 1 : 0;
  a.narrow = page_size * max_pages < (1LL << 31) ? 1 : 0;
  a.scale = scale;
  a.tokens = static_cast<int>(tokens);
  a.scratch = nullptr;
  p->q = q, p->k_cache = static_cast<const uint8_t*>(k_cache), p->v_cache = static_cast<const uint8_t*>(v_cache);
  p->k_scale = k_scale, p->v_scale = v_scale;
  p->group = static_cast<int>(q_heads / kv_heads), p->dtype = dtype;
  return XDK_OK;
}
// Splits of the items over the CTAs of a cluster: one wave of the SMs, no more than `tiles`, at most the portable cluster size.
int cluster_splits(int64_t tokens, int64_t kv_heads, int64_t dim, int64_t tiles) {
  int64_t splits = resident(dim) * sm_count() / (tokens * kv_heads);
  if (splits > tiles) splits = tiles;
  if (splits > kMaxSplits) splits = kMaxSplits;
  return splits < 1 ? 1 : static_cast<int>(splits);
}

}  // namespace
}  // namespace xdk

extern "C" size_t xdk_kv8_decode_attention_scratch_bytes(int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                                         int64_t context_hint) {
  using namespace xdk;
  if (tokens < 1 || q_heads < 1 || kv_heads < 1 || kv_heads > 65535 || q_heads % kv_heads != 0 || q_heads / kv_heads > kMaxGroup) return 0;
  if (!kv8_head_dim(head_dim)) return 0;
  if (context_hint <= 0 || context_hint > kMaxContextHint) context_hint = kMaxContextHint;
  return static_cast<size_t>(kv8_even_grid(tokens, kv_heads, head_dim, context_hint)) *
         partial_words(static_cast<size_t>(q_heads / kv_heads), static_cast<size_t>(head_dim)) * 4;
}

extern "C" int xdk_kv8_decode_attention(const void* q, const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                                        const int64_t* positions, const int64_t* page_table, const int64_t* sequence_ids,
                                        const xdk_peer_out* out_dst, int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                        int64_t max_pages_per_seq, int64_t page_size, int cache_is_hnd, float scale, int64_t context_hint,
                                        int dtype, int codes, void* scratch, size_t scratch_bytes, unsigned flags, void* stream) {
  using namespace xdk;
  Kv8Args p;
  PeerOut out;
  if (int st = kv8_arguments(q, k_cache, v_cache, k_scale, v_scale, positions, page_table, sequence_ids, out_dst, tokens, q_heads, kv_heads,
                             head_dim, max_pages_per_seq, page_size, cache_is_hnd, scale, dtype, codes, flags, &p, &out))
    return st;
  CallFlagsScope scope(flags);
  // no bound from the caller: a row of the page table has one
  const int64_t most = max_pages_per_seq * page_size;  // at most 2^41
  if (context_hint <= 0) context_hint = most;
  if (context_hint > kMaxContextHint) context_hint = kMaxContextHint;
  int splits = 0;
  if (scratch && aligned16(scratch)) {
    const size_t need = xdk_kv8_decode_attention_scratch_bytes(tokens, q_heads, kv_heads, head_dim, context_hint);
    if (need > 0 && scratch_bytes >= need) {
      p.at.scratch = static_cast<float*>(scratch);
      splits = kv8_even_grid(tokens, kv_heads, head_dim, context_hint);
    }
  }
  if (!p.at.scratch) splits = cluster_splits(tokens, kv_heads, head_dim, (context_hint + kAttnThreads - 1) / kAttnThreads);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return codes == XDK_KV8_INT8 ? dispatch_kv8<Int8Codes, false>(head_dim, p, out, splits, s)
                               : dispatch_kv8<E4m3Codes, false>(head_dim, p, out, splits, s);
}

extern "C" int xdk_kv8_sparse_attention(const void* q, const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                                        const int32_t* pages, const int64_t* positions, const int64_t* page_table,
                                        const int64_t* sequence_ids, const xdk_peer_out* out_dst, int64_t tokens, int64_t q_heads,
                                        int64_t kv_heads, int64_t head_dim, int64_t max_pages_per_seq, int64_t page_size, int64_t n_pages,
                                        int cache_is_hnd, float scale, int dtype, int codes, unsigned flags, void* stream) {
  using namespace xdk;
  Kv8Args p;
  PeerOut out;
  if (!pages || n_pages < 1) return XDK_ERR_ARG;
  if (n_pages > 2147483647LL / kKV8MaxPage) return XDK_ERR_LIMIT;
  if (int st = kv8_arguments(q, k_cache, v_cache, k_scale, v_scale, positions, page_table, sequence_ids, out_dst, tokens, q_heads, kv_heads,
                             head_dim, max_pages_per_seq, page_size, cache_is_hnd, scale, dtype, codes, flags, &p, &out))
    return st;
  CallFlagsScope scope(flags);
  p.pages = pages, p.n_pages = static_cast<int>(n_pages);
  const int splits = cluster_splits(tokens, kv_heads, head_dim, (n_pages * page_size + kAttnThreads - 1) / kAttnThreads);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return codes == XDK_KV8_INT8 ? dispatch_kv8<Int8Codes, true>(head_dim, p, out, splits, s)
                               : dispatch_kv8<E4m3Codes, true>(head_dim, p, out, splits, s);
}
