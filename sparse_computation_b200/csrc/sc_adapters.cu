// Low-rank adapters of many requests beside a shared projection.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <memory>
#include <type_traits>
#include <vector>

#include <cooperative_groups.h>

#include "sc_mma.cuh"
#include "sc_serve.h"

using namespace sc::serve;
namespace cg = cooperative_groups;
namespace mma = sc::mma;

namespace {

constexpr int64_t kMaxRank = 256;

// What the kernels read of a set.  Rows first[i] .. first[i+1] of `down`
// (rank rows of in_features) and of `up` (rank rows of out_features: up is
// stored transposed) are adapter i's.  Rows are padded with zeros to a
// multiple of kPad elements, so that each of a cluster's blocks finds its
// share of a row on a 16-byte boundary.
constexpr int64_t kPad = 64;
struct SetView {
  const void *down, *up;
  const int32_t *first;  // [count + 1]
  const float *scale;    // [count]
  int64_t in, out;
  int64_t in_row, out_row;  // padded
  int count, rank_max;
  int *status;
};

// Copies matrix blockIdx.y of `list` into rows of dst_row elements, padded with zeros.
struct PackItem {
  const void *src;
  int64_t row_stride, col_stride, cols, dst_row, dst;  // dst: first element
  int rows;
};
template <class W>
__global__ void __launch_bounds__(256) pack_rows(const PackItem *list, W *dst) {
  const PackItem p = list[blockIdx.y];
  const W *src = static_cast<const W *>(p.src);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < p.rows * p.dst_row; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / p.dst_row, c = i % p.dst_row;
    dst[p.dst + i] = c < p.cols ? src[r * p.row_stride + c * p.col_stride] : W(0);
  }
}

// ------------------------------------------------------ a few tokens ----
//
// Up to kFewTokens tokens (a decoding step): what counts is reading each
// adapter's weights once and at once.  A cluster of two to eight blocks takes
// up to kGroup tokens that share an adapter: the cluster of a token whose
// place among its adapter's tokens is a multiple of kGroup takes that one and
// the next ones, the others leave.  Each block multiplies its part of the
// columns of `down` with its part of x, so that x is read once; the parts of
// v = down x are added up through distributed shared memory, in block order;
// then each block makes its part of the rows of up v.  One launch, no scratch
// memory.  Bound by latency (a chain of ids, weights, two cluster barriers,
// weights) and fp32 instructions; the tensor-core tiles below cost more before
// they start, and less for each further token of an adapter.  us here / there
// for 1, 2, 4, 8, 16 and 64 tokens an adapter, 512 x 2048 of rank 16 in bf16:
//   64 tokens  12.5/16.1   9.3/15.6 10.5/14.9 10.6/14.3 11.3/14.7 10.7/14.4
//   128        15.8/22.9  12.2/17.1 13.8/16.1 14.5/15.8 15.8/15.3 15.5/14.5
//   256        23.4/42.6  19.2/24.6 30.3/23.1 30.5/18.3 28.6/19.0 28.9/16.0
// and 4096 x 4096 of ranks 16 to 64 in bf16:
//   128        56.5/93.9  46.1/53.5 27.1/38.3 27.5/27.7 27.6/28.5 24.1/27.6
//   256       105.9/171.6 70.8/96.5 61.1/91.7 54.1/46.7 45.5/35.5 45.5/35.9
// How tokens spread over adapters is known on the device only, so the rule goes
// by their number: up to 256, where a thread of a block looks at each token's
// id.  From about 8 tokens an adapter and 200 tokens on the tiles would be faster.
constexpr int kFewTokens = 256, kGroup = 4 /* a float4 of v */, kFewChunk = 512, kFewThreads = 256, kFewBlocks = 3;

// Eight weights, as they lie.
template <class W>
struct Eight {
  uint4 w[sizeof(W) / 2];
  __device__ __forceinline__ void load(const W *p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(W) / 2; ++i) w[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const W *v = reinterpret_cast<const W *>(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(v[i]);
  }
};

// 16-byte aligned: x, sums and v are read in fours.
struct alignas(16) FewShared {
  union alignas(16) {
    float x[kGroup][kFewChunk];           // this block's part of the tokens' x
    float sums[kGroup][kFewThreads * 8];  // parts of up v
  };
  float part[kMaxRank][kGroup];  // its part of v, read by the whole cluster
  alignas(16) float v[kMaxRank][kGroup];  // scale * v
  int tokens[kGroup];
  int count[kFewThreads / 32], n;
};

// Where column k of a token lies: lower and upper fours of the eights apart, so that the lanes' fours are neighbours.
__device__ __forceinline__ int x_place(int k) { return (k & 4 ? kFewChunk / 2 : 0) + (k >> 3) * 4 + (k & 3); }

// v parts of the rows of one adapter from `width` columns: a warp takes rows, LANES lanes a row.
template <int NT, class W>
__device__ __forceinline__ void few_shrink(FewShared &sh, const W *down, int64_t row, int rank, int width) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  // lanes of a row: a power of two, eight columns each
  int lanes = 32;
  while (lanes > 1 && lanes * 4 >= width) lanes >>= 1;
  const int sub = lane / lanes, in = lane % lanes, rows = 32 / lanes;
  constexpr int B = 3, warps = kFewThreads / 32;  // B rows of a lane at a time (96 tokens of 40
  // adapters of 4096 x 4096: 21.4 us with 3, 22.7 with 4, 21.7 with 6)
  for (int r0 = warp * rows; r0 < rank; r0 += B * warps * rows) {
    float acc[B][NT] = {};
    for (int k = in * 8; k < width; k += lanes * 8) {
      Eight<W> w[B];
#pragma unroll
      for (int i = 0; i < B; ++i) {
        const int r = r0 + i * warps * rows + sub;
        w[i].load(down + min(r, rank - 1) * row + k);
      }
      float x[NT][8];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 8; e += 4) *reinterpret_cast<float4 *>(&x[t][e]) = *reinterpret_cast<const float4 *>(&sh.x[t][x_place(k + e)]);
#pragma unroll
      for (int i = 0; i < B; ++i) {
        if (r0 + i * warps * rows >= rank) break;
        float f[8];
        w[i].get(f);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[i][t] += f[e] * x[t][e];
      }
    }
#pragma unroll
    for (int i = 0; i < B; ++i) {
      const int r = r0 + i * warps * rows + sub;
      if (r - sub >= rank) break;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        for (int d = lanes / 2; d; d >>= 1) acc[i][t] += __shfl_xor_sync(~0u, acc[i][t], d);
        if (in == 0 && r < rank) sh.part[r][t] += acc[i][t];
      }
    }
  }
}

// Rows [m0, m0 + rows) of up v for NT tokens; groups of threads take every so-manieth rank row, their sums are added
// up token by token.
template <int NT, class T, class W>
__device__ __forceinline__ void few_expand(FewShared &sh, const sc_adapters_args &a, const W *up, int64_t row, int rank, int m0,
                                           int rows) {
  constexpr int kEarly = 2;  // values of base that a thread asks for ahead
  float early[NT][kEarly] = {};
  if (a.base.ptr)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < kEarly; ++j) {
        const int i = threadIdx.x + j * kFewThreads;
        if (t < sh.n && i < rows)
          early[t][j] = to_f32(static_cast<const T *>(a.base.ptr)[(int64_t)(m0 + i) * a.base.stride[0] +
                                                                  (int64_t)sh.tokens[t] * a.base.stride[1]]);
      }
  for (int base = 0; base < rows; base += kFewThreads * 8) {
    const int here = min(rows - base, kFewThreads * 8), eights = (here + 7) / 8;
    const int sets = kFewThreads / eights, set = threadIdx.x / eights, at = base + threadIdx.x % eights * 8;
    float acc[NT][8] = {};
    constexpr int B = NT <= 2 && sizeof(W) == 2 ? 8 : 4;  // rank rows of a thread at a time
    if (set < sets)
      for (int r0 = set; r0 < rank; r0 += B * sets) {
        Eight<W> w[B];
#pragma unroll
        for (int i = 0; i < B; ++i) w[i].load(up + min(r0 + i * sets, rank - 1) * row + m0 + at);
#pragma unroll
        for (int i = 0; i < B; ++i) {
          if (r0 + i * sets >= rank) break;
          float f[8];
          w[i].get(f);
          const float4 v4 = *reinterpret_cast<const float4 *>(sh.v[r0 + i * sets]);
          const float v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[t][e] += f[e] * v[t];
        }
      }
    __syncthreads();
    if (set < sets)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 8; e += 4)
          *reinterpret_cast<float4 *>(&sh.sums[t][set * eights * 8 + at - base + e]) =
              make_float4(acc[t][e], acc[t][e + 1], acc[t][e + 2], acc[t][e + 3]);
    __syncthreads();
    for (int i = threadIdx.x, j = 0; i < here; i += kFewThreads, ++j) {
      const int64_t m = m0 + base + i;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (t >= sh.n) break;
        const int64_t token = sh.tokens[t];
        float y = 0.f;
        for (int s = 0; s < sets; ++s) y += sh.sums[t][s * eights * 8 + i];
        if (a.base.ptr)
          y += j < kEarly && base == 0
                   ? early[t][j < kEarly ? j : 0]
                   : to_f32(static_cast<const T *>(a.base.ptr)[m * a.base.stride[0] + token * a.base.stride[1]]);
        static_cast<T *>(a.out.ptr)[m * a.out.stride[0] + token * a.out.stride[1]] = from_f32<T>(y);
      }
    }
    __syncthreads();
  }
}

template <class T, class W>
__global__ void __launch_bounds__(kFewThreads, kFewBlocks) few_kernel(const __grid_constant__ SetView s, const __grid_constant__ sc_adapters_args a) {
  __shared__ FewShared sh;
  const int c = blockIdx.x, blocks = gridDim.x, t = blockIdx.y, tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int n_tokens = (int)a.tokens;
  const int id = a.ids[t];
  const int other = tid < n_tokens ? a.ids[tid] : -1;
  const int rank = id >= 0 && id < s.count ? s.first[id + 1] - s.first[id] : 0;
  // this block's columns of x and rows of out
  const int k0 = (int)(s.in_row / blocks) * c, k1 = min((int)s.in, k0 + (int)(s.in_row / blocks));
  const int m0 = (int)(s.out_row / blocks) * c, m1 = min((int)s.out, m0 + (int)(s.out_row / blocks));
  if (rank == 0) {
    if (id >= s.count && c == 0 && tid == 0) set_status(s.status, 10);
    if (a.out.ptr != a.base.ptr)
      for (int64_t m = m0 + tid; m < m1; m += kFewThreads)
        static_cast<T *>(a.out.ptr)[m * a.out.stride[0] + t * a.out.stride[1]] =
            a.base.ptr ? static_cast<const T *>(a.base.ptr)[m * a.base.stride[0] + t * a.base.stride[1]] : from_f32<T>(0.f);
    return;
  }
  // the adapter's tokens in order; this cluster's are those at places [t's place, + kGroup)
  const uint32_t mine = __ballot_sync(~0u, other == id);
  if (lane == 0) sh.count[warp] = __popc(mine);
  __syncthreads();
  int place = __popc(mine & ((1u << lane) - 1)), at = 0, all = 0;
  for (int w = 0; w < kFewThreads / 32; ++w) {
    if (w < warp) place += sh.count[w];
    if (w < t / 32) at += sh.count[w];
    all += sh.count[w];
  }
  if (tid / 32 == t / 32 && tid % 32 == t % 32) sh.n = place;
  __syncthreads();
  at = sh.n;
  if (at % kGroup) return;  // the whole cluster
  __syncthreads();
  if (other == id && place >= at && place < at + kGroup) sh.tokens[place - at] = tid;
  if (tid == 0) sh.n = min(kGroup, all - at);
  for (int i = tid; i < rank * kGroup; i += kFewThreads) sh.part[i / kGroup][i % kGroup] = 0.f;
  __syncthreads();
  const int n = sh.n;
  const W *down = static_cast<const W *>(s.down) + s.first[id] * s.in_row,
          *up = static_cast<const W *>(s.up) + s.first[id] * s.out_row;
  // the second product's weights on their way to L2 while the first one runs
  if (m1 > m0) {
    const int lines = (int)((m1 - m0) * sizeof(W) + 127) / 128;
    for (int i = tid; i < rank * lines; i += kFewThreads)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const uint8_t *>(up + (int64_t)(i / lines) * s.out_row + m0) +
                                                   i % lines * 128));
  }
  for (int k = k0; k < k1; k += kFewChunk) {
    const int width = min(kFewChunk, k1 - k), wide = (width + 7) / 8 * 8;
    constexpr int per = kFewChunk / kFewThreads;
    float x[kGroup][per];  // all loads at once
#pragma unroll
    for (int g = 0; g < kGroup; ++g)
#pragma unroll
      for (int i = 0; i < per; ++i) {
        const int kk = tid + i * kFewThreads;
        x[g][i] = g < n && kk < width
                      ? to_f32(static_cast<const T *>(a.x.ptr)[(k + kk) * a.x.stride[0] + sh.tokens[g] * a.x.stride[1]])
                      : 0.f;
      }
#pragma unroll
    for (int g = 0; g < kGroup; ++g)
#pragma unroll
      for (int i = 0; i < per; ++i)
        if (tid + i * kFewThreads < wide) sh.x[g][x_place(tid + i * kFewThreads)] = x[g][i];
    __syncthreads();
    if (n == 1)
      few_shrink<1>(sh, down + k, s.in_row, rank, wide);
    else if (n == 2)
      few_shrink<2>(sh, down + k, s.in_row, rank, wide);
    else if (n == 3)
      few_shrink<3>(sh, down + k, s.in_row, rank, wide);
    else
      few_shrink<kGroup>(sh, down + k, s.in_row, rank, wide);
    __syncthreads();
  }
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  const float scale = s.scale[id];
  for (int i = tid; i < rank * kGroup; i += kFewThreads) {
    float v = 0.f;
    for (int b = 0; b < blocks; ++b) v += cluster.map_shared_rank(&sh.part[0][0], b)[i];
    sh.v[i / kGroup][i % kGroup] = v * scale;
  }
  cluster.sync();  // no block leaves, or goes on, before all have read
  if (m1 <= m0) return;
  if (n == 1)
    few_expand<1, T>(sh, a, up, s.out_row, rank, m0, m1 - m0);
  else if (n == 2)
    few_expand<2, T>(sh, a, up, s.out_row, rank, m0, m1 - m0);
  else if (n == 3)
    few_expand<3, T>(sh, a, up, s.out_row, rank, m0, m1 - m0);
  else
    few_expand<kGroup, T>(sh, a, up, s.out_row, rank, m0, m1 - m0);
}

// ---------------------------------------------------- prompts ----
//
// A cluster of two to eight blocks takes a tile: up to kTile tokens that share
// an adapter.  Each block multiplies its part of the columns of `down` with its
// part of x, so that x is read once; the parts of v = down x are added up
// through distributed shared memory, in block order; then each block makes its
// part of the rows of up v.  One launch; v never leaves the chip.
//
// Both products are mma.sync with the tokens as the 16 rows and the weights
// straight from global memory into B fragments, as whole 16-byte pieces per
// lane (the sum over columns may run in any order, and so may the rows of the
// result): of `down`, piece t + 4j of rank row g; of `up` (stored transposed),
// the piece at rows 8g.. of ranks 2t, 2t+1 (+8).  What a 16-bit operand loses
// of x and v goes into further parts, one instruction each (two TF32 parts on
// both sides for fp32 weights, heads and tails added up apart, as an instruction
// cuts its sums off at their size), fp16 parts scaled by a power of two.
//
// A block sorts the tokens by adapter first (group_kernel, 7 us for 2049
// tokens); tokens without one are copied.  x and out bound it at best; at
// present the latencies between the phases of a tile do, two blocks a SM:
// 2049 fp32 tokens of 6 adapters, 2048 x 2048 in fp16, 54.9 us (one warp per
// token and rank row, then one thread per result: 387).
constexpr int kMaxCluster = 8, kTile = 16, kChunk = 512, kThreads = 256, kWarps = kThreads / 32;
constexpr int kXRow = kChunk + 4, kSpan = 64;  // floats of a token's chunk in shared memory; columns of a warp

struct Tile {
  int adapter, first, n;  // first: in the sorted tokens
};

// The tokens sorted by adapter, and the tiles that they are cut into.
struct Sorted {
  const Tile *tiles;  // *n of them
  const int *tokens, *n;
};

template <class T, class W>
struct Kind {
  static constexpr bool f32 = sizeof(W) == 4, f16 = std::is_same<W, __half>::value, same = std::is_same<T, W>::value && !f32;
  static constexpr int mode = f32 ? mma::kTF32 : f16 ? mma::kF16Wide : mma::kBF16Wide;
  static constexpr int px = same ? 1 : f32 || f16 ? 2 : 3;                      // parts of x
  static constexpr int pv = f32 || f16 ? 2 : sizeof(T) == 2 ? 2 : 3;            // of v
  static constexpr int epc = 16 / sizeof(W), J = kSpan / (4 * epc);             // elements of a piece, pieces of a lane
  static constexpr int unit = 8 * epc;                                          // rows of `up` that a warp makes at a time
  static constexpr int step = f32 ? 8 : 16;                                     // ranks of an instruction
  static constexpr bool scaled = f16 && !same;
};

// Two neighbouring values of rows g and g + 8 as parts of A: a[part][0] row g, [1] row g + 8.
template <int MODE, int PARTS>
__device__ __forceinline__ void split2(float x0, float x1, float y0, float y1, uint32_t (&a)[PARTS][2]) {
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
    a[p][0] = mma::pack2<MODE>(x0, x1);
    a[p][1] = mma::pack2<MODE>(y0, y1);
  }
}

// A sum of products in plain fp32: what stands in for a result of split operands that is not finite, as their parts make
// NaN of an infinity.  Out of line: hardly any call takes it.
template <class X, class W>
__device__ __noinline__ float plain_dot(const X *x, int64_t x_step, const W *w, int64_t w_step, int n) {
  float sum = 0.f;
#pragma unroll 4
  for (int i = 0; i < n; ++i) sum += to_f32(x[i * x_step]) * to_f32(w[i * w_step]);
  return sum;
}

template <class T, class W>
__global__ void __launch_bounds__(kThreads, 2)
    tile_kernel(const __grid_constant__ SetView s, const __grid_constant__ sc_adapters_args a, const Sorted sorted) {
  using K = Kind<T, W>;
  extern __shared__ __align__(16) float smem[];
  __shared__ int s_tokens[kTile];
  const int c = blockIdx.x, blocks = gridDim.x, tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, t = lane % 4;
  // this block's columns of x and rows of out
  const int k0 = (int)(s.in_row / blocks) * c, k1 = min((int)s.in, k0 + (int)(s.in_row / blocks));
  const int m0 = (int)(s.out_row / blocks) * c, m1 = min((int)s.out, m0 + (int)(s.out_row / blocks));
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if ((int)blockIdx.y >= *sorted.n) return;  // the whole cluster
  const Tile tile = sorted.tiles[blockIdx.y];
  const int n = tile.n;
  if (tid < n) s_tokens[tid] = sorted.tokens[tile.first + tid];
  const int id = tile.adapter >= 0 && s.first[tile.adapter + 1] > s.first[tile.adapter] ? tile.adapter : -1;
  __syncthreads();
  if (id < 0) {
    if (a.out.ptr == a.base.ptr) return;
    const bool by_token = a.out.stride[1] == 1;
    const int rows = m1 - m0;
    for (int i = tid; i < rows * n; i += kThreads) {
      const int64_t m = m0 + (by_token ? i / n : i % rows), tok = s_tokens[by_token ? i % n : i / rows];
      static_cast<T *>(a.out.ptr)[m * a.out.stride[0] + tok * a.out.stride[1]] =
          a.base.ptr ? static_cast<const T *>(a.base.ptr)[m * a.base.stride[0] + tok * a.base.stride[1]] : from_f32<T>(0.f);
    }
    return;
  }
  const int first = s.first[id], rank = s.first[id + 1] - first;
  const float scale = s.scale[id];
  const W *down = static_cast<const W *>(s.down) + first * s.in_row, *up = static_cast<const W *>(s.up) + first * s.out_row;
  // the second product's weights on their way to L2 while the first one runs
  if (m1 > m0) {
    const int lines = (int)((m1 - m0) * sizeof(W) + 127) / 128;
    for (int i = tid; i < rank * lines; i += kThreads)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const uint8_t *>(up + (int64_t)(i / lines) * s.out_row + m0) +
                                                   i % lines * 128));
  }
  const int v_row = (rank + 15) / 16 * 16 + 4;  // floats; ranks up to a multiple of 16 are zeros
  float *part = smem + 2 * kTile * kXRow, *v_part = part + kWarps * kTile * 64;
  float *v = part;  // after the parts are added up
  for (int i = tid; i < kTile * v_row; i += kThreads) v_part[i] = 0.f;

  // base on its way to L2: rows m0.. of the tile's tokens
  if (a.base.ptr) {
    const bool by_token = a.base.stride[1] == 1;  // then the tokens of a row mostly share a line
    const int per = by_token ? 1 : (m1 - m0 + 31) / 32, count = by_token ? m1 - m0 : per * n;
    for (int i = tid; i < count; i += kThreads) {
      const int64_t m = by_token ? m0 + i : min(m0 + i % per * 32, m1 - 1), tok = s_tokens[by_token ? 0 : i / per];
      asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const T *>(a.base.ptr) + m * a.base.stride[0] +
                                                   tok * a.base.stride[1]));
    }
  }

  // ---- v = down x over this block's columns, kChunk at a time; x is asked for two chunks ahead
  const bool by_token = a.x.stride[1] == 1;  // neighbouring threads on neighbouring tokens, else on neighbouring features
  auto stage = [&](int chunk) {
    const int k = k0 + chunk * kChunk, width = min(kChunk, k1 - k), wide = (width + kSpan - 1) / kSpan * kSpan;
    float *to = smem + (chunk & 1) * (kTile * kXRow);
    if (width > 0) {
      // a thread keeps to a token (by_token: its columns are kThreads / kTile apart) or walks a token's columns; pointers
      // move by additions only, as index arithmetic for each element took as long as the rest of the kernel
      const T *x = static_cast<const T *>(a.x.ptr) + k * a.x.stride[0];
      const int across = by_token ? kThreads / kTile : kThreads, rows = by_token ? 1 : kTile;
      const int first = by_token ? tid / kTile : tid;
      const int64_t step = across * a.x.stride[0];
      for (int r = 0; r < rows; ++r) {
        const int row = by_token ? tid % kTile : r;
        const T *src = x + first * a.x.stride[0] + (row < n ? s_tokens[row] * a.x.stride[1] : 0);
        float *dst = to + row * kXRow + first;
        if (sizeof(T) == 4) {
          uint32_t at = (uint32_t)__cvta_generic_to_shared(dst);
#pragma unroll 4
          for (int col = first; col < wide; col += across, src += step, at += across * 4) {
            const bool in = row < n && col < width;
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(at), "l"(in ? src : x), "r"(in ? 4 : 0)
                         : "memory");
          }
        } else {
          for (int col0 = first; col0 < wide; col0 += 8 * across, src += 8 * step, dst += 8 * across) {
            T v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u)
              if (row < n && col0 + u * across < width) v[u] = src[u * step];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              const int col = col0 + u * across;
              if (col < wide) dst[u * across] = row < n && col < width ? to_f32(v[u]) : 0.f;
            }
          }
        }
      }
    }
    asm volatile("cp.async.commit_group;");
  };
  stage(0);
  stage(1);
  for (int k = k0, chunk = 0; k < k1; k += kChunk, ++chunk) {
    const int width = min(kChunk, k1 - k);
    float *x_tile = smem + (chunk & 1) * (kTile * kXRow);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncthreads();
    // warps: kw of them along the columns, kSpan each, the others along the ranks
    const int spans = (width + kSpan - 1) / kSpan, kw = spans > 4 ? 8 : spans > 2 ? 4 : spans;
    const int col0 = warp % kw * kSpan;
    const bool busy = col0 < spans * kSpan;
    uint32_t ax[K::J][2][K::px][4];  // A fragments: of pieces, their two k-steps
    float up_g = 1.f, up_g8 = 1.f;
    if (busy) {
      float xs[K::J][2][K::epc];
#pragma unroll
      for (int j = 0; j < K::J; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < K::epc; e += 4) {
            const float4 y = *reinterpret_cast<const float4 *>(&x_tile[(g + 8 * h) * kXRow + col0 + (t + 4 * j) * K::epc + e]);
            xs[j][h][e] = y.x, xs[j][h][e + 1] = y.y, xs[j][h][e + 2] = y.z, xs[j][h][e + 3] = y.w;
          }
      if (K::scaled) {
        float top[2] = {0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int j = 0; j < K::J; ++j)
#pragma unroll
            for (int e = 0; e < K::epc; ++e) top[h] = fmaxf(top[h], fabsf(xs[j][h][e]));
          top[h] = fmaxf(top[h], __shfl_xor_sync(~0u, top[h], 1));
          top[h] = fmaxf(top[h], __shfl_xor_sync(~0u, top[h], 2));
        }
        up_g = mma::f16_scale(top[0]);
        up_g8 = mma::f16_scale(top[1]);
#pragma unroll
        for (int j = 0; j < K::J; ++j)
#pragma unroll
          for (int e = 0; e < K::epc; ++e) xs[j][0][e] *= 1.f / up_g, xs[j][1][e] *= 1.f / up_g8;
      }
#pragma unroll
      for (int j = 0; j < K::J; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (K::f32) {
            const float x0 = xs[j][0][2 * h], x1 = xs[j][0][2 * h + 1], y0 = xs[j][1][2 * h], y1 = xs[j][1][2 * h + 1];
            ax[j][h][0][0] = mma::tf32_head(x0), ax[j][h][0][1] = mma::tf32_head(y0);
            ax[j][h][0][2] = mma::tf32_head(x1), ax[j][h][0][3] = mma::tf32_head(y1);
            ax[j][h][K::px - 1][0] = mma::tf32_tail(x0), ax[j][h][K::px - 1][1] = mma::tf32_tail(y0);
            ax[j][h][K::px - 1][2] = mma::tf32_tail(x1), ax[j][h][K::px - 1][3] = mma::tf32_tail(y1);
          } else {
            constexpr int q = K::epc / 2;
            uint32_t lo[K::px][2], hi[K::px][2];
            split2<K::mode>(xs[j][0][q * h], xs[j][0][q * h + 1], xs[j][1][q * h], xs[j][1][q * h + 1], lo);
            split2<K::mode>(xs[j][0][q * h + q - 2], xs[j][0][q * h + q - 1], xs[j][1][q * h + q - 2], xs[j][1][q * h + q - 1], hi);
#pragma unroll
            for (int p = 0; p < K::px; ++p) {
              ax[j][h][p][0] = lo[p][0], ax[j][h][p][1] = lo[p][1];
              ax[j][h][p][2] = hi[p][0], ax[j][h][p][3] = hi[p][1];
            }
          }
        }
    }
    const int row_end = (int)s.in_row - k;  // columns from k on that a weight row has
    for (int r64 = 0; r64 < rank; r64 += 64) {
      const int tiles = (min(64, rank - r64) + 7) / 8, across = kWarps / kw, mine = warp / kw;
      if (busy) {
        constexpr int B = 4;  // rank tiles whose weights are in flight
#pragma unroll 1
        for (int nt0 = mine; nt0 < tiles; nt0 += B * across) {
          uint4 w[B][K::J];
#pragma unroll
          for (int i = 0; i < B; ++i) {
            const W *row = down + (int64_t)min(r64 + (nt0 + i * across) * 8 + g, rank - 1) * s.in_row + k;
#pragma unroll
            for (int j = 0; j < K::J; ++j) {
              const int col = col0 + (t + 4 * j) * K::epc;
              w[i][j] = __ldg(reinterpret_cast<const uint4 *>(row + (col < row_end ? col : 0)));  // beyond: x is zero
            }
          }
#pragma unroll
          for (int i = 0; i < B; ++i) {
            if (nt0 + i * across >= tiles) break;
            float acc[2][4] = {};
#pragma unroll
            for (int j = 0; j < K::J; ++j) {
              const uint32_t b[4] = {w[i][j].x, w[i][j].y, w[i][j].z, w[i][j].w};
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int p = 0; p < K::px; ++p) {
                  const uint32_t(&f)[4] = ax[j][h][p];
                  if (K::f32) {
                    const float b0 = __uint_as_float(b[2 * h]), b1 = __uint_as_float(b[2 * h + 1]);
                    mma::mma16<K::mode>(acc[p], f[0], f[1], f[2], f[3], mma::tf32_head(b0), mma::tf32_head(b1));
                    if (p == 0) mma::mma16<K::mode>(acc[1], f[0], f[1], f[2], f[3], mma::tf32_tail(b0), mma::tf32_tail(b1));
                  } else {
                    mma::mma16<K::mode>(acc[h], f[0], f[1], f[2], f[3], b[2 * h], b[2 * h + 1]);
                  }
                }
            }
            float *to = part + ((warp % kw) * kTile + g) * 64 + (nt0 + i * across) * 8 + 2 * t;
            *reinterpret_cast<float2 *>(to) = make_float2((acc[0][0] + acc[1][0]) * up_g, (acc[0][1] + acc[1][1]) * up_g);
            *reinterpret_cast<float2 *>(to + 8 * 64) =
                make_float2((acc[0][2] + acc[1][2]) * up_g8, (acc[0][3] + acc[1][3]) * up_g8);
          }
        }
      }
      __syncthreads();
      const int live = min(kw, spans);
      for (int i = tid; i < kTile * 64; i += kThreads) {
        const int r = i % 64;
        if (r64 + r < rank) {
          float sum = 0.f;
          for (int w = 0; w < live; ++w) sum += part[w * kTile * 64 + i];
          sum += v_part[i / 64 * v_row + r64 + r];
          if (k + kChunk >= k1 && !isfinite(sum) && i / 64 < n)
            sum = plain_dot(static_cast<const T *>(a.x.ptr) + k0 * a.x.stride[0] + s_tokens[i / 64] * a.x.stride[1], a.x.stride[0],
                            down + (r64 + r) * s.in_row + k0, 1, k1 - k0);
          v_part[i / 64 * v_row + r64 + r] = sum;
        }
      }
      __syncthreads();
    }
    stage(chunk + 2);  // every warp has its fragments of this chunk
  }
  asm volatile("cp.async.wait_all;" ::: "memory");

  // ---- the cluster's v
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  for (int i = tid; i < kTile * v_row; i += kThreads) {
    float sum = 0.f;
    for (int b = 0; b < blocks; ++b) sum += cluster.map_shared_rank(v_part, b)[i];
    v[i] = sum * scale;
  }
  cluster.sync();  // no block leaves before all have read

  // ---- out = base + up v, K::unit rows a warp
  const int token_g = g < n ? s_tokens[g] : -1, token_g8 = g + 8 < n ? s_tokens[g + 8] : -1;
  float vs[2] = {1.f, 1.f};
  if (K::f16) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float top = 0.f;
      for (int r = t; r < rank; r += 4) top = fmaxf(top, fabsf(v[(g + 8 * h) * v_row + r]));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
      vs[h] = mma::f16_scale(top);
    }
  }
  const float vi[2] = {1.f / vs[0], 1.f / vs[1]};
#pragma unroll 1
  for (int mu = m0 + warp * K::unit; mu < m1; mu += kWarps * K::unit) {
    float acc[K::epc][4];
#pragma unroll
    for (int e = 0; e < K::epc; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[e][i] = 0.f;
    float tails[K::f32 ? K::epc : 1][4] = {};
    // this lane's results: the 2 epc rows from mu + 2t epc on of tokens g and g + 8
    const int row0 = mu + 2 * t * K::epc;
    float base[2][2 * K::epc];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int tok = h ? token_g8 : token_g;
      const T *p = static_cast<const T *>(a.base.ptr) + row0 * a.base.stride[0] + tok * a.base.stride[1];
#pragma unroll
      for (int r = 0; r < 2 * K::epc; ++r, p += a.base.stride[0])
        base[h][r] = a.base.ptr && tok >= 0 && row0 + r < m1 ? to_f32(*p) : 0.f;
    }
    const int piece = mu + g * K::epc < s.out_row ? mu + g * K::epc : 0;
    constexpr int R = K::f32 ? 2 : 4;  // rank rows of a lane in a step
#pragma unroll 2
    for (int r0 = 0; r0 < rank; r0 += K::step) {
      uint4 w[R];
      float va[2][R];
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int r = r0 + 2 * t + (i & 1) + (i & 2) * 4;
        w[i] = __ldg(reinterpret_cast<const uint4 *>(up + (int64_t)min(r, rank - 1) * s.out_row + piece));  // beyond: v is zero
        va[0][i] = v[g * v_row + r] * vi[0];
        va[1][i] = v[(g + 8) * v_row + r] * vi[1];
      }
      uint32_t f[K::pv][4];
      if (K::f32) {
        f[0][0] = mma::tf32_head(va[0][0]), f[0][1] = mma::tf32_head(va[1][0]);
        f[0][2] = mma::tf32_head(va[0][1]), f[0][3] = mma::tf32_head(va[1][1]);
        f[K::pv - 1][0] = mma::tf32_tail(va[0][0]), f[K::pv - 1][1] = mma::tf32_tail(va[1][0]);
        f[K::pv - 1][2] = mma::tf32_tail(va[0][1]), f[K::pv - 1][3] = mma::tf32_tail(va[1][1]);
      } else {
        uint32_t lo[K::pv][2], hi[K::pv][2];
        split2<K::mode>(va[0][0], va[0][1], va[1][0], va[1][1], lo);
        split2<K::mode>(va[0][R - 2], va[0][R - 1], va[1][R - 2], va[1][R - 1], hi);
#pragma unroll
        for (int p = 0; p < K::pv; ++p) f[p][0] = lo[p][0], f[p][1] = lo[p][1], f[p][2] = hi[p][0], f[p][3] = hi[p][1];
      }
#pragma unroll
      for (int e = 0; e < K::epc; ++e) {
        auto word = [&](int i) {
          const int k = K::f32 ? e : e / 2;
          return k == 0 ? w[i].x : k == 1 ? w[i].y : k == 2 ? w[i].z : w[i].w;
        };
        if (K::f32) {
          const float b0 = __uint_as_float(word(0)), b1 = __uint_as_float(word(1));
          float(&low)[4] = tails[e % (K::f32 ? K::epc : 1)];
          mma::mma16<K::mode>(acc[e], f[0][0], f[0][1], f[0][2], f[0][3], mma::tf32_head(b0), mma::tf32_head(b1));
          mma::mma16<K::mode>(low, f[K::pv - 1][0], f[K::pv - 1][1], f[K::pv - 1][2], f[K::pv - 1][3], mma::tf32_head(b0),
                              mma::tf32_head(b1));
          mma::mma16<K::mode>(low, f[0][0], f[0][1], f[0][2], f[0][3], mma::tf32_tail(b0), mma::tf32_tail(b1));
        } else {
          const uint32_t sel = e % 2 ? 0x7632 : 0x5410;
          const uint32_t b0 = __byte_perm(word(0), word(1), sel), b1 = __byte_perm(word(R - 2), word(R - 1), sel);
#pragma unroll
          for (int p = 0; p < K::pv; ++p) mma::mma16<K::mode>(acc[e], f[p][0], f[p][1], f[p][2], f[p][3], b0, b1);
        }
      }
    }
    uint32_t bad = 0;  // results that are not finite, and not written yet
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int tok = h ? token_g8 : token_g;
      T *p = static_cast<T *>(a.out.ptr) + row0 * a.out.stride[0] + tok * a.out.stride[1];
#pragma unroll
      for (int r = 0; r < 2 * K::epc; ++r, p += a.out.stride[0]) {
        float sum = acc[r % K::epc][2 * h + r / K::epc];
        if (K::f32) sum += tails[r % (K::f32 ? K::epc : 1)][2 * h + r / K::epc];
        const float y = fmaf(sum, vs[h], base[h][r]);
        if (tok >= 0 && row0 + r < m1) {
          if (isfinite(y))
            *p = from_f32<T>(y);
          else
            bad |= 1u << (2 * K::epc * h + r);
        }
      }
    }
    for (; bad; bad &= bad - 1) {
      const int i = __ffs(bad) - 1, h = i / (2 * K::epc);
      const int64_t m = row0 + i % (2 * K::epc), tok = h ? token_g8 : token_g;
      float y = plain_dot(v + (g + 8 * h) * v_row, 1, up + m, s.out_row, rank);
      if (a.base.ptr) y += to_f32(static_cast<const T *>(a.base.ptr)[m * a.base.stride[0] + tok * a.base.stride[1]]);
      static_cast<T *>(a.out.ptr)[m * a.out.stride[0] + tok * a.out.stride[1]] = from_f32<T>(y);
    }
  }
}

// Sorts the tokens by adapter (those without one last) and cuts them into tiles; one block.  Tokens of 32 at a time
// keep their order, so that neighbouring tokens of a prompt stay neighbours.
__global__ void __launch_bounds__(1024) group_kernel(const __grid_constant__ SetView s, const int32_t *ids, int n, int *heads,
                                                     int *tokens, Tile *tiles, int *n_tiles) {
  constexpr int kBins = 2048;  // so many counters fit shared memory
  __shared__ int s_a[32], s_b[32], s_tokens, s_tiles, s_heads[kBins];
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, bins = s.count + 1;
  if (bins <= kBins) heads = s_heads;
  auto bin_of = [&](int i) {
    const int id = ids[i];
    if (id >= s.count) set_status(s.status, 10);
    return id < 0 || id >= s.count ? s.count : id;
  };
  asm volatile("griddepcontrol.launch_dependents;");  // the tiles' blocks may take their places, and wait there
  for (int i = tid; i < bins; i += 1024) heads[i] = 0;
  if (tid == 0) s_tokens = s_tiles = 0;
  __syncthreads();
  for (int i = tid; i < n; i += 1024) atomicAdd(&heads[bin_of(i)], 1);
  __syncthreads();
  // running sums of tokens and tiles over the bins
  for (int b0 = 0; b0 < bins; b0 += 1024) {
    const int b = b0 + tid, count = b < bins ? heads[b] : 0, cut = (count + kTile - 1) / kTile;
    int x = count, y = cut;
    for (int d = 1; d < 32; d <<= 1) {
      const int ux = __shfl_up_sync(~0u, x, d), uy = __shfl_up_sync(~0u, y, d);
      if (lane >= d) x += ux, y += uy;
    }
    if (lane == 31) s_a[warp] = x, s_b[warp] = y;
    __syncthreads();
    const int all = __reduce_add_sync(~0u, s_a[lane]), cuts = __reduce_add_sync(~0u, s_b[lane]);
    const int px = s_tokens + __reduce_add_sync(~0u, lane < warp ? s_a[lane] : 0);
    const int py = s_tiles + __reduce_add_sync(~0u, lane < warp ? s_b[lane] : 0);
    const int first = px + x - count;
    if (b < bins) heads[b] = first;
    for (int k = 0; k < cut; ++k)
      tiles[py + y - cut + k] = Tile{b == s.count ? -1 : b, first + k * kTile, min(kTile, count - k * kTile)};
    __syncthreads();
    if (tid == 0) s_tokens += all, s_tiles += cuts;
    __syncthreads();
  }
  for (int i0 = 0; i0 < n; i0 += 1024) {
    const int i = i0 + tid;
    const int bin = i < n ? bin_of(i) : -1;
    const uint32_t peers = __match_any_sync(~0u, bin);
    const int leader = __ffs(peers) - 1;
    int at = 0;
    if (lane == leader && bin >= 0) at = atomicAdd(&heads[bin], __popc(peers));
    at = __shfl_sync(~0u, at, leader);
    if (bin >= 0) tokens[at + __popc(peers & ((1u << lane) - 1))] = i;
  }
  if (tid == 0) *n_tiles = s_tiles;
}

template <class F>
void with_types(int64_t rows, int64_t weights, F f) {
  auto inner = [&](auto t) {
    if (weights == SC_TYPE_F32)
      f(t, float());
    else if (weights == SC_TYPE_F16)
      f(t, __half());
    else
      f(t, __nv_bfloat16());
  };
  if (rows == SC_TYPE_F32)
    inner(float());
  else if (rows == SC_TYPE_F16)
    inner(__half());
  else
    inner(__nv_bfloat16());
}

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

// The scratch of a call with many tokens.
struct Scratch {
  int *n_tiles, *heads, *tokens;
  Tile *tiles;
  int64_t most_tiles;
  size_t bytes;
};
Scratch scratch_of(const SetView &v, int64_t tokens, void *at) {
  uint8_t *p = static_cast<uint8_t *>(at);
  size_t used = 0;
  auto take = [&](size_t n) {
    uint8_t *q = p + used;
    used += align256(n);
    return q;
  };
  Scratch s;
  s.most_tiles = tokens / kTile + std::min<int64_t>(v.count + 1, tokens);
  s.n_tiles = reinterpret_cast<int *>(take(4));
  s.heads = reinterpret_cast<int *>(take((v.count + 1) * sizeof(int)));
  s.tokens = reinterpret_cast<int *>(take(tokens * sizeof(int)));
  s.tiles = reinterpret_cast<Tile *>(take(s.most_tiles * sizeof(Tile)));
  s.bytes = used;
  return s;
}

// Shared memory of the tile kernel: x, the warps' parts of v (later v), the block's part of v.
int tile_smem(int rank_max) {
  const int v = kTile * ((rank_max + 15) / 16 * 16 + 4);
  return 4 * (2 * kTile * kXRow + std::max(kWarps * kTile * 64, v) + v);
}

}  // namespace

struct sc_adapters {
  int device = 0;
  int64_t type = 0;
  SetView view{};
  int64_t mean_bytes = 0;  // of an adapter's weights
  DeviceBlock mem;  // its own memory, if any
};

namespace {

// Where a set's parts lie in its memory.
struct SetLayout {
  std::vector<int32_t> first;
  int64_t total = 0, most = 0, in_row = 0, out_row = 0, filled = 0;  // filled: adapters with ranks
  size_t e = 0, up = 0, firsts = 0, scales = 0, status = 0, list = 0, bytes = 0;
};

SetLayout lay_out(int64_t in_features, int64_t out_features, int64_t count, const int64_t *ranks, int64_t type) {
  require(count > 0 && count < (1 << 24), SC_ERR_ARG, "a set has 1 to 2^24 adapters");
  require(in_features > 0 && out_features > 0 && in_features < (1 << 24) && out_features < (1 << 24), SC_ERR_ARG,
          "features must be 1 to 2^24");
  require(type_ok(type), SC_ERR_ARG, "unknown element type");
  SetLayout l;
  l.first.assign(count + 1, 0);
  for (int64_t i = 0; i < count; ++i) {
    require(ranks[i] >= 0 && ranks[i] <= kMaxRank, SC_ERR_UNSUPPORTED, "ranks must be 0 to 256");
    l.total += ranks[i];
    l.most = std::max(l.most, ranks[i]);
    l.filled += ranks[i] > 0;
    require(l.total < INT32_MAX, SC_ERR_UNSUPPORTED, "too many rank rows in one set");
    l.first[i + 1] = (int32_t)l.total;
  }
  l.e = (size_t)type_bytes(type);
  l.in_row = (in_features + kPad - 1) / kPad * kPad;
  l.out_row = (out_features + kPad - 1) / kPad * kPad;
  l.up = align256(l.total * l.in_row * l.e + 16);
  l.firsts = l.up + align256(l.total * l.out_row * l.e + 16);
  l.scales = l.firsts + align256((count + 1) * 4);
  l.status = l.scales + align256(count * 4);
  l.list = l.status + 256;
  l.bytes = l.list + align256(2 * l.filled * sizeof(PackItem));
  return l;
}

// memory null: the set allocates it.
sc_adapters *make_set(int32_t device, int64_t in_features, int64_t out_features, int64_t count, const int64_t *ranks,
                      int64_t type, const void *const *down, const int64_t *down_ld, const void *const *up,
                      const int64_t *up_ld, const float *scales, cudaStream_t st, void *memory, int64_t bytes) {
  require(ranks && down && down_ld && up && up_ld && scales, SC_ERR_ARG, "null argument");
  require(device >= 0 && device < 64, SC_ERR_ARG, "bad device");
  const SetLayout l = lay_out(in_features, out_features, count, ranks, type);
  for (int64_t i = 0; i < count; ++i)
    require(ranks[i] == 0 || (down[i] && up[i] && down_ld[i] >= in_features && up_ld[i] >= ranks[i]), SC_ERR_ARG,
            "null adapter weights or row stride too small");
  require(!memory || (bytes >= (int64_t)l.bytes && reinterpret_cast<uintptr_t>(memory) % 256 == 0), SC_ERR_ARG,
          "memory too small or not 256-byte aligned");
  std::unique_ptr<sc_adapters> s(new sc_adapters);
  s->device = device;
  s->type = type;
  DeviceGuard dg(device);
  if (!memory) {
    s->mem.alloc(device, l.bytes, "allocate adapters");
    memory = s->mem.p;
  }
  uint8_t *p = static_cast<uint8_t *>(memory);
  cuda_check(cudaMemcpyAsync(p + l.firsts, l.first.data(), (count + 1) * 4, cudaMemcpyHostToDevice, st), "upload adapters");
  cuda_check(cudaMemcpyAsync(p + l.scales, scales, count * 4, cudaMemcpyHostToDevice, st), "upload adapters");
  cuda_check(cudaMemsetAsync(p + l.status, 0, 256, st), "clear status word");
  std::vector<PackItem> list;
  list.reserve(2 * l.filled);
  for (int64_t i = 0; i < count; ++i) {
    if (!ranks[i]) continue;
    list.push_back({down[i], down_ld[i], 1, in_features, l.in_row, l.first[i] * l.in_row, (int)ranks[i]});
    list.push_back({up[i], 1, up_ld[i], out_features, l.out_row, (int64_t)(l.up / l.e) + l.first[i] * l.out_row, (int)ranks[i]});
  }
  if (!list.empty())
    cuda_check(cudaMemcpyAsync(p + l.list, list.data(), list.size() * sizeof(PackItem), cudaMemcpyHostToDevice, st),
               "upload packing list");
  const unsigned across = (unsigned)std::max<int64_t>(1, std::min<int64_t>(64, l.most * std::max(l.in_row, l.out_row) / 1024));
  for (size_t at = 0; at < list.size(); at += 65535) {
    const dim3 grid(across, (unsigned)std::min<size_t>(65535, list.size() - at));
    const PackItem *items = reinterpret_cast<const PackItem *>(p + l.list) + at;
    if (l.e == 4)
      pack_rows<<<grid, 256, 0, st>>>(items, reinterpret_cast<uint32_t *>(p));
    else
      pack_rows<<<grid, 256, 0, st>>>(items, reinterpret_cast<uint16_t *>(p));
  }
  cuda_check(cudaGetLastError(), "launch adapter packing");
  cuda_check(cudaStreamSynchronize(st), "stream synchronize");
  s->view = SetView{p,           p + l.up,     reinterpret_cast<int32_t *>(p + l.firsts), reinterpret_cast<float *>(p + l.scales),
                    in_features, out_features, l.in_row, l.out_row, (int)count, (int)l.most, reinterpret_cast<int *>(p + l.status)};
  s->mean_bytes = (int64_t)(l.firsts / count);
  return s.release();
}

}  // namespace

extern "C" {

int sc_adapters_size(int64_t in_features, int64_t out_features, int64_t count, const int64_t *ranks, int64_t type,
                     int64_t *bytes) {
  SC_SERVE_BEGIN
  require(ranks && bytes, SC_ERR_ARG, "null argument");
  *bytes = (int64_t)lay_out(in_features, out_features, count, ranks, type).bytes;
  SC_SERVE_END
}

int sc_adapters_create(int32_t device, int64_t in_features, int64_t out_features, int64_t count,
                       const int64_t *ranks, int64_t type, const void *const *down, const int64_t *down_ld,
                       const void *const *up, const int64_t *up_ld, const float *scales, void *stream,
                       sc_adapters **out) {
  SC_SERVE_BEGIN
  require(out, SC_ERR_ARG, "null argument");
  *out = nullptr;
  *out = make_set(device, in_features, out_features, count, ranks, type, down, down_ld, up, up_ld, scales,
                  static_cast<cudaStream_t>(stream), nullptr, 0);
  SC_SERVE_END
}

int sc_adapters_create_in(int32_t device, int64_t in_features, int64_t out_features, int64_t count,
                          const int64_t *ranks, int64_t type, const void *const *down, const int64_t *down_ld,
                          const void *const *up, const int64_t *up_ld, const float *scales, void *stream,
                          void *memory, int64_t memory_bytes, sc_adapters **out) {
  SC_SERVE_BEGIN
  require(out && memory, SC_ERR_ARG, "null argument");
  *out = nullptr;
  *out = make_set(device, in_features, out_features, count, ranks, type, down, down_ld, up, up_ld, scales,
                  static_cast<cudaStream_t>(stream), memory, memory_bytes);
  SC_SERVE_END
}

void sc_adapters_free(sc_adapters *s) { delete s; }

int sc_adapters_workspace(const sc_adapters *s, int64_t tokens, int64_t *bytes) {
  SC_SERVE_BEGIN
  require(s && bytes && tokens >= 0, SC_ERR_ARG, "null argument or negative token count");
  *bytes = tokens <= kFewTokens ? 0 : (int64_t)scratch_of(s->view, tokens, nullptr).bytes;
  SC_SERVE_END
}

int sc_adapters_status(sc_adapters *s, int32_t *status) {
  SC_SERVE_BEGIN
  require(s && status, SC_ERR_ARG, "null argument");
  *status = take_status(s->device, s->view.status);
  SC_SERVE_END
}

int sc_adapters_apply(sc_adapters *s, const sc_adapters_args *a, void *stream) {
  SC_SERVE_BEGIN
  require(s && a, SC_ERR_ARG, "null argument");
  require(a->tokens >= 0 && a->tokens < (1 << 24), SC_ERR_ARG, "0 to 2^24 tokens a call");
  if (a->tokens == 0) return SC_OK;
  require(type_ok(a->type), SC_ERR_ARG, "unknown element type");
  require(a->x.ptr && a->out.ptr && a->ids, SC_ERR_ARG, "null x, out or ids");
  int64_t need = 0;
  sc_adapters_workspace(s, a->tokens, &need);
  require(need == 0 || (a->workspace && a->workspace_bytes >= need &&
                        reinterpret_cast<uintptr_t>(a->workspace) % 16 == 0),
          SC_ERR_ARG, "workspace missing, too small or not 16-byte aligned");
  DeviceGuard dg(s->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  with_types(a->type, s->type, [&](auto t, auto w) {
    using T = decltype(t);
    using W = decltype(w);
    const bool few = a->tokens <= kFewTokens;
    const Scratch sc = few ? Scratch{} : scratch_of(s->view, a->tokens, a->workspace);
    const int64_t clusters = few ? a->tokens : sc.most_tiles;
    require(clusters <= 65535, SC_ERR_UNSUPPORTED, "too many tokens in one call");
    if (!few) group_kernel<<<1, 1024, 0, st>>>(s->view, a->ids, (int)a->tokens, sc.heads, sc.tokens, sc.tiles, sc.n_tiles);
    // Blocks a cluster.  Few tokens: eight, fewer while they would not all run at once (the clusters of tokens that lead
    // no group come and go, but each costs its turn) and a block's share of an adapter stays below 32 KB: 4 x 148 blocks
    // of 22 KB instead of 7 x 148 of 44 KB took 15.6 us instead of 22.4 (128 tokens, 100 adapters of 512 x 2048), but
    // 38 us instead of 23 where they hold 147 and 74 KB (96 tokens, 40 adapters of 4096 x 4096).  Prompts: two a SM.
    int blocks = kMaxCluster;
    if (few)
      while (blocks > 2 && clusters * blocks > 4 * 148 && s->mean_bytes / blocks < 32 << 10) blocks /= 2;
    else
      while (blocks > 2 && clusters * blocks > 2 * 148) blocks /= 2;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = blocks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // the tiles are launched while they are sorted
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(blocks, (unsigned)clusters);
    cfg.blockDim = dim3(few ? kFewThreads : kThreads);
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = few ? 1 : 2;
    if (few) {
      cuda_check(cudaLaunchKernelEx(&cfg, few_kernel<T, W>, s->view, *a), "launch adapters");
      return;
    }
    cfg.dynamicSmemBytes = tile_smem(s->view.rank_max);
    auto kernel = tile_kernel<T, W>;
    static std::atomic<uint64_t> ready{0};  // devices where the kernel may use this much shared memory
    if (!(ready.load() >> s->device & 1)) {
      cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, tile_smem(kMaxRank)),
                 "set shared memory size");
      ready |= (uint64_t)1 << s->device;
    }
    cuda_check(cudaLaunchKernelEx(&cfg, kernel, s->view, *a, Sorted{sc.tiles, sc.tokens, sc.n_tiles}), "launch adapters");
  });
  cuda_check(cudaGetLastError(), "launch adapters");
  SC_SERVE_END
}

}  // extern "C"
