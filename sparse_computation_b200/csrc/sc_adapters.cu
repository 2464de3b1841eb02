// Low-rank adapters of many requests beside a shared projection.
#include <algorithm>
#include <cmath>
#include <memory>
#include <vector>

#include <cooperative_groups.h>

#include "sc_serve.h"

using namespace sc::serve;
namespace cg = cooperative_groups;

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

template <class W>
__global__ void pack_rows(const W *src, int64_t row_stride, int64_t col_stride, int64_t rows, int64_t cols, W *dst,
                          int64_t dst_row) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, r = i / dst_row, c = i % dst_row;
  if (r < rows) dst[i] = c < cols ? src[r * row_stride + c * col_stride] : W(0);
}

__device__ __forceinline__ int adapter_of(const SetView &s, const int32_t *ids, int64_t t) {
  const int a = ids[t];
  if (a >= s.count) {
    set_status(s.status, 10);
    return -1;
  }
  return a;
}

// One warp per (token, rank row): v = scale * down x.
template <class T, class W>
__global__ void __launch_bounds__(256) shrink_kernel(const SetView s, const sc_adapters_args a, float *v) {
  const int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / 32;
  const int lane = threadIdx.x % 32;
  if (i >= a.tokens * s.rank_max) return;
  const int64_t t = i / s.rank_max, r = i % s.rank_max;
  const int ad = adapter_of(s, a.ids, t);
  if (ad < 0 || r >= s.first[ad + 1] - s.first[ad]) return;
  const W *w = static_cast<const W *>(s.down) + (s.first[ad] + r) * s.in_row;
  const T *x = static_cast<const T *>(a.x.ptr) + t * a.x.stride[1];
  float sum = 0.f;
  for (int64_t k = lane; k < s.in; k += 32) sum += to_f32(w[k]) * to_f32(x[k * a.x.stride[0]]);
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
  if (lane == 0) v[i] = sum * s.scale[ad];
}

// One thread per output element: out = base + up v.
template <class T, class W>
__global__ void __launch_bounds__(256) expand_kernel(const SetView s, const sc_adapters_args a, const float *v) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= a.tokens * s.out) return;
  const int64_t t = i / s.out, m = i % s.out;
  float y = 0.f;
  if (a.base.ptr) y = to_f32(static_cast<const T *>(a.base.ptr)[m * a.base.stride[0] + t * a.base.stride[1]]);
  const int ad = adapter_of(s, a.ids, t);
  if (ad >= 0) {
    const int r0 = s.first[ad], n = s.first[ad + 1] - r0;
    float sum = 0.f;
    for (int r = 0; r < n; ++r)
      sum += v[t * s.rank_max + r] * to_f32(static_cast<const W *>(s.up)[(int64_t)(r0 + r) * s.out_row + m]);
    y += sum;
  }
  static_cast<T *>(a.out.ptr)[m * a.out.stride[0] + t * a.out.stride[1]] = from_f32<T>(y);
}

// ------------------------------------------------------ a few tokens ----
//
// Up to kFewTokens tokens (a decoding step): what counts is reading each
// adapter's weights once and at once.  A cluster of eight blocks takes up to
// eight tokens that share an adapter: the cluster of a token whose place among
// its adapter's tokens is a multiple of eight takes that one and the next
// seven, the others' clusters leave.  Block c multiplies columns c of eight
// parts of `down` with its part of x, so that x is read once, too; the eight
// parts of v = down x are added up through distributed shared memory, in block
// order; then block c makes rows c of eight parts of up v.  One launch, no
// scratch memory.  Bound by the weights' bytes, and by latency below some MB.
constexpr int kFewTokens = 256, kCluster = 8, kGroup = 8, kChunk = 512, kFewThreads = 256;

// Eight weights as floats.
template <class W>
__device__ __forceinline__ void load8(const W *p, float (&x)[8]) {
  uint4 w[sizeof(W) / 2];
#pragma unroll
  for (int i = 0; i < (int)sizeof(W) / 2; ++i) w[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
  const W *v = reinterpret_cast<const W *>(w);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = to_f32(v[i]);
}

struct FewShared {
  float x[kGroup][kChunk];          // this block's part of the tokens' x
  float part[kMaxRank][kGroup];     // its part of v, read by the whole cluster
  float v[kMaxRank][kGroup];        // scale * v
  float sums[kFewThreads * 8];
  int tokens[kGroup];
  int count[kFewThreads / 32], n;
};

// v parts of the rows of one adapter from `width` columns: a warp takes rows, LANES lanes a row.
template <int NT, class W>
__device__ __forceinline__ void few_shrink(FewShared &sh, const W *down, int64_t row, int rank, int width) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  // lanes of a row: a power of two, eight columns each
  int lanes = 32;
  while (lanes > 1 && lanes * 4 >= width) lanes >>= 1;
  const int sub = lane / lanes, in = lane % lanes, rows = 32 / lanes;
  for (int r0 = warp * rows; r0 < rank; r0 += kFewThreads / 32 * rows) {
    const int r = r0 + sub;
    float acc[NT] = {};
    if (r < rank)
      for (int k = in * 8; k < width; k += lanes * 8) {
        float w[8];
        load8(down + r * row + k, w);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const float4 a = *reinterpret_cast<const float4 *>(&sh.x[t][k]);
          const float4 b = *reinterpret_cast<const float4 *>(&sh.x[t][k + 4]);
          acc[t] += w[0] * a.x + w[1] * a.y + w[2] * a.z + w[3] * a.w + w[4] * b.x + w[5] * b.y + w[6] * b.z + w[7] * b.w;
        }
      }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      for (int d = lanes / 2; d; d >>= 1) acc[t] += __shfl_xor_sync(~0u, acc[t], d);
      if (in == 0 && r < rank) sh.part[r][t] += acc[t];
    }
  }
}

// Rows [m0, m0 + rows) of up v for NT tokens; groups of threads take every so-manieth rank row, their sums are added
// up token by token.
template <int NT, class T, class W>
__device__ __forceinline__ void few_expand(FewShared &sh, const sc_adapters_args &a, const W *up, int64_t row, int rank, int m0,
                                           int rows) {
  for (int base = 0; base < rows; base += kFewThreads * 8) {
    const int here = min(rows - base, kFewThreads * 8), eights = (here + 7) / 8;
    const int sets = kFewThreads / eights, set = threadIdx.x / eights, at = base + threadIdx.x % eights * 8;
    float acc[NT][8] = {};
    if (set < sets)
#pragma unroll 4
      for (int r = set; r < rank; r += sets) {
        float w[8];
        load8(up + r * row + m0 + at, w);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const float v = sh.v[r][t];
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[t][e] += w[e] * v;
        }
      }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (t >= sh.n) break;
      __syncthreads();
      if (set < sets)
#pragma unroll
        for (int e = 0; e < 8; e += 4)
          *reinterpret_cast<float4 *>(&sh.sums[set * eights * 8 + at - base + e]) =
              make_float4(acc[t][e], acc[t][e + 1], acc[t][e + 2], acc[t][e + 3]);
      __syncthreads();
      const int64_t token = sh.tokens[t];
      for (int i = threadIdx.x; i < here; i += kFewThreads) {
        const int64_t m = m0 + base + i;
        float y = 0.f;
        for (int s = 0; s < sets; ++s) y += sh.sums[s * eights * 8 + i];
        if (a.base.ptr) y += to_f32(static_cast<const T *>(a.base.ptr)[m * a.base.stride[0] + token * a.base.stride[1]]);
        static_cast<T *>(a.out.ptr)[m * a.out.stride[0] + token * a.out.stride[1]] = from_f32<T>(y);
      }
    }
  }
}

template <class T, class W>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kFewThreads)
    few_kernel(const __grid_constant__ SetView s, const __grid_constant__ sc_adapters_args a) {
  __shared__ FewShared sh;
  const int c = blockIdx.x, t = blockIdx.y, tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int n_tokens = (int)a.tokens;
  const int id = a.ids[t];
  const int other = tid < n_tokens ? a.ids[tid] : -1;
  const int rank = id >= 0 && id < s.count ? s.first[id + 1] - s.first[id] : 0;
  // this block's columns of x and rows of out
  const int k0 = (int)(s.in_row / kCluster) * c, k1 = min((int)s.in, k0 + (int)(s.in_row / kCluster));
  const int m0 = (int)(s.out_row / kCluster) * c, m1 = min((int)s.out, m0 + (int)(s.out_row / kCluster));
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
  const W *down = static_cast<const W *>(s.down) + s.first[id] * s.in_row, *up = static_cast<const W *>(s.up) + s.first[id] * s.out_row;
  for (int k = k0; k < k1; k += kChunk) {
    const int width = min(kChunk, k1 - k), wide = (width + 7) / 8 * 8;
    for (int i = tid; i < kGroup * wide; i += kFewThreads) {
      const int g = i / wide, kk = i - g * wide;
      sh.x[g][kk] = g < n && kk < width
                        ? to_f32(static_cast<const T *>(a.x.ptr)[(k + kk) * a.x.stride[0] + sh.tokens[g] * a.x.stride[1]])
                        : 0.f;
    }
    __syncthreads();
    if (n == 1)
      few_shrink<1>(sh, down + k, s.in_row, rank, wide);
    else if (n == 2)
      few_shrink<2>(sh, down + k, s.in_row, rank, wide);
    else if (n <= 4)
      few_shrink<4>(sh, down + k, s.in_row, rank, wide);
    else
      few_shrink<8>(sh, down + k, s.in_row, rank, wide);
    __syncthreads();
  }
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  const float scale = s.scale[id];
  for (int i = tid; i < rank * kGroup; i += kFewThreads) {
    float v = 0.f;
    for (int b = 0; b < kCluster; ++b) v += cluster.map_shared_rank(&sh.part[0][0], b)[i];
    sh.v[i / kGroup][i % kGroup] = v * scale;
  }
  cluster.sync();  // no block leaves, or goes on, before all have read
  if (m1 <= m0) return;
  if (n == 1)
    few_expand<1, T>(sh, a, up, s.out_row, rank, m0, m1 - m0);
  else if (n == 2)
    few_expand<2, T>(sh, a, up, s.out_row, rank, m0, m1 - m0);
  else if (n <= 4)
    few_expand<4, T>(sh, a, up, s.out_row, rank, m0, m1 - m0);
  else
    few_expand<8, T>(sh, a, up, s.out_row, rank, m0, m1 - m0);
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

}  // namespace

struct sc_adapters {
  int device = 0;
  int64_t type = 0;
  SetView view{};
  DeviceBlock mem;
};

extern "C" {

int sc_adapters_create(int32_t device, int64_t in_features, int64_t out_features, int64_t count,
                       const int64_t *ranks, int64_t type, const void *const *down, const int64_t *down_ld,
                       const void *const *up, const int64_t *up_ld, const float *scales, void *stream,
                       sc_adapters **out) {
  SC_SERVE_BEGIN
  require(out && ranks && down && down_ld && up && up_ld && scales, SC_ERR_ARG, "null argument");
  *out = nullptr;
  require(count > 0 && count < (1 << 24), SC_ERR_ARG, "a set has 1 to 2^24 adapters");
  require(in_features > 0 && out_features > 0 && in_features < (1 << 24) && out_features < (1 << 24), SC_ERR_ARG,
          "features must be 1 to 2^24");
  require(type_ok(type), SC_ERR_ARG, "unknown element type");
  std::vector<int32_t> first(count + 1, 0);
  int64_t total = 0, most = 0;
  for (int64_t i = 0; i < count; ++i) {
    require(ranks[i] >= 0 && ranks[i] <= kMaxRank, SC_ERR_UNSUPPORTED, "ranks must be 0 to 256");
    require(ranks[i] == 0 || (down[i] && up[i] && down_ld[i] >= in_features && up_ld[i] >= ranks[i]), SC_ERR_ARG,
            "null adapter weights or row stride too small");
    total += ranks[i];
    most = std::max(most, ranks[i]);
    require(total < INT32_MAX, SC_ERR_UNSUPPORTED, "too many rank rows in one set");
    first[i + 1] = (int32_t)total;
  }
  const size_t e = (size_t)type_bytes(type);
  const int64_t in_row = (in_features + kPad - 1) / kPad * kPad, out_row = (out_features + kPad - 1) / kPad * kPad;
  const size_t b_down = align256(total * in_row * e + 16), b_up = align256(total * out_row * e + 16);
  const size_t b_first = align256((count + 1) * 4), b_scale = align256(count * 4);
  std::unique_ptr<sc_adapters> s(new sc_adapters);
  s->device = device;
  s->type = type;
  DeviceGuard dg(device);
  s->mem.alloc(device, b_down + b_up + b_first + b_scale + 256, "allocate adapters");
  uint8_t *p = static_cast<uint8_t *>(s->mem.p);
  uint8_t *d_down = p, *d_up = d_down + b_down, *d_first = d_up + b_up, *d_scale = d_first + b_first,
          *d_status = d_scale + b_scale;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cuda_check(cudaMemcpyAsync(d_first, first.data(), (count + 1) * 4, cudaMemcpyHostToDevice, st), "upload adapters");
  cuda_check(cudaMemcpyAsync(d_scale, scales, count * 4, cudaMemcpyHostToDevice, st), "upload adapters");
  cuda_check(cudaMemsetAsync(d_status, 0, 256, st), "clear status word");
  auto pack = [&](const void *src, int64_t rs, int64_t cs, int64_t rows, int64_t cols, uint8_t *dst, int64_t dst_row) {
    const unsigned blocks = (unsigned)((rows * dst_row + 255) / 256);
    if (e == 4)
      pack_rows<<<blocks, 256, 0, st>>>(static_cast<const uint32_t *>(src), rs, cs, rows, cols,
                                        reinterpret_cast<uint32_t *>(dst), dst_row);
    else
      pack_rows<<<blocks, 256, 0, st>>>(static_cast<const uint16_t *>(src), rs, cs, rows, cols,
                                        reinterpret_cast<uint16_t *>(dst), dst_row);
  };
  for (int64_t i = 0; i < count; ++i) {
    if (!ranks[i]) continue;
    pack(down[i], down_ld[i], 1, ranks[i], in_features, d_down + (size_t)first[i] * in_row * e, in_row);
    pack(up[i], 1, up_ld[i], ranks[i], out_features, d_up + (size_t)first[i] * out_row * e, out_row);
  }
  cuda_check(cudaGetLastError(), "launch adapter packing");
  cuda_check(cudaStreamSynchronize(st), "stream synchronize");
  s->view = SetView{d_down,          d_up,        reinterpret_cast<int32_t *>(d_first), reinterpret_cast<float *>(d_scale),
                    in_features,     out_features, in_row, out_row, (int)count, (int)most, reinterpret_cast<int *>(d_status)};
  *out = s.release();
  SC_SERVE_END
}

void sc_adapters_free(sc_adapters *s) { delete s; }

int sc_adapters_workspace(const sc_adapters *s, int64_t tokens, int64_t *bytes) {
  SC_SERVE_BEGIN
  require(s && bytes && tokens >= 0, SC_ERR_ARG, "null argument or negative token count");
  *bytes = tokens <= kFewTokens ? 0 : (int64_t)align256((size_t)tokens * s->view.rank_max * 4);
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
  float *v = static_cast<float *>(a->workspace);
  with_types(a->type, s->type, [&](auto t, auto w) {
    using T = decltype(t);
    using W = decltype(w);
    if (a->tokens <= kFewTokens) {
      few_kernel<T, W><<<dim3(kCluster, (unsigned)a->tokens), kFewThreads, 0, st>>>(s->view, *a);
      return;
    }
    const int64_t warps = a->tokens * s->view.rank_max, elems = a->tokens * s->view.out;
    if (warps) shrink_kernel<decltype(t), decltype(w)><<<(unsigned)((warps + 7) / 8), 256, 0, st>>>(s->view, *a, v);
    expand_kernel<decltype(t), decltype(w)><<<(unsigned)((elems + 255) / 256), 256, 0, st>>>(s->view, *a, v);
  });
  cuda_check(cudaGetLastError(), "launch adapters");
  SC_SERVE_END
}

}  // extern "C"
