// Low-rank adapters of many requests beside a shared projection.
#include <cmath>
#include <memory>
#include <vector>

#include "sc_serve.h"

using namespace sc::serve;

namespace {

constexpr int64_t kMaxRank = 256;

// What the kernels read of a set.  Rows first[i] .. first[i+1] of `down`
// (rank rows of in_features) and of `up` (rank rows of out_features: up is
// stored transposed) are adapter i's.
struct SetView {
  const void *down, *up;
  const int32_t *first;  // [count + 1]
  const float *scale;    // [count]
  int64_t in, out;
  int count, rank_max;
  int *status;
};

template <class W>
__global__ void pack_rows(const W *src, int64_t row_stride, int64_t col_stride, int64_t rows, int64_t cols, W *dst) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i < rows * cols) dst[i] = src[(i / cols) * row_stride + (i % cols) * col_stride];
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
  const W *w = static_cast<const W *>(s.down) + (s.first[ad] + r) * s.in;
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
      sum += v[t * s.rank_max + r] * to_f32(static_cast<const W *>(s.up)[(int64_t)(r0 + r) * s.out + m]);
    y += sum;
  }
  static_cast<T *>(a.out.ptr)[m * a.out.stride[0] + t * a.out.stride[1]] = from_f32<T>(y);
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
  const size_t b_down = align256(total * in_features * e + 16), b_up = align256(total * out_features * e + 16);
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
  auto pack = [&](const void *src, int64_t rs, int64_t cs, int64_t rows, int64_t cols, uint8_t *dst) {
    const unsigned blocks = (unsigned)((rows * cols + 255) / 256);
    if (e == 4)
      pack_rows<<<blocks, 256, 0, st>>>(static_cast<const uint32_t *>(src), rs, cs, rows, cols,
                                        reinterpret_cast<uint32_t *>(dst));
    else
      pack_rows<<<blocks, 256, 0, st>>>(static_cast<const uint16_t *>(src), rs, cs, rows, cols,
                                        reinterpret_cast<uint16_t *>(dst));
  };
  for (int64_t i = 0; i < count; ++i) {
    if (!ranks[i]) continue;
    pack(down[i], down_ld[i], 1, ranks[i], in_features, d_down + (size_t)first[i] * in_features * e);
    pack(up[i], 1, up_ld[i], ranks[i], out_features, d_up + (size_t)first[i] * out_features * e);
  }
  cuda_check(cudaGetLastError(), "launch adapter packing");
  cuda_check(cudaStreamSynchronize(st), "stream synchronize");
  s->view = SetView{d_down,          d_up,        reinterpret_cast<int32_t *>(d_first), reinterpret_cast<float *>(d_scale),
                    in_features,     out_features, (int)count, (int)most, reinterpret_cast<int *>(d_status)};
  *out = s.release();
  SC_SERVE_END
}

void sc_adapters_free(sc_adapters *s) { delete s; }

int sc_adapters_workspace(const sc_adapters *s, int64_t tokens, int64_t *bytes) {
  SC_SERVE_BEGIN
  require(s && bytes && tokens >= 0, SC_ERR_ARG, "null argument or negative token count");
  *bytes = (int64_t)align256((size_t)tokens * s->view.rank_max * 4);
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
    const int64_t warps = a->tokens * s->view.rank_max, elems = a->tokens * s->view.out;
    if (warps) shrink_kernel<decltype(t), decltype(w)><<<(unsigned)((warps + 7) / 8), 256, 0, st>>>(s->view, *a, v);
    expand_kernel<decltype(t), decltype(w)><<<(unsigned)((elems + 255) / 256), 256, 0, st>>>(s->view, *a, v);
  });
  cuda_check(cudaGetLastError(), "launch adapters");
  SC_SERVE_END
}

}  // extern "C"
