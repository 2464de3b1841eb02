// Decode attention: plan, workspace and launch (the kernel is in sc_attn.cuh).
#include <algorithm>
#include <cmath>
#include <memory>

#include "sc_attn.cuh"

using namespace sc::serve;
using namespace sc::attn;

namespace {

// One instantiation of the kernel and what its launch needs.
struct Variant {
  void (*kernel)(Params);
  int smem, tile, record, per_sm;
};

template <int MODE, int DP>
Variant variant() {
  using C = Cfg<MODE, DP>;
  Variant v{attend_kernel<MODE, DP>, C::smem, C::tile, C::record, 0};
  cuda_check(cudaFuncSetAttribute(v.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, v.smem),
             "set shared memory size");
  cuda_check(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&v.per_sm, v.kernel, kThreads, v.smem), "occupancy");
  require(v.per_sm > 0, SC_ERR_CUDA, "the attention kernel does not fit this GPU");
  return v;
}

template <int MODE>
Variant variant_for(int64_t head_dim) {
  return head_dim <= 64 ? variant<MODE, 64>() : head_dim <= 128 ? variant<MODE, 128>() : variant<MODE, 256>();
}

}  // namespace

struct sc_attn {
  sc_kv_pool pool;
  int device = 0;
  int64_t q_heads = 0, max_seqs = 0, window = 0;
  float scale = 0.f;
  int qtiles = 0, sms = 0, min_tiles = 1;
  Variant same, other;  // q of the cache's type; q of another type
  DeviceBlock mem;      // status | arrivals | partial records
  int *status = nullptr, *arrivals = nullptr;
  float *partials = nullptr;
};

extern "C" {

int sc_attn_create(const sc_kv_cache *cache, int64_t q_heads, int64_t max_seqs, double scale, int64_t window,
                   sc_attn **out) {
  SC_SERVE_BEGIN
  require(cache && out, SC_ERR_ARG, "null argument");
  *out = nullptr;
  const sc_kv_pool &pool = cache->pool;
  require(q_heads > 0 && q_heads % pool.kv_heads == 0 && q_heads <= 65535, SC_ERR_ARG,
          "q_heads must be a positive multiple of kv_heads");
  require(max_seqs > 0 && max_seqs <= (1 << 20), SC_ERR_ARG, "max_seqs must be 1 to 2^20");
  require(std::isfinite(scale) && scale >= 0, SC_ERR_ARG, "scale must be positive and finite");
  require(window >= 0, SC_ERR_ARG, "negative window");
  std::unique_ptr<sc_attn> p(new sc_attn);
  p->pool = pool;
  p->device = cache->device;
  p->q_heads = q_heads;
  p->max_seqs = max_seqs;
  p->window = std::min<int64_t>(window, INT32_MAX);
  p->scale = (float)(scale > 0 ? scale : 1.0 / std::sqrt((double)pool.head_dim));
  p->qtiles = (int)((q_heads / pool.kv_heads + kQT - 1) / kQT);
  const int64_t segments = max_seqs * pool.kv_heads * p->qtiles;
  require(segments < INT32_MAX, SC_ERR_UNSUPPORTED, "max_seqs times heads reaches 2^31");
  DeviceGuard dg(p->device);
  cuda_check(cudaDeviceGetAttribute(&p->sms, cudaDevAttrMultiProcessorCount, p->device), "device attribute");
  if (pool.type == SC_TYPE_F32) {
    p->same = p->other = variant_for<kTF32>(pool.head_dim);
  } else if (pool.type == SC_TYPE_F16) {
    p->same = variant_for<kF16>(pool.head_dim);
    p->other = variant_for<kF16Wide>(pool.head_dim);
  } else {
    p->same = variant_for<kBF16>(pool.head_dim);
    p->other = variant_for<kBF16Wide>(pool.head_dim);
  }
  const size_t blocks = (size_t)std::max(p->same.per_sm, p->other.per_sm) * p->sms;
  require(blocks * kQT * 4 <= (size_t)std::min(p->same.smem, p->other.smem), SC_ERR_UNSUPPORTED,
          "more blocks than the join has room for");
  const size_t words = 64 + ((size_t)segments + 63) / 64 * 64;
  p->mem.alloc(p->device, words * 4 + blocks * 2 * p->same.record * 4, "allocate attention workspace");
  cuda_check(cudaMemset(p->mem.p, 0, words * 4), "clear attention workspace");
  cuda_check(cudaDeviceSynchronize(), "device synchronize");
  p->status = static_cast<int *>(p->mem.p);
  p->arrivals = p->status + 64;
  p->partials = reinterpret_cast<float *>(p->status + words);
  *out = p.release();
  SC_SERVE_END
}

void sc_attn_free(sc_attn *p) { delete p; }

int sc_attn_status(sc_attn *p, int32_t *status) {
  SC_SERVE_BEGIN
  require(p && status, SC_ERR_ARG, "null argument");
  *status = take_status(p->device, p->status);
  SC_SERVE_END
}

int sc_attn_decode(sc_attn *p, const sc_attn_args *a, void *stream) {
  SC_SERVE_BEGIN
  require(p && a, SC_ERR_ARG, "null argument");
  require(a->seqs >= 0 && a->seqs <= p->max_seqs, SC_ERR_ARG, "more sequences than the plan's max_seqs");
  if (a->seqs == 0) return SC_OK;
  require(type_ok(a->type), SC_ERR_ARG, "unknown element type");
  require(a->q.ptr && a->out.ptr && a->page_table && a->seq_lens, SC_ERR_ARG,
          "null q, out, page table or lengths");
  require(a->table_cols >= 0 && a->table_stride >= 0, SC_ERR_ARG, "bad page table sizes");
  const Variant &v = a->type == p->pool.type ? p->same : p->other;
  Params k{*a,           p->pool,    (int)p->q_heads, (int)(p->q_heads / p->pool.kv_heads), p->qtiles, p->min_tiles,
           (float)(p->scale * 1.4426950408889634), p->window, p->status, p->arrivals, p->partials};
  // the most tiles that these lengths can have; the true number is known on the device only
  int64_t keys = std::min<int64_t>(a->table_cols, INT32_MAX / p->pool.page_size) * p->pool.page_size;
  if (p->window) keys = std::min(keys, p->window + 15);
  const int64_t tiles = std::max<int64_t>(1, (keys + v.tile - 1) / v.tile) * a->seqs * p->pool.kv_heads * p->qtiles;
  const int64_t blocks = std::min<int64_t>(tiles, (int64_t)v.per_sm * p->sms);
  DeviceGuard dg(p->device);
  v.kernel<<<(unsigned)blocks, kThreads, v.smem, static_cast<cudaStream_t>(stream)>>>(k);
  cuda_check(cudaGetLastError(), "launch decode attention");
  SC_SERVE_END
}

}  // extern "C"
