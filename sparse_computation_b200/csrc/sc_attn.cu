// Decode attention: plan, workspace and launch (the kernel is in sc_attn.cuh).
#include <algorithm>
#include <cmath>
#include <memory>

#include "sc_attn.cuh"

using namespace sc::serve;
using namespace sc::attn;

struct sc_attn {
  sc_kv_pool pool;
  int device = 0;
  int64_t q_heads = 0, max_seqs = 0, window = 0;
  float scale_log2 = 0.f;
  int qtiles = 0, q_rows = 0, sms = 0;
  uint32_t page_mul = 0, page_shift = 0;
  Variant same, other;  // q of the cache's type; q of another type
  DeviceBlock mem;      // its own workspace, if any: status | 1 KB of zeros | arrivals | doubtful rows | pieces | records
  int *status = nullptr, *arrivals = nullptr;
  uint32_t *doubtful = nullptr;
  float *heads = nullptr, *records = nullptr;
};

namespace {

// A plan without its workspace, and the layout of that in 4-byte words.
struct Layout {
  size_t segments, words, heads, total;  // arrivals; status, zeros, arrivals and doubtful rows; pieces; all
};

std::unique_ptr<sc_attn> set_up(const sc_kv_cache *cache, int64_t q_heads, int64_t max_seqs, double scale, int64_t window,
                                Layout &layout) {
  const sc_kv_pool &pool = cache->pool;
  require(q_heads > 0 && q_heads % pool.kv_heads == 0 && q_heads <= 65535, SC_ERR_ARG,
          "q_heads must be a positive multiple of kv_heads");
  require(max_seqs > 0 && max_seqs <= (1 << 20), SC_ERR_ARG, "max_seqs must be 1 to 2^20");
  require(std::isfinite((float)(scale * 1.4426950408889634)) && scale >= 0, SC_ERR_ARG,
          "scale must be positive and finite, in fp32 too");
  require(window >= 0, SC_ERR_ARG, "negative window");
  std::unique_ptr<sc_attn> p(new sc_attn);
  p->pool = pool;
  p->device = cache->device;
  p->q_heads = q_heads;
  p->max_seqs = max_seqs;
  p->window = std::min<int64_t>(window, INT32_MAX);
  p->scale_log2 = (float)((scale > 0 ? scale : 1.0 / std::sqrt((double)pool.head_dim)) * 1.4426950408889634);
  p->qtiles = (int)((q_heads / pool.kv_heads + kQT - 1) / kQT);
  const int64_t segments = max_seqs * pool.kv_heads * p->qtiles;
  // a run of one block is counted in 32 bits
  require(segments < INT32_MAX, SC_ERR_UNSUPPORTED, "max_seqs times heads reaches 2^31");
  p->q_rows = (int)std::min<int64_t>(q_heads / pool.kv_heads, kQT);
  // key / page_size for keys below 2^31: multiply by 2^(31 + bits) / page_size, rounded up
  for (int bits = 1; pool.page_size > 1; ++bits)
    if (((int64_t)1 << bits) >= pool.page_size) {
      p->page_mul = (uint32_t)((((uint64_t)1 << (31 + bits)) + pool.page_size - 1) / pool.page_size);
      p->page_shift = bits - 1;
      break;
    }
  const int64_t unit = 16 / type_bytes(pool.type);
  for (const int64_t *st : {pool.k_stride, pool.v_stride})
    require(((pool.num_pages - 1) * st[0] + (pool.page_size - 1) * st[2]) / unit <= UINT32_MAX, SC_ERR_UNSUPPORTED,
            "a cache pool of 64 GB or more");
  DeviceGuard dg(p->device);
  int limit = 0;
  cuda_check(cudaDeviceGetAttribute(&p->sms, cudaDevAttrMultiProcessorCount, p->device), "device attribute");
  cuda_check(cudaDeviceGetAttribute(&limit, cudaDevAttrMaxSharedMemoryPerBlockOptin, p->device), "device attribute");
  if (pool.type == SC_TYPE_F32) {
    p->same = p->other = variant_for<kTF32>(pool.head_dim, p->q_rows, limit);
  } else if (pool.type == SC_TYPE_F16) {
    p->same = variant_for<kF16>(pool.head_dim, p->q_rows, limit);
    p->other = variant_for<kF16Wide>(pool.head_dim, p->q_rows, limit);
  } else {
    p->same = variant_for<kBF16>(pool.head_dim, p->q_rows, limit);
    // three parts of up to four query heads share an instruction's 16 rows
    p->other = p->q_rows <= 4 ? variant_for<kBF16Wide4>(pool.head_dim, p->q_rows, limit)
                              : variant_for<kBF16Wide>(pool.head_dim, p->q_rows, limit);
  }
  const size_t piece = (size_t)p->same.piece;
  layout.segments = ((size_t)segments + 63) / 64 * 64;
  layout.words = 64 + 256 + 2 * layout.segments;
  layout.heads = (size_t)p->sms * std::max(p->same.warps, p->other.warps) * piece;
  layout.total = layout.words + layout.heads + (size_t)p->sms * 2 * piece;
  return p;
}

void give_workspace(sc_attn &p, void *at, const Layout &layout) {
  clear_words(at, layout.words * 4);
  p.status = static_cast<int *>(at);
  p.arrivals = p.status + 64 + 256;
  p.doubtful = reinterpret_cast<uint32_t *>(p.arrivals + layout.segments);
  p.heads = reinterpret_cast<float *>(p.status + layout.words);
  p.records = p.heads + layout.heads;
}

}  // namespace

extern "C" {

int sc_attn_workspace(const sc_kv_cache *cache, int64_t q_heads, int64_t max_seqs, int64_t *bytes) {
  SC_SERVE_BEGIN
  require(cache && bytes, SC_ERR_ARG, "null argument");
  Layout layout;
  set_up(cache, q_heads, max_seqs, 1.0, 0, layout);
  *bytes = (int64_t)layout.total * 4;
  SC_SERVE_END
}

int sc_attn_create(const sc_kv_cache *cache, int64_t q_heads, int64_t max_seqs, double scale, int64_t window,
                   sc_attn **out) {
  SC_SERVE_BEGIN
  require(cache && out, SC_ERR_ARG, "null argument");
  *out = nullptr;
  Layout layout;
  auto p = set_up(cache, q_heads, max_seqs, scale, window, layout);
  DeviceGuard dg(p->device);
  p->mem.alloc(p->device, layout.total * 4, "allocate attention workspace");
  give_workspace(*p, p->mem.p, layout);
  *out = p.release();
  SC_SERVE_END
}

int sc_attn_create_in(const sc_kv_cache *cache, int64_t q_heads, int64_t max_seqs, double scale, int64_t window,
                      void *workspace, int64_t workspace_bytes, sc_attn **out) {
  SC_SERVE_BEGIN
  require(cache && out && workspace, SC_ERR_ARG, "null argument");
  *out = nullptr;
  Layout layout;
  auto p = set_up(cache, q_heads, max_seqs, scale, window, layout);
  require(workspace_bytes >= (int64_t)layout.total * 4 && reinterpret_cast<uintptr_t>(workspace) % 256 == 0, SC_ERR_ARG,
          "workspace too small or not 256-byte aligned");
  DeviceGuard dg(p->device);
  give_workspace(*p, workspace, layout);
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
  const int64_t unit = 16 / type_bytes(p->pool.type);  // elements in 16 bytes
  const int64_t qe = type_bytes(a->type);
  const int q_vec = a->q.stride[2] == 1 && a->q.stride[1] * qe % 16 == 0 && a->q.stride[0] * qe % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(a->q.ptr) % 16 == 0 && p->pool.head_dim * qe % 16 == 0;
  Params k{*a, p->pool, (int)p->q_heads, (int)(p->q_heads / p->pool.kv_heads), p->qtiles, p->q_rows, v.warps, q_vec,
           p->page_mul, p->page_shift, (uint32_t)(p->pool.k_stride[0] / unit), (uint32_t)(p->pool.k_stride[2] / unit),
           (uint32_t)(p->pool.v_stride[0] / unit), (uint32_t)(p->pool.v_stride[2] / unit),
           p->scale_log2, p->window, p->status,
           reinterpret_cast<const uint8_t *>(p->status + 64), p->arrivals, p->doubtful, p->heads, p->records};
  // the most steps that these lengths can have; the true number is known on the device only
  int64_t keys = std::min<int64_t>(a->table_cols, INT32_MAX / p->pool.page_size) * p->pool.page_size;
  if (p->window) keys = std::min(keys, p->window + 15);
  const int64_t per_seq = std::max<int64_t>(1, (keys + v.keys - 1) / v.keys) + v.change, units = p->pool.kv_heads * p->qtiles;
  // places are counted in 32 bits, and a block's run may end one run beyond the last
  require(per_seq * a->seqs * units < INT32_MAX / 2, SC_ERR_UNSUPPORTED,
          "the page table names more keys than one call can take");
  const int64_t blocks = std::min<int64_t>((per_seq * a->seqs * units + v.warps - 1) / v.warps, p->sms);
  DeviceGuard dg(p->device);
  v.kernel<<<(unsigned)blocks, v.warps * 32, v.smem, static_cast<cudaStream_t>(stream)>>>(k);
  cuda_check(cudaGetLastError(), "launch decode attention");
  SC_SERVE_END
}

}  // extern "C"
