// Cache append with the rotary rotation.
#include <cmath>
#include <memory>

#include "sc_serve.h"

using namespace sc::serve;

namespace {

constexpr int64_t kMaxHeadDim = 256;  // the widest tile of the attention kernel

// --------------------------------------------------------------- append ----

struct AppendParams {
  sc_kv_append_args a;
  sc_kv_pool pool;
  int *status;
};

// The cache place of token t: page and slot, or page -1 when it is skipped.
__device__ __forceinline__ void token_place(const AppendParams &p, int64_t t, int &pos, int &page, int &slot) {
  const sc_kv_append_args &a = p.a;
  page = -1;
  slot = 0;
  pos = a.positions[t];
  if (pos < 0) return;
  const int64_t seq = a.seq_ids ? a.seq_ids[t] : t;
  const int col = pos / (int)p.pool.page_size;
  if (seq < 0 || seq >= a.seqs || col >= a.table_cols) {
    set_status(p.status, 8);
    return;
  }
  const int e = a.page_table[seq * a.table_stride + col];
  if (e < 0 || e >= p.pool.num_pages) {
    set_status(p.status, 8);
    return;
  }
  if (a.cos && pos >= a.rope_rows) {
    set_status(p.status, 9);
    return;
  }
  page = e;
  slot = pos - col * (int)p.pool.page_size;
}

// One thread per pair of dims that rotate together (or two neighbouring ones
// that do not) of one head of one token.
template <class T, class C>
__global__ void __launch_bounds__(256) append_kernel(const AppendParams p) {
  const sc_kv_append_args &a = p.a;
  const int pairs = (int)p.pool.head_dim / 2;
  const int hk = (int)p.pool.kv_heads, hq = a.q.ptr ? (int)a.q_heads : 0;
  const int64_t per_token = (int64_t)(hq + 2 * hk) * pairs;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= a.tokens * per_token) return;
  const int64_t t = i / per_token;
  const int rest = (int)(i - t * per_token);
  int head = rest / pairs;
  const int pr = rest - head * pairs;
  int pos, page, slot;
  token_place(p, t, pos, page, slot);
  const int half = a.cos ? (int)a.rotary / 2 : 0;
  int d0, d1;
  if (pr >= half) {
    d0 = 2 * pr;
    d1 = d0 + 1;
  } else if (a.interleaved) {
    d0 = 2 * pr;
    d1 = d0 + 1;
  } else {
    d0 = pr;
    d1 = pr + half;
  }
  const bool is_q = head < hq, is_v = head >= hq + hk;
  const sc_rows &src = is_q ? a.q : is_v ? a.v : a.k;
  if (!is_q) head -= is_v ? hq + hk : hq;
  const T *x = static_cast<const T *>(src.ptr) + t * src.stride[0] + head * src.stride[1];
  float u = to_f32(x[d0 * src.stride[2]]), w = to_f32(x[d1 * src.stride[2]]);
  if (page >= 0 && pr < half && !is_v) {
    const float c = a.cos[pos * a.rope_stride + pr], s = a.sin[pos * a.rope_stride + pr];
    const float ru = u * c - w * s;
    w = w * c + u * s;
    u = ru;
  }
  if (is_q) {
    T *y = static_cast<T *>(a.q_out.ptr) + t * a.q_out.stride[0] + head * a.q_out.stride[1];
    y[d0 * a.q_out.stride[2]] = from_f32<T>(page >= 0 ? u : 0.f);
    y[d1 * a.q_out.stride[2]] = from_f32<T>(page >= 0 ? w : 0.f);
  } else if (page >= 0) {
    const int64_t *st = is_v ? p.pool.v_stride : p.pool.k_stride;
    C *y = static_cast<C *>(is_v ? p.pool.v : p.pool.k) + page * st[0] + head * st[1] + slot * st[2];
    y[d0] = from_f32<C>(u);
    y[d1] = from_f32<C>(w);
  }
}

template <class F>
void with_types(int64_t rows, int64_t cache, F f) {
  auto inner = [&](auto t) {
    if (cache == SC_TYPE_F32)
      f(t, float());
    else if (cache == SC_TYPE_F16)
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

void check_pool(const sc_kv_pool &p) {
  require(p.k && p.v, SC_ERR_ARG, "null cache pool");
  require(type_ok(p.type), SC_ERR_ARG, "unknown cache element type");
  require(p.num_pages > 0 && p.page_size > 0 && p.kv_heads > 0 && p.head_dim > 0, SC_ERR_ARG,
          "cache sizes must be positive");
  require(p.num_pages <= INT32_MAX / p.page_size, SC_ERR_UNSUPPORTED, "the cache has 2^31 slots or more");
  require(p.kv_heads <= 65535, SC_ERR_UNSUPPORTED, "more than 65535 kv heads");
  require(p.head_dim <= kMaxHeadDim, SC_ERR_UNSUPPORTED, "head_dim above 256");
  const int64_t e = type_bytes(p.type);
  require(p.head_dim * e % 16 == 0, SC_ERR_UNSUPPORTED, "head_dim rows of the cache must be multiples of 16 bytes");
  for (int i = 0; i < 3; ++i)
    require(p.k_stride[i] >= 0 && p.v_stride[i] >= 0 && p.k_stride[i] * e % 16 == 0 && p.v_stride[i] * e % 16 == 0,
            SC_ERR_UNSUPPORTED, "cache strides must be non-negative multiples of 16 bytes");
  require(reinterpret_cast<uintptr_t>(p.k) % 16 == 0 && reinterpret_cast<uintptr_t>(p.v) % 16 == 0,
          SC_ERR_UNSUPPORTED, "cache pools must be 16-byte aligned");
}

}  // namespace

extern "C" {

int sc_kv_cache_create(const sc_kv_pool *pool, int32_t device, sc_kv_cache **out) {
  SC_SERVE_BEGIN
  require(pool && out, SC_ERR_ARG, "null argument");
  *out = nullptr;
  check_pool(*pool);
  std::unique_ptr<sc_kv_cache> c(new sc_kv_cache);
  c->pool = *pool;
  c->device = device;
  DeviceGuard dg(device);
  c->status.alloc(device, 256, "allocate status word");
  cuda_check(cudaMemset(c->status.p, 0, 256), "clear status word");
  *out = c.release();
  SC_SERVE_END
}

void sc_kv_cache_free(sc_kv_cache *c) { delete c; }

int sc_kv_cache_status(sc_kv_cache *c, int32_t *status) {
  SC_SERVE_BEGIN
  require(c && status, SC_ERR_ARG, "null argument");
  *status = take_status(c->device, static_cast<int *>(c->status.p));
  SC_SERVE_END
}

int sc_kv_append(sc_kv_cache *c, const sc_kv_append_args *a, void *stream) {
  SC_SERVE_BEGIN
  require(c && a, SC_ERR_ARG, "null argument");
  require(a->tokens >= 0, SC_ERR_ARG, "negative token count");
  if (a->tokens == 0) return SC_OK;
  require(type_ok(a->type), SC_ERR_ARG, "unknown element type");
  require(a->k.ptr && a->v.ptr && a->positions && a->page_table, SC_ERR_ARG, "null k, v, positions or page table");
  require(a->seqs > 0 && a->table_cols >= 0 && a->table_stride >= 0, SC_ERR_ARG, "bad page table sizes");
  require(a->tokens < (int64_t)1 << 31 && a->q_heads >= 0 && a->q_heads <= 65535, SC_ERR_UNSUPPORTED,
          "too many tokens or query heads");
  require(!a->q.ptr || (a->q_out.ptr && a->q_heads > 0), SC_ERR_ARG, "queries need q_heads and an output");
  require(!a->cos == !a->sin, SC_ERR_ARG, "the rotation needs both cos and sin");
  if (a->cos)
    require(a->rotary > 0 && a->rotary % 2 == 0 && a->rotary <= c->pool.head_dim && a->rope_rows > 0, SC_ERR_ARG,
            "rotary must be even and at most head_dim");
  AppendParams p{*a, c->pool, static_cast<int *>(c->status.p)};
  DeviceGuard dg(c->device);
  const int64_t n = a->tokens * ((a->q.ptr ? a->q_heads : 0) + 2 * c->pool.kv_heads) * (c->pool.head_dim / 2);
  require((n + 255) / 256 <= INT32_MAX, SC_ERR_UNSUPPORTED, "too many rows in one call");
  with_types(a->type, c->pool.type, [&](auto t, auto e) {
    append_kernel<decltype(t), decltype(e)>
        <<<(unsigned)((n + 255) / 256), 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
  });
  cuda_check(cudaGetLastError(), "launch cache append");
  SC_SERVE_END
}

}  // extern "C"
