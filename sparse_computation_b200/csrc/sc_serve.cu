// Cache append with the rotary rotation.
#include <algorithm>
#include <cmath>
#include <memory>
#include <type_traits>

#include "sc_serve.h"

using namespace sc::serve;

namespace {

constexpr int64_t kMaxHeadDim = 256;  // the widest tile of the attention kernel

// --------------------------------------------------------------- append ----

// n / by for n below 2^31, as umulhi(n, mul) >> shift (mul 0: by is 1).
struct Divider {
  uint32_t by = 1, mul = 0, shift = 0;
  Divider() = default;
  explicit Divider(int64_t d) : by((uint32_t)d) {
    for (int bits = 1; d > 1; ++bits)
      if (((int64_t)1 << bits) >= d) {
        mul = (uint32_t)((((uint64_t)1 << (31 + bits)) + d - 1) / d);
        shift = bits - 1;
        return;
      }
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return mul ? __umulhi(n, mul) >> shift : n; }
};

struct AppendParams {
  sc_kv_append_args a;
  sc_kv_pool pool;
  int *status;
  uint32_t page_mul, page_shift;    // divider by the page size
  uint32_t pairs_mul, pairs_shift;  // divider by the pairs of a head
  int tile_bits, parts, eights, rope4;
  Divider plain, turned;            // eights of a head; without the partners' in the half style
};

// The cache place of token t: page and slot, or page -1 when it is skipped.
__device__ __forceinline__ void token_place(const AppendParams &p, int64_t t, int &pos, int &page, int &slot) {
  const sc_kv_append_args &a = p.a;
  page = -1;
  slot = 0;
  pos = a.positions[t];
  if (pos < 0) return;
  const int64_t seq = a.seq_ids ? a.seq_ids[t] : t;
  const int col = p.page_mul ? (int)(__umulhi((uint32_t)pos, p.page_mul) >> p.page_shift) : pos;
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

// Any strides: one thread per pair of dims that rotate together (or two
// neighbouring ones that do not) of one head of one token.
template <class T, class C>
__global__ void __launch_bounds__(256) append_any_kernel(const AppendParams p) {
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

// Eight neighbouring elements, as they lie.
template <class T>
struct Eight {
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T *p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4 *>(p)[i];
  }
  __device__ __forceinline__ void store(T *p) const {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4 *>(p)[i] = w[i];
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const T *v = reinterpret_cast<const T *>(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(v[i]);
  }
  __device__ __forceinline__ void set(const float (&x)[8]) {
    T *v = reinterpret_cast<T *>(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = from_f32<T>(x[i]);
  }
};

// Token-major activations (the heads of a token contiguous): a warp takes a
// token, or 1/p.parts of it, so that position, page and rotation row are its
// own scalars.  It walks the heads of v, k and q in jobs of eight dims (with
// their eight partners in the half style), and asks for the first jobs of all
// three before the place of the token is known.  Bound by memory latency and,
// at 16 bits, by the instructions of a job: walking v, k and q one after the
// other took 16.3 us for 4099 tokens of 20 + 2 x 4 heads of 80 in bf16 (one
// thread per pair 45.0), this 13.9: 2.7 TB/s.
struct RowJobs {
  Divider jobs;  // of a head
  int half;      // distance of partners, 0: none
};

struct Turn {  // the rotation of a token
  const float *cos, *sin;
  int rotary;  // 0: none
  bool four;   // rows can be read in fours
};

// Turns dims d .. d + 7 (x), in the half style with their partners (z).
__device__ __forceinline__ void turn8(float (&x)[8], float (&z)[8], int d, int half, const Turn &turn) {
  const float *cp = turn.cos + (half ? d : d / 2), *sp = turn.sin + (half ? d : d / 2);
  float c[8], s[8];
#pragma unroll
  for (int e = 0; e < 8; e += 4)
    if (e == 0 || half) {
      if (turn.four) {
        *reinterpret_cast<float4 *>(c + e) = *reinterpret_cast<const float4 *>(cp + e);
        *reinterpret_cast<float4 *>(s + e) = *reinterpret_cast<const float4 *>(sp + e);
      } else {
#pragma unroll
        for (int f = e; f < e + 4; ++f) c[f] = cp[f], s[f] = sp[f];
      }
    }
  if (half) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = x[e] * c[e] - z[e] * s[e];
      z[e] = z[e] * c[e] + x[e] * s[e];
      x[e] = v;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float v = x[e] * c[e / 2] - x[e + 1] * s[e / 2];
      x[e + 1] = x[e + 1] * c[e / 2] + x[e] * s[e / 2];
      x[e] = v;
    }
  }
}

// BATCH jobs of one lane, `step` apart.
template <class T, int BATCH>
struct HeadJobs {
  Eight<T> u[BATCH], w[BATCH];

  __device__ __forceinline__ void load(const T *src, const RowJobs &r, int heads, int first, int step) {
    const int n = heads * (int)r.jobs.by, D = (int)r.jobs.by * 8 + r.half;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int j = first + i * step;
      if (j < n) {
        const int head = (int)r.jobs(j);
        int d = (j - head * (int)r.jobs.by) * 8;
        if (d >= r.half) d += r.half;  // the partners' eights go with the first ones
        const T *p = src + head * D + d;
        u[i].load(p);
        if (d < r.half) w[i].load(p + r.half);
      }
    }
  }

  // dst_head 0: heads lie as in the source
  template <class C>
  __device__ __forceinline__ void finish(C *dst, int64_t dst_head, const RowJobs &r, int heads, const Turn &turn, bool zero, int first,
                                         int step) {
    const int n = heads * (int)r.jobs.by, D = (int)r.jobs.by * 8 + r.half;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int j = first + i * step;
      if (j >= n) break;
      const int head = (int)r.jobs(j);
      int d = (j - head * (int)r.jobs.by) * 8;
      if (d >= r.half) d += r.half;
      const bool two = d < r.half;
      C *y = dst + (dst_head ? head * dst_head : head * D) + d;
      if (std::is_same<T, C>::value && d >= turn.rotary && !zero) {  // the bits move as they are
        u[i].store(reinterpret_cast<T *>(y));
        if (two) w[i].store(reinterpret_cast<T *>(y + r.half));
        continue;
      }
      float x[8], z[8] = {};
      u[i].get(x);
      if (two) w[i].get(z);
      if (d < turn.rotary) turn8(x, z, d, r.half, turn);
      if (zero)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = z[e] = 0.f;
      Eight<C> o;
      o.set(x);
      o.store(y);
      if (two) {
        o.set(z);
        o.store(y + r.half);
      }
    }
  }
};

template <class T, class C>
__global__ void __launch_bounds__(128, 4) append_rows_kernel(const __grid_constant__ AppendParams p,
                                                             const __grid_constant__ RowJobs turned,
                                                             const __grid_constant__ RowJobs plain, int rope4) {
  constexpr int BK = sizeof(T) == 4 ? 1 : 2, BQ = sizeof(T) == 4 ? 2 : 4;
  const sc_kv_append_args &a = p.a;
  const int64_t t = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / 32;
  if (t >= a.tokens) return;
  const int first = blockIdx.y * 32 + threadIdx.x % 32, step = 32 * p.parts, hk = (int)p.pool.kv_heads;
  const int hq = a.q.ptr ? (int)a.q_heads : 0;
  const T *sv = static_cast<const T *>(a.v.ptr) + t * a.v.stride[0], *sk = static_cast<const T *>(a.k.ptr) + t * a.k.stride[0];
  const T *sq = static_cast<const T *>(a.q.ptr) + t * a.q.stride[0];
  HeadJobs<T, BK> v, k;
  HeadJobs<T, BQ> q;
  v.load(sv, plain, hk, first, step);
  k.load(sk, turned, hk, first, step);
  q.load(sq, turned, hq, first, step);
  int pos, page, slot;
  token_place(p, t, pos, page, slot);
  const Turn none{nullptr, nullptr, 0, false};
  const Turn turn{a.cos + pos * a.rope_stride, a.sin + pos * a.rope_stride, a.cos && page >= 0 ? (int)a.rotary : 0, rope4 != 0};
  if (page >= 0) {
    C *dv = static_cast<C *>(p.pool.v) + page * p.pool.v_stride[0] + slot * p.pool.v_stride[2];
    C *dk = static_cast<C *>(p.pool.k) + page * p.pool.k_stride[0] + slot * p.pool.k_stride[2];
    const int64_t vh = hk > 1 ? p.pool.v_stride[1] : 0, kh = hk > 1 ? p.pool.k_stride[1] : 0;
    v.finish(dv, vh, plain, hk, none, false, first, step);
    k.finish(dk, kh, turned, hk, turn, false, first, step);
#pragma unroll 1
    for (int j = first + BK * step; j < hk * (int)plain.jobs.by; j += BK * step) {
      v.load(sv, plain, hk, j, step);
      k.load(sk, turned, hk, j, step);
      v.finish(dv, vh, plain, hk, none, false, j, step);
      k.finish(dk, kh, turned, hk, turn, false, j, step);
    }
  }
  T *dq = static_cast<T *>(a.q_out.ptr) + t * a.q_out.stride[0];
  for (int j = first; j < hq * (int)turned.jobs.by; j += BQ * step) {
    if (j != first) q.load(sq, turned, hq, j, step);
    q.finish(dq, 0, turned, hq, turn, page < 0, j, step);
  }
}

// Feature-major activations, as a product leaves them (tokens contiguous): a
// block takes one head of 2^p.tile_bits tokens, reads it along the tokens,
// turns it in shared memory and writes it along the dims, two to a thread, or
// eight for prompts.  Bound by the chain of latencies (position, page entry,
// rotation row, store) at decoding sizes: 128 tokens of 32 + 2 x 8 heads of 128,
// fp32 into bf16, 5.7 us against 0.9 for their bytes; 4 tokens of 3 x 8 heads
// of 64 2.4 us.  2000 tokens of the former 36 us against 14.
template <class T, class C>
__global__ void __launch_bounds__(256) append_columns_kernel(const __grid_constant__ AppendParams p) {
  const sc_kv_append_args &a = p.a;
  __shared__ float tile[kMaxHeadDim * 33 + kMaxHeadDim / 8];
  __shared__ int s_pos[32], s_slot[32], s_page[32];
  const int hk = (int)p.pool.kv_heads, hq = a.q.ptr ? (int)a.q_heads : 0, D = (int)p.pool.head_dim;
  const int TT = 1 << p.tile_bits;
  // a word more for each dim and each eight: neither the tokens of a dim nor every eighth dim of a token share a bank
  auto place = [&](int d, int t) { return d * (TT + 1) + d / 8 + t; };
  const int64_t t0 = (int64_t)blockIdx.y << p.tile_bits;
  const int here = (int)min((int64_t)TT, a.tokens - t0);
  int head = blockIdx.x;
  const bool is_q = head < hq, is_v = head >= hq + hk;
  const sc_rows &src = is_q ? a.q : is_v ? a.v : a.k;
  if (!is_q) head -= is_v ? hq + hk : hq;
  const T *x = static_cast<const T *>(src.ptr) + t0 + head * src.stride[1];
  // the first loads are on their way while the places, two dependent loads, are worked out
  constexpr int B = 4;
  auto load = [&](int i0, T (&v)[B]) {
#pragma unroll
    for (int k = 0; k < B; ++k) {
      const int i = i0 + 256 * k, d = i >> p.tile_bits, t = i & (TT - 1);
      if (d < D && t < here) v[k] = x[d * src.stride[2] + t];
    }
  };
  auto keep = [&](int i0, const T (&v)[B]) {
#pragma unroll
    for (int k = 0; k < B; ++k) {
      const int i = i0 + 256 * k, d = i >> p.tile_bits, t = i & (TT - 1);
      if (d < D && t < here) tile[place(d, t)] = to_f32(v[k]);
    }
  };
  T v[B];
  load(threadIdx.x, v);
  if ((int)threadIdx.x < here) {
    int pos, page, slot;
    token_place(p, t0 + threadIdx.x, pos, page, slot);
    s_pos[threadIdx.x] = pos, s_page[threadIdx.x] = page, s_slot[threadIdx.x] = slot;
  }
  keep(threadIdx.x, v);
#pragma unroll 1
  for (int i0 = threadIdx.x + B * 256; i0 < D << p.tile_bits; i0 += B * 256) {
    load(i0, v);
    keep(i0, v);
  }
  __syncthreads();
  const int rotary = a.cos && !is_v ? (int)a.rotary : 0, half = rotary / 2, pairs = D / 2;
  const bool halves = !a.interleaved;
  if (p.eights) {
    const int h = halves ? half : 0;
    const Divider &by = h ? p.turned : p.plain;  // eights of a head, partners' apart
    for (int i = threadIdx.x; i < (int)by.by * here; i += 256) {
      const int t = (int)by(i), e = i - t * (int)by.by, d = e * 8 < h ? e * 8 : e * 8 + h;
      const int page = s_page[t], pos = s_pos[t];
      if (page < 0 && !is_q) continue;
      const bool two = d < h;
      float u[8], w[8] = {};
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        u[k] = page < 0 ? 0.f : tile[place(d + k, t)];
        if (two && page >= 0) w[k] = tile[place(d + h + k, t)];
      }
      if (d < rotary && page >= 0)
        turn8(u, w, d, h, Turn{a.cos + pos * a.rope_stride, a.sin + pos * a.rope_stride, rotary, p.rope4 != 0});
      auto put = [&](auto *y) {
        Eight<std::remove_reference_t<decltype(*y)>> o;
        o.set(u);
        o.store(y);
        if (two) {
          o.set(w);
          o.store(y + h);
        }
      };
      if (is_q) {
        put(static_cast<T *>(a.q_out.ptr) + (t0 + t) * a.q_out.stride[0] + head * a.q_out.stride[1] + d);
      } else {
        const int64_t *st = is_v ? p.pool.v_stride : p.pool.k_stride;
        put(static_cast<C *>(is_v ? p.pool.v : p.pool.k) + page * st[0] + head * st[1] + s_slot[t] * st[2] + d);
      }
    }
    return;
  }
  for (int i = threadIdx.x; i < pairs * here; i += 256) {
    const int t = p.pairs_mul ? (int)(__umulhi(i, p.pairs_mul) >> p.pairs_shift) : i, d = 2 * (i - t * pairs);
    const int page = s_page[t], pos = s_pos[t];
    if (page < 0 && !is_q) continue;
    float u = tile[place(d, t)], w = tile[place(d + 1, t)];
    if (page < 0) {
      u = w = 0.f;
    } else if (d < rotary) {
      const float *c = a.cos + pos * a.rope_stride, *s = a.sin + pos * a.rope_stride;
      if (halves) {  // half is even: both dims lie on one side
        const bool upper = d >= half;
        const int i0 = upper ? d - half : d, other = upper ? d - half : d + half;
        const float sign = upper ? 1.f : -1.f;
        u = u * c[i0] + sign * (tile[place(other, t)] * s[i0]);
        w = w * c[i0 + 1] + sign * (tile[place(other + 1, t)] * s[i0 + 1]);
      } else {
        const float ci = c[d / 2], si = s[d / 2], ru = u * ci - w * si;
        w = w * ci + u * si;
        u = ru;
      }
    }
    auto put = [&](auto *y) {
      using E = std::remove_reference_t<decltype(*y)>;
      struct alignas(2 * sizeof(E)) Two {
        E a, b;
      };
      *reinterpret_cast<Two *>(y) = Two{from_f32<E>(u), from_f32<E>(w)};
    };
    if (is_q) {
      put(static_cast<T *>(a.q_out.ptr) + (t0 + t) * a.q_out.stride[0] + head * a.q_out.stride[1] + d);
    } else {
      const int64_t *st = is_v ? p.pool.v_stride : p.pool.k_stride;
      put(static_cast<C *>(is_v ? p.pool.v : p.pool.k) + page * st[0] + head * st[1] + s_slot[t] * st[2] + d);
    }
  }
}

// Whether rows of `type` are contiguous along the dims with every `elems`-th element aligned to a vector of that many.
bool along_dims(const sc_rows &r, int64_t tokens, int64_t type, int64_t elems) {
  const int64_t e = type_bytes(type), n = elems * e < 16 ? elems * e : 16;
  return r.stride[2] == 1 && (tokens == 1 || r.stride[0] * e % n == 0) && r.stride[1] * e % n == 0 &&
         reinterpret_cast<uintptr_t>(r.ptr) % n == 0;
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
  make_status(c->status, device);
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
  const Divider by_page(c->pool.page_size);
  AppendParams p{*a, c->pool, static_cast<int *>(c->status.p), by_page.mul, by_page.shift, 0, 0, 0, 0, 0, 0, Divider(), Divider()};
  DeviceGuard dg(c->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool q = a->q.ptr != nullptr, rotates = a->cos != nullptr, halves = rotates && !a->interleaved;
  const int64_t D = c->pool.head_dim, heads = (q ? a->q_heads : 0) + 2 * c->pool.kv_heads;
  const int64_t half = rotates ? a->rotary / 2 : 0;
  auto packed = [&](const sc_rows &r, int64_t h) { return h == 1 || r.stride[1] == D; };
  // Token-major rows with packed heads move in eights, feature-major ones through shared memory; what fits neither
  // (odd strides, a rotation that splits an eight) goes element by element.
  const bool rows = D % 8 == 0 && half % 8 == 0 && heads <= 65535 && packed(a->k, c->pool.kv_heads) && packed(a->v, c->pool.kv_heads) &&
                    along_dims(a->k, a->tokens, a->type, 8) && along_dims(a->v, a->tokens, a->type, 8) &&
                    (!q || (packed(a->q, a->q_heads) && packed(a->q_out, a->q_heads) &&
                            along_dims(a->q, a->tokens, a->type, 8) && along_dims(a->q_out, a->tokens, a->type, 8)));
  const bool columns = half % 2 == 0 && (!q || (a->q.stride[0] == 1 && along_dims(a->q_out, a->tokens, a->type, 2))) &&
                       a->k.stride[0] == 1 && a->v.stride[0] == 1 && heads <= 65535;
  const int rope4 = rotates && a->rope_stride % 4 == 0 && reinterpret_cast<uintptr_t>(a->cos) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(a->sin) % 16 == 0;
  p.rope4 = rope4;
  p.plain = Divider(std::max<int64_t>(1, D / 8));
  p.turned = Divider(std::max<int64_t>(1, (D - (halves ? half : 0)) / 8));
  // results in eights, unless the rotation splits one or q_out is not laid out for it
  p.eights = D % 8 == 0 && half % 8 == 0 && (!q || along_dims(a->q_out, a->tokens, a->type, 8));
  const int64_t n = a->tokens * heads * (D / 2);
  require((n + 255) / 256 <= INT32_MAX, SC_ERR_UNSUPPORTED, "too many rows in one call");
  with_types(a->type, c->pool.type, [&](auto t, auto e) {
    using T = decltype(t);
    using C = decltype(e);
    if (rows) {
      const int h = halves ? (int)half : 0;
      const RowJobs turned{Divider((D - h) / 8), h}, plain{Divider(D / 8), 0};
      // one warp a token when that fills the SMs (16 warps each), else up to 8 warps
      p.parts = (int)std::max<int64_t>(1, std::min<int64_t>(8, 148 * 16 / a->tokens));
      append_rows_kernel<T, C><<<dim3((unsigned)((a->tokens + 3) / 4), p.parts), 128, 0, st>>>(p, turned, plain, rope4);
    } else if (columns && a->tokens <= 65535 * 32) {
      // at most 32 tokens a block, fewer for more blocks, but whole 32-byte sectors of a feature's tokens
      const int fewest = sizeof(T) == 4 ? 3 : 4;
      p.tile_bits = 5;
      while (p.tile_bits > fewest && heads * (a->tokens >> p.tile_bits) < 4 * 148) --p.tile_bits;
      while (p.tile_bits > 2 && a->tokens <= 1 << (p.tile_bits - 1)) --p.tile_bits;
      // Eights have fewer instructions, pairs more threads.  us in eights / in pairs for 4, 64, 256, 512 and 2000 fp32
      // tokens into bf16, 32 + 2 x 8 heads of 128: 3.0/2.5 3.8/4.0 7.3/8.6 10.9/14.8 36.2/46.5; 3 x 8 heads of 64:
      // 3.1/2.4 3.4/3.1 5.5/4.8 5.7/5.9 10.9/13.2.
      if (p.tile_bits < 5) p.eights = 0;
      const Divider pairs(D / 2);
      p.pairs_mul = pairs.mul, p.pairs_shift = pairs.shift;
      append_columns_kernel<T, C>
          <<<dim3((unsigned)heads, (unsigned)((a->tokens + (1 << p.tile_bits) - 1) >> p.tile_bits)), 256, 0, st>>>(p);
    } else {
      append_any_kernel<T, C><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(p);
    }
  });
  cuda_check(cudaGetLastError(), "launch cache append");
  SC_SERVE_END
}

}  // extern "C"
