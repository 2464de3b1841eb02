// Decode attention over a paged cache: one query token per sequence.
//
// For each kv head, the keys of a sequence are read once for the whole group
// of query heads that share it; o = sum_j exp(z_j - m) v_j / sum_j exp(z_j - m)
// is built in one pass with a running maximum m.  Per key and kv head that is
// 2 head_dim elements read and 4 group head_dim flops, a few flops per byte:
// the bound is the memory read, and everything here serves to keep enough
// reads in flight.
//
// Matrix instructions.  A warp takes kKeys keys at a time and computes
// S = Q K^T and O += P V with mma.sync, the 8 query heads of a tile in rows
// 0-7.  Rows 8-15 carry what a single 16-bit or TF32 operand loses: Q and P
// are split into a head (rows 0-7) and a tail (rows 8-15), and the two halves
// of the result are added, so the split costs no further instructions.
//
// Fragments without shared-memory transposition.  The sum over head_dim may
// run in any order and the columns of O may be any permutation, so each lane
// takes whole 16-byte pieces: of K, piece t + 4j of key g (g = lane / 4,
// t = lane % 4) is a B fragment of 2 k-steps; of V, piece g + 8j of keys
// 2t, 2t+1 (+8) holds one column of O per element.  K and V go from global
// memory straight into the registers that feed the matrix instructions: the
// next K is asked for as soon as the scores are done, the next V after the
// product with P.  At 8 KB a warp step and 12 or 16 warps a SM that is
// 64-128 KB in flight, more than latency times bandwidth asks for.  (The same
// through cp.async and shared memory was bound by the extra 16 shared loads a
// step: 147 us against TODO at 131071 keys, 8 kv heads of 128, bf16.)
//
// Work.  All (sequence, kv head, query tile) segments are cut into steps of
// kKeys keys and laid end to end.  Every block takes one equal, contiguous
// run of steps, found by a scan over the sequence lengths on the device (the
// host never sees them), and every warp an equal share of its block's run.
// Warps do not wait for one another until all are done: a segment that one
// warp covers is written directly, the others leave pieces (m, l, O) that the
// block adds up at its end.  A segment that passes the end of a block's run
// goes into a record in the workspace, and the last of its blocks to arrive
// adds the records up.  Pieces and records are added in the order of the
// keys, so results do not depend on the order of arrival.
#pragma once

#include "sc_serve.h"

namespace sc {
namespace attn {

using serve::to_f32;

constexpr int kQT = 8, kMaxWarps = 12;

enum Mode { kTF32, kBF16, kBF16Wide, kF16, kF16Wide };

struct Params {
  sc_attn_args a;
  sc_kv_pool pool;
  int q_heads, group, qtiles, q_rows;  // q_rows: rows of a query tile, min(group, kQT)
  int min_run;                         // fewest steps of a block
  uint32_t page_mul, page_shift;       // key / page_size = umulhi(key, mul) >> shift (mul 0: page_size 1)
  int q_vec;                           // query rows are contiguous and 16-byte aligned
  int64_t k_page, k_head, k_slot, v_page, v_head, v_slot;  // strides in bytes
  float scale_log2;                    // scale * log2(e)
  int64_t window;
  int *status;
  int *arrivals;   // [seqs * kv_heads * qtiles], zero between calls
  float *heads;    // [blocks][warps] pieces whose warp went on after them
  float *records;  // [blocks][2]
};

template <int MODE, int DP>
struct Cfg {
  static constexpr bool f32 = MODE == kTF32;
  static constexpr int es = f32 ? 4 : 2, epc = 16 / es;  // bytes per element, elements per 16-byte piece
  // 8-key columns of S per step: 8 KB of K and V (16 KB from head_dim 129 on)
  static constexpr int NT = f32 ? (DP > 64 ? 1 : 2) : (DP > 64 ? 2 : 4);
  static constexpr int KJ = DP / (4 * epc), VJ = (DP + 8 * epc - 1) / (8 * epc);
  static constexpr int parts = MODE == kBF16Wide ? 3 : MODE == kBF16 || MODE == kF16 ? 1 : 2;  // of Q
  static constexpr int keys = NT * 8;
  static constexpr int sub = keys < 16 ? keys : 16;  // keys that lie in one page when page_size is a multiple of 16
  static constexpr int q_row = KJ * parts * 64;      // bytes of one query row in fragment order
  static constexpr int max_warps = DP > 128 ? 8 : 12;  // by the registers of a step
  static constexpr bool ahead = DP <= 128;  // registers suffice to load a step ahead
  static constexpr int o_row = DP + 4;               // floats; the pad spreads rows over the banks
  static constexpr int piece = kQT * o_row + 2 * kQT;  // O | m | l
  // shared memory of a warp: its query tile, later its last piece
  __host__ __device__ static constexpr int warp_bytes(int q_rows) { return (q_row * q_rows > piece * 4 ? q_row * q_rows : piece * 4); }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 16 bytes that are read once: past L1, 128-byte requests to L2
__device__ __forceinline__ uint4 ldg16(const void *p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::128B.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

__device__ __forceinline__ uint4 lds(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}

template <int MODE>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  if (MODE == kTF32)
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else if (MODE == kF16 || MODE == kF16Wide)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The TF32 head of x: its upper 11 significant bits; x - head is exact.
__device__ __forceinline__ uint32_t tf32_head(float x) { return __float_as_uint(x) & 0xffffe000u; }
__device__ __forceinline__ uint32_t tf32_tail(float x) {
  return __float_as_uint(x - __uint_as_float(__float_as_uint(x) & 0xffffe000u));
}

// Two floats as packed 16-bit values, and what the packing lost of them.
template <int MODE>
__device__ __forceinline__ uint32_t pack2(float &a, float &b) {
  if (MODE == kF16 || MODE == kF16Wide) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    a -= f.x;
    b -= f.y;
    return *reinterpret_cast<const uint32_t *>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    const float2 f = __bfloat1622float2(h);
    a -= f.x;
    b -= f.y;
    return *reinterpret_cast<const uint32_t *>(&h);
  }
}

__device__ __forceinline__ void store_row(void *p, int64_t type, int64_t i, float x) {
  if (type == SC_TYPE_F32)
    static_cast<float *>(p)[i] = x;
  else if (type == SC_TYPE_F16)
    static_cast<__half *>(p)[i] = __float2half_rn(x);
  else
    static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(x);
}

// Keys [first, len) of a sequence; steps start at `start`, first rounded down
// to a multiple of 16 so that no step straddles a page whose size is one.
struct Span {
  int first, len, start, steps;
};

template <int KEYS>
__device__ __forceinline__ Span span_of(const Params &p, int64_t s) {
  Span r;
  r.len = max(p.a.seq_lens[s], 0);
  const int64_t most = p.a.table_cols * p.pool.page_size;
  if (r.len > most) {
    serve::set_status(p.status, 8);
    r.len = (int)most;
  }
  r.first = p.window && r.len > p.window ? r.len - (int)p.window : 0;
  r.start = r.first & ~15;
  r.steps = (r.len - r.start) / KEYS + ((r.len - r.start) % KEYS != 0);
  return r;
}

__device__ __forceinline__ int page_of(const Params &p, int key) {
  return p.page_mul ? (int)(__umulhi((uint32_t)key, p.page_mul) >> p.page_shift) : key;
}

// Four neighbouring outputs from dim d on of one head.
__device__ __forceinline__ void store4(const Params &p, int64_t seq, int head, int d, float4 y) {
  const int64_t st = p.a.out.stride[2];
  const int64_t i = seq * p.a.out.stride[0] + head * p.a.out.stride[1] + d * st;
  const float v[4] = {y.x, y.y, y.z, y.w};
  for (int e = 0; e < 4; ++e) store_row(p.a.out.ptr, p.a.type, i + e * st, v[e]);
}

__device__ __forceinline__ float lse_of(float ref, float sum) { return (ref + log2f(sum)) * 0.69314718055994531f; }

// A boundary between two blocks' runs: the place that an equal cut gives,
// moved to an end of its segment when that is near, which saves a join.
struct Cut {
  int64_t at, seq, seq_begin, seg_begin, seg_end;
};

__device__ __forceinline__ int64_t snapped(int64_t b, int64_t x, int64_t y, int64_t near) {
  const int64_t lo = b - x, hi = y - b;
  return lo <= near && lo <= hi ? x : hi <= near ? y : b;
}

// N neighbouring elements of a query row from dim d on, as floats; zeros from head_dim on.
template <int N, class T>
__device__ __forceinline__ void load_dims(const T *q, const Params &p, int d, float (&x)[N]) {
  const int D = (int)p.pool.head_dim;
  if (p.q_vec) {  // contiguous and aligned: head_dim is a multiple of N then
    if (d >= D) {
#pragma unroll
      for (int e = 0; e < N; ++e) x[e] = 0.f;
    } else {
      constexpr int words = N * (int)sizeof(T) / 8;
      uint2 w[words];
#pragma unroll
      for (int i = 0; i < words; ++i) w[i] = reinterpret_cast<const uint2 *>(q + d)[i];
      const T *v = reinterpret_cast<const T *>(w);
#pragma unroll
      for (int e = 0; e < N; ++e) x[e] = to_f32(v[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = d + e < D ? to_f32(q[(d + e) * p.a.q.stride[2]]) : 0.f;
  }
}

// Puts a lane's share of query row q (pieces t, t + 4, ...) into fragment
// order, split into parts.  For fp16 parts a row is scaled by a power of two
// to below 2, so that no part overflows and the tails stay above fp16's
// smallest values; returns that factor.  The four lanes of a row call it together.
template <int MODE, int DP, class T>
__device__ __forceinline__ float fill_q(const T *q, const Params &p, int t, uint32_t sq, int q_step, uint32_t group) {
  using C = Cfg<MODE, DP>;
  float x[C::KJ][C::epc], up = 1.f;
#pragma unroll
  for (int j = 0; j < C::KJ; ++j) load_dims<C::epc>(q, p, (t + 4 * j) * C::epc, x[j]);
  if (MODE == kF16Wide) {
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < C::KJ; ++j)
#pragma unroll
      for (int e = 0; e < C::epc; ++e) top = fmaxf(top, fabsf(x[j][e]));
    top = fmaxf(top, __shfl_xor_sync(group, top, 1));
    top = fmaxf(top, __shfl_xor_sync(group, top, 2));
    const int e = (int)(__float_as_uint(top) >> 23) - 127;  // floor(log2(top)) of a normal number
    if (e > -120 && e < 127) up = __uint_as_float((uint32_t)(e + 127) << 23);
  }
#pragma unroll
  for (int j = 0; j < C::KJ; ++j) {
    if (MODE == kF16Wide)
#pragma unroll
      for (int e = 0; e < C::epc; ++e) x[j][e] *= 1.f / up;
#pragma unroll
    for (int part = 0; part < C::parts; ++part) {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (C::f32)
          w[e] = part ? tf32_tail(x[j][e]) : tf32_head(x[j][e]);
        else
          w[e] = pack2<MODE>(x[j][(2 * e) % C::epc], x[j][(2 * e + 1) % C::epc]);
      }
      asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(sq + (j * C::parts + part) * q_step), "r"(w[0]),
                   "r"(w[1]), "r"(w[2]), "r"(w[3])
                   : "memory");
    }
  }
  return up;
}

// Adds up row r of up to 32 pieces (m, l, O) at a time: lane i weighs piece i, then every lane adds dims
// 4 lane, 4 lane + 128, ... of all pieces, eight loads in flight.  List: how many, and where piece i is.
template <int DP, class List>
__device__ __forceinline__ void add_up(const List &list, int r, float4 (&y)[(DP + 127) / 128], float &ref, float &sum) {
  constexpr int ND = (DP + 127) / 128, o_row = DP + 4;
  const int lane = threadIdx.x % 32, n = list.count();
  float top = -INFINITY;
  for (int i = lane; i < n; i += 32) top = fmaxf(top, list.load(list.at(i) + kQT * o_row + r));
  for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
  ref = top == -INFINITY ? 0.f : top;
  sum = 0.f;
#pragma unroll
  for (int k = 0; k < ND; ++k) y[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int base = 0; base < n; base += 32) {
    float weight = 0.f;
    const float *mine = nullptr;
    if (base + lane < n) {
      mine = list.at(base + lane);
      const float *q = mine + kQT * o_row + r;
      weight = ex2(list.load(q) - ref);
      sum += weight * list.load(q + kQT);
    }
    const int here = min(32, n - base);
    for (int i0 = 0; i0 < here; i0 += 8) {
      float4 v[8][ND];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float *q = reinterpret_cast<const float *>(__shfl_sync(~0u, reinterpret_cast<uint64_t>(mine), i0 + i));
#pragma unroll
        for (int k = 0; k < ND; ++k) {
          const int d = 4 * lane + 128 * k;
          v[i][k] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (i0 + i < here && d < DP) v[i][k] = list.load(reinterpret_cast<const float4 *>(q + r * o_row + d));
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float f = __shfl_sync(~0u, weight, i0 + i);
        if (i0 + i < here) {
#pragma unroll
          for (int k = 0; k < ND; ++k)
            y[k].x += f * v[i][k].x, y[k].y += f * v[i][k].y, y[k].z += f * v[i][k].z, y[k].w += f * v[i][k].w;
        }
      }
    }
  }
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
}

// The pieces of one segment in a block: even numbers in the workspace, odd ones in the warps' shared memory.
struct PieceList {
  uint32_t members;
  const float *heads;  // of the block
  const uint8_t *smem;
  int piece, warp_bytes;
  template <class T>
  __device__ T load(const T *q) const { return *q; }  // shared or global memory, of this block's own writing
  __device__ int count() const { return __popc(members); }
  __device__ const float *at(int n) const {
    const int i = __fns(members, 0, n + 1);
    return i % 2 ? reinterpret_cast<const float *>(smem + (i / 2) * warp_bytes) : heads + (i / 2) * piece;
  }
};

// The records of a segment: of the block where it begins, then of those that it runs through.
struct RecordList {
  const float *records;
  int piece, from, to;
  template <class T>
  __device__ T load(const T *q) const { return __ldcg(q); }  // written by other blocks
  __device__ int count() const { return to - from + 1; }
  __device__ const float *at(int n) const { return records + ((int64_t)(from + n) * 2 + (n == 0)) * piece; }
};

template <int MODE, int DP>
__global__ void __launch_bounds__(Cfg<MODE, DP>::max_warps * 32, 1) attend_kernel(const Params p) {
  using C = Cfg<MODE, DP>;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int64_t s_scan[kMaxWarps];
  __shared__ Cut s_cut[2];
  // pieces: sequence (-1: none), segment of it, and whether that began before (1) or only ends after (2) this run
  __shared__ int s_seq[2 * kMaxWarps], s_unit[2 * kMaxWarps], s_open[2 * kMaxWarps];
  __shared__ uint32_t s_masks[2];
  __shared__ int s_last;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, t = lane % 4;
  const int W = blockDim.x / 32, D = (int)p.pool.head_dim;
  const int ps = (int)p.pool.page_size;
  const int64_t units = p.pool.kv_heads * p.qtiles;  // segments of a sequence

  // ---- this block's run of steps
  int64_t mine = 0;
  for (int64_t s = tid; s < p.a.seqs; s += blockDim.x) mine += span_of<C::keys>(p, s).steps;
  for (int d = 16; d; d >>= 1) mine += __shfl_xor_sync(~0u, mine, d);
  if (lane == 0) s_scan[warp] = mine;
  __syncthreads();
  int64_t total = 0;
  for (int w = 0; w < W; ++w) total += s_scan[w];
  total *= units;
  int64_t per = (total + gridDim.x - 1) / gridDim.x;
  if (per < p.min_run) per = p.min_run;
  const int64_t near = max(per / 8, min(per, (int64_t)W) / 2);

  // sequences without keys
  for (int64_t s = blockIdx.x; s < p.a.seqs; s += gridDim.x)
    if (span_of<C::keys>(p, s).steps == 0) {
      for (int i = tid; i < p.q_heads * D; i += blockDim.x)
        store_row(p.a.out.ptr, p.a.type,
                  s * p.a.out.stride[0] + (i / D) * p.a.out.stride[1] + (i % D) * p.a.out.stride[2], 0.f);
      if (p.a.lse)
        for (int i = tid; i < p.q_heads; i += blockDim.x) p.a.lse[s * p.q_heads + i] = -INFINITY;
    }
  const int64_t nominal0 = per * blockIdx.x, nominal1 = nominal0 + per;
  if (nominal0 >= total) return;
  if (nominal1 >= total && tid == 0) s_cut[1] = Cut{total, p.a.seqs, total, total, total};
  int64_t before = 0;
  for (int64_t base = 0; before <= nominal1 && base < p.a.seqs; base += blockDim.x) {
    const int64_t s = base + tid;
    const int steps = s < p.a.seqs ? span_of<C::keys>(p, s).steps : 0;
    const int64_t n = steps * units;
    int64_t sum = n;
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t up = __shfl_up_sync(~0u, sum, d);
      if (lane >= d) sum += up;
    }
    __syncthreads();
    if (lane == 31) s_scan[warp] = sum;
    __syncthreads();
    sum += before;
    for (int w = 0; w < W; ++w) {
      if (w < warp) sum += s_scan[w];
      before += s_scan[w];
    }
    for (int k = 0; k < 2; ++k) {
      const int64_t b = k ? nominal1 : nominal0, from = sum - n;
      if (b >= from && b < sum) {
        const int64_t x = from + (b - from) / steps * steps;
        s_cut[k] = Cut{snapped(b, x, x + steps, near), s, from, x, x + steps};
      }
    }
  }
  __syncthreads();
  const int64_t begin = s_cut[0].at, end = s_cut[1].at;
  if (begin >= end) return;

  // ---- this warp's share of it; places in the run are counted from its begin from here on
  const int run = (int)(end - begin);
  const int wb = (int)((int64_t)run * warp / W), we = (int)((int64_t)run * (warp + 1) / W);
  int seq = (int)s_cut[0].seq;
  int64_t seq_begin = s_cut[0].seq_begin - begin;
  Span sp = span_of<C::keys>(p, seq);
  if (lane < 2) s_seq[2 * warp + lane] = -1;

  const int warp_bytes = C::warp_bytes(p.q_rows);
  uint8_t *own = smem + warp * warp_bytes;
  // query row g in fragment order; lanes beyond the tile's rows repeat its last one, their results go nowhere
  const uint32_t sq = (uint32_t)__cvta_generic_to_shared(own) + min(g, p.q_rows - 1) * 64 + t * 16;
  const int q_step = p.q_rows * 64;
  const bool paged16 = ps % 16 == 0, full_dim = D == DP;
  const uint8_t *kbase = static_cast<const uint8_t *>(p.pool.k), *vbase = static_cast<const uint8_t *>(p.pool.v);

  for (int at = wb; at < we;) {
    while (at >= seq_begin + sp.steps * units) {  // next sequence with keys
      seq_begin += sp.steps * units;
      sp = span_of<C::keys>(p, ++seq);
    }
    const int64_t off = at - seq_begin;
    const int unit = (int)(off / sp.steps), step0 = (int)(off - (int64_t)unit * sp.steps);
    const int h = unit / p.qtiles, qt = unit - h * p.qtiles;
    const int n = min(sp.steps - step0, we - at);
    const bool whole = step0 == 0 && n == sp.steps;
    const int rows = min(kQT, p.group - qt * kQT), head0 = h * p.group + qt * kQT;
    const int32_t *table = p.a.page_table + seq * p.a.table_stride;
    const int key0 = sp.start + step0 * C::keys;
    const uint8_t *kh = kbase + h * p.k_head, *vh = vbase + h * p.v_head;

    // ---- places of a step's keys: a page entry per 16 keys, or one per key
    constexpr int NS = C::keys / C::sub;
    int entry[NS];  // paged16: of each 16 keys; else entry[0], of key lane % keys
    auto look_up = [&](int key) {
      if (paged16) {
#pragma unroll
        for (int i = 0; i < NS; ++i)
          entry[i] = key + i * 16 < sp.len ? table[page_of(p, key + i * 16)] : 0;
      } else {
        const int k = key + lane % C::keys;
        entry[0] = k >= sp.first && k < sp.len ? table[page_of(p, k)] : 0;
      }
    };
    // present keys of the step at `key`, by entries as looked up
    auto present_of = [&](int key) -> uint32_t {
      const int hi = min(sp.len - key, C::keys), lo = min(max(sp.first - key, 0), C::keys);
      uint32_t mask = (uint32_t)((1ull << hi) - 1) & ~(uint32_t)((1ull << lo) - 1);
      bool bad = false;
      if (paged16) {
#pragma unroll
        for (int i = 0; i < NS; ++i)
          if (key + i * 16 < sp.len && (uint32_t)entry[i] >= (uint32_t)p.pool.num_pages) {
            bad = true;
            mask &= ~(0xffffu << (16 * i));
            entry[i] = 0;
          }
      } else {
        const bool ok = (uint32_t)entry[0] < (uint32_t)p.pool.num_pages;
        const uint32_t good = __ballot_sync(~0u, ok);
        bad = !ok;
        mask &= good;
        if (!ok) entry[0] = 0;
      }
      if (bad) serve::set_status(p.status, 8);
      return mask;
    };
    // Loads this lane's pieces of the keys of the step at `key`: of K, piece t + 4j of key 8 nt + g; of V, piece
    // g + 8j of keys 8 nt + 2t + (0, 1).  Absent keys and pieces beyond head_dim are zeros.
    uint4 kf[C::NT][C::KJ], vf[2 * C::NT][C::VJ];
    auto load = [&](auto &f, const uint8_t *base, int64_t page, int64_t slot, int key, uint32_t mask, bool is_k) {
      constexpr int rows = sizeof(f) / sizeof(f[0]), J = sizeof(f[0]) / sizeof(f[0][0]);
      const int lane_row = is_k ? g : 2 * t, first_piece = is_k ? t : g, piece_step = is_k ? 4 : 8;
      const bool full = full_dim && mask == (uint32_t)((1ull << C::keys) - 1);
      const uint8_t *block = base;
#pragma unroll
      for (int r = 0; r < rows; ++r) {
        const int k8 = is_k ? r * 8 : r / 2 * 8, k = is_k ? g : 2 * t + r % 2;  // key k8 + k
        const uint8_t *src;
        if (paged16) {
          const int first = key + k8 / 16 * 16;
          if (k8 % 16 == 0 && (is_k || r % 2 == 0))
            block = base + entry[k8 / 16] * page + (first - page_of(p, first) * ps + lane_row) * slot + first_piece * 16;
          src = block + (k8 % 16 + (is_k ? 0 : r % 2)) * slot;
        } else {
          const int e = __shfl_sync(~0u, entry[0], k8 + k), kk = key + k8 + k;
          src = base + e * page + (kk - page_of(p, kk) * ps) * slot + first_piece * 16;
        }
        if (full) {
#pragma unroll
          for (int j = 0; j < J; ++j) f[r][j] = ldg16(src + j * piece_step * 16);
        } else {
          const bool ok = mask >> (k8 + k) & 1;
#pragma unroll
          for (int j = 0; j < J; ++j) {
            f[r][j] = make_uint4(0, 0, 0, 0);
            if (ok && (first_piece + piece_step * j) * C::epc < D) f[r][j] = ldg16(src + j * piece_step * 16);
          }
        }
      }
    };
    auto load_k = [&](int key, uint32_t mask) { load(kf, kh, p.k_page, p.k_slot, key, mask, true); };
    auto load_v = [&](int key, uint32_t mask) { load(vf, vh, p.v_page, p.v_slot, key, mask, false); };
    look_up(key0);
    uint32_t mask = present_of(key0);
    load_k(key0, mask);
    load_v(key0, mask);

    // ---- the query tile, split into parts, in fragment order
    const int64_t q0 = seq * p.a.q.stride[0] + (head0 + min(g, rows - 1)) * p.a.q.stride[1];
    float up = 1.f;
    if (g < p.q_rows) {
      const uint32_t group = p.q_rows == kQT ? ~0u : (1u << (4 * p.q_rows)) - 1;
      if (p.a.type == SC_TYPE_F32)
        up = fill_q<MODE, DP>(static_cast<const float *>(p.a.q.ptr) + q0, p, t, sq, q_step, group);
      else if (p.a.type == SC_TYPE_F16)
        up = fill_q<MODE, DP>(static_cast<const __half *>(p.a.q.ptr) + q0, p, t, sq, q_step, group);
      else
        up = fill_q<MODE, DP>(static_cast<const __nv_bfloat16 *>(p.a.q.ptr) + q0, p, t, sq, q_step, group);
    }
    __syncwarp();
    const float c = p.scale_log2 * __shfl_sync(~0u, up, 4 * min(g, p.q_rows - 1));

    // ---- one pass over the keys
    float m = -INFINITY, l = 0.f;
    constexpr int ON = C::VJ * C::epc;
    float o[ON][2];
#pragma unroll
    for (int i = 0; i < ON; ++i) o[i][0] = o[i][1] = 0.f;
    if (n > 1) look_up(key0 + C::keys);
    for (int i = 0; i < n; ++i) {
      const int next = key0 + (i + 1) * C::keys;
      float s[C::NT][2][4] = {};
#pragma unroll
      for (int j = 0; j < C::KJ; ++j) {
        uint4 q[C::parts];
#pragma unroll
        for (int part = 0; part < C::parts; ++part) q[part] = lds(sq + (j * C::parts + part) * q_step);
#pragma unroll
        for (int nt = 0; nt < C::NT; ++nt) {
          const uint4 k = kf[nt][j];
          if (C::f32) {
            const uint32_t kw[4] = {k.x, k.y, k.z, k.w};
            const uint32_t qh[4] = {q[0].x, q[0].y, q[0].z, q[0].w};
            const uint4 ql4 = q[C::parts - 1];
            const uint32_t ql[4] = {ql4.x, ql4.y, ql4.z, ql4.w};
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
              const float k0 = __uint_as_float(kw[e]), k1 = __uint_as_float(kw[e + 1]);
              mma<MODE>(s[nt][0], qh[e], ql[e], qh[e + 1], ql[e + 1], tf32_head(k0), tf32_head(k1));
              mma<MODE>(s[nt][1], qh[e], ql[e], qh[e + 1], ql[e + 1], tf32_tail(k0), tf32_tail(k1));
            }
          } else {
            const uint4 q1 = C::parts > 1 ? q[C::parts > 1 ? 1 : 0] : make_uint4(0, 0, 0, 0);
            mma<MODE>(s[nt][0], q[0].x, q1.x, q[0].y, q1.y, k.x, k.y);
            mma<MODE>(s[nt][1], q[0].z, q1.z, q[0].w, q1.w, k.z, k.w);
            if (C::parts > 2) {
              mma<MODE>(s[nt][0], q[C::parts - 1].x, 0, q[C::parts - 1].y, 0, k.x, k.y);
              mma<MODE>(s[nt][1], q[C::parts - 1].z, 0, q[C::parts - 1].w, 0, k.z, k.w);
            }
          }
        }
      }
      const uint32_t now = mask;
      if (i + 1 < n) {
        mask = present_of(next);
        if (C::ahead) load_k(next, mask);
      }
      // running maximum and sum; a lane has query g and keys 2t, 2t+1 of every 8
      float x[C::NT][2], top = -INFINITY;
#pragma unroll
      for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          x[nt][e] = s[nt][0][e] + s[nt][1][e];
          if (C::parts > 1) x[nt][e] += s[nt][0][2 + e] + s[nt][1][2 + e];
          if (!(now >> (nt * 8 + 2 * t + e) & 1)) x[nt][e] = -INFINITY;
          top = fmaxf(top, x[nt][e]);
        }
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
      top = fmaxf(m, top * c);
      const float ref = top == -INFINITY ? 0.f : top;
      const float shrink = ex2(m - ref);
      m = top;
      l *= shrink;
#pragma unroll
      for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          x[nt][e] = ex2(fmaf(x[nt][e], c, -ref));
          l += x[nt][e];
        }
      constexpr int PN = C::f32 ? C::NT : C::NT / 2;  // A fragments of P: of 8 keys (f32) or 16
      uint32_t pa[PN][4], p3[PN][2];
#pragma unroll
      for (int k = 0; k < PN; ++k) {
        if (C::f32) {
          pa[k][0] = tf32_head(x[k][0]);
          pa[k][1] = tf32_tail(x[k][0]);
          pa[k][2] = tf32_head(x[k][1]);
          pa[k][3] = tf32_tail(x[k][1]);
        } else {
          constexpr int two = C::f32 ? 0 : 1;
          float(&xa)[2] = x[two * 2 * k], (&xb)[2] = x[two * (2 * k + 1)];
          pa[k][0] = pack2<MODE>(xa[0], xa[1]);
          pa[k][2] = pack2<MODE>(xb[0], xb[1]);
          pa[k][1] = pack2<MODE>(xa[0], xa[1]);
          pa[k][3] = pack2<MODE>(xb[0], xb[1]);
          if (MODE == kBF16Wide) {
            p3[k][0] = pack2<MODE>(xa[0], xa[1]);
            p3[k][1] = pack2<MODE>(xb[0], xb[1]);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < C::VJ; ++j) {
        uint32_t v[2 * C::NT][4];
#pragma unroll
        for (int kk = 0; kk < 2 * C::NT; ++kk) {
          const uint4 w = vf[kk][j];
          v[kk][0] = w.x, v[kk][1] = w.y, v[kk][2] = w.z, v[kk][3] = w.w;
        }
#pragma unroll
        for (int e = 0; e < C::epc; ++e) {
          float acc[4] = {};
#pragma unroll
          for (int k = 0; k < PN; ++k) {
            if (C::f32) {
              const float v0 = __uint_as_float(v[2 * k][e % 4]), v1 = __uint_as_float(v[2 * k + 1][e % 4]);
              mma<MODE>(acc, pa[k][0], pa[k][1], pa[k][2], pa[k][3], tf32_head(v0), tf32_head(v1));
              mma<MODE>(acc, pa[k][0], pa[k][1], pa[k][2], pa[k][3], tf32_tail(v0), tf32_tail(v1));
            } else {
              const uint32_t sel = e % 2 ? 0x7632 : 0x5410;
              constexpr int two = C::f32 ? 0 : 4;
              const uint32_t b0 = __byte_perm(v[two * k][e / 2], v[two * k + 1][e / 2], sel);
              const uint32_t b1 = __byte_perm(v[two * k + two / 2][e / 2], v[two * k + two / 2 + 1][e / 2], sel);
              mma<MODE>(acc, pa[k][0], pa[k][1], pa[k][2], pa[k][3], b0, b1);
              if (MODE == kBF16Wide) mma<MODE>(acc, p3[k][0], 0, p3[k][1], 0, b0, b1);
            }
          }
          float *oo = o[j * C::epc + e];
          oo[0] = fmaf(oo[0], shrink, acc[0] + acc[2]);
          oo[1] = fmaf(oo[1], shrink, acc[1] + acc[3]);
        }
      }
      if (i + 1 < n) {
        if (!C::ahead) load_k(next, mask);
        load_v(next, mask);
        if (i + 2 < n) look_up(next + C::keys);
      }
    }
    l += __shfl_xor_sync(~0u, l, 1);
    l += __shfl_xor_sync(~0u, l, 2);
    __syncwarp();  // every lane is done with the query tile
    if (whole) {
      if (g < rows) {
        const float scale = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int j = 0; j < C::VJ; ++j)
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int e = 0; e < C::epc; e += 4) {
              const int d = (8 * j + 2 * t + k) * C::epc + e;
              const int b = j * C::epc + e;
              if (d < D)
                store4(p, seq, head0 + g, d,
                       make_float4(o[b][k] * scale, o[b + 1][k] * scale, o[b + 2][k] * scale, o[b + 3][k] * scale));
            }
        if (p.a.lse && t == 0) p.a.lse[seq * p.q_heads + head0 + g] = lse_of(m == -INFINITY ? 0.f : m, l);
      }
    } else {
      // the last piece of a run stays in shared memory, an earlier one goes to the workspace
      const int tail = at + n == we;
      float *to = tail ? reinterpret_cast<float *>(own) : p.heads + ((int64_t)blockIdx.x * W + warp) * C::piece;
#pragma unroll
      for (int j = 0; j < C::VJ; ++j)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int e = 0; e < C::epc; e += 4) {
            const int d = (8 * j + 2 * t + k) * C::epc + e, b = j * C::epc + e;
            if (d < DP && g < rows)
              *reinterpret_cast<float4 *>(to + g * C::o_row + d) =
                  make_float4(o[b][k], o[b + 1][k], o[b + 2][k], o[b + 3][k]);
          }
      if (t == 0) {
        to[kQT * C::o_row + g] = m;
        to[kQT * C::o_row + kQT + g] = l;
      }
      if (lane == 0) {
        const int i = 2 * warp + tail;
        s_seq[i] = seq, s_unit[i] = unit, s_open[i] = at - step0 < 0 ? 1 : at - step0 + sp.steps > run ? 2 : 0;
      }
    }
    at += n;
  }

  // ---- the block's pieces, one warp per segment and row
  __syncthreads();
  if (warp == 0) {
    const bool has = lane < 2 * W && s_seq[lane] >= 0;
    const uint32_t valid = __ballot_sync(~0u, has), earlier = valid & ((1u << lane) - 1);
    const int prev = 31 - __clz(earlier);
    const bool leads = has && (!earlier || s_seq[prev] != s_seq[lane] || s_unit[prev] != s_unit[lane]);
    const uint32_t leaders = __ballot_sync(~0u, leads);
    if (lane == 0) s_masks[0] = valid, s_masks[1] = leaders;
  }
  __syncthreads();
  const uint32_t valid = s_masks[0];
  constexpr int ND = (DP + 127) / 128;
  auto write_row = [&](int64_t seq, int head, const float4 (&y)[ND], float ref, float sum) {
    const float scale = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int k = 0; k < ND; ++k) {
      const int d = 4 * lane + 128 * k;
      if (d < D)
        store4(p, seq, head, d, make_float4(y[k].x * scale, y[k].y * scale, y[k].z * scale, y[k].w * scale));
    }
    if (p.a.lse && lane == 0) p.a.lse[seq * p.q_heads + head] = lse_of(ref, sum);
  };
  const int groups = __popc(s_masks[1]);
  for (int task = warp; task < groups * p.q_rows; task += W) {
    const int r = task % p.q_rows;
    uint32_t leaders = s_masks[1];
    for (int k = task / p.q_rows; k; --k) leaders &= leaders - 1;
    const int lead = __ffs(leaders) - 1;
    leaders &= leaders - 1;
    const uint32_t members = valid & ~((1u << lead) - 1) & (leaders ? (1u << (__ffs(leaders) - 1)) - 1 : ~0u);
    const int unit = s_unit[lead], qt = unit % p.qtiles, head = unit / p.qtiles * p.group + qt * kQT + r;
    if (qt * kQT + r >= p.group) continue;
    float4 y[ND];
    float ref, sum;
    add_up<DP>(PieceList{members, p.heads + (int64_t)blockIdx.x * W * C::piece, smem, C::piece, warp_bytes}, r, y, ref,
               sum);
    if (s_open[lead] == 0) {
      write_row(s_seq[lead], head, y, ref, sum);
    } else {
      float *rec = p.records + ((int64_t)blockIdx.x * 2 + s_open[lead] - 1) * C::piece;
#pragma unroll
      for (int k = 0; k < ND; ++k)
        if (4 * lane + 128 * k < DP) *reinterpret_cast<float4 *>(rec + r * C::o_row + 4 * lane + 128 * k) = y[k];
      if (lane == 0) {
        rec[kQT * C::o_row + r] = sum == 0.f ? -INFINITY : ref;
        rec[kQT * C::o_row + kQT + r] = sum;
      }
    }
  }

  // ---- segments that pass this run's ends: the last block to arrive adds the records up
  for (int k = 0; k < 2; ++k) {
    const Cut cut = s_cut[k];
    const int64_t x = cut.seg_begin, y_end = cut.seg_end;
    if (cut.at <= x || cut.at >= y_end || (k && x < begin)) continue;
    // the blocks of the segment: cuts inside it, by the same rule as above
    int64_t lo = x / per + 1, hi = (y_end + per - 1) / per - 1;
    while (snapped(lo * per, x, y_end, near) == x) ++lo;
    while (snapped(hi * per, x, y_end, near) == y_end) --hi;
    const int first = (int)lo - 1, last = (int)hi;
    const int64_t unit = (x - cut.seq_begin) / (y_end - x);
    __threadfence();
    __syncthreads();
    if (tid == 0) {
      int *word = p.arrivals + cut.seq * units + unit;
      s_last = atomicAdd(word, 1) == last - first;
      if (s_last) *word = 0;
    }
    __syncthreads();
    if (s_last) {
      __threadfence();
      const int qt = (int)(unit % p.qtiles), rows = min(kQT, p.group - qt * kQT);
      for (int r = warp; r < rows; r += W) {
        float4 y[ND];
        float ref, sum;
        add_up<DP>(RecordList{p.records, C::piece, first, last}, r, y, ref, sum);
        write_row(cut.seq, (int)(unit / p.qtiles) * p.group + qt * kQT + r, y, ref, sum);
      }
    }
    __syncthreads();
  }
}

}  // namespace attn
}  // namespace sc
