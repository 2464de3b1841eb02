// Decode attention over a paged cache: one query token per sequence.
//
// For each kv head, the keys of a sequence are read once for the whole group
// of query heads that share it; o = sum_j exp(z_j - m) v_j / sum_j exp(z_j - m)
// is built in one pass with a running maximum m.  Per key and kv head that is
// 2 head_dim elements read and 4 group head_dim flops, a few flops per byte:
// the bound is the memory read, and everything here serves to keep enough
// reads in flight.
//
// Matrix instructions.  A warp takes 16 (or 8) keys at a time and computes
// S = Q K^T and O += P V with mma.sync, the 8 query heads of a tile in rows
// 0-7.  Rows 8-15 carry what a single 16-bit or TF32 operand loses: Q and P
// are split into a head (rows 0-7) and a tail (rows 8-15), and the two halves
// of the result are added, so the split costs no further instructions.
//
// Fragments without shared-memory transposition.  The sum over head_dim may
// run in any order and the columns of O may be any permutation, so each lane
// takes whole 16-byte pieces: of K, piece t + 4j of key g (g = lane / 4,
// t = lane % 4) is a B fragment of 2 k-steps; of V, piece g + 8j of keys
// 2t, 2t+1 (+8) holds one column of O per element.  A lane therefore only
// ever reads back what it copied itself: its cp.async ring in shared memory
// needs no barrier, only its own wait_group.
//
// Work.  All (sequence, kv head, query tile) segments are cut into tiles of
// kTile keys and laid end to end; every block takes one equal, contiguous run
// of tiles, found by a scan over the sequence lengths on the device (the host
// never sees them).  A segment that one block covers is written directly;
// otherwise its blocks leave partial (m, l, O) records in the workspace and
// the last one to arrive adds them up in block order, so results do not
// depend on the order of arrival.
#pragma once

#include "sc_serve.h"

namespace sc {
namespace attn {

using serve::to_f32;

constexpr int kWarps = 4, kThreads = kWarps * 32, kQT = 8;

enum Mode { kTF32, kBF16, kBF16Wide, kF16, kF16Wide };

struct Params {
  sc_attn_args a;
  sc_kv_pool pool;
  int q_heads, group, qtiles, min_tiles;
  float scale_log2;  // scale * log2(e)
  int64_t window;
  int *status;
  int *arrivals;    // [seqs * kv_heads * qtiles], zero between calls
  float *partials;  // [blocks][2][kQT * (DP + 2)]
};

template <int MODE, int DP>
struct Cfg {
  static constexpr bool f32 = MODE == kTF32;
  static constexpr int es = f32 ? 4 : 2, epc = 16 / es;  // bytes per element, elements per 16-byte piece
  static constexpr int NT = f32 && DP > 64 ? 1 : 2;      // 8-key columns of S per warp step
  static constexpr int KJ = DP / (4 * epc), VJ = (DP + 8 * epc - 1) / (8 * epc);
  static constexpr int slots = NT * KJ + 2 * NT * VJ, stage = slots * 512;
  static constexpr int NST = stage <= 4096 ? 4 : stage <= 8192 ? 3 : 2;
  static constexpr int parts = MODE == kBF16Wide ? 3 : MODE == kBF16 || MODE == kF16 ? 1 : 2;  // of Q
  static constexpr int keys = NT * 8, tile = keys * kWarps;
  static constexpr int q_bytes = KJ * parts * 512;
  static constexpr int ring = kWarps * NST * stage;
  static constexpr int smem = ring + q_bytes;
  static constexpr int o_row = DP + 4;
  static constexpr int record = kQT * (DP + 2);  // floats of a partial record
  static_assert(NST * stage >= kQT * o_row * 4, "a warp's ring holds its O for the join");
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool ok) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0));
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

__device__ __forceinline__ float load_row(const void *p, int64_t type, int64_t i) {
  if (type == SC_TYPE_F32) return static_cast<const float *>(p)[i];
  if (type == SC_TYPE_F16) return to_f32(static_cast<const __half *>(p)[i]);
  return to_f32(static_cast<const __nv_bfloat16 *>(p)[i]);
}
__device__ __forceinline__ void store_row(void *p, int64_t type, int64_t i, float x) {
  if (type == SC_TYPE_F32)
    static_cast<float *>(p)[i] = x;
  else if (type == SC_TYPE_F16)
    static_cast<__half *>(p)[i] = __float2half_rn(x);
  else
    static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(x);
}

// Keys [first, len) of a sequence; the tiles start at `start`, first rounded
// down to a multiple of 16 so that no warp step straddles a page whose size is one.
struct Span {
  int first, len, start, tiles;
};

template <int TILE>
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
  r.tiles = (r.len - r.start) / TILE + ((r.len - r.start) % TILE != 0);
  return r;
}

template <int MODE, int DP>
__global__ void __launch_bounds__(kThreads) attend_kernel(const Params p) {
  using C = Cfg<MODE, DP>;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int64_t s_scan[kWarps];
  __shared__ int64_t s_found[2];
  __shared__ float s_scale[kQT], s_m[kWarps][kQT], s_l[kWarps][kQT], s_top[kQT], s_sum[kQT];
  __shared__ int s_last;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, t = lane % 4;
  const int D = (int)p.pool.head_dim, H = (int)p.pool.kv_heads;
  const int ps = (int)p.pool.page_size;
  const int64_t units = (int64_t)H * p.qtiles;  // segments of a sequence

  // ---- this block's run of tiles
  int64_t mine = 0;
  for (int64_t s = tid; s < p.a.seqs; s += kThreads) mine += span_of<C::tile>(p, s).tiles;
  for (int d = 16; d; d >>= 1) mine += __shfl_xor_sync(~0u, mine, d);
  if (lane == 0) s_scan[warp] = mine;
  __syncthreads();
  int64_t total = 0;
  for (int w = 0; w < kWarps; ++w) total += s_scan[w];
  total *= units;
  int64_t per = (total + gridDim.x - 1) / gridDim.x;
  if (per < p.min_tiles) per = p.min_tiles;
  const int64_t begin = per * blockIdx.x, end = begin + per < total ? begin + per : total;

  // sequences without keys
  for (int64_t s = blockIdx.x; s < p.a.seqs; s += gridDim.x)
    if (span_of<C::tile>(p, s).tiles == 0) {
      for (int i = tid; i < p.q_heads * D; i += kThreads)
        store_row(p.a.out.ptr, p.a.type,
                  s * p.a.out.stride[0] + (i / D) * p.a.out.stride[1] + (i % D) * p.a.out.stride[2], 0.f);
      if (p.a.lse)
        for (int i = tid; i < p.q_heads; i += kThreads) p.a.lse[s * p.q_heads + i] = -INFINITY;
    }
  if (begin >= end) return;

  // the sequence that holds tile `begin`
  int64_t before = 0;
  for (int64_t base = 0;; base += kThreads) {
    const int64_t s = base + tid;
    const int64_t n = s < p.a.seqs ? span_of<C::tile>(p, s).tiles * units : 0;
    int64_t sum = n;
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t up = __shfl_up_sync(~0u, sum, d);
      if (lane >= d) sum += up;
    }
    __syncthreads();
    if (lane == 31) s_scan[warp] = sum;
    if (tid == 0) s_found[0] = -1;
    __syncthreads();
    int64_t here = before;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) here += s_scan[w];
      before += s_scan[w];
    }
    if (begin >= here + sum - n && begin < here + sum) {
      s_found[0] = s;
      s_found[1] = here + sum - n;
    }
    __syncthreads();
    if (s_found[0] >= 0) break;
  }
  int64_t seq = s_found[0], seq_begin = s_found[1];
  Span sp = span_of<C::tile>(p, seq);

  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * (C::NST * C::stage) + lane * 16;
  const uint32_t sq = (uint32_t)__cvta_generic_to_shared(smem) + C::ring;
  const bool paged16 = ps % 16 == 0;
  const uint8_t *kbase = static_cast<const uint8_t *>(p.pool.k), *vbase = static_cast<const uint8_t *>(p.pool.v);
  const int64_t kslot = p.pool.k_stride[2] * C::es, vslot = p.pool.v_stride[2] * C::es;

  for (int64_t at = begin; at < end;) {
    while (at >= seq_begin + sp.tiles * units) {  // next sequence with keys
      seq_begin += sp.tiles * units;
      sp = span_of<C::tile>(p, ++seq);
    }
    const int64_t off = at - seq_begin, unit = off / sp.tiles;
    const int tile0 = (int)(off - unit * sp.tiles);
    const int h = (int)(unit / p.qtiles), qt = (int)(unit % p.qtiles);
    const int64_t seg_begin = seq_begin + unit * sp.tiles, seg_end = seg_begin + sp.tiles;
    const int n = (int)((seg_end < end ? seg_end : end) - at);
    const int rows = min(kQT, p.group - qt * kQT), head0 = h * p.group + qt * kQT;
    const int32_t *table = p.a.page_table + seq * p.a.table_stride;
    const int key0 = sp.start + tile0 * C::tile + warp * C::keys;

    // ---- copies of one warp step: 16-byte pieces of K, then of V
    uint64_t present = 0;  // 16 bits per ring stage: which of its keys there are
    auto entry_of = [&](int key) -> int { return key < sp.len ? table[key / ps] : 0; };
    int next_entry = paged16 ? entry_of(key0) : 0;
    auto issue = [&](int i) {
      const int key = key0 + i * C::tile;
      const uint32_t st = ring + (i % C::NST) * C::stage;
      uint32_t mask = 0;
      if (i < n && key < sp.len) {
        const int hi = min(sp.len - key, C::keys), lo = min(max(sp.first - key, 0), C::keys);
        mask = ((1u << hi) - 1) & ~((1u << lo) - 1);
        int64_t koff, voff;  // of key `key` (paged16), or of this lane's key
        if (paged16) {
          const int e = next_entry;
          if (e < 0 || e >= p.pool.num_pages) {
            if (lane == 0) serve::set_status(p.status, 8);
            mask = 0;
          }
          const int64_t page = mask ? e : 0;
          const int in = key % ps;
          koff = (page * p.pool.k_stride[0] + h * p.pool.k_stride[1]) * C::es + in * kslot;
          voff = (page * p.pool.v_stride[0] + h * p.pool.v_stride[1]) * C::es + in * vslot;
          next_entry = entry_of(key + C::tile);
        } else {
          int e = 0;
          const int mykey = key + (lane % C::keys);
          const bool want = mask >> (lane % C::keys) & 1;
          if (want) e = table[mykey / ps];
          const bool ok = want && e >= 0 && e < p.pool.num_pages;
          if (want && !ok) serve::set_status(p.status, 8);
          mask = __ballot_sync(~0u, ok) & ((1u << C::keys) - 1);
          const int64_t page = ok ? e : 0;
          const int in = ok ? mykey % ps : 0;
          koff = (page * p.pool.k_stride[0] + h * p.pool.k_stride[1]) * C::es + in * kslot;
          voff = (page * p.pool.v_stride[0] + h * p.pool.v_stride[1]) * C::es + in * vslot;
        }
        if (mask) {
#pragma unroll
          for (int nt = 0; nt < C::NT; ++nt) {
            const int k = nt * 8 + g;
            const uint8_t *src = kbase + (paged16 ? koff + k * kslot : __shfl_sync(~0u, koff, k));
            const bool ok = mask >> k & 1;
#pragma unroll
            for (int j = 0; j < C::KJ; ++j) {
              const int piece = t + 4 * j;
              const bool in = ok && piece * C::epc < D;
              copy16(st + (nt * C::KJ + j) * 512, in ? src + piece * 16 : kbase, in);
            }
          }
#pragma unroll
          for (int kk = 0; kk < 2 * C::NT; ++kk) {
            const int k = (kk / 2) * 8 + 2 * t + kk % 2;
            const uint8_t *src = vbase + (paged16 ? voff + k * vslot : __shfl_sync(~0u, voff, k));
            const bool ok = mask >> k & 1;
#pragma unroll
            for (int j = 0; j < C::VJ; ++j) {
              const int piece = g + 8 * j;
              const bool in = ok && piece * C::epc < D;
              copy16(st + (C::NT * C::KJ + kk * C::VJ + j) * 512, in ? src + piece * 16 : vbase, in);
            }
          }
        }
      }
      const int sh = (i % C::NST) * 16;
      present = (present & ~(0xffffull << sh)) | ((uint64_t)mask << sh);
      asm volatile("cp.async.commit_group;");
    };
    for (int i = 0; i < C::NST - 1; ++i) issue(i);

    // ---- the query tile, split into parts, in fragment order
    auto q_at = [&](int r, int d) {
      return r < rows && d < D ? load_row(p.a.q.ptr, p.a.type,
                                          seq * p.a.q.stride[0] + (head0 + r) * p.a.q.stride[1] + d * p.a.q.stride[2])
                               : 0.f;
    };
    for (int r = warp; r < kQT; r += kWarps) {
      // fp16 parts: rows are scaled by a power of two to below 2, so that no
      // part overflows and the tails stay above fp16's smallest values
      float up = 1.f;
      if (MODE == kF16Wide) {
        float top = 0.f;
        for (int d = lane; d < D; d += 32) top = fmaxf(top, fabsf(q_at(r, d)));
        for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
        const int e = (int)(__float_as_uint(top) >> 23) - 127;  // floor(log2(top)) of a normal number
        if (e > -120 && e < 127) up = __uint_as_float((uint32_t)(e + 127) << 23);
      }
      if (lane == 0) s_scale[r] = up;
    }
    if (MODE == kF16Wide) __syncthreads();
    for (int i = tid; i < C::KJ * 32; i += kThreads) {
      const int l = i % 32, r = l / 4, d0 = (l % 4 + 4 * (i / 32)) * C::epc;
      float x[C::epc];
#pragma unroll
      for (int e = 0; e < C::epc; ++e) {
        x[e] = q_at(r, d0 + e);
        if (MODE == kF16Wide) x[e] *= 1.f / s_scale[r];
      }
#pragma unroll
      for (int part = 0; part < C::parts; ++part) {
        uint32_t w[4];
        for (int e = 0; e < 4; ++e) {
          if (C::f32)
            w[e] = part ? tf32_tail(x[e]) : tf32_head(x[e]);
          else
            w[e] = pack2<MODE>(x[(2 * e) % C::epc], x[(2 * e + 1) % C::epc]);
        }
        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(sq + ((i / 32) * C::parts + part) * 512 + l * 16),
                     "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                     : "memory");
      }
    }
    __syncthreads();
    const float c = p.scale_log2 * s_scale[g];

    // ---- one pass over the keys
    float m = -INFINITY, l = 0.f;
    constexpr int ON = C::VJ * C::epc;
    float o[ON][2];
#pragma unroll
    for (int i = 0; i < ON; ++i) o[i][0] = o[i][1] = 0.f;
    for (int i = 0; i < n; ++i) {
      issue(i + C::NST - 1);
      asm volatile("cp.async.wait_group %0;" ::"n"(C::NST - 1) : "memory");
      const uint32_t mask = (uint32_t)(present >> ((i % C::NST) * 16)) & 0xffffu;
      if (!mask) continue;
      const uint32_t st = ring + (i % C::NST) * C::stage;
      float s[C::NT][2][4] = {};
#pragma unroll
      for (int j = 0; j < C::KJ; ++j) {
        uint4 q[C::parts];
#pragma unroll
        for (int part = 0; part < C::parts; ++part) q[part] = lds(sq + (j * C::parts + part) * 512 + lane * 16);
#pragma unroll
        for (int nt = 0; nt < C::NT; ++nt) {
          const uint4 k = lds(st + (nt * C::KJ + j) * 512);
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
      // running maximum and sum; a lane has query g and keys 2t, 2t+1 (+8)
      float x[C::NT][2], top = -INFINITY;
#pragma unroll
      for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          x[nt][e] = s[nt][0][e] + s[nt][1][e];
          if (C::parts > 1) x[nt][e] += s[nt][0][2 + e] + s[nt][1][2 + e];
          if (!(mask >> (nt * 8 + 2 * t + e) & 1)) x[nt][e] = -INFINITY;
          top = fmaxf(top, x[nt][e]);
        }
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
      top = fmaxf(m, top * c);
      const float ref = top == -INFINITY ? 0.f : top;
      const float shrink = ex2(m - ref);
      m = top;
      l *= shrink;
      uint32_t pa[C::NT][4];  // P as A fragments: one per 8 keys (f32) or pa[0]
#pragma unroll
      for (int nt = 0; nt < C::NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          x[nt][e] = ex2(fmaf(x[nt][e], c, -ref));
          l += x[nt][e];
        }
      }
      if (C::f32) {
#pragma unroll
        for (int nt = 0; nt < C::NT; ++nt) {
          pa[nt][0] = tf32_head(x[nt][0]);
          pa[nt][1] = tf32_tail(x[nt][0]);
          pa[nt][2] = tf32_head(x[nt][1]);
          pa[nt][3] = tf32_tail(x[nt][1]);
        }
      } else {
        pa[0][0] = pack2<MODE>(x[0][0], x[0][1]);
        pa[0][2] = pack2<MODE>(x[C::NT - 1][0], x[C::NT - 1][1]);
        pa[0][1] = pack2<MODE>(x[0][0], x[0][1]);
        pa[0][3] = pack2<MODE>(x[C::NT - 1][0], x[C::NT - 1][1]);
      }
      uint32_t p3a = 0, p3b = 0;
      if (MODE == kBF16Wide) {
        p3a = pack2<MODE>(x[0][0], x[0][1]);
        p3b = pack2<MODE>(x[C::NT - 1][0], x[C::NT - 1][1]);
      }
      const uint32_t sv = st + C::NT * C::KJ * 512;
#pragma unroll
      for (int j = 0; j < C::VJ; ++j) {
        uint32_t v[2 * C::NT][4];
#pragma unroll
        for (int kk = 0; kk < 2 * C::NT; ++kk) {
          const uint4 w = lds(sv + (kk * C::VJ + j) * 512);
          v[kk][0] = w.x, v[kk][1] = w.y, v[kk][2] = w.z, v[kk][3] = w.w;
        }
#pragma unroll
        for (int e = 0; e < C::epc; ++e) {
          float acc[4] = {};
          if (C::f32) {
#pragma unroll
            for (int nt = 0; nt < C::NT; ++nt) {
              const float v0 = __uint_as_float(v[2 * nt][e % 4]), v1 = __uint_as_float(v[2 * nt + 1][e % 4]);
              mma<MODE>(acc, pa[nt][0], pa[nt][1], pa[nt][2], pa[nt][3], tf32_head(v0), tf32_head(v1));
              mma<MODE>(acc, pa[nt][0], pa[nt][1], pa[nt][2], pa[nt][3], tf32_tail(v0), tf32_tail(v1));
            }
          } else {
            const uint32_t sel = e % 2 ? 0x7632 : 0x5410;
            const uint32_t b0 = __byte_perm(v[0][e / 2], v[1][e / 2], sel);
            const uint32_t b1 = __byte_perm(v[2 * C::NT - 2][e / 2], v[2 * C::NT - 1][e / 2], sel);
            mma<MODE>(acc, pa[0][0], pa[0][1], pa[0][2], pa[0][3], b0, b1);
            if (MODE == kBF16Wide) mma<MODE>(acc, p3a, 0, p3b, 0, b0, b1);
          }
          float *oo = o[j * C::epc + e];
          oo[0] = fmaf(oo[0], shrink, acc[0] + acc[2]);
          oo[1] = fmaf(oo[1], shrink, acc[1] + acc[3]);
        }
      }
    }

    // ---- join the warps
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    l += __shfl_xor_sync(~0u, l, 1);
    l += __shfl_xor_sync(~0u, l, 2);
    if (t == 0) s_m[warp][g] = m, s_l[warp][g] = l;
    __syncwarp();  // every lane has read its last stage before O goes into the warp's ring
    float *so = reinterpret_cast<float *>(smem) + warp * (C::NST * C::stage / 4);
#pragma unroll
    for (int j = 0; j < C::VJ; ++j)
#pragma unroll
      for (int e = 0; e < C::epc; ++e)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int d = (8 * j + 2 * t + k) * C::epc + e;
          if (d < DP) so[g * C::o_row + d] = o[j * C::epc + e][k];
        }
    __syncthreads();
    const float *all = reinterpret_cast<const float *>(smem);
    const bool whole = at == seg_begin && at + n == seg_end;
    float *record = p.partials + ((int64_t)blockIdx.x * 2 + (at == seg_begin)) * C::record;
    if (tid < rows) {
      float top = -INFINITY, sum = 0.f;
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w][tid]);
      const float ref = top == -INFINITY ? 0.f : top;
      for (int w = 0; w < kWarps; ++w) sum += s_l[w][tid] * ex2(s_m[w][tid] - ref);
      s_top[tid] = ref;
      s_sum[tid] = sum;
      if (whole) {
        if (p.a.lse) p.a.lse[seq * p.q_heads + head0 + tid] = (ref + log2f(sum)) * 0.69314718055994531f;
      } else {
        record[kQT * DP + tid] = top;
        record[kQT * DP + kQT + tid] = sum;
      }
    }
    __syncthreads();
    for (int i = tid; i < rows * D; i += kThreads) {
      const int r = i / D, d = i - r * D;
      float y = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w)
        y += all[w * (C::NST * C::stage / 4) + r * C::o_row + d] * ex2(s_m[w][r] - s_top[r]);
      if (whole)
        store_row(p.a.out.ptr, p.a.type,
                  seq * p.a.out.stride[0] + (head0 + r) * p.a.out.stride[1] + d * p.a.out.stride[2],
                  s_sum[r] == 0.f ? 0.f : y / s_sum[r]);
      else
        record[r * DP + d] = y;
    }
    if (!whole) {
      // the last of the segment's blocks adds their records up in block order
      const int first = (int)(seg_begin / per), last = (int)((seg_end - 1) / per);
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        int *word = p.arrivals + seq * units + unit;
        s_last = atomicAdd(word, 1) == last - first;
        if (s_last) *word = 0;
      }
      __syncthreads();
      if (s_last) {
        __threadfence();
        auto rec = [&](int b) { return p.partials + ((int64_t)b * 2 + (b == first)) * C::record; };
        float *w = reinterpret_cast<float *>(smem);  // [blocks of the segment][kQT] weights
        const int parts = last - first + 1;
        for (int i = tid; i < parts * rows; i += kThreads)
          w[(i / rows) * kQT + i % rows] = __ldcg(rec(first + i / rows) + kQT * DP + i % rows);
        __syncthreads();
        if (tid < rows) {
          float top = -INFINITY, sum = 0.f;
          for (int b = 0; b < parts; ++b) top = fmaxf(top, w[b * kQT + tid]);
          const float ref = top == -INFINITY ? 0.f : top;
          for (int b = 0; b < parts; ++b) {
            const float f = ex2(w[b * kQT + tid] - ref);
            w[b * kQT + tid] = f;
            sum += f * __ldcg(rec(first + b) + kQT * DP + kQT + tid);
          }
          s_sum[tid] = sum;
          if (p.a.lse) p.a.lse[seq * p.q_heads + head0 + tid] = (ref + log2f(sum)) * 0.69314718055994531f;
        }
        __syncthreads();
        for (int i = tid; i < rows * D; i += kThreads) {
          const int r = i / D, d = i - r * D;
          float y = 0.f;
#pragma unroll 8
          for (int b = 0; b < parts; ++b) y += w[b * kQT + r] * __ldcg(rec(first + b) + r * DP + d);
          store_row(p.a.out.ptr, p.a.type,
                    seq * p.a.out.stride[0] + (head0 + r) * p.a.out.stride[1] + d * p.a.out.stride[2],
                    s_sum[r] == 0.f ? 0.f : y / s_sum[r]);
        }
      }
    }
    __syncthreads();
    at += n;
  }
}

}  // namespace attn
}  // namespace sc
