// Decode attention over a paged cache: one query token per sequence.
//
// For each kv head, the keys of a sequence are read once for the whole group
// of query heads that share it; o = sum_j exp(z_j - m) v_j / sum_j exp(z_j - m)
// is built in one pass with a running maximum m.  Per key and kv head that is
// 2 head_dim elements read and 4 group head_dim flops, a few flops per byte:
// the bound is the memory read, and everything here serves to keep enough
// reads in flight.
//
// Matrix instructions.  A warp takes `keys` keys at a time and computes
// S = Q K^T and O += P V with mma.sync, the query heads of a tile in the first
// rows.  Rows that a group of heads leaves free carry what a single 16-bit or
// TF32 operand loses: Q and P are split into parts that share one instruction
// (head in rows 0-7, tail in rows 8-15), and the parts of the result are
// added.  16-bit queries of the cache's type need no parts (P has two for them:
// 16 bits or more, below the rounding of their results); fp32 queries over
// fp16 two, over bf16 three: those fit one instruction for groups of up to
// four (rows 0-3, 4-7, 8-11: kBF16Wide4) and take two for larger ones.  An fp32
// cache is split too, into TF32 heads and tails: two instructions.
//
// Fragments without shared-memory transposition.  The sum over head_dim may
// run in any order and the columns of O may be any permutation, so each lane
// takes whole 16-byte pieces: of K, piece t + 4j of key g (g = lane / 4,
// t = lane % 4) is a B fragment of 2 k-steps; of V, piece g + 8j of keys
// 2t, 2t+1 (+8) holds one column of O per element.  K and V go from global
// memory straight into the registers that feed the matrix instructions: the
// next K is asked for as soon as the scores are done, the next V after the
// product with P.  At 8 KB a warp step and 12 warps a SM that is 48-96 KB in
// flight, more than latency times bandwidth asks for.  A version with 16 warps
// that went through cp.async and shared memory took 147 us at 131071 keys (8
// kv heads of 128, bf16), a fifth of it in a slower join; this takes 94, 5.7
// TB/s.  Row addresses are computed where they are needed: handing them round
// by shuffles cost a fifth of the loop's speed.
//
// Work.  All (sequence, kv head, query tile) segments are cut into steps of
// `keys` keys and laid end to end.  Every block takes one equal, contiguous
// run of steps, found by a scan over the sequence lengths on the device (the
// host never sees them), and every warp an equal share of its block's run.
// Warps do not wait for one another until all are done: a segment that one
// warp covers is written directly, the others leave pieces (m, l, O) that the
// block adds up at its end.  A segment that passes the end of a block's run
// goes into a record in the workspace, and the last of its blocks to arrive
// adds the records up.  Pieces and records are added in the order of the
// keys, so results do not depend on the order of arrival.
//
// What is left over the read: the scan, the first loads, and the two joins, 5
// to 10 us in all, most of it fetching code that each block runs once (25
// cycles an instruction while the memory is busy).  128 fp32 requests of 16 to
// 1024 keys, 8 heads of 64: 40 us against 19 for the bytes; 32 requests of 100
// to 8192 keys, 32 / 8 heads of 128, fp32 queries over bf16: 63 against 39.
#pragma once

#include "sc_mma.cuh"
#include "sc_serve.h"

namespace sc {
namespace attn {

using serve::to_f32;
using namespace mma;

constexpr int kQT = 8, kMaxWarps = 12, kWindow = 128;

struct Params {
  sc_attn_args a;
  sc_kv_pool pool;
  int q_heads, group, qtiles, q_rows;  // q_rows: rows of a query tile, min(group, kQT)
  int min_run;                         // fewest places of a block
  int q_vec;                           // query rows are contiguous and 16-byte aligned
  uint32_t page_mul, page_shift;       // key / page_size = umulhi(key, mul) >> shift (mul 0: page_size 1)
  uint32_t k_page, k_slot, v_page, v_slot;  // strides in 16-byte units
  float scale_log2;                    // scale * log2(e)
  int64_t window;
  int *status;
  const uint8_t *zeros;  // 1 KB
  int *arrivals;   // [seqs * kv_heads * qtiles], zero between calls
  uint32_t *doubtful;  // as many: rows (bits) of a query tile whose results are not finite, and the block (+ 1) that wrote them
  float *heads;    // [blocks][warps] pieces whose warp went on after them
  float *records;  // [blocks][2]
};

// One instantiation of the kernel and what its launch needs.
struct Variant {
  void (*kernel)(Params);
  int warps, smem, keys, piece, change;
};

// The instantiation for a head_dim, made ready on the current device.
template <Mode MODE>
Variant variant_for(int64_t head_dim, int q_rows, int smem_limit);

// DP: head_dim rounded up to what the kernel is laid out for; FULL: head_dim is DP.
template <int MODE, int DP>
struct Cfg {
  static constexpr bool f32 = MODE == kTF32, quarter = MODE == kBF16Wide4;
  static constexpr int es = f32 ? 4 : 2, epc = 16 / es;  // bytes per element, elements per 16-byte piece
  // 8-key columns of S per step: 8 KB of K and V (16 KB from head_dim 129 on)
  static constexpr int NT = f32 ? (DP > 64 ? 1 : 2) : (DP > 64 ? 2 : 4);
  static constexpr int KJ = (DP + 4 * epc - 1) / (4 * epc), VJ = (DP + 8 * epc - 1) / (8 * epc);
  static constexpr int parts = MODE == kBF16Wide || quarter ? 3 : MODE == kBF16 || MODE == kF16 ? 1 : 2;  // of Q
  static constexpr int keys = NT * 8, sub = keys < 16 ? keys : 16;
  static constexpr int q_row = KJ * parts * 64;              // bytes of one query row in fragment order
  static constexpr int max_warps = DP > 128 ? 8 : kMaxWarps;  // by the registers of a step
  // Segments are laid end to end with this many places after each that hold no keys: they stand for what changing to
  // another segment costs a warp (its query, its pages, its result) in steps.  us with 1 / 2 / 3 / 4, fp32 caches: 128
  // requests of 16-1024 keys 40.0 41.2 41.9 43.8, 64 of 50-3000 50.6 51.3 51.4 52.5, 37 of 1-700 (4 kv heads of 128)
  // 22.0 23.4 23.2 23.2; 16 bits: 32 of 100-8192 70.1 65.5 62.6 62.6, 48 of 1-2500 39.1 33.6 32.6 32.8, 61 windows of
  // 1000 30.0 27.3 27.2 28.0, 100 windows of 500 22.2 22.3 22.5 22.6.
  static constexpr int change = f32 ? 1 : 3;
  // P (1 at most) as it is split into fp16 parts: two parts then keep weights down to 2^-38 of the largest, where fp16's
  // smallest value would cut those of e^-16 to a single bit.  Taken off again where a portion's result is written.
  static constexpr float lift = is_f16(MODE) ? 16384.f : 1.f;
  static constexpr bool ahead = DP <= 128;                   // registers suffice to load K a phase ahead
  static constexpr int o_row = DP + 4;                       // floats; the pad spreads rows over the banks
  static constexpr int piece = kQT * o_row + 2 * kQT;        // O | m | l
  // shared memory of a warp: a result or its last piece, a query tile as it is and in fragment order, page entries
  __host__ __device__ static constexpr int warp_bytes(int q_rows) { return piece * 4 + (o_row * 4 + q_row) * q_rows + kWindow * 4; }
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

__device__ __forceinline__ void copy_async(uint32_t dst, const void *src, bool four) {
  if (four)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
  else
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// Code that a block runs once costs more to fetch than to execute, so what is
// not in the loop over the keys is kept small: no unrolled loops, 32-bit
// places, one copy of each part.

// Generic loads that see other blocks' writes.
__device__ __forceinline__ float ld_relaxed(const float *p) {
  float v;
  asm volatile("ld.relaxed.gpu.f32 %0, [%1];" : "=f"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ float4 ld_relaxed4(const float *p) {
  float4 v;
  asm volatile("ld.relaxed.gpu.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
  return v;
}

// Four neighbouring outputs; whether they are finite.  Out of line: it is not worth a copy at each of its uses.
static __device__ __noinline__ bool store4(void *ptr, int type, int64_t i, int64_t stride, float4 y) {
  const float v[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (type == SC_TYPE_F32)
      static_cast<float *>(ptr)[i + e * stride] = v[e];
    else if (type == SC_TYPE_F16)
      static_cast<__half *>(ptr)[i + e * stride] = __float2half_rn(v[e]);
    else
      static_cast<__nv_bfloat16 *>(ptr)[i + e * stride] = __float2bfloat16_rn(v[e]);
  }
  return fabsf(y.x) + fabsf(y.y) + fabsf(y.z) + fabsf(y.w) < INFINITY;
}

// Keys [first, len) of a sequence; steps start at `start`, first rounded down
// to a multiple of 16.
struct Span {
  int first, len, start, steps;
};

template <int KEYS>
__device__ __forceinline__ Span span_of(const Params &p, int s) {
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

__device__ __forceinline__ float lse_of(float ref, float sum) { return (ref + log2f(sum)) * 0.69314718055994531f; }

// Element i of an array of a type known at run time.
__device__ __forceinline__ float element(const void *p, int type, int64_t i) {
  return type == SC_TYPE_F32   ? static_cast<const float *>(p)[i]
         : type == SC_TYPE_F16 ? __half2float(static_cast<const __half *>(p)[i])
                               : __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}

// A boundary between two blocks' runs: the place that an equal cut gives,
// moved to an end of its segment when that is near, which saves a join, or
// when no keys are left there.
struct Cut {
  int at, seq_begin, seg_begin, seg_end, seq;
};

template <int CHANGE>
__device__ __forceinline__ int snapped(int b, int x, int y, int near) {
  const int lo = b - x, hi = y - b;
  return lo <= near && lo <= hi ? x : hi <= near || hi <= CHANGE ? y : b;
}

template <int MODE, int DP, bool FULL>
__global__ void __launch_bounds__(Cfg<MODE, DP>::max_warps * 32, 1) attend_kernel(const __grid_constant__ Params p) {
  using C = Cfg<MODE, DP>;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int s_scan[kMaxWarps], s_more[kMaxWarps];
  __shared__ Cut s_cut[2];
  // pieces: sequence (-1: none), segment of it, and whether that began before (1) or only ends after (2) this run
  __shared__ int s_seq[2 * kMaxWarps], s_unit[2 * kMaxWarps], s_open[2 * kMaxWarps];
  __shared__ int s_last, s_doubt;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, t = lane % 4;
  const int W = blockDim.x / 32, D = FULL ? DP : (int)p.pool.head_dim;
  const int seqs = (int)p.a.seqs;
  const int units = (int)p.pool.kv_heads * p.qtiles;  // segments of a sequence

  // A result that is not finite: its row is computed again at the end.
  auto doubt = [&](int seq, int unit, int row) {
    atomicOr(p.doubtful + (int64_t)seq * units + unit, (blockIdx.x + 1) << kQT | 1u << row);
    s_doubt = 1;
  };
  auto work = [&] {
  // ---- this block's run: a scan over the sequences, blockDim of them at a time
  auto places_of = [&](int s) {  // of one of its segments
    const int n = s < seqs ? span_of<C::keys>(p, s).steps : 0;
    return n ? n + C::change : 0;
  };
  int n = places_of(tid), more = 0;
#pragma unroll 1
  for (int s = tid + blockDim.x; s < seqs; s += blockDim.x) more += places_of(s);
  auto scan = [&](int v) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(~0u, v, d);
      if (lane >= d) v += up;
    }
    if (lane == 31) s_scan[warp] = v;
    return v;
  };
  int incl = scan(n);
  more = __reduce_add_sync(~0u, more);
  if (lane == 0) s_more[warp] = more;
  if (tid < 2 * W) s_seq[tid] = -1;
  if (tid == 0) s_doubt = 0;
  __syncthreads();
  auto sum_of = [&](const int *v, int below) {  // of the first `below` warps' sums
    return __reduce_add_sync(~0u, lane < below ? v[lane] : 0);
  };
  int before = sum_of(s_scan, warp), chunk = sum_of(s_scan, W);
  const int total = (chunk + sum_of(s_more, W)) * units;
  const int per = max((int)((total + gridDim.x - 1) / gridDim.x), p.min_run);
  // A join costs about what a block's eighth does, or half a step of every warp: with a quarter of either the smallest
  // batch took 14.2 us instead of 11.8 and 48 requests of 1-2500 keys 34.6 instead of 32.5; with twice the eighth 32 of
  // 100-8192 keys 66.8 instead of 62.6 and 64 fp32 ones of 50-3000 56.4 instead of 50.5 (61 windows 26.3, not 27.2).
  const int near = max(per / 8, min(per, W) / 2);
  const int nominal0 = per * blockIdx.x, nominal1 = nominal0 + per;
  if (nominal0 >= total) return;
  if (nominal1 >= total && tid == 0) s_cut[1] = Cut{total, total, total, total, seqs};
#pragma unroll 1
  for (int base = 0;;) {
    const int from = (before + incl - n) * units, to = from + n * units;
#pragma unroll 1
    for (int k = 0; k < 2; ++k) {
      const int b = k ? nominal1 : nominal0;
      if (b >= from && b < to) {
        const int x = from + (b - from) / n * n;
        s_cut[k] = Cut{snapped<C::change>(b, x, x + n, near), from, x, x + n, base + tid};
      }
    }
    base += blockDim.x;
    if (base >= seqs || chunk * units > nominal1) break;
    __syncthreads();
    n = places_of(base + tid);
    incl = scan(n);
    __syncthreads();
    before = chunk + sum_of(s_scan, warp);
    chunk += sum_of(s_scan, W);
  }
  __syncthreads();
  const int begin = s_cut[0].at, end = s_cut[1].at;
  if (begin >= end) return;

  // ---- this warp's share of it; places in the run are counted from its begin from here on
  const int run = end - begin, share = run / W, rest = run - share * W;
  const int wb = share * warp + min(warp, rest), we = wb + share + (warp < rest);
  const int warp_bytes = C::warp_bytes(p.q_rows);
  float *own = reinterpret_cast<float *>(smem + warp * warp_bytes);
  // query row g in fragment order; lanes beyond the tile's rows repeat its last one, their results go nowhere
  const int qg = min(C::quarter ? g % 4 : g, p.q_rows - 1), q_step = p.q_rows * 64;
  const uint32_t raw = (uint32_t)__cvta_generic_to_shared(own) + C::piece * 4;
  const uint32_t sq = raw + C::o_row * 4 * p.q_rows + qg * 64 + t * 16;

  const bool paged16 = p.pool.page_size % 16 == 0;
  // the step whose keys are looked up: its sequence, segment and key, and how many follow in this portion of a segment
  int seq = s_cut[0].seq, unit = 0, key = 0, left = 0, at = wb;
  int seq_begin = s_cut[0].seq_begin - begin;
  Span sp = span_of<C::keys>(p, seq);
  bool whole = false;
  int open = 0;
  const uint8_t *k_head = nullptr, *v_head = nullptr;  // the segment's kv head in the first page
  const int32_t *table = nullptr;
  // Moves `at` to the next place that holds keys and describes the portion that begins there; at >= we: none left.
  auto open_portion = [&] {
    int step0 = 0;
#pragma unroll 1
    for (;;) {
#pragma unroll 1
      while (sp.steps == 0 || at >= seq_begin + (sp.steps + C::change) * units) {  // next sequence with keys
        if (at >= we) return;
        if (sp.steps) seq_begin += (sp.steps + C::change) * units;
        sp = span_of<C::keys>(p, ++seq);
      }
      const uint32_t off = (uint32_t)(at - seq_begin), each = sp.steps + C::change;
      unit = (int)(off / each);
      step0 = (int)(off - unit * each);
      if (step0 < sp.steps || at >= we) break;
      at += each - step0;
    }
    if (at >= we) return;
    left = min(sp.steps - step0, we - at);
    whole = left == sp.steps;
    open = at < step0 ? 1 : at - step0 + sp.steps > run ? 2 : 0;
    key = sp.start + step0 * C::keys;
    k_head = static_cast<const uint8_t *>(p.pool.k) + unit / p.qtiles * p.pool.k_stride[1] * C::es;
    v_head = static_cast<const uint8_t *>(p.pool.v) + unit / p.qtiles * p.pool.v_stride[1] * C::es;
    table = p.a.page_table + seq * p.a.table_stride;
  };
  // Page entries of the portion, kWindow of them at a time in shared memory: those of pages window, window + 1, ...
  // A load per step would make every step wait for it, and for the V loads that were asked for before it.
  int window = 0;
  int *entries = reinterpret_cast<int *>(reinterpret_cast<uint8_t *>(own) + warp_bytes) - kWindow;
  auto open_window = [&](int first) {
    const int end_page = page_of(p, sp.len - 1);
    int e[kWindow / 32];
#pragma unroll
    for (int i = 0; i < kWindow / 32; ++i) {
      const int page = first + lane + 32 * i;
      e[i] = page <= end_page ? __ldg(table + page) : -1;
    }
    window = first;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kWindow / 32; ++i) entries[lane + 32 * i] = e[i];
    __syncwarp();
  };
  // Present keys of the step at `key`, and the rows of this lane in 16-byte units: of K, key 8 nt + g; of V, keys
  // 8 nt + 2t + (0, 1).  In place of an absent key a present one is read (its weight becomes zero).  Without any (a bad
  // page entry) all lanes read a row of zeros, and the step goes its way: a branch around the use of the loaded
  // registers makes copies of them that wait for the loads (126 us against 100 at 131071 keys).
  uint32_t mask = 0, row_k[C::NT], row_v[2 * C::NT];
  bool empty = true;
  auto place = [&] {
    const int first = page_of(p, key);
    if (first - window > kWindow - C::keys) open_window(first);
    const int hi = min(sp.len - key, C::keys), lo = min(max(sp.first - key, 0), C::keys);
    mask = (uint32_t)((1ull << hi) - 1) & ~(uint32_t)((1ull << lo) - 1);
    if (paged16) {  // whole 16s of keys lie in a page
      uint32_t e[C::keys / C::sub], in[C::keys / C::sub];
      bool bad = false;
#pragma unroll
      for (int i = 0; i < C::keys / C::sub; ++i) {
        const int page = page_of(p, key + 16 * i);
        e[i] = entries[page - window];
        in[i] = key + 16 * i - page * (int)p.pool.page_size;
        if (mask >> (16 * i) & 0xffffu && e[i] >= (uint32_t)p.pool.num_pages) {
          bad = true;
          mask &= ~(0xffffu << (16 * i));
        }
      }
      if (bad) serve::set_status(p.status, 8);
      // the present keys are a range but for bad pages; then a lane may need another 16's page
      const int a = __ffs(mask | 1u << 31) - 1, b = 31 - __clz(mask | 1);
      auto row = [&](int k8, int k, uint32_t page, uint32_t slot) -> uint32_t {
        if (C::keys / C::sub == 1) return e[0] * page + (in[0] + min(max(k8 + k, a), b)) * slot;
        const int kk = min(max(k8 + k, a), b), i = kk >> 4;
        return (i ? e[C::keys / C::sub - 1] : e[0]) * page + ((i ? in[C::keys / C::sub - 1] : in[0]) + (kk & 15)) * slot;
      };
#pragma unroll
      for (int nt = 0; nt < C::NT; ++nt) row_k[nt] = row(nt * 8, g, p.k_page, p.k_slot);
#pragma unroll
      for (int kk = 0; kk < 2 * C::NT; ++kk) row_v[kk] = row(kk / 2 * 8, 2 * t + kk % 2, p.v_page, p.v_slot);
    } else {
      const int k = key + lane % C::keys, page = page_of(p, k);
      const bool there = mask >> (lane % C::keys) & 1;
      uint32_t e = there ? entries[page - window] : 0;
      const bool ok = there && e < (uint32_t)p.pool.num_pages;
      if (there && !ok) serve::set_status(p.status, 8);
      mask = __ballot_sync(~0u, ok) & (uint32_t)((1ull << C::keys) - 1);
      if (!ok) e = 0;
      const uint32_t in = (uint32_t)(k - page * (int)p.pool.page_size);
      const uint32_t at_k = e * p.k_page + in * p.k_slot, at_v = e * p.v_page + in * p.v_slot;
      const int spare = __ffs(mask | 1u << 31) - 1;
#pragma unroll
      for (int nt = 0; nt < C::NT; ++nt)
        row_k[nt] = __shfl_sync(~0u, at_k, mask >> (nt * 8 + g) & 1 ? nt * 8 + g : spare);
#pragma unroll
      for (int kk = 0; kk < 2 * C::NT; ++kk) {
        const int i = kk / 2 * 8 + 2 * t + kk % 2;
        row_v[kk] = __shfl_sync(~0u, at_v, mask >> i & 1 ? i : spare);
      }
    }
    empty = !mask;
    if (empty) {
#pragma unroll
      for (int nt = 0; nt < C::NT; ++nt) row_k[nt] = 0;
#pragma unroll
      for (int kk = 0; kk < 2 * C::NT; ++kk) row_v[kk] = 0;
    }
  };
  // This lane's 16-byte pieces: of K, piece t + 4j; of V, piece g + 8j.  In place of a piece beyond head_dim the first
  // one is read (it meets zeros of Q, or makes columns of O that go nowhere).
  uint4 kf[C::NT][C::KJ], vf[2 * C::NT][C::VJ];
  // Without any (a bad page entry) all lanes read a row of zeros, and the step goes its way: a branch around the use of
  // these registers makes copies of them that wait for the loads (126 us against 100 at 131071 keys).
  auto load_k = [&] {
    const uint8_t *base = empty ? p.zeros : k_head;
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt) {
      const uint8_t *row = base + (uint64_t)row_k[nt] * 16 + (FULL ? t * 16 : 0);
#pragma unroll
      for (int j = 0; j < C::KJ; ++j)
        kf[nt][j] = ldg16(row + (FULL ? j * 64 : (t + 4 * j) * C::epc < D ? (t + 4 * j) * 16 : 0));
    }
  };
  auto load_v = [&] {
    constexpr bool all = FULL && DP % (8 * C::epc) == 0;
    const uint8_t *base = empty ? p.zeros : v_head;
#pragma unroll
    for (int kk = 0; kk < 2 * C::NT; ++kk) {
      const uint8_t *row = base + (uint64_t)row_v[kk] * 16 + (all ? g * 16 : 0);
#pragma unroll
      for (int j = 0; j < C::VJ; ++j)
        vf[kk][j] = ldg16(row + (all ? j * 128 : (g + 8 * j) * C::epc < D ? (g + 8 * j) * 16 : 0));
    }
  };
  // The query tile of the portion at hand: its raw rows into shared memory, then split into parts in fragment order.
  auto copy_q = [&] {
    const int h = unit / p.qtiles, qt = unit - h * p.qtiles, rows = min(kQT, p.group - qt * kQT);
    const int es = p.a.type == SC_TYPE_F32 ? 4 : 2, n = p.q_vec ? D * es / 16 : D;
    const int64_t step = p.q_vec ? 16 : p.a.q.stride[2] * es;
    const uint8_t *src = static_cast<const uint8_t *>(p.a.q.ptr) +
                         (seq * p.a.q.stride[0] + (h * p.group + qt * kQT) * p.a.q.stride[1]) * es;
    __syncwarp();
#pragma unroll 1
    for (int r = 0; r < rows; ++r, src += p.a.q.stride[1] * es)
#pragma unroll 1
      for (int i = lane; i < n; i += 32) {
        const uint32_t to = raw + r * C::o_row * 4 + i * (p.q_vec ? 16 : es);
        if (p.q_vec || es == 4) {
          copy_async(to, src + i * step, !p.q_vec);
        } else {
          asm volatile("st.shared.u16 [%0], %1;" ::"r"(to), "h"(*reinterpret_cast<const uint16_t *>(src + i * step))
                       : "memory");
        }
      }
  };
  float c = 1.f;
  auto split_q = [&] {
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
    const uint32_t row = raw + qg * C::o_row * 4;
    auto piece = [&](int j, float (&x)[C::epc]) {  // elements of piece t + 4j
      const int d = (t + 4 * j) * C::epc;
      if (d >= D) {
#pragma unroll
        for (int e = 0; e < C::epc; ++e) x[e] = 0.f;
      } else if (p.a.type == SC_TYPE_F32) {
#pragma unroll
        for (int e = 0; e < C::epc; e += 4) {
          const uint4 w = lds(row + (d + e) * 4);
          x[e] = __uint_as_float(w.x), x[e + 1] = __uint_as_float(w.y);
          x[e + 2] = __uint_as_float(w.z), x[e + 3] = __uint_as_float(w.w);
        }
      } else {
        const uint4 w = lds(row + (d * 2 & ~15));
        const uint32_t v[4] = {C::epc == 4 && d % 8 ? w.z : w.x, C::epc == 4 && d % 8 ? w.w : w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < C::epc; ++e) {
          const uint32_t bits = e % 2 ? v[e / 2] >> 16 : v[e / 2] & 0xffffu;
          x[e] = p.a.type == SC_TYPE_BF16 ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half((uint16_t)bits));
        }
      }
    };
    float up = 1.f;  // fp16 parts are of scaled rows
    if (MODE == kF16Wide) {
      float top = 0.f;
#pragma unroll 1
      for (int j = 0; j < C::KJ; ++j) {
        float x[C::epc];
        piece(j, x);
#pragma unroll
        for (int e = 0; e < C::epc; ++e) top = fmaxf(top, fabsf(x[e]));
      }
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
      up = f16_scale(top);
    }
    // not zero: the -inf of a masked key stays one; scores of so small a factor are zero in any case
    c = fmaxf(p.scale_log2 * up, 1.17549435e-38f);
#pragma unroll 1
    for (int j = 0; j < C::KJ; ++j) {
      float x[C::epc];
      piece(j, x);
      if (MODE == kF16Wide)
#pragma unroll
        for (int e = 0; e < C::epc; ++e) x[e] *= 1.f / up;
#pragma unroll
      for (int part = 0; part < C::parts; ++part) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (C::f32)
            w[e] = part ? tf32_tail(x[e]) : tf32_head(x[e]);
          else
            w[e] = pack2<MODE>(x[(2 * e) % C::epc], x[(2 * e + 1) % C::epc]);
        }
        if (g < p.q_rows)
          asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(sq + (j * C::parts + part) * q_step), "r"(w[0]),
                       "r"(w[1]), "r"(w[2]), "r"(w[3])
                       : "memory");
      }
    }
    __syncwarp();
  };

  constexpr int ON = C::VJ * C::epc;
#pragma unroll 1
  for (;;) {
    open_portion();
    if (at >= we) break;
    float m = -INFINITY, l = 0.f, o[ON][2];
#pragma unroll
    for (int i = 0; i < ON; ++i) o[i][0] = o[i][1] = 0.f;
    copy_q();
    open_window(page_of(p, key));
    place();
    load_k();
    load_v();
    split_q();
    at += left;
#pragma unroll 1
    for (; left > 0; --left) {
    const uint32_t now = mask;
    const bool more_keys = left > 1;
    // scores
    float s[C::NT][2][4] = {};
    {
#pragma unroll
      for (int j = 0; j < C::KJ; ++j) {
        uint4 q[C::parts];
#pragma unroll
        for (int part = 0; part < C::parts; ++part) q[part] = lds(sq + (j * C::parts + part) * q_step);
        // rows 0-7 and 8-15 of A
        uint4 a0 = q[0], a1 = make_uint4(0, 0, 0, 0);
        if (C::parts == 2) a1 = q[C::parts - 1];
        if (MODE == kBF16Wide) a1 = q[C::parts > 1 ? 1 : 0];
        if (C::quarter) {
          if (g < 4)
            a1 = q[C::parts - 1];
          else
            a0 = q[C::parts > 1 ? 1 : 0];
        }
#pragma unroll
        for (int nt = 0; nt < C::NT; ++nt) {
          const uint4 k = kf[nt][j];
          if (C::f32) {
            const uint32_t kw[4] = {k.x, k.y, k.z, k.w}, qh[4] = {a0.x, a0.y, a0.z, a0.w},
                           ql[4] = {a1.x, a1.y, a1.z, a1.w};
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
              const float k0 = __uint_as_float(kw[e]), k1 = __uint_as_float(kw[e + 1]);
              mma16<MODE>(s[nt][0], qh[e], ql[e], qh[e + 1], ql[e + 1], tf32_head(k0), tf32_head(k1));
              mma16<MODE>(s[nt][1], qh[e], ql[e], qh[e + 1], ql[e + 1], tf32_tail(k0), tf32_tail(k1));
            }
          } else {
            mma16<MODE>(s[nt][0], a0.x, a1.x, a0.y, a1.y, k.x, k.y);
            mma16<MODE>(s[nt][1], a0.z, a1.z, a0.w, a1.w, k.z, k.w);
            if (MODE == kBF16Wide) {
              mma16<MODE>(s[nt][0], q[C::parts - 1].x, 0, q[C::parts - 1].y, 0, k.x, k.y);
              mma16<MODE>(s[nt][1], q[C::parts - 1].z, 0, q[C::parts - 1].w, 0, k.z, k.w);
            }
          }
        }
      }
    }
    if (more_keys) {
      key += C::keys;
      place();
      if (C::ahead) load_k();
    }
    {
      // running maximum and sum; a lane has query g and keys 2t, 2t+1 of every 8
      float x[C::NT][2], top = -INFINITY;
#pragma unroll
      for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          x[nt][e] = s[nt][0][e] + s[nt][1][e];
          if (C::parts > 1) x[nt][e] += s[nt][0][2 + e] + s[nt][1][2 + e];
          if (C::quarter) x[nt][e] += __shfl_xor_sync(~0u, x[nt][e], 16);
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
          x[nt][e] *= C::lift;
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
          if (C::parts == 3) {
            p3[k][0] = pack2<MODE>(xa[0], xa[1]);
            p3[k][1] = pack2<MODE>(xb[0], xb[1]);
          }
          if (C::quarter) {  // rows 4-7 take the second parts, rows 8-11 the third, rows 12-15 nothing
            if (g >= 4) pa[k][0] = pa[k][1], pa[k][2] = pa[k][3], p3[k][0] = p3[k][1] = 0;
            pa[k][1] = p3[k][0];
            pa[k][3] = p3[k][1];
          }
        }
      }
#pragma unroll
      for (int j = 0; j < C::VJ; ++j)
#pragma unroll
        for (int e = 0; e < C::epc; ++e) {
          auto word = [&](int kk) {
            const uint4 w = vf[kk][j];
            const int i = C::f32 ? e : e / 2;
            return i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w;
          };
          float acc[4] = {};
#pragma unroll
          for (int kt = 0; kt < (C::f32 ? 2 * PN : PN); ++kt) {
            const int k = C::f32 ? kt % PN : kt;
            if (C::f32) {  // tails first: the instruction cuts its sums off, small ones lose less
              const float v0 = __uint_as_float(word(2 * k)), v1 = __uint_as_float(word(2 * k + 1));
              if (kt < PN)
                mma16<MODE>(acc, pa[k][0], pa[k][1], pa[k][2], pa[k][3], tf32_tail(v0), tf32_tail(v1));
              else
                mma16<MODE>(acc, pa[k][0], pa[k][1], pa[k][2], pa[k][3], tf32_head(v0), tf32_head(v1));
            } else {
              const uint32_t sel = e % 2 ? 0x7632 : 0x5410;
              constexpr int two = C::f32 ? 0 : 4;
              const uint32_t b0 = __byte_perm(word(two * k), word(two * k + 1 % (two + 1)), sel);
              const uint32_t b1 = __byte_perm(word(two * k + two / 2), word(two * k + two / 2 + 1 % (two + 1)), sel);
              mma16<MODE>(acc, pa[k][0], pa[k][1], pa[k][2], pa[k][3], b0, b1);
              if (MODE == kBF16Wide) mma16<MODE>(acc, p3[k][0], 0, p3[k][1], 0, b0, b1);
            }
          }
          float *oo = o[j * C::epc + e];
          oo[0] = fmaf(oo[0], shrink, acc[0] + acc[2]);
          oo[1] = fmaf(oo[1], shrink, acc[1] + acc[3]);
        }
    }
    if (more_keys) {
      if (!C::ahead) load_k();
      load_v();
    }
    }

    // ---- the portion's result
    l += __shfl_xor_sync(~0u, l, 1);
    l += __shfl_xor_sync(~0u, l, 2);
    const int h = unit / p.qtiles, qt = unit - h * p.qtiles;
    const int rows = min(kQT, p.group - qt * kQT), head0 = h * p.group + qt * kQT;
    // a whole segment is written from shared memory; the last piece of a run stays there, an earlier one goes to the
    // workspace
    const bool tail = at >= we;
    float *to = whole || tail ? own : p.heads + ((int64_t)blockIdx.x * W + warp) * C::piece;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < C::VJ; ++j)
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < C::epc; e += 4) {
          const int d = (8 * j + 2 * t + k) * C::epc + e, b = j * C::epc + e;
          constexpr float down = 1.f / C::lift;
          float4 y = make_float4(o[b][k] * down, o[b + 1][k] * down, o[b + 2][k] * down, o[b + 3][k] * down);
          if (C::quarter) {
            y.x += __shfl_xor_sync(~0u, y.x, 16);
            y.y += __shfl_xor_sync(~0u, y.y, 16);
            y.z += __shfl_xor_sync(~0u, y.z, 16);
            y.w += __shfl_xor_sync(~0u, y.w, 16);
          }
          if (d < DP && g < rows) *reinterpret_cast<float4 *>(to + g * C::o_row + d) = y;
        }
    if (t == 0 && g < rows) {
      to[kQT * C::o_row + g] = m;
      to[kQT * C::o_row + kQT + g] = l;
    }
    if (whole) {
      __syncwarp();
#pragma unroll 1
      for (int i = lane; i < rows * (D / 4); i += 32) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        const float sum = to[kQT * C::o_row + kQT + r], scale = sum == 0.f ? 0.f : 1.f / sum;
        const float4 y = *reinterpret_cast<const float4 *>(to + r * C::o_row + d);
        if (!store4(p.a.out.ptr, (int)p.a.type,
                    seq * p.a.out.stride[0] + (head0 + r) * p.a.out.stride[1] + d * p.a.out.stride[2], p.a.out.stride[2],
                    make_float4(y.x * scale, y.y * scale, y.z * scale, y.w * scale)))
          doubt(seq, unit, r);
      }
      if (p.a.lse && t == 0 && g < rows)
        p.a.lse[(int64_t)seq * p.q_heads + head0 + g] = lse_of(m == -INFINITY ? 0.f : m, l);
    } else if (lane == 0) {
      const int i = 2 * warp + tail;
      s_seq[i] = seq, s_unit[i] = unit, s_open[i] = open;
    }
  }

  __syncthreads();
  // ---- Phase 0: the block's pieces, a warp per segment and row; the sums of segments that pass the run's ends become
  // records.  Phases 1 and 2: for the segments that pass its begin and its end, the last block to arrive adds their
  // records up.
  const bool has = lane < 2 * W && s_seq[lane] >= 0;
  const uint32_t valid = __ballot_sync(~0u, has), earlier = valid & ((1u << lane) - 1);
  const int prev = earlier ? 31 - __clz(earlier) : 0;
  const uint32_t lead_mask =
      __ballot_sync(~0u, has && (!earlier || s_seq[prev] != s_seq[lane] || s_unit[prev] != s_unit[lane]));
  constexpr int ND = (DP + 127) / 128;
#pragma unroll 1
  for (int phase = 0; phase < 3; ++phase) {
    int tasks = __popc(lead_mask) * p.q_rows, first = 0, last = 0, at_seq = 0, at_unit = 0;
    if (phase) {
      const Cut cut = s_cut[phase - 1];
      const int x = cut.seg_begin, y_end = cut.seg_end;
      if (cut.at <= x || cut.at >= y_end || (phase == 2 && x < begin)) continue;
      // the blocks of the segment: cuts inside it, by the same rule as above
      int lo = x / per + 1, hi = (y_end - 1) / per;
#pragma unroll 1
      while (snapped<C::change>(lo * per, x, y_end, near) == x) ++lo;
#pragma unroll 1
      while (snapped<C::change>(hi * per, x, y_end, near) == y_end) --hi;
      first = lo - 1;
      last = hi;
      at_seq = cut.seq;
      at_unit = (x - cut.seq_begin) / (y_end - x);
      tasks = p.q_rows;
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        int *word = p.arrivals + (int64_t)at_seq * units + at_unit;
        s_last = atomicAdd(word, 1) == last - first;
        if (s_last) *word = 0;
      }
      __syncthreads();
      if (!s_last) continue;
      __threadfence();
    }
#pragma unroll 1
    for (int task = warp; task < tasks; task += W) {
      int r = task, record = 0;
      uint32_t members = 0;
      if (!phase) {
        r = task % p.q_rows;
        uint32_t leaders = lead_mask;
#pragma unroll 1
        for (int k = task / p.q_rows; k; --k) leaders &= leaders - 1;
        const int lead = __ffs(leaders) - 1;
        leaders &= leaders - 1;
        members = valid & ~((1u << lead) - 1) & (leaders ? (1u << (__ffs(leaders) - 1)) - 1 : ~0u);
        at_seq = s_seq[lead];
        at_unit = s_unit[lead];
        record = s_open[lead];
      }
      const int h = at_unit / p.qtiles, qt = at_unit - h * p.qtiles;
      if (qt * kQT + r >= p.group) continue;
      // 32 pieces at a time: lane i weighs the i-th, then every lane adds dims 4 lane, 4 lane + 128, ... of all, four
      // loads in flight
      float top = -INFINITY, sum = 0.f;
      float4 y[ND];
#pragma unroll
      for (int k = 0; k < ND; ++k) y[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
      for (int b = first; b <= last; b += 32) {
        const float *mine = nullptr;
        int here = 32;
        if (phase) {
          here = min(32, last - b + 1);
          if (lane < here) mine = p.records + ((int64_t)(b + lane) * 2 + (b + lane == first)) * C::piece;
        } else if (members >> lane & 1) {
          mine = lane % 2 ? reinterpret_cast<const float *>(smem + lane / 2 * warp_bytes)
                          : p.heads + ((int64_t)blockIdx.x * W + lane / 2) * C::piece;
        }
        float mm = -INFINITY, ll = 0.f;
        if (mine) {
          mm = ld_relaxed(mine + kQT * C::o_row + r);
          ll = ld_relaxed(mine + kQT * C::o_row + kQT + r);
        }
        float ref = fmaxf(top, mm);
#pragma unroll
        for (int d = 16; d; d >>= 1) ref = fmaxf(ref, __shfl_xor_sync(~0u, ref, d));
        const float from = ref == -INFINITY ? 0.f : ref, keep = ex2(top - from), weight = ex2(mm - from);
        top = ref;
        sum = sum * keep + weight * ll;  // of this lane's pieces
#pragma unroll
        for (int k = 0; k < ND; ++k) y[k].x *= keep, y[k].y *= keep, y[k].z *= keep, y[k].w *= keep;
#pragma unroll 1
        for (int i0 = 0; i0 < here; i0 += 4) {
          float4 v[4][ND];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float *q = reinterpret_cast<const float *>(__shfl_sync(~0u, reinterpret_cast<uint64_t>(mine), i0 + i));
#pragma unroll
            for (int k = 0; k < ND; ++k) {
              v[i][k] = make_float4(0.f, 0.f, 0.f, 0.f);
              if (q && 4 * lane + 128 * k < DP) v[i][k] = ld_relaxed4(q + r * C::o_row + 4 * lane + 128 * k);
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float f = __shfl_sync(~0u, weight, i0 + i);
#pragma unroll
            for (int k = 0; k < ND; ++k)
              y[k].x += f * v[i][k].x, y[k].y += f * v[i][k].y, y[k].z += f * v[i][k].z, y[k].w += f * v[i][k].w;
          }
        }
      }
#pragma unroll
      for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
      const int head = h * p.group + qt * kQT + r;
      float *rec = p.records + ((int64_t)blockIdx.x * 2 + record - 1) * C::piece;
      const float scale = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
      for (int k = 0; k < ND; ++k) {
        const int d = 4 * lane + 128 * k;
        if (record) {
          if (d < DP) *reinterpret_cast<float4 *>(rec + r * C::o_row + d) = y[k];
        } else if (d < D) {
          if (!store4(p.a.out.ptr, (int)p.a.type,
                      at_seq * p.a.out.stride[0] + head * p.a.out.stride[1] + d * p.a.out.stride[2], p.a.out.stride[2],
                      make_float4(y[k].x * scale, y[k].y * scale, y[k].z * scale, y[k].w * scale)))
            doubt(at_seq, at_unit, r);
        }
      }
      if (lane == 0) {
        if (record) {
          rec[kQT * C::o_row + r] = top;
          rec[kQT * C::o_row + kQT + r] = sum;
        } else if (p.a.lse) {
          p.a.lse[(int64_t)at_seq * p.q_heads + head] = lse_of(top == -INFINITY ? 0.f : top, sum);
        }
      }
    }
  }
  };
  work();

  // Doubtful rows that this block wrote, once more by plain fp32 products.  An infinity among keys, values or queries
  // makes NaN of split operands (the parts of one side meet it with either sign, or zero) where the formula has a weight
  // of zero or an infinite result.  A warp takes a row, 32 keys at a time: a lane its key's score, then four dims of the sum.
  // It takes 0.7 us a key (88 ms for a long document of 131071 keys with a NaN among its values), for memory that is
  // broken as a rule.  It stands here and calls nothing: with a function call more, the loop over the keys spills (fp32
  // queries over fp16 3 to 6 % slower).
  __syncthreads();
  if (s_doubt) {
    const int words = (min(s_cut[1].seq, seqs - 1) - s_cut[0].seq + 1) * units;
    uint32_t *const notes = p.doubtful + (int64_t)s_cut[0].seq * units;
#pragma unroll 1
    for (int64_t i = warp; i < (int64_t)words * p.q_rows; i += W) {
      const int word = (int)(i / p.q_rows), r = (int)(i - (int64_t)word * p.q_rows);
      const int s = s_cut[0].seq + word / units, unit = word % units, h = unit / p.qtiles;
      const uint32_t note = *static_cast<volatile uint32_t *>(notes + word);
      if (note >> kQT != blockIdx.x + 1 || !(note >> r & 1)) continue;
      const Span sp = span_of<C::keys>(p, s);
      const int head = h * p.group + (unit - h * p.qtiles) * kQT + r, type = (int)p.pool.type;
      const int64_t q0 = s * p.a.q.stride[0] + head * p.a.q.stride[1];
#pragma unroll 1
      for (int d0 = 0; d0 < D; d0 += 128) {
        const int dim = d0 + lane;  // and 32, 64, 96 on
        float top = -INFINITY, sum = 0.f, y[4] = {};
#pragma unroll 1
        for (int key0 = sp.first; key0 < sp.len && !isnan(sum); key0 += 32) {  // a NaN there is one in every result
          float z = -INFINITY;
          int64_t at_v = -1;
          if (key0 + lane < sp.len) {
            const int page = page_of(p, key0 + lane), e = p.a.page_table[s * p.a.table_stride + page];
            const int64_t slot = key0 + lane - page * (int)p.pool.page_size;
            if (e >= 0 && e < p.pool.num_pages) {
              at_v = e * p.pool.v_stride[0] + h * p.pool.v_stride[1] + slot * p.pool.v_stride[2];
              const uint4 *k = reinterpret_cast<const uint4 *>(
                  static_cast<const uint8_t *>(p.pool.k) +
                  (e * p.pool.k_stride[0] + h * p.pool.k_stride[1] + slot * p.pool.k_stride[2]) * C::es);
              z = 0.f;
#pragma unroll 1
              for (int d = 0; d < D; d += C::epc) {
                const uint4 w = k[d / C::epc];
#pragma unroll
                for (int c = 0; c < C::epc; ++c)
                  z += element(p.a.q.ptr, (int)p.a.type, q0 + (d + c) * p.a.q.stride[2]) * element(&w, type, c);
              }
              z *= p.scale_log2;
            }
          }
          float m = fmaxf(top, z);
#pragma unroll
          for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
          const float ref = m == -INFINITY ? 0.f : m, shrink = ex2(top - ref), weight = at_v < 0 ? 0.f : ex2(z - ref);
          float all = weight;
#pragma unroll
          for (int d = 16; d; d >>= 1) all += __shfl_xor_sync(~0u, all, d);
          top = m;
          sum = sum * shrink + all;
#pragma unroll
          for (int c = 0; c < 4; ++c) y[c] *= shrink;
#pragma unroll 2
          for (int k = 0; k < 32; ++k) {
            const int64_t at = __shfl_sync(~0u, at_v, k);
            const float w = __shfl_sync(~0u, weight, k);
            if (at >= 0)
#pragma unroll
              for (int c = 0; c < 4; ++c) y[c] += w * element(p.pool.v, type, at + min(dim + 32 * c, D - 1));
          }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float x = sum == 0.f ? 0.f : y[c] / sum;
          const int64_t to = s * p.a.out.stride[0] + head * p.a.out.stride[1] + min(dim + 32 * c, D - 1) * p.a.out.stride[2];
          if (p.a.type == SC_TYPE_F32)
            static_cast<float *>(p.a.out.ptr)[to] = x;
          else if (p.a.type == SC_TYPE_F16)
            static_cast<__half *>(p.a.out.ptr)[to] = __float2half_rn(x);
          else
            static_cast<__nv_bfloat16 *>(p.a.out.ptr)[to] = __float2bfloat16_rn(x);
        }
        if (p.a.lse && lane == 0) p.a.lse[(int64_t)s * p.q_heads + head] = lse_of(top == -INFINITY ? 0.f : top, sum);
      }
    }
    __syncthreads();
#pragma unroll 1
    for (int i = tid; i < words; i += blockDim.x)
      if (notes[i] >> kQT == blockIdx.x + 1) notes[i] = 0;
  }

  // sequences without keys; the blocks share them
#pragma unroll 1
  for (int s = blockIdx.x; s < seqs; s += gridDim.x)
    if (span_of<C::keys>(p, s).steps == 0) {
#pragma unroll 1
      for (int i = tid; i < p.q_heads * (D / 4); i += blockDim.x)
        store4(p.a.out.ptr, (int)p.a.type,
               s * p.a.out.stride[0] + i / (D / 4) * p.a.out.stride[1] + i % (D / 4) * 4 * p.a.out.stride[2],
               p.a.out.stride[2], make_float4(0.f, 0.f, 0.f, 0.f));
      if (p.a.lse)
#pragma unroll 1
        for (int i = tid; i < p.q_heads; i += blockDim.x) p.a.lse[(int64_t)s * p.q_heads + i] = -INFINITY;
    }
}

}  // namespace attn
}  // namespace sc
