// fs_rows.cuh -- kernels over the rows of a batch of logits: sampling one
// token of every row, and the n best log-probabilities of every row.
//
// A row x of V logits belongs to one thread-block cluster.  Its CTAs split the
// row, read it from HBM once, keep it in shared memory and walk it there as
// often as the row's parameters need.
//
// Mathematics.  With m = max x, c = log2(e) / T and y_j = (m - x_j) c >= 0 the
// weight of entry j is w_j = 2^-y_j, and softmax(x / T)_j = w_j / sum w.  Each
// w_j is rounded once, to a whole multiple q_j of 2^-40 (w_j has 24 bits, so
// weights above 2^-16 keep all of them; what is below 2^-41 of the maximum
// counts as nothing).  Every sum, cut and draw is then one of whole numbers:
// it does not depend on the order of the additions, on the number of CTAs or
// on atomics, and a batch gives the same tokens however it is split.  Sums of
// 2^19 entries stay below 2^60.
#pragma once

#include <cooperative_groups.h>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "fs_device.cuh"

namespace fs {

namespace cg = cooperative_groups;

constexpr int ROW_THREADS = 512;
constexpr int ROW_WARPS = ROW_THREADS / 32;
constexpr int ROW_MAX_CLUSTER = 16;
constexpr uint32_t ROW_MAX_COLS = 1u << 19;
constexpr int ROW_BINS = 2048;
constexpr int ROW_BEST_MAX = 1024;
// Level-0 bins of a selection: linear in y, 1/48 of an octave of weight each,
// so that the bins 0..2046 cover every entry with q > 0 (y < 41) and the last
// one the rest.
constexpr float ROW_BIN_SCALE = 48.0f;
// Shared-memory bytes of row data a CTA may hold.
constexpr uint32_t ROW_PART_MAX = 160u << 10;

constexpr float ROW_LOG2E = 1.4426950408889634f;
constexpr float ROW_LN2 = 0.6931471805599453f;

struct RowArgs {
  const void* x;        // rows x cols logits
  int64_t stride;       // elements between rows
  uint32_t rows, cols;
  uint32_t part_vecs;   // 16-byte vectors of a row per CTA of its cluster
  // sampling (null: off)
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  const float* uniform;
  int* tokens;
  float* logprobs;      // may be null
  // best n
  int n;
  int* best_idx;
  float* best_logprob;
  float* lse;           // may be null
};

// ---- elements -------------------------------------------------------------------
// A 16-byte vector of logits with NaN read as -inf and +inf as the type's
// largest finite value: -inf is then the only value that is not finite.
template <typename T> struct RowElem;
template <> struct RowElem<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ uint32_t clean(uint32_t v) {
    return __float_as_uint(fminf(fmaxf(__uint_as_float(v), -INFINITY), 3.402823466e+38f));
  }
  static __device__ __forceinline__ float get(const uint4& v, int e) {
    return __uint_as_float(e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w);
  }
  static constexpr uint32_t NEG_INF = 0xff800000u;  // fills a 32-bit word
};
template <> struct RowElem<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ uint32_t clean(uint32_t v) {
    __nv_bfloat162 b = *reinterpret_cast<__nv_bfloat162*>(&v);
    const uint32_t lo = 0xff80ff80u, hi = 0x7f7f7f7fu;
    b = __hmin2(__hmax2(b, *reinterpret_cast<const __nv_bfloat162*>(&lo)), *reinterpret_cast<const __nv_bfloat162*>(&hi));
    return *reinterpret_cast<uint32_t*>(&b);
  }
  static __device__ __forceinline__ float get(const uint4& v, int e) {
    const uint32_t w = e < 2 ? v.x : e < 4 ? v.y : e < 6 ? v.z : v.w;
    return __uint_as_float((e & 1) ? (w & 0xffff0000u) : (w << 16));
  }
  static constexpr uint32_t NEG_INF = 0xff80ff80u;
};
template <> struct RowElem<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ uint32_t clean(uint32_t v) {
    __half2 b = *reinterpret_cast<__half2*>(&v);
    const uint32_t lo = 0xfc00fc00u, hi = 0x7bff7bffu;
    b = __hmin2(__hmax2(b, *reinterpret_cast<const __half2*>(&lo)), *reinterpret_cast<const __half2*>(&hi));
    return *reinterpret_cast<uint32_t*>(&b);
  }
  static __device__ __forceinline__ float get(const uint4& v, int e) {
    const uint32_t w = e < 2 ? v.x : e < 4 ? v.y : e < 6 ? v.z : v.w;
    return __half2float(__ushort_as_half((unsigned short)((e & 1) ? (w >> 16) : (w & 0xffffu))));
  }
  static constexpr uint32_t NEG_INF = 0xfc00fc00u;
};

__device__ __forceinline__ uint4 row_load(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// Descending order of x as ascending unsigned order; -0 and +0 are equal.
__device__ __forceinline__ uint32_t row_key(float x) {
  return ~to_ordered<uint32_t, XF_FLOAT>(__float_as_uint(x + 0.0f));
}
__device__ __forceinline__ float row_unkey(uint32_t k) {
  return __uint_as_float(from_ordered<uint32_t, XF_FLOAT>(~k));
}

__device__ __forceinline__ float row_exp2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// y = (m - x) c, each step rounded (no fused multiply-add).
__device__ __forceinline__ float row_y(float x, float m, float c) { return __fmul_rn(__fsub_rn(m, x), c); }

// q = round(w 2^40) of 0 <= w <= 1 in two 32-bit parts, by two additions that
// push the unwanted bits out of the mantissa: hi = w to a multiple of 2^-23
// (the mantissa bits of w + 1), lo = the rest to a multiple of 2^-40 (the
// mantissa bits of rest + 1.5 2^-17).  Each addition rounds half to even and
// w - hi is exact.  (A conversion to a 64-bit integer would run at the rate
// of the exponential; these are ordinary additions.)
struct RowQ {
  uint32_t hi;  // units of 2^-23
  int lo;       // units of 2^-40
};
__device__ __forceinline__ RowQ row_quant(float w) {
  constexpr float MAGIC = 1.5f / 131072.0f;
  const float a = __fadd_rn(w, 1.0f);
  const float r = __fsub_rn(w, __fsub_rn(a, 1.0f));
  const float b = __fadd_rn(r, MAGIC);
  return RowQ{__float_as_uint(a) - 0x3f800000u, __float_as_int(b) - __float_as_int(MAGIC)};
}
__device__ __forceinline__ uint64_t row_mass(uint64_t hi, int64_t lo) { return (hi << 17) + (uint64_t)lo; }
__device__ __forceinline__ uint64_t row_q(float w) {
  const RowQ q = row_quant(w);
  return row_mass(q.hi, q.lo);
}

__device__ __forceinline__ uint64_t warp_sum_u64(uint64_t v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
  return v;
}
__device__ __forceinline__ uint64_t warp_scan_u64(uint64_t v, int lane) {  // inclusive
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint64_t o = __shfl_up_sync(~0u, v, d);
    if (lane >= d) v += o;
  }
  return v;
}

// ---- shared state ---------------------------------------------------------------
struct RowPick {     // what the cluster's first CTA found in a histogram
  uint32_t bin;      // ROW_BINS: the target is beyond the last entry
  uint32_t above_n;  // entries of the bins before it
  uint32_t bin_n;
  uint64_t above_q;  // mass of the bins before it
  uint64_t bin_q;
};
struct RowCut {  // entries before or at (key, idx) in (key, index) order
  uint32_t key;
  uint32_t idx;
  uint64_t mass;  // their mass
};

struct RowShared {
  uint64_t q[ROW_BINS];  // bin masses; the list of the best
  uint32_t n[ROW_BINS];  // bin counts
  uint64_t warp_q[ROW_WARPS];
  uint32_t warp_n[ROW_WARPS];
  uint64_t cta_q[ROW_MAX_CLUSTER];
  float cta_max[ROW_MAX_CLUSTER];
  RowPick pick;
  uint32_t found;
  uint32_t count;
};

// ---- one row --------------------------------------------------------------------
template <typename T> struct Row {
  using E = RowElem<T>;
  static constexpr int N = E::N;

  cg::cluster_group cluster;
  RowShared& sh;
  uint4* data;
  const int tid, lane, wid;
  const uint32_t rank, ctas;
  uint32_t seg0, seg1;  // this warp's vectors of the CTA's part
  int first;            // index of the part's element 0 (negative inside the row's leading fill)
  float m, c;

  __device__ __forceinline__ Row(RowShared& s, uint4* d)
      : cluster(cg::this_cluster()),
        sh(s),
        data(d),
        tid(threadIdx.x),
        lane(threadIdx.x & 31),
        wid(threadIdx.x >> 5),
        rank(cluster.block_rank()),
        ctas(cluster.num_blocks()) {
    cluster.barrier_arrive();  // waited for in load(): no CTA writes into one that has not started
  }

  // Reads this CTA's part into shared memory and finds the row's maximum.  The
  // part is cut at 16-byte boundaries of memory, wherever the row begins;
  // slots outside the row hold -inf.
  __device__ __forceinline__ void load(const RowArgs& a, uint32_t row) {
    const T* x = static_cast<const T*>(a.x) + (int64_t)row * a.stride;
    const uint32_t lead = (uint32_t)(reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T);
    const uint32_t total = (lead + a.cols + N - 1) / N;
    const uint32_t v0 = min(rank * a.part_vecs, total), v1 = min(v0 + a.part_vecs, total);
    const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(x) & ~(uintptr_t)15) + v0;
    first = (int)(v0 * N) - (int)lead;
    const uint32_t nv = v1 - v0, sv = (nv + ROW_WARPS - 1) / ROW_WARPS;
    seg0 = min(wid * sv, nv);
    seg1 = min(seg0 + sv, nv);
    float mx = -INFINITY;
    for (uint32_t i = seg0 + lane; i < seg1; i += 32) {
      const int j0 = first + (int)(i * N);
      uint4 v;
      if (j0 >= 0 && j0 + N <= (int)a.cols) {
        v = row_load(src + i);
      } else {  // the row's first or last vector
        union { uint4 v; T e[N]; } u;
        u.v = make_uint4(E::NEG_INF, E::NEG_INF, E::NEG_INF, E::NEG_INF);
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (j0 + e >= 0 && j0 + e < (int)a.cols) u.e[e] = x[j0 + e];
        v = u.v;
      }
      v.x = E::clean(v.x), v.y = E::clean(v.y), v.z = E::clean(v.z), v.w = E::clean(v.w);
      data[i] = v;
#pragma unroll
      for (int e = 0; e < N; ++e) mx = fmaxf(mx, E::get(v, e));
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, d));
    float* warp_max = reinterpret_cast<float*>(sh.warp_n);
    if (lane == 0) warp_max[wid] = mx;
    __syncthreads();
    cluster.barrier_wait();
    if (tid < (int)ctas) {  // thread t tells CTA t
      float b = -INFINITY;
      for (int w = 0; w < ROW_WARPS; ++w) b = fmaxf(b, warp_max[w]);
      *cluster.map_shared_rank(&sh.cta_max[rank], tid) = b;
    }
    cluster.sync();
    m = -INFINITY;
    for (uint32_t k = 0; k < ctas; ++k) m = fmaxf(m, sh.cta_max[k]);
  }

  // f(x, index) for every entry of this thread
  template <typename F> __device__ __forceinline__ void each(F f) const {
    for (uint32_t i = seg0 + lane; i < seg1; i += 32) {
      const uint4 v = data[i];
      const int j0 = first + (int)(i * N);
#pragma unroll
      for (int e = 0; e < N; ++e) f(E::get(v, e), j0 + e);
    }
  }

  // Sums `mine` over the cluster; leaves the warps' sums in sh.warp_q and the
  // CTAs' in sh.cta_q.
  __device__ __forceinline__ uint64_t sum(uint64_t mine) {
    const uint64_t w = warp_sum_u64(mine);
    if (lane == 0) sh.warp_q[wid] = w;
    __syncthreads();
    if (tid < (int)ctas) {
      uint64_t t = 0;
      for (int k = 0; k < ROW_WARPS; ++k) t += sh.warp_q[k];
      *cluster.map_shared_rank(&sh.cta_q[rank], tid) = t;
    }
    cluster.sync();
    uint64_t t = 0;
    for (uint32_t k = 0; k < ctas; ++k) t += sh.cta_q[k];
    return t;
  }

  // After sum() of value(x, index): the entry at which the running sum in
  // index order first exceeds t calls hit(x, index), on one thread of the cluster.
  template <typename V, typename H> __device__ __forceinline__ void locate(uint64_t t, V value, H hit) {
    uint64_t before = 0;
    for (uint32_t k = 0; k < rank; ++k) before += sh.cta_q[k];
    if (t < before || t - before >= sh.cta_q[rank]) return;
    t -= before;
    for (int k = 0; k < wid; ++k) {
      if (t < sh.warp_q[k]) return;
      t -= sh.warp_q[k];
    }
    if (t >= sh.warp_q[wid]) return;
    for (uint32_t i0 = seg0; i0 < seg1; i0 += 32) {
      const uint32_t i = i0 + lane;
      uint64_t mine = 0;
      uint4 v = make_uint4(E::NEG_INF, E::NEG_INF, E::NEG_INF, E::NEG_INF);
      const int j0 = first + (int)(i * N);
      if (i < seg1) {
        v = data[i];
#pragma unroll
        for (int e = 0; e < N; ++e) mine += value(E::get(v, e), j0 + e);
      }
      const uint64_t upto = warp_scan_u64(mine, lane);
      const uint64_t all = __shfl_sync(~0u, upto, 31);
      if (t >= all) {
        t -= all;
        continue;
      }
      if (t < upto && t >= upto - mine) {
        uint64_t left = t - (upto - mine);
        bool done = false;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float x = E::get(v, e);
          const uint64_t q = value(x, j0 + e);
          if (!done && left < q) {
            hit(x, j0 + e);
            done = true;
          }
          left -= q;
        }
      }
      return;
    }
  }

  __device__ __forceinline__ float weight(float x) const { return row_exp2(-row_y(x, m, c)); }
  __device__ __forceinline__ uint64_t mass(float x) const { return row_q(weight(x)); }
  __device__ __forceinline__ uint32_t bin0(float x) const {
    return (uint32_t)fminf(__fmul_rn(row_y(x, m, c), ROW_BIN_SCALE), (float)(ROW_BINS - 1));
  }

  // Histogram of the entries for which digit(x, key) gives a bin, over the
  // whole row; then the bin where the running count (BY_MASS: mass) reaches
  // `target`.
  template <bool BY_MASS, typename D> __device__ __forceinline__ RowPick pick(uint64_t target, D digit) {
    for (int b = tid; b < ROW_BINS; b += ROW_THREADS) sh.n[b] = 0, sh.q[b] = 0;
    cluster.sync();
    each([&](float x, int) {
      if (x == -INFINITY) return;
      const uint32_t b = digit(x, row_key(x));
      if (b >= (uint32_t)ROW_BINS) return;
      atomicAdd(&sh.n[b], 1u);
      const uint64_t q = mass(x);
      if (q) atomicAdd(reinterpret_cast<unsigned long long*>(&sh.q[b]), (unsigned long long)q);
    });
    __syncthreads();
    if (rank) {
      uint32_t* n0 = cluster.map_shared_rank(sh.n, 0);
      uint64_t* q0 = cluster.map_shared_rank(sh.q, 0);
      for (int b = tid; b < ROW_BINS; b += ROW_THREADS)
        if (sh.n[b]) {
          atomicAdd(&n0[b], sh.n[b]);
          atomicAdd(reinterpret_cast<unsigned long long*>(&q0[b]), (unsigned long long)sh.q[b]);
        }
    }
    cluster.sync();
    if (rank == 0) {
      constexpr int PER = ROW_BINS / ROW_THREADS;
      uint64_t tq = 0;
      uint32_t tn = 0;
      for (int k = 0; k < PER; ++k) tq += sh.q[tid * PER + k], tn += sh.n[tid * PER + k];
      uint64_t iq = warp_scan_u64(tq, lane);
      uint32_t in = tn;
      for (int d = 1; d < 32; d <<= 1) {
        const uint32_t o = __shfl_up_sync(~0u, in, d);
        if (lane >= d) in += o;
      }
      if (lane == 31) sh.warp_q[wid] = iq, sh.warp_n[wid] = in;
      if (tid == 0) sh.pick = RowPick{(uint32_t)ROW_BINS, 0, 0, 0, 0};
      __syncthreads();
      for (int k = 0; k < wid; ++k) iq += sh.warp_q[k], in += sh.warp_n[k];
      uint64_t bq = iq - tq;
      uint32_t bn = in - tn;
      for (int k = 0; k < PER; ++k) {
        const uint64_t q = sh.q[tid * PER + k];
        const uint32_t n = sh.n[tid * PER + k];
        const uint64_t lo = BY_MASS ? bq : bn, hi = BY_MASS ? bq + q : bn + n;
        if (lo < target && target <= hi) sh.pick = RowPick{(uint32_t)(tid * PER + k), bn, n, bq, q};
        bq += q, bn += n;
      }
      __syncthreads();
      if (tid > 0 && tid < (int)ctas) *cluster.map_shared_rank(&sh.pick, tid) = sh.pick;
    }
    cluster.sync();
    return sh.pick;
  }

  // The shortest prefix of (descending x, ascending index) order with at
  // least `target` entries (BY_MASS: mass), target >= 1; where the row has
  // less than that, all of it, with mass ~0.
  template <bool BY_MASS> __device__ __noinline__ RowCut select(uint64_t target) {
    RowPick p = pick<BY_MASS>(target, [&](float x, uint32_t) { return bin0(x); });
    if (p.bin == (uint32_t)ROW_BINS) return RowCut{~0u, ~0u, ~0ull};
    const uint32_t b0 = p.bin;
    uint64_t left = target, above_q = 0;
    left -= BY_MASS ? p.above_q : p.above_n;
    above_q += p.above_q;
    // Keys of the bin's entries, as far as its bounds tell; keys outside them
    // fall into the first or the last digit, whose interval is then open.
    const float step = 1.0f / (ROW_BIN_SCALE * c);
    uint32_t lo = row_key(fminf(m, m - (float)b0 * step));
    uint32_t hi = b0 == (uint32_t)ROW_BINS - 1 ? ~0u : row_key(fmaxf(m - (float)(b0 + 1) * step, -3.402823466e+38f));
    hi = max(hi, lo);
    bool open_lo = true, open_hi = true;
    for (int level = 0; level < 8; ++level) {  // at most one open and three closed intervals
      const int shift = max(0, 32 - __clz((int)((hi - lo) | 1)) - 11);
      const uint32_t last = (hi - lo) >> shift;
      p = pick<BY_MASS>(left, [&](float x, uint32_t k) -> uint32_t {
        if (bin0(x) != b0) return ~0u;
        if (k < lo) return open_lo ? 0u : ~0u;
        if (k > hi) return open_hi ? last : ~0u;
        return (k - lo) >> shift;
      });
      if (p.bin == (uint32_t)ROW_BINS) return RowCut{~0u, ~0u, ~0ull};
      left -= BY_MASS ? p.above_q : p.above_n;
      above_q += p.above_q;
      const uint32_t base = lo;
      const bool was_lo = open_lo, was_hi = open_hi;
      open_lo = was_lo && p.bin == 0;
      open_hi = was_hi && p.bin == last;
      lo = open_lo ? 0u : base + (p.bin << shift);
      const uint32_t top = base + (p.bin << shift) + ((1u << shift) - 1);
      hi = open_hi ? ~0u : min(top, hi);
      // an interval that was closed on both sides is now one key, or is cut again
      if (open_lo || open_hi) {
        open_lo = open_hi = false;
        continue;
      }
      if (shift == 0) break;
    }
    // p.bin_n entries share the key; the first `ties` of them in index order belong
    const uint64_t each_q = p.bin_q / p.bin_n;
    const uint64_t ties = BY_MASS ? (left + each_q - 1) / each_q : left;
    RowCut cut{lo, ~0u, above_q + ties * each_q};
    if (ties < p.bin_n) {
      auto is = [&](float x, int) -> uint64_t { return x != -INFINITY && row_key(x) == cut.key; };
      uint64_t mine = 0;
      each([&](float x, int j) { mine += is(x, j); });
      sum(mine);
      locate(ties - 1, is, [&](float, int j) {
        for (uint32_t k = 0; k < ctas; ++k) *cluster.map_shared_rank(&sh.found, k) = (uint32_t)j;
      });
      cluster.sync();
      cut.idx = sh.found;
    }
    return cut;
  }
};

// ---- sampling ---------------------------------------------------------------------
template <typename T> __global__ void __launch_bounds__(ROW_THREADS) k_row_sample(const RowArgs a) {
  extern __shared__ __align__(16) unsigned char row_smem[];
  RowShared& sh = *reinterpret_cast<RowShared*>(row_smem);
  Row<T> r(sh, reinterpret_cast<uint4*>(row_smem + (sizeof(RowShared) + 15) / 16 * 16));
  const uint32_t row = blockIdx.x / r.ctas;
  r.load(a, row);

  if (r.m == -INFINITY) {
    if (r.rank == 0 && r.tid == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = -INFINITY;
    }
    return;
  }
  const float t = a.temperature ? a.temperature[row] : 1.0f;
  const bool greedy = !(t > 0.0f);
  // within the finite numbers above 0: 0 * c and (max + inf) * c stay what they are for the smallest and infinite t
  r.c = greedy ? ROW_LOG2E : fminf(fmaxf(__fdiv_rn(ROW_LOG2E, t), 1.175494351e-38f), 3.402823466e+38f);
  uint64_t mine = 0;
  r.each([&](float x, int) { mine += r.mass(x); });
  const uint64_t total = r.sum(mine);

  auto store = [&](float x, int j) {
    a.tokens[row] = j;
    if (a.logprobs) a.logprobs[row] = -(row_y(x, r.m, r.c) * ROW_LN2) - logf((float)total * 0x1p-40f);
  };
  if (greedy) {
    auto top = [&](float x, int) -> uint64_t { return x == r.m; };
    mine = 0;
    r.cluster.sync();
    r.each([&](float x, int j) { mine += top(x, j); });
    r.sum(mine);
    r.locate(0, top, store);
    return;
  }
  RowCut cut{~0u, ~0u, total};
  const int k = a.top_k ? a.top_k[row] : 0;
  if (k > 0 && (uint32_t)k < a.cols) {
    cut = r.template select<false>((uint64_t)k);
    if (cut.mass == ~0ull) cut.mass = total;
  }
  const float p = a.top_p ? a.top_p[row] : 1.0f;
  if (p < 1.0f) {
    const double least = ceil((double)fmaxf(p, 0.0f) * (double)cut.mass);
    cut = r.template select<true>(least < 1.0 ? 1ull : (uint64_t)least);
  }
  const float least_w = fminf(a.min_p ? a.min_p[row] : 0.0f, 1.0f);
  auto kept = [&](float x, int j) -> uint64_t {
    const float w = r.weight(x);
    const uint32_t key = row_key(x);
    if (w < least_w || key > cut.key || (key == cut.key && (uint32_t)j > cut.idx)) return 0;
    return row_q(w);
  };
  mine = 0;
  r.cluster.sync();
  r.each([&](float x, int j) { mine += kept(x, j); });
  const uint64_t mass = r.sum(mine);
  const float u = a.uniform[row];
  const double at = floor((double)(u > 0.0f ? u : 0.0f) * (double)mass);
  const uint64_t draw = at < (double)mass ? min((uint64_t)at, mass - 1) : mass - 1;
  r.locate(draw, kept, store);
}

// Ascending sort of n (a power of two) 64-bit numbers in shared memory.
__device__ __forceinline__ void row_bitonic(uint64_t* v, int n) {
  for (int k = 2; k <= n; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < n / 2; i += ROW_THREADS) {
        const int a = 2 * i - (i & (j - 1)), b = a + j;
        const uint64_t x = v[a], y = v[b];
        if ((x > y) == ((a & k) == 0)) v[a] = y, v[b] = x;
      }
    }
  __syncthreads();
}

// ---- the n best ---------------------------------------------------------------------
template <typename T> __global__ void __launch_bounds__(ROW_THREADS) k_row_best(const RowArgs a) {
  extern __shared__ __align__(16) unsigned char row_smem[];
  RowShared& sh = *reinterpret_cast<RowShared*>(row_smem);
  Row<T> r(sh, reinterpret_cast<uint4*>(row_smem + (sizeof(RowShared) + 15) / 16 * 16));
  const uint32_t row = blockIdx.x / r.ctas;
  if (r.tid == 0) sh.count = 0;
  r.load(a, row);
  if (r.m == -INFINITY) {
    if (r.rank == 0) {
      for (int i = r.tid; i < a.n; i += ROW_THREADS) {
        a.best_idx[(int64_t)row * a.n + i] = -1;
        a.best_logprob[(int64_t)row * a.n + i] = -INFINITY;
      }
      if (a.lse && r.tid == 0) a.lse[row] = -INFINITY;
    }
    return;
  }
  r.c = ROW_LOG2E;
  uint64_t mine = 0;
  r.each([&](float x, int) { mine += r.mass(x); });
  const float ln = logf((float)r.sum(mine) * 0x1p-40f);
  if (a.lse && r.rank == 0 && r.tid == 0) a.lse[row] = r.m + ln;
  const RowCut cut = r.template select<false>((uint64_t)a.n);
  r.cluster.sync();
  uint32_t* count = r.cluster.map_shared_rank(&sh.count, 0);
  uint64_t* list = r.cluster.map_shared_rank(sh.q, 0);
  r.each([&](float x, int j) {
    const uint32_t key = row_key(x);
    if (x == -INFINITY || key > cut.key || (key == cut.key && (uint32_t)j > cut.idx)) return;
    list[atomicAdd(count, 1u)] = (uint64_t)key << 32 | (uint32_t)j;
  });
  r.cluster.sync();
  if (r.rank) return;
  int n2 = 1;
  while (n2 < a.n) n2 <<= 1;
  const int have = (int)sh.count;
  for (int i = have + r.tid; i < n2; i += ROW_THREADS) sh.q[i] = ~0ull;
  row_bitonic(sh.q, n2);
  for (int i = r.tid; i < a.n; i += ROW_THREADS) {
    const uint64_t e = sh.q[i];
    const bool in = i < have;
    a.best_idx[(int64_t)row * a.n + i] = in ? (int)(uint32_t)e : -1;
    a.best_logprob[(int64_t)row * a.n + i] = in ? (row_unkey((uint32_t)(e >> 32)) - r.m) - ln : -INFINITY;
  }
}

}  // namespace fs
