// fs_rows.cuh -- kernels over the rows of a batch of logits: sampling one
// token of every row, and the n best log-probabilities of every row.
//
// A row x of V logits belongs to one thread-block cluster, whose CTAs split it,
// read it from HBM once, keep it in shared memory and walk it there as often as
// the row's parameters need; or, in large batches, to one CTA that streams it
// twice or more, from HBM and then from L2.
//
// Mathematics.  With m = max x, c = log2(e) / T and y_j = (m - x_j) c >= 0 the
// weight of entry j is w_j = 2^-y_j, and softmax(x / T)_j = w_j / sum w.  Each
// w_j is rounded once, to a whole multiple q_j of 2^-40 (w_j has 24 bits, so
// weights above 2^-16 keep all of them; what is below 2^-41 of the maximum
// counts as nothing).  Every sum, cut and draw is then one of whole numbers:
// it does not depend on the order of the additions, on the number of CTAs or
// on atomics, and a batch gives the same tokens however it is split.  Sums of
// 2^19 entries stay below 2^60.
//
// What bounds them.  A row has to be read (at 6.55 TB/s: 10.2 us for 256 x 131072
// bf16) and costs an exponential an entry, which is cheap; what takes the time
// is the chain of a row's phases -- load, edge, weigh, list, cut, draw, each
// with a barrier of the cluster -- of 15,000 cycles for one row of 32768 (9.7 us
// with the launch) and 20 to 40,000 beside two other CTAs on the SM, and 35,000
// more where a nucleus lies beyond the candidates.  Each phase runs once or
// twice per CTA, from a cold instruction cache: cutting the code of the sampling kernel from
// 287 KB to 124 KB (loops rolled, one copy of each search) made every case 10
// to 35% faster, so loops are unrolled where a pass over the row is hot and
// nowhere else.
#pragma once

#include <cooperative_groups.h>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "fs_device.cuh"

namespace fs {

namespace cg = cooperative_groups;

constexpr int ROW_MAX_CLUSTER = 16;
constexpr int ROW_IDX_BITS = 19;
constexpr uint32_t ROW_MAX_COLS = 1u << ROW_IDX_BITS;
constexpr int ROW_LIST = 640;   // candidates of a row above its edge
constexpr int ROW_POOL = 1024;  // undecided entries of a row that narrowing leaves
constexpr int ROW_FEW = 256;    // entries that are ranked in place, by comparing all of them
constexpr int ROW_BEST_MAX = 1024;
constexpr int ROW_TOPS = 512;   // thread maxima that a cluster's warps publish
// A nucleus is first looked for among about this many entries: few nuclei of a
// model's rows that hold more than that end before thousands (256 x 131072 bf16:
// 192 entries 68.8 us, 128 entries 68.1, 64 entries 65.8).
constexpr uint32_t ROW_NUCLEUS_GUESS = 64;
// Bins linear in y: of the published maxima (1/6 octave of weight each, 42 in
// all; entries with q > 0 have y < 41), and of all entries (1/42 octave).
constexpr int ROW_EDGE_BINS = 256;
constexpr float ROW_EDGE_SCALE = 6.0f;
constexpr int ROW_BINS = 1792;
constexpr int ROW_BINS_END = ROW_BINS - 28;  // of weights
constexpr float ROW_BIN_SCALE = 42.0f;        // of counts, an octave
constexpr float ROW_MASS_END = 42.0f;  // octaves: no mass beyond
constexpr int ROW_SORT_BINS = 1024;

constexpr float ROW_LOG2E = 1.4426950408889634f;
constexpr float ROW_LN2 = 0.6931471805599453f;
constexpr float ROW_F32_MAX = 3.402823466e+38f;

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
// 16-byte vectors of logits.  top() is the maximum with NaN passed on, so that
// a thread whose running maximum is NaN or +inf knows that it has values to
// clean: NaN becomes -inf and +inf the type's largest finite value, after
// which -inf is the only value that is not finite.
__device__ __forceinline__ float fmax_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ uint4 smem_load(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
// Word k of a vector, by selections (an index would put it in local memory).
__device__ __forceinline__ uint32_t row_word(const uint4& v, int k) {
  uint32_t w = v.x;
  asm("{\n .reg .pred p, q, r;\n setp.eq.s32 p, %4, 1;\n setp.eq.s32 q, %4, 2;\n setp.eq.s32 r, %4, 3;\n"
      " @p mov.b32 %0, %1;\n @q mov.b32 %0, %2;\n @r mov.b32 %0, %3;\n}"
      : "+r"(w)
      : "r"(v.y), "r"(v.z), "r"(v.w), "r"(k));
  return w;
}

// The same word replaced.
__device__ __forceinline__ void row_put_word(uint4& v, int k, uint32_t w) {
  v.x = k == 0 ? w : v.x, v.y = k == 1 ? w : v.y, v.z = k == 2 ? w : v.z, v.w = k == 3 ? w : v.w;
}
__device__ __forceinline__ void row_put_half(uint4& v, int e, uint32_t h) {
  const uint32_t w = row_word(v, e >> 1);
  row_put_word(v, e >> 1, e & 1 ? (w & 0xffffu) | h << 16 : (w & 0xffff0000u) | h);
}

template <typename T> struct RowElem;
template <> struct RowElem<float> {
  static constexpr int N = 4;
  static constexpr uint32_t NEG_INF = 0xff800000u;  // fills a 32-bit word
  static constexpr int ZEROS = 0;                   // low bits of its 32-bit form that are always 0
  using Top = float;                                // running maximum
  static __device__ __forceinline__ Top top0() { return -INFINITY; }
  static __device__ __forceinline__ Top top(Top t, const uint4& v) {
    return fmax_nan(fmax_nan(fmax_nan(t, __uint_as_float(v.x)), fmax_nan(__uint_as_float(v.y), __uint_as_float(v.z))),
                    __uint_as_float(v.w));
  }
  static __device__ __forceinline__ float value(Top t) { return t; }
  static __device__ __forceinline__ uint32_t clean(uint32_t v) {
    return __float_as_uint(fminf(fmaxf(__uint_as_float(v), -INFINITY), ROW_F32_MAX));
  }
  static __device__ __forceinline__ float at(const uint4& v, int e) { return __uint_as_float(row_word(v, e)); }
  static __device__ __forceinline__ void put(uint4& v, int e, const float* x) { row_put_word(v, e, __float_as_uint(*x)); }
  static __device__ __forceinline__ void get(const uint4& v, float (&x)[N]) {
    x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
  }
};
template <> struct RowElem<__nv_bfloat16> {
  static constexpr int N = 8;
  static constexpr uint32_t NEG_INF = 0xff80ff80u;
  static constexpr int ZEROS = 16;
  using Top = uint32_t;
  static __device__ __forceinline__ Top top0() { return NEG_INF; }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ Top top(Top t, const uint4& v) {
    return max2(max2(t, v.x), max2(max2(v.y, v.z), v.w));
  }
  static __device__ __forceinline__ float value(Top t) {
    return fmax_nan(__uint_as_float(t << 16), __uint_as_float(t & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t clean(uint32_t v) {
    asm("max.bf16x2 %0, %0, %1;" : "+r"(v) : "r"(NEG_INF));
    asm("min.bf16x2 %0, %0, %1;" : "+r"(v) : "r"(0x7f7f7f7fu));
    return v;
  }
  static __device__ __forceinline__ float at(const uint4& v, int e) {
    const uint32_t w = row_word(v, e >> 1);
    return __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
  }
  static __device__ __forceinline__ void put(uint4& v, int e, const __nv_bfloat16* x) {
    row_put_half(v, e, *reinterpret_cast<const unsigned short*>(x));
  }
  static __device__ __forceinline__ void get(const uint4& v, float (&x)[N]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) x[2 * k] = __uint_as_float(w[k] << 16), x[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
  }
};
template <> struct RowElem<__half> {
  static constexpr int N = 8;
  static constexpr uint32_t NEG_INF = 0xfc00fc00u;
  static constexpr int ZEROS = 13;
  using Top = uint32_t;
  static __device__ __forceinline__ Top top0() { return NEG_INF; }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ Top top(Top t, const uint4& v) {
    return max2(max2(t, v.x), max2(max2(v.y, v.z), v.w));
  }
  static __device__ __forceinline__ float2 both(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
  static __device__ __forceinline__ float value(Top t) {
    const float2 f = both(t);
    return fmax_nan(f.x, f.y);
  }
  static __device__ __forceinline__ uint32_t clean(uint32_t v) {
    asm("max.f16x2 %0, %0, %1;" : "+r"(v) : "r"(NEG_INF));
    asm("min.f16x2 %0, %0, %1;" : "+r"(v) : "r"(0x7bff7bffu));
    return v;
  }
  static __device__ __forceinline__ float at(const uint4& v, int e) {
    const uint32_t w = row_word(v, e >> 1);
    return __half2float(__ushort_as_half((unsigned short)(e & 1 ? w >> 16 : w)));
  }
  static __device__ __forceinline__ void put(uint4& v, int e, const __half* x) {
    row_put_half(v, e, *reinterpret_cast<const unsigned short*>(x));
  }
  static __device__ __forceinline__ void get(const uint4& v, float (&x)[N]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = both(w[k]);
      x[2 * k] = f.x, x[2 * k + 1] = f.y;
    }
  }
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

// -y = (x - m) c, each step rounded (no fused multiply-add).
__device__ __forceinline__ float row_neg_y(float x, float m, float c) { return __fmul_rn(__fsub_rn(x, m), c); }

// q = round(w 2^40) of 0 <= w <= 1 in two 32-bit parts, by two additions that
// push the unwanted bits out of the mantissa: hi = w to a multiple of 2^-23
// (the mantissa bits of w + 1), lo = the rest to a multiple of 2^-40 (the
// mantissa bits of rest + 1.5 2^-17).  Each addition rounds half to even and
// w - hi, and 1 + 1.5 2^-17 - (w + 1), are exact.  (A conversion to an integer runs at the rate of the
// exponential, an eighth of that of these additions.)
constexpr float ROW_MAGIC = 1.5f / 131072.0f;
constexpr uint32_t ROW_ONE_BITS = 0x3f800000u;    // 1.0f
constexpr uint32_t ROW_MAGIC_BITS = 0x37400000u;  // 1.5 2^-17
__device__ __forceinline__ uint64_t row_mass(uint32_t hi, int lo) { return ((uint64_t)hi << 17) + (int64_t)lo; }
__device__ __forceinline__ uint64_t row_q(float w) {
  const float a = __fadd_rn(w, 1.0f);
  const float b = __fadd_rn(__fsub_rn(w, __fsub_rn(a, 1.0f)), ROW_MAGIC);
  return row_mass(__float_as_uint(a) - ROW_ONE_BITS, __float_as_int(b) - (int)ROW_MAGIC_BITS);
}

// Two 32-bit numbers in one instruction.
__device__ __forceinline__ uint64_t f2_pack(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2_unpack(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// In three parts of 27 bits, whose sums over a warp fit 32: three reductions of
// one instruction each against five exchanges of both halves.
__device__ __forceinline__ uint64_t warp_sum_u64(uint64_t v) {
  const uint32_t a = __reduce_add_sync(~0u, (uint32_t)v & 0x7ffffffu), b = __reduce_add_sync(~0u, (uint32_t)(v >> 27) & 0x7ffffffu);
  const uint32_t c = __reduce_add_sync(~0u, (uint32_t)(v >> 54));
  return a + ((uint64_t)b << 27) + ((uint64_t)c << 54);
}
template <typename V> __device__ __forceinline__ V warp_scan(V v, int lane) {  // inclusive
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const V o = __shfl_up_sync(~0u, v, d);
    if (lane >= d) v += o;
  }
  return v;
}
// Adds v to a word in shared memory where yes, without a branch.
__device__ __forceinline__ void smem_add_if(bool yes, uint32_t at, uint32_t v) {
  asm volatile("{\n .reg .pred q;\n setp.ne.u32 q, %2, 0;\n @q red.shared.add.u32 [%0], %1;\n}" ::"r"(at), "r"(v), "r"((uint32_t)yes)
               : "memory");
}
__device__ __forceinline__ uint32_t smem_of(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ uint64_t row_target(float p, uint64_t mass) {  // ceil(p mass), at least 1
  const double least = ceil((double)fmaxf(p, 0.0f) * (double)mass);
  return least < 1.0 ? 1ull : (uint64_t)least;
}
__device__ __forceinline__ uint64_t row_draw(float u, uint64_t mass) {  // floor(u mass), below mass
  const double at = floor((double)(u > 0.0f ? u : 0.0f) * (double)mass);
  return at < (double)mass ? min((uint64_t)at, mass - 1) : mass - 1;
}

// A row's sampling parameters.
struct RowParams {
  float t, p, least_w, u;
  uint32_t k;
  bool greedy, by_k, by_p, by_w;

  __device__ __forceinline__ RowParams(const RowArgs& a, uint32_t row) {
    t = a.temperature ? a.temperature[row] : 1.0f;
    const int k_arg = a.top_k ? a.top_k[row] : 0;
    p = a.top_p ? a.top_p[row] : 1.0f;
    least_w = a.min_p ? __saturatef(a.min_p[row]) : 0.0f;  // NaN: 0, off
    u = a.uniform[row];
    k = (uint32_t)k_arg;
    greedy = !(t > 0.0f);
    by_k = !greedy && k_arg > 0 && k < a.cols;
    by_p = !greedy && p < 1.0f;
    by_w = !greedy && least_w > 0.0f;
  }
  __device__ __forceinline__ bool cuts() const { return by_k || by_p || by_w; }
  // log2(e) / t, within the finite numbers above 0: 0 * c and (max + inf) * c stay what they are for the smallest and
  // infinite t
  __device__ __forceinline__ float c() const {
    return greedy ? ROW_LOG2E : fminf(fmaxf(__fdiv_rn(ROW_LOG2E, t), 1.175494351e-38f), ROW_F32_MAX);
  }
};

// ---- shared state ---------------------------------------------------------------
template <int CTAS, int WARPS> struct RowShared {
  union {
    struct {
      uint64_t list[ROW_LIST];         // candidates: key << 19 | index
      uint32_t tops[ROW_TOPS];         // keys of the largest thread maxima of each warp of the cluster
      uint32_t edge_n[ROW_EDGE_BINS];  // those by bin
    };
    uint32_t bins[ROW_BINS];  // while a cut is narrowed down: weights or counts,
    uint64_t pool[ROW_POOL];  // then the undecided entries
  };
  uint64_t mass[CTAS][WARPS];  // of each warp of the cluster
  uint64_t part[CTAS][WARPS];  // of its candidates; of its kept entries
  uint64_t scan_q[WARPS];
  uint32_t scan_n[WARPS];
  uint32_t n[CTAS];
  uint64_t lo, hi, mid, cut_q, cut_c;
  uint32_t cut_n, count, above, first, b1, b2, last, dirty;
};
constexpr int ROW_SUMS = 128;  // warps of the CTAs that share a row

// What the first CTA lays over its part of the row when only the listed
// entries (or the copy in memory) matter any more.
struct RowFinish {
  uint32_t start[ROW_SORT_BINS + 4];
  uint64_t loose[ROW_POOL];
  uint64_t sorted[ROW_POOL];
  uint64_t input[ROW_POOL];
  uint32_t part[ROW_SUMS][2];  // masses of a stretch's entries in the interval: their low 20 bits, the rest
};

// ---- one row --------------------------------------------------------------------
// NT threads a CTA.  MEM: one CTA has the row to itself and streams it from
// memory (L2) as often as it looks at it; else a cluster shares it and each CTA
// keeps its part in shared memory.
template <typename T, int NT, bool MEM> struct Row {
  using E = RowElem<T>;
  static constexpr int WARPS = NT / 32;
  static constexpr int CTAS = MEM ? 1 : ROW_MAX_CLUSTER;
  static_assert(CTAS * WARPS <= ROW_SUMS, "sums");
  using Shared = RowShared<CTAS, WARPS>;
  // the row begins at a whole line of shared memory behind it (at 16-byte boundaries, by the state's size: 512 x 131072
  // f32 mixed 123.6 us against 113.8, n = 20 of 128 x 131072 bf16 18.5 to 19.4 against 18.1)
  static constexpr size_t SHARED_BYTES = (sizeof(Shared) + 127) / 128 * 128;
  using Sums = uint64_t[CTAS][WARPS];
  // vectors that each thread keeps in flight, in slots of its own in shared memory
  static constexpr int AHEAD = 8;
  static constexpr size_t RING_BYTES = MEM ? (size_t)AHEAD * NT * 16 : 0;
  static constexpr int N = E::N;

  cg::cluster_group cluster;
  Shared& sh;
  uint4* data;
  const int tid, lane, wid;
  const uint32_t rank, ctas;
  const uint32_t lists;  // of published maxima
  const uint32_t per;    // how many of its 32 sorted thread maxima a warp publishes
  const uint32_t room;   // a CTA's share of the first CTA's list of candidates
  // the row in memory, cut into 16-byte vectors at memory's boundaries
  const T* x;
  const uint4* vecs;
  uint32_t cols, part_vecs;
  int lead;             // elements of the first vector that are not the row's
  uint32_t total_vecs;
  uint32_t seg0, seg1;  // this warp's vectors of the CTA's part
  int first;            // index of the part's element 0 (negative inside the row's leading fill)
  float mine;           // this thread's maximum
  bool dirty = false;   // the row has NaN or +inf (MEM)
  float m, c;

  // CTA `part` of the `parts` of a row; d: where it keeps its part (null: nowhere).
  __device__ __forceinline__ Row(Shared& s, uint4* d, const RowArgs& a, uint32_t row, uint32_t part, uint32_t parts, uint32_t lists_a_warp = 1)
      : cluster(cg::this_cluster()),
        sh(s),
        data(d),
        tid(threadIdx.x),
        lane(threadIdx.x & 31),
        wid(threadIdx.x >> 5),
        rank(part),
        ctas(parts),
        lists(parts * WARPS * lists_a_warp),
        per(min(32u, (uint32_t)ROW_TOPS / lists)),
        room(ROW_LIST / parts) {
#pragma unroll 1
    for (int b = tid; b < ROW_EDGE_BINS; b += NT) sh.edge_n[b] = 0;
    if (tid == 0) sh.count = 0, sh.first = ~0u, sh.dirty = 0;
    if constexpr (MEM) __syncthreads();
    x = static_cast<const T*>(a.x) + (int64_t)row * a.stride;
    cols = a.cols;
    part_vecs = a.part_vecs;
    lead = (int)((uint32_t)(reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    total_vecs = ((uint32_t)lead + cols + N - 1) / N;
    vecs = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(x) & ~(uintptr_t)15);
  }

  static __device__ __forceinline__ uint4 nothing() {
    return make_uint4(E::NEG_INF, E::NEG_INF, E::NEG_INF, E::NEG_INF);
  }
  static __device__ __forceinline__ uint4 cleaned(uint4 v) {
    v.x = E::clean(v.x), v.y = E::clean(v.y), v.z = E::clean(v.z), v.w = E::clean(v.w);
    return v;
  }
  __device__ __forceinline__ bool inside(uint32_t v) const {  // all of the row's vector v belongs to the row
    const int j0 = (int)(v * N) - lead;
    return j0 >= 0 && j0 + N <= (int)cols;
  }
  __device__ __forceinline__ uint4 ragged(uint32_t i) const {  // the row's first or last vector
    const int j0 = (int)(i * N) - lead;
    uint4 v = nothing();
#pragma unroll 1
    for (int e = 0; e < N; ++e)
      if (j0 + e >= 0 && j0 + e < (int)cols) E::put(v, e, x + j0 + e);
    return v;
  }
  __device__ __forceinline__ uint4 from_memory(uint32_t v) const {
    return cleaned(inside(v) ? __ldg(vecs + v) : ragged(v));
  }
  // vectors [v0, v1) of warp w's stretch of CTA r's part
  __device__ __forceinline__ void stretch(uint32_t r, uint32_t w, uint32_t& v0, uint32_t& v1) const {
    const uint32_t p0 = min(r * part_vecs, total_vecs), p1 = min(p0 + part_vecs, total_vecs);
    const uint32_t sv = (p1 - p0 + WARPS - 1) / WARPS;
    v0 = min(p0 + w * sv, p1);
    v1 = min(v0 + sv, p1);
  }

  // Finds the row's maximum from memory; two maxima a thread, of every other
  // vector each.
  __device__ __forceinline__ void load_memory(bool tops) {
    first = -lead;
    typename E::Top top[2] = {E::top0(), E::top0()};
    stream<false, false, true>([&](const uint4& v, uint32_t) {  // the two take turns
      const typename E::Top t = E::top(top[0], v);
      top[0] = top[1];
      top[1] = t;
    }, [] {});
    const bool bad = !(E::value(top[0]) <= ROW_F32_MAX && E::value(top[1]) <= ROW_F32_MAX);
    if (__any_sync(~0u, bad)) {  // NaN or +inf: the warp looks through its stretch again
      sh.dirty = 1;
      top[0] = top[1] = E::top0();
      stream<true, false, false>([&](const uint4& v, uint32_t) { top[0] = E::top(top[0], v); }, [] {});
    }
#pragma unroll
    for (int l = 0; l < 2; ++l) {
      mine = E::value(top[l]);
      const uint32_t k = tops ? sorted_tops() : __reduce_min_sync(~0u, row_key(mine));
      if (lane < (int)(tops ? per : 1)) sh.tops[(wid * 2 + l) * per + lane] = k;
    }
    __syncthreads();
    dirty = sh.dirty != 0;
    find_max();
  }

  // Reads this CTA's part into shared memory and finds the row's maximum.
  // Each warp has a stretch of its own, in index order; each thread copies the
  // vectors that it will work on itself, all of them in flight at once, so
  // nothing but its own copies has to be waited for.
  // With `tops`, the warps also publish their threads' largest maxima.
  __device__ __forceinline__ void load(bool tops) {
    if constexpr (MEM) {
      load_memory(tops);
      return;
    }
    cluster.barrier_arrive();  // waited for below: no CTA writes into one that has not started
    const uint32_t p0 = min(rank * part_vecs, total_vecs);
    stretch(rank, wid, seg0, seg1);
    seg0 -= p0, seg1 -= p0;
    first = (int)(p0 * N) - lead;
    // the row's first and last vector, where they are not its own alone; the others are copied
    const bool head = seg0 < seg1 && !inside(p0 + seg0), tail = seg0 + head < seg1 && !inside(p0 + seg1 - 1);
    const uint32_t i0 = seg0 + lane, from = i0 + (head && lane == 0 ? 32 : 0), end = seg1 - tail;
    uint32_t to = smem_of(data + from);
    const uint4* of = vecs + p0 + from;
#pragma unroll 4
    for (uint32_t i = from; i < end; i += 32, to += 32 * 16, of += 32)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(of) : "memory");
    const uint32_t last = seg1 - 1 - seg0;  // the last vector's thread copies it, too
    if (head && lane == 0) data[seg0] = ragged(p0 + seg0);
    if (tail && lane == (int)(last % 32)) data[seg1 - 1] = ragged(p0 + seg1 - 1);
    asm volatile("cp.async.wait_all;" ::: "memory");
    typename E::Top top = E::top0();
#pragma unroll 4
    for (uint32_t i = seg0 + lane; i < seg1; i += 32) top = E::top(top, data[i]);
    mine = E::value(top);
    if (!(mine <= ROW_F32_MAX)) {  // NaN or +inf among this thread's entries
      top = E::top0();
#pragma unroll 1
      for (uint32_t i = seg0 + lane; i < seg1; i += 32) {
        const uint4 v = cleaned(data[i]);
        data[i] = v;
        top = E::top(top, v);
      }
      mine = E::value(top);
    }
    const uint32_t k = tops ? sorted_tops() : __reduce_min_sync(~0u, row_key(mine));
    cluster.barrier_wait();
#pragma unroll 1
    for (uint32_t i0 = 0; i0 < per * ctas; i0 += 32) {
      const uint32_t to = (i0 + lane) / per, e = i0 + lane - to * per, v = __shfl_sync(~0u, k, e);
      if (to < ctas && (tops || e == 0)) *cluster.map_shared_rank(&sh.tops[(rank * WARPS + wid) * per + e], to) = v;
    }
    cluster.sync();
    find_max();
  }
  // The keys of the warp's thread maxima in ascending order: lane 0 has the
  // largest entry's.
  __device__ __forceinline__ uint32_t sorted_tops() const {
    uint32_t k = row_key(mine);
#pragma unroll
    for (int n = 2; n <= 32; n <<= 1)
#pragma unroll
      for (int d = n >> 1; d; d >>= 1) {
        const uint32_t o = __shfl_xor_sync(~0u, k, d);
        k = ((lane & d) == 0) == ((lane & n) == 0) ? min(k, o) : max(k, o);
      }
    return k;
  }
  // The row's maximum from the published ones.
  __device__ __forceinline__ void find_max() {
    uint32_t best = ~0u;
#pragma unroll 1
    for (uint32_t i = lane; i < lists; i += 32) best = min(best, sh.tops[i * per]);
    m = row_unkey(__reduce_min_sync(~0u, best));
  }
  // The edge of the candidates of a cut; infinity where they are too many to list.
  __device__ __forceinline__ float edge_for(const RowParams& q) {
    if (q.by_k || q.by_p) {
      const uint32_t want = q.by_k ? q.k : ROW_NUCLEUS_GUESS;
      return want <= most_tops() ? edge_of(want, ROW_EDGE_SCALE * c, mass_end()) : INFINITY;
    }
    return fmaxf(m + (log2f(q.least_w) - 0x1p-10f) / c - fabsf(m) * 0x1p-21f, mass_end());
  }
  __device__ __forceinline__ float edge_for_best(uint32_t n) {
    if (n > most_tops()) return INFINITY;
    const float edge = edge_of(n, ROW_EDGE_SCALE * ROW_LOG2E, -ROW_F32_MAX);
    return edge == -ROW_F32_MAX ? edge_of(n, far_scale(), -ROW_F32_MAX) : edge;
  }
  __device__ __forceinline__ uint32_t most_tops() const { return per * lists * 3 / 4; }

  // f(vector, number in the part) for this thread's vectors, two side by side;
  // from memory, with +inf and NaN as they are unless CLEAN; now_and_then() is
  // called every 32 vectors.  BACK: from the
  // stretch's end, which was read last and is in L2 for the longest.  f appears
  // in the code once or twice (WIDE) in the loop and once behind it: the code of
  // a row is run once or twice by a CTA, so its size is time.
  template <bool CLEAN, bool BACK, bool WIDE, typename F, typename G> __device__ __forceinline__ void stream(F f, G now_and_then) const {
    uint32_t v0, v1;
    stretch(0, wid, v0, v1);
    const bool head = v0 < v1 && !inside(v0), tail = v0 + head < v1 && !inside(v1 - 1);
    const uint32_t lo = v0 + head, end = v1 - tail;
    uint32_t i = lo + lane, next = i;
    auto number = [&](uint32_t n) { return BACK ? lo + end - 1 - n : n; };
    constexpr uint32_t STEP = NT * 16;
    const uint32_t slots = smem_of(data + tid);
    auto fetch = [&](uint32_t slot) {
      if (next < end)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slot), "l"(vecs + number(next)) : "memory");
      next += 32;
    };
    auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
    auto get = [&](uint32_t slot) {
      const uint4 v = smem_load(slot);
      return CLEAN ? cleaned(v) : v;
    };
#pragma unroll
    for (int k = 0; k < AHEAD; k += 2) fetch(slots + k * STEP), fetch(slots + (k + 1) * STEP), commit();
    uint32_t slot = slots, turns = 0;
#pragma unroll 1
    for (; i + 32 < end; i += 64) {
      asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD / 2 - 1) : "memory");
      if constexpr (WIDE) {
        const uint4 a = get(slot), b = get(slot + STEP);
        f(a, number(i));
        f(b, number(i + 32));
      } else {
#pragma unroll 1
        for (int k = 0; k < 2; ++k) f(get(slot + k * STEP), number(i + 32 * k));
      }
      fetch(slot), fetch(slot + STEP), commit();
      slot += 2 * STEP;
      if (slot == slots + AHEAD * STEP) slot = slots;
      if (++turns % 16 == 0) now_and_then();
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    // what is left: a vector of the loop's, then on one thread each the row's ends
    const bool at_head = head && lane == 0, at_tail = tail && lane == 1;
    const uint32_t ragged_at = at_head ? v0 : v1 - 1;
#pragma unroll 1
    for (int k = i < end ? 0 : 1; k < (at_head || at_tail ? 2 : 1); ++k)
      f(k ? cleaned(ragged(ragged_at)) : get(slot), k ? ragged_at : number(i));
  }
  template <bool WIDE, typename F, typename G> __device__ __forceinline__ void vectors(F f, G now_and_then) const {
    if constexpr (MEM) {
      stream<true, true, WIDE>(f, now_and_then);
    } else if constexpr (WIDE) {
#pragma unroll 2
      for (uint32_t i = seg0 + lane; i < seg1; i += 32) f(data[i], i);
    } else {
#pragma unroll 1
      for (uint32_t i = seg0 + lane; i < seg1; i += 32) f(data[i], i);
    }
  }

  __device__ __forceinline__ float weight(float v) const { return row_exp2(row_neg_y(v, m, c)); }
  __device__ __forceinline__ uint64_t mass(float v) const { return row_q(weight(v)); }
  __device__ __forceinline__ uint32_t bin_of(float v, float scale, int bins) const {
    return (uint32_t)fminf(__fmul_rn(-row_neg_y(v, m, c), scale), (float)(bins - 1));
  }

  // Exclusive sum over the block, and the block's sum.
  template <typename V> static __device__ __forceinline__ V block_scan(V v, V* scratch, V& all) {
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    const V in = warp_scan(v, lane);
    if (lane == 31) scratch[wid] = in;
    __syncthreads();
    V before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const V s = scratch[w];
      if (w < wid) before += s;
      all += s;
    }
    return before + in - v;
  }

  // ---- the one pass over all weights ----
  // The mass of this thread's entries (ABOVE: of those over `over`, and
  // f(x, index) for those from `low` to `over`; HEAVY: of those over
  // `over` with w >= least_w).  Per entry: a half of four
  // packed additions, a half of one packed multiplication, the exponential and
  // one integer addition.  Fewer than 512 entries
  // come between folds (a part in shared memory has fewer a thread), so that
  // neither 32-bit sum of hi < 2^23 or |lo| <= 2^17 wraps.
  enum { ALL, ABOVE, HEAVY };
  struct Sum {
    uint64_t m2, c2;
    uint64_t folded = 0;
    uint32_t hi = 0, lo = 0, n = 0;
    __device__ __forceinline__ Sum(float m, float c) : m2(f2_pack(-m, -m)), c2(f2_pack(c, c)) {}
    template <int KIND> __device__ __forceinline__ void add(const uint4& v, float over, float least_w, float* below = nullptr) {
      const uint64_t one = f2_pack(1.0f, 1.0f), none = f2_pack(-1.0f, -1.0f), both = f2_pack(1.0f + ROW_MAGIC, 1.0f + ROW_MAGIC);
      float z[N];
      E::get(v, z);
#pragma unroll
      for (int e = 0; e < N; e += 2) {
        float w0, w1, a0, a1, b0, b1;
        f2_unpack(f2_mul(f2_add(f2_pack(z[e], z[e + 1]), m2), c2), w0, w1);
        w0 = row_exp2(w0), w1 = row_exp2(w1);
        if (KIND == HEAVY) w0 = w0 >= least_w ? w0 : 0.0f, w1 = w1 >= least_w ? w1 : 0.0f;
        if (KIND != ALL) {
          const bool in0 = z[e] > over, in1 = z[e + 1] > over;
          w0 = in0 ? w0 : 0.0f, w1 = in1 ? w1 : 0.0f;
          if (KIND == ABOVE) *below = fmaxf(fmaxf(*below, in0 ? -INFINITY : z[e]), in1 ? -INFINITY : z[e + 1]);
        }
        const uint64_t w = f2_pack(w0, w1);
        const uint64_t a = f2_add(w, one);
        const uint64_t b = f2_add(w, f2_fma(a, none, both));  // 1 + MAGIC - a is exact
        f2_unpack(a, a0, a1);
        f2_unpack(b, b0, b1);
        hi += __float_as_uint(a0) + __float_as_uint(a1);
        lo += __float_as_uint(b0) + __float_as_uint(b1);
      }
      n += N;
    }
    __device__ __forceinline__ void fold() {
      folded = mass();
      hi = lo = n = 0;
    }
    __device__ __forceinline__ uint64_t mass() const {
      return folded + row_mass(hi - n * ROW_ONE_BITS, (int)(lo - n * ROW_MAGIC_BITS));
    }
  };
  template <int KIND, typename F> __device__ __forceinline__ uint64_t weigh(float over, float low, float least_w, F f) const {
    Sum sum(m, c);
    // which of the thread's vectors f wants (the last bit: any of the 32nd and later ones): they are looked at again
    // afterwards, few and together
    uint32_t has = 0, bit = 1;
    vectors<KIND == ALL>([&](const uint4& v, uint32_t i) {
      float below = -INFINITY;  // the largest that is not above
      sum.template add<KIND>(v, over, least_w, &below);
      if (KIND == ABOVE && MEM && below >= low) each_of(hits(v, low, over), v, i, f);
      if (KIND == ABOVE && !MEM) {
        if (below >= low) has |= bit;
        bit = bit << 1 | (bit & 0x80000000u);
      }
    }, [&] { sum.fold(); });
#pragma unroll 1
    while (KIND == ABOVE && !MEM && has) {
      const uint32_t k = __ffs((int)has) - 1;
      has &= has - 1;
#pragma unroll 1
      for (uint32_t i = seg0 + lane + 32 * k; i < seg1; i += k == 31 ? 32 : part_vecs) {
        const uint4 v = data[i];
        each_of(hits(v, low, over), v, i, f);
      }
    }
    return sum.mass();
  }
  __device__ __forceinline__ uint64_t heavy(float over, float least_w) const {
    return weigh<HEAVY>(over, 0.0f, least_w, [](float, int) {});
  }

  // The same pass also lists the entries of at least `edge` in this CTA's share
  // of the first CTA's list (sh.count = 0 before), or only finds the first of
  // them.  Infinity: none.
  __device__ __forceinline__ void list_entry(float z, int j, bool only_first) const {
    if (only_first) {
      atomicMin(cluster.map_shared_rank(&sh.first, 0), (uint32_t)j);
    } else {
      const uint32_t at = atomicAdd(&sh.count, 1u);
      if (at < room) sh.list[at] = (uint64_t)row_key(z) << ROW_IDX_BITS | (uint32_t)j;
    }
  }
  template <bool CLEAN> __device__ __forceinline__ uint64_t weigh_and_list_of(float edge, bool only_first) {
    Sum sum(m, c);
    const bool lists_any = edge < INFINITY;
    stream<CLEAN, true, !CLEAN>([&](const uint4& v, uint32_t i) {
      sum.template add<ALL>(v, 0.0f, 0.0f);
      if (lists_any && E::value(E::top(E::top0(), v)) >= edge)
        each_of(hits(v, edge, INFINITY), v, i, [&](float z, int j) { list_entry(z, j, only_first); });
    }, [&] { sum.fold(); });
    return sum.mass();
  }
  __device__ __forceinline__ uint64_t weigh_and_list(float edge, bool only_first) {
    if constexpr (MEM) {
      return dirty ? weigh_and_list_of<true>(edge, only_first) : weigh_and_list_of<false>(edge, only_first);
    } else {
      Sum sum(m, c);
      const bool lists_any = mine >= edge;
      // which of the thread's vectors have any (the last bit: any of the 32nd and later ones): they are looked at again
      uint32_t has = 0, bit = 1;
#pragma unroll 2
      for (uint32_t i = seg0 + lane; i < seg1; i += 32) {
        const uint4 v = data[i];
        sum.template add<ALL>(v, 0.0f, 0.0f);
        if (lists_any) {
          if (E::value(E::top(E::top0(), v)) >= edge) has |= bit;
          bit = bit << 1 | (bit & 0x80000000u);
        }
      }
#pragma unroll 1
      while (has) {
        const uint32_t k = __ffs((int)has) - 1;
        has &= has - 1;
#pragma unroll 1
        for (uint32_t i = seg0 + lane + 32 * k; i < seg1; i += k == 31 ? 32 : part_vecs) {
          const uint4 v = data[i];
          each_of(hits(v, edge, INFINITY), v, i, [&](float z, int j) { list_entry(z, j, only_first); });
        }
      }
      return sum.mass();
    }
  }

  // Bits of the entries of a vector in [low, high].
  static __device__ __forceinline__ uint32_t hits(const uint4& v, float low, float high) {
    float z[N];
    E::get(v, z);
    uint32_t mask = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) mask |= (uint32_t)(z[e] >= low && z[e] <= high) << e;
    return mask;
  }
  // f(x, index) for the entries of vector i of this CTA's part that mask names
  template <typename F> __device__ __forceinline__ void each_of(uint32_t mask, const uint4& v, uint32_t i, F f) const {
#pragma unroll 1
    while (mask) {
      const int e = __ffs((int)mask) - 1;
      mask &= mask - 1;
      f(E::at(v, e), first + (int)(i * N) + e);
    }
  }
  // Calls f(x, index) for the warp's entries in [low, high], many of them.
  template <typename F> __device__ __forceinline__ void between(float low, float high, F f) const {
    vectors<false>([&](const uint4& v, uint32_t i) { each_of(hits(v, low, high), v, i, f); }, [] {});
  }
  // A value with at least `k` of the row's entries at or above it: the k-th
  // largest of the published thread maxima, rounded down to the bound of a bin
  // of 1 / scale and by more than the bound's rounding.  Where fewer are within
  // the bins: `last`.  Of entries in no particular order, and maxima of G
  // groups, about G ln(G / (G - k)) lie above the k-th largest maximum: hardly
  // more than k.  Every warp scans the histogram for itself, which spares a
  // barrier.
  __device__ __forceinline__ float edge_of(uint32_t k, float scale, float last) {
    const uint32_t tops = per * lists;
    scale = fminf(scale, ROW_F32_MAX);
#pragma unroll 1
    for (uint32_t i = tid; i < tops; i += NT) {
      const float z = row_unkey(sh.tops[i]);
      if (z > -INFINITY)
        atomicAdd(&sh.edge_n[(uint32_t)fminf(__fmul_rn(__fsub_rn(m, z), scale), (float)(ROW_EDGE_BINS - 1))], 1u);
    }
    __syncthreads();
    constexpr int PER = ROW_EDGE_BINS / 32;
    uint32_t n[PER], t = 0;
#pragma unroll
    for (int b = 0; b < PER; ++b) n[b] = sh.edge_n[lane * PER + b], t += n[b];
    const uint32_t upto = warp_scan(t, lane);
    const uint32_t has = __ballot_sync(~0u, upto >= k);
    if (!has) return last;
    uint32_t bin = lane * PER, run = upto - t;
#pragma unroll
    for (int b = 0; b + 1 < PER; ++b) {
      run += n[b];
      bin += run < k;
    }
    bin = __shfl_sync(~0u, bin, __ffs((int)has) - 1);
    if (bin >= (uint32_t)ROW_EDGE_BINS - 1) return last;
    const float d = (float)(bin + 1) / scale;
    return fmaxf(m - d * (1.0f + 0x1p-18f) - fabsf(m) * 0x1p-21f, last);
  }
  // Its scale where 42 octaves of weight are too short: up to the smallest
  // maximum, or 512.  Empties the bins again.
  __device__ __forceinline__ float far_scale() {
    const uint32_t tops = per * lists;
    float low = m;
#pragma unroll 1
    for (uint32_t i = lane; i < tops; i += 32) {
      const float z = row_unkey(sh.tops[i]);
      if (z > m - 512.0f) low = fminf(low, z);
    }
    low = row_unkey(__reduce_max_sync(~0u, row_key(low)));
    __syncthreads();
#pragma unroll 1
    for (int b = tid; b < ROW_EDGE_BINS; b += NT) sh.edge_n[b] = 0;
    __syncthreads();
    return (ROW_EDGE_BINS - 2) / fmaxf(m - low, 0x1p-20f);
  }
  // Below this no entry has mass.
  __device__ __forceinline__ float mass_end() const {
    return fmaxf(m - ROW_MASS_END / c - fabsf(m) * 0x1p-21f, -ROW_F32_MAX);
  }

  // Hands this warp's masses to the first CTA (ALL: to every CTA).
  template <bool ALL> __device__ __forceinline__ void hand(Sums& to, uint64_t own) {
    own = warp_sum_u64(own);
    if (lane < (ALL ? (int)ctas : 1)) *cluster.map_shared_rank(&to[rank][wid], lane) = own;
  }
  // Sums of what was handed over.
  __device__ __forceinline__ uint64_t handed(const Sums& of) const {
    uint64_t t = 0;
#pragma unroll 1
    for (uint32_t i = lane; i < ctas * WARPS; i += 32) t += (&of[0][0])[i];
    return warp_sum_u64(t);
  }
  // Hands them to the first CTA and tells every CTA their number.
  __device__ __forceinline__ void tell_list() {
    __syncthreads();
    if (tid < (int)ctas) *cluster.map_shared_rank(&sh.n[rank], tid) = sh.count;
    if (rank) {
      uint64_t* const to = cluster.map_shared_rank(sh.list, 0) + rank * room;
#pragma unroll 1
      for (uint32_t i = tid; i < min(sh.count, room); i += NT) to[i] = sh.list[i];
    }
  }
  // Whether the candidates of all CTAs fit their shares; their total.
  __device__ __forceinline__ bool all_listed(uint32_t& n) const {
    const uint32_t of = lane < (int)ctas ? sh.n[lane] : 0;
    n = __reduce_add_sync(~0u, of);
    return __all_sync(~0u, of <= room);
  }
  // f(number, entry) for this thread's candidates, on the first CTA.
  template <typename F> __device__ __forceinline__ void each_listed(F f) const {
    const uint32_t of = lane < (int)ctas ? sh.n[lane] : 0, upto = warp_scan(of, lane);
#pragma unroll 1
    for (uint32_t r = MEM ? 0 : wid; r < ctas; r += WARPS) {
      const uint32_t have = __shfl_sync(~0u, of, r), before = __shfl_sync(~0u, upto, r) - have;
#pragma unroll 1
      for (uint32_t i = MEM ? tid : lane; i < have; i += MEM ? NT : 32) f(before + i, sh.list[r * room + i]);
    }
  }
  // Tells every CTA the number of entries that this one has put at the start
  // of its pool.
  __device__ __forceinline__ void tell_pool() {
    __syncthreads();
    if (tid < (int)ctas) *cluster.map_shared_rank(&sh.n[rank], tid) = sh.count;
  }
  // After tell_pool() on every CTA and a cluster barrier: their total, and
  // where they are at most `room`, the others' go behind the first CTA's.
  __device__ __forceinline__ uint32_t pooled(uint32_t room) {
    uint32_t n = 0, base = 0;
#pragma unroll 1
    for (uint32_t i = 0; i < ctas; ++i) {
      if (i == rank) base = n;
      n += sh.n[i];
    }
    if (n <= room && rank) {
      uint64_t* const to = cluster.map_shared_rank(sh.pool, 0) + base;
#pragma unroll 1
      for (uint32_t i = tid; i < sh.n[rank]; i += NT) to[i] = sh.pool[i];
    }
    return n;
  }
  // The end of the cluster's common work: true on the first CTA, once the
  // others' writes into it are there; the others are done.
  __device__ __forceinline__ bool last_part() {
    cluster.barrier_arrive();
    if (rank) return false;
    cluster.barrier_wait();
    return true;
  }

  // ---- narrowing a cut down, by the whole cluster ----
  // Bins of weight: (m - x) cs, that is y by the bins an octave, to the nearest
  // whole number, by an addition that pushes the fraction out of the mantissa.
  __device__ __forceinline__ float place_of(float v, float cs) const { return __fmul_rn(__fsub_rn(m, v), cs); }
  static __device__ __forceinline__ uint32_t bin_at(float place) {
    return __float_as_uint(__fadd_rn(fminf(place, (float)(ROW_BINS - 1)), 0x1p23f)) & 0x7fffffu;
  }
  // The smallest key from the maximum's on whose bin is b or later; one warp,
  // 32 probes at a time.
  __device__ __forceinline__ uint32_t first_key(uint32_t b, float cs) const {
    uint32_t lo = row_key(m), hi = row_key(-ROW_F32_MAX) + 1;
#pragma unroll 1
    while (lo < hi) {
      const uint32_t step = max(1u, (hi - lo) / 32), at = lo + lane * step;
      const bool past = at - lo >= hi - lo || bin_at(place_of(row_unkey(at), cs)) >= b;
      const uint32_t has = __ballot_sync(~0u, past);
      if (has & 1) break;
      const int f = has ? __ffs((int)has) - 1 : 32;
      if (has) hi = min(hi, lo + f * step);
      lo += (f - 1) * step + 1;
    }
    return lo;
  }

  // The unit of a weight in its bin: with it 32 bits hold the sum of every
  // entry that a CTA has, of up to twice the unit less a little.  (The tangents
  // are within 1% of the unit; what q holds is up to 4/3 of the weight, and
  // below 2^-40, where it is up to twice the weight, the unit is that of 2^-40.)
  static constexpr float UNIT = MEM ? 0x1p12f : 0x1p16f;
  static constexpr int UNIT_BITS = MEM ? 12 : 16;
  // A vector's entries by bin.  Their weights, up to the last bin, as
  // UNIT 2^-(y - b) / per_octave by the power's tangent, made a whole number by
  // another addition of 2^23.  Two entries an instruction, and all of a vector's places
  // before the first addition: few warps share an SM here, so what counts is
  // the length of the chain.
  __device__ __forceinline__ void weigh_bins(const uint4& v, uint32_t bins, float cs, float per_octave) const {
    constexpr uint32_t MAGIC = 0x4b000000u;  // 2^23
    const uint64_t magic = f2_pack(0x1p23f, 0x1p23f), minus = f2_pack(-0x1p23f, -0x1p23f), none = f2_pack(-1.0f, -1.0f);
    const float slope = -UNIT * ROW_LN2 / per_octave;
    const uint64_t tangent = f2_pack(slope, slope);
    const uint64_t unit = f2_pack(0x1p23f + UNIT, 0x1p23f + UNIT), m2 = f2_pack(m, m), c2 = f2_pack(cs, cs);
    float z[N], y[N], b[N], w[N];
    E::get(v, z);
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const uint64_t place = f2_mul(f2_fma(f2_pack(z[e], z[e + 1]), none, m2), c2);
      const uint64_t bin = f2_add(place, magic);
      f2_unpack(place, y[e], y[e + 1]);
      f2_unpack(bin, b[e], b[e + 1]);
      f2_unpack(f2_fma(f2_fma(f2_add(bin, minus), none, place), tangent, unit), w[e], w[e + 1]);
    }
#pragma unroll
    for (int e = 0; e < N; ++e)
      smem_add_if(y[e] < (float)ROW_BINS_END, bins + (__float_as_uint(b[e]) - MAGIC) * 4, __float_as_uint(w[e]) - MAGIC);
  }
  // Their numbers.
  __device__ __forceinline__ void count_bins(const uint4& v, uint32_t bins, float cs) const {
#pragma unroll 1
    for (int e = 0; e < N; ++e) {
      const float z = E::at(v, e);
      smem_add_if(z > -INFINITY, bins + bin_at(place_of(z, cs)) * 4, 1u);
    }
  }
  // From the bins' sums over the row, by one CTA: the bins sh.b1 to sh.b2 that
  // the prefix ends in (both ~0 before, and at most sh.last, 0 before), and for
  // counts the entries before them, sh.above.  The prefix ends in b1 or later, and in b2 or before: where a sum of
  // estimates, its slack and in the first round 2^-20 of the largest weight
  // added, and taken off, reaches the goal.  (An estimate is off by half a unit
  // and, a tangent at most half a bin from where it touches, by a 16th of the
  // bin's width squared; the weights' rounding to q by at most 2^-22 together;
  // from the second round on estimates follow q.  Counts are exact.)
  // Else it ends in the last bin with anything; a count that is not reached,
  // beyond all of them.
  __device__ __forceinline__ void end_bins(bool by_mass, bool first_round, float goal, uint32_t above_n, float octaves) {
    constexpr int PER = (ROW_BINS + NT - 1) / NT;
    const int at = tid * PER;
    float v[PER], own = 0, all;
    uint32_t filled = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = at + i < ROW_BINS ? __uint_as_float(sh.bins[at + i]) : 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (v[i] > 0.0f) filled = at + i;
      own += v[i];
    }
    filled = __reduce_max_sync(~0u, filled);
    if (lane == 0) atomicMax(&sh.last, filled);
    float run = block_scan(own, reinterpret_cast<float*>(sh.scan_n), all);
    const float slack = by_mass ? 1.25f / UNIT + 0.0625f * octaves * octaves : 0.0f, more = by_mass && first_round ? UNIT * 0x1p-20f : 0.0f;
    uint32_t b1 = ~0u, b2 = ~0u;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int b = at + i;
      if (b >= ROW_BINS) break;
      if (run < goal && (run + v[i] >= goal || b == ROW_BINS - 1)) sh.above = above_n + (uint32_t)run;  // read for counts alone
      run += v[i];
      if (run * (1.0f + slack) + more >= goal) b1 = min(b1, (uint32_t)b);
      if (run * (1.0f - slack) - more >= goal) b2 = min(b2, (uint32_t)b);
    }
    b1 = __reduce_min_sync(~0u, b1), b2 = __reduce_min_sync(~0u, b2);
    if (lane == 0) {
      if (b1 != ~0u) atomicMin(&sh.b1, b1);
      if (b2 != ~0u) atomicMin(&sh.b2, b2);
    }
    __syncthreads();
  }
  // Of the interval of those bins: warp 0 gets the first entry, warp 1 the last,
  // warp 2 the last of bin b1.
  // In the first round by mass a little before and behind them, by more than
  // the rounding of a bin's bound, which spares the search; counts, and the
  // rounds that have to shorten the interval, need the bounds themselves.
  __device__ __forceinline__ uint64_t end_of(bool by_mass, bool by_weight, bool first_round, float cs, int shift, uint64_t lo,
                                             uint64_t hi) {
    if (wid >= 3) return 0;
    const uint32_t end = by_mass ? sh.last : (uint32_t)ROW_BINS - 1;
    const uint32_t b = min(wid == 1 ? sh.b2 : sh.b1, end) + (wid ? 1 : 0);
    uint64_t at;
    if (by_mass && first_round) {
      const float d = __fdiv_rn((float)b - 0.5f, cs), by = fabsf(m) * 0x1p-21f;
      if (wid) {
        const float z = m - d * (1.0f + 0x1p-18f) - by;
        return b < (uint32_t)ROW_BINS && z > -ROW_F32_MAX ? (uint64_t)row_key(z) << ROW_IDX_BITS | (ROW_MAX_COLS - 1) : hi;
      }
      return b ? max(lo, (uint64_t)row_key(fminf(fmaxf(m - d * (1.0f - 0x1p-18f) + by, -ROW_F32_MAX), m)) << ROW_IDX_BITS) : lo;
    }
    if (by_weight)
      at = b < (uint32_t)ROW_BINS ? max(lo, (uint64_t)first_key(b, cs) << ROW_IDX_BITS) : hi + 1;
    else
      at = lo + ((uint64_t)b << shift);
    at = min(at, hi + 1);
    return wid ? at - 1 : at;
  }

  // Finds an interval [sh.lo, sh.hi] of (key, index) order, with at most
  // `most` <= ROW_POOL entries, in which the prefix of `target` entries
  // (by_mass: mass) ends, and leaves
  //   those entries in the first CTA's sh.pool, their number in n,
  //   every warp's mass before the interval in sh.mass, and of that the mass
  //   of entries with w >= least_w in sh.part, on all CTAs,
  //   the number of entries before it in above_n (counts alone).
  // Each round counts the undecided entries by bin, or sums their weights, each
  // to 13 or 17 bits of its bin's, which tells the bin b1 that the prefix ends in or,
  // where it ends closer to b1's end than the sums' error, a range of bins from b1 on.  A
  // second pass takes the exact masses of what comes before b1 and of b1, which
  // tell b1 from what lies behind it: the next round has b1 alone, or has b1
  // among what comes before, and its estimates err by a part of the rest alone.
  // Bins are of a 42nd octave of weight or less, by how far
  // the nucleus may reach, and of a 2^-10th of the interval once it is shorter
  // than three of those (for counts: after the first round).
  // Most rows take two or three rounds.  A round that leaves b1 alone shortens the
  // interval of 51-bit (key, index) to a bin: once by weight, then by 2^9 at
  // least, so at most seven do.  One that leaves what lies behind b1
  // shrinks the goal, below 2^59, to twice the estimates' error of it, 2^-10
  // or less, so at most six do.
  // A weight as q holds it.
  static __device__ __forceinline__ float held(float w) {
    return w < 0x1p-17f ? __fsub_rn(__fadd_rn(w, ROW_MAGIC), ROW_MAGIC) : w;
  }
  struct Left {
    uint32_t n, above_n;
  };
  __device__ __forceinline__ Left narrow(bool by_mass, uint64_t target, uint64_t rest, float least_w, uint32_t most) const {
    return narrow_copy(*this, by_mass, target, rest, least_w, most);
  }
  // Not inlined, for its size; on a copy, so that the row's own members may
  // stay in registers everywhere else.
  static __device__ __noinline__ Left narrow_copy(Row r, bool by_mass, uint64_t target, uint64_t rest, float least_w, uint32_t most) {
    Left left;
    r.narrow_into(by_mass, target, rest, least_w, most, left.n, left.above_n);
    return left;
  }
  __device__ __forceinline__ void narrow_into(bool by_mass, uint64_t target, uint64_t rest, float least_w, uint32_t most,
                                              uint32_t& n, uint32_t& above_n) {
    uint64_t lo = (uint64_t)row_key(m) << ROW_IDX_BITS, hi = (uint64_t)row_key(-ROW_F32_MAX) << ROW_IDX_BITS | (ROW_MAX_COLS - 1);
    uint64_t above_q = 0;
    above_n = 0;
    // Bins an octave of weight.  What a nucleus leaves is at least `rest`, and so its last entry has at least rest / cols:
    // the bins of weights end an octave further on (or at the last weight that q holds).
    const float per_octave =
        by_mass ? ROW_BINS_END / fminf(ROW_MASS_END, 41.125f - log2f(fmaxf((float)rest / (float)cols, 0x1p-8f))) : ROW_BIN_SCALE;
    const float octaves = 1.0f / per_octave, cs = fminf(c * per_octave, ROW_F32_MAX);
    constexpr int ROUNDS = 16;
    __syncthreads();  // what was there has been read, by this CTA alone since the last barrier
#pragma unroll 1
    for (int round = 0; round < ROUNDS; ++round) {
#pragma unroll 1
      for (int b = tid; b < ROW_BINS; b += NT) sh.bins[b] = 0;
      if (tid == 0) sh.count = 0, sh.b1 = sh.b2 = ~0u, sh.last = 0;
      __syncthreads();
      const int shift = max(0, 64 - __clzll((long long)((hi - lo) | 1)) - 10);
      const float top_w = fmaxf(weight(value_of(lo)), 0x1p-40f), scale = UNIT / top_w;
      // octaves down to the weight whose unit bin b has
      auto down = [&](uint32_t b) { return round ? fminf((float)b * octaves, 40.0f) : (float)b * octaves; };
      const bool by_weight = round == 0 || (by_mass && bin_at(place_of(value_of(hi), cs)) >= bin_at(place_of(value_of(lo), cs)) + 3);
      if (round == 0) {
        const uint32_t bins = smem_of(sh.bins);
        vectors<false>([&](const uint4& v, uint32_t) {
          if (by_mass)
            weigh_bins(v, bins, cs, per_octave);
          else
            count_bins(v, bins, cs);
        }, [] {});
      } else {
        between(value_of(hi), value_of(lo), [&](float z, int j) {
          const uint64_t e = (uint64_t)row_key(z) << ROW_IDX_BITS | (uint32_t)j;
          if (e < lo || e > hi) return;
          if (!by_mass) {
            atomicAdd(&sh.bins[(uint32_t)((e - lo) >> shift)], 1u);
          } else if (by_weight) {
            const uint32_t b = bin_at(place_of(z, cs));
            atomicAdd(&sh.bins[b], (uint32_t)(held(weight(z)) * row_exp2(down(b) + (float)UNIT_BITS) + 0.5f));
          } else {
            atomicAdd(&sh.bins[(uint32_t)((e - lo) >> shift)], (uint32_t)(held(weight(z)) * scale + 0.5f));
          }
        });
      }
      cluster.sync();
      // each CTA sums a slice of the bins over the cluster, into the first CTA's
      const uint32_t slice = (ROW_BINS + ctas - 1) / ctas;
#pragma unroll 1
      for (uint32_t i = tid; i < slice; i += NT) {
        const uint32_t b = rank * slice + i;
        if (b < ROW_BINS) {
          float v = 0;
#pragma unroll 8
          for (uint32_t k = 0; k < ctas; ++k) v += (float)cluster.map_shared_rank(sh.bins, k)[b];
          if (by_mass) v *= by_weight ? row_exp2(-down(b)) : top_w;
          cluster.map_shared_rank(sh.bins, 0)[b] = __float_as_uint(v);
        }
      }
      cluster.sync();
      if (rank == 0) {
        const float goal = by_mass ? (float)(target - above_q) * (UNIT * 0x1p-40f) : (float)(target - above_n);
        end_bins(by_mass, round == 0, goal, above_n, octaves);
        const uint64_t at = end_of(by_mass, by_weight, round == 0, cs, shift, lo, hi);
        if (wid < 3 && lane < (int)ctas) {
          *cluster.map_shared_rank(wid == 0 ? &sh.lo : wid == 1 ? &sh.hi : &sh.mid, lane) = at;
          if (wid == 1 && lane) *cluster.map_shared_rank(&sh.above, lane) = sh.above;
        }
      }
      cluster.sync();
      lo = sh.lo, hi = sh.hi;
      // exact sums of what comes before, and the entries of the interval
      above_n = by_mass ? 0 : sh.above;
      const uint64_t mid = sh.mid;
      uint64_t before = 0, kept, in_b1 = 0;
      const float over = value_of(lo);
      const bool cuts_equals = (lo & (ROW_MAX_COLS - 1)) != 0;  // equal values lie on both sides of lo
      before = weigh<ABOVE>(over, value_of(hi), 0.0f, [&](float z, int j) {
        const uint64_t e = (uint64_t)row_key(z) << ROW_IDX_BITS | (uint32_t)j;
        if (e < lo || e > hi) return;
        if (by_mass && e <= mid) in_b1 += mass(z);
        const uint32_t at = atomicAdd(&sh.count, 1u);
        if (at < ROW_POOL) sh.pool[at] = e;
      });
      // where the weight there is clearly more, all that comes before has at least least_w
      kept = weight(over) * (1.0f - 0x1p-12f) >= least_w ? before : heavy(over, least_w);
      if (cuts_equals) {
        const float w = weight(over);
        between(over, over, [&](float, int j) {
          if ((uint32_t)j < ((uint32_t)lo & (ROW_MAX_COLS - 1))) before += row_q(w), kept += w >= least_w ? row_q(w) : 0;
        });
      }
      hand<true>(sh.mass, before);
      hand<true>(sh.part, kept);
      tell_pool();
      cluster.sync();
      above_q = handed(sh.mass);
      n = pooled(most);
      if (n <= most) return;
      if (by_mass) hand<true>(sh.part, in_b1);  // nobody reads its masses before the last round's
      cluster.sync();
      if (by_mass) {
        in_b1 = handed(sh.part);
        if (above_q + in_b1 >= target)
          hi = mid;
        else
          lo = mid + 1, above_q += in_b1;
      }
    }
    n = 0;  // by the count above, never; a row without a kept mass would say so
  }

  // ---- ordering the candidates, on the first CTA alone ----
  // Sorts the places c (all different) of up to ROW_POOL entries, entry i of
  // thread tid + 256 i: in(i, c, bin) says whether there is one, its place and
  // its bin, which grows with c.  A counting sort by bin; what shares a bin is
  // then ranked by comparing.  Returns their number.
  template <typename F> __device__ __forceinline__ uint32_t order(RowFinish& f, F in) {
    constexpr int PER = ROW_POOL / NT;
    uint64_t c[PER];
    uint32_t bin[PER], at[PER];
    constexpr int BINS = ROW_SORT_BINS / NT;
    static_assert(BINS * NT == ROW_SORT_BINS && PER * NT == ROW_POOL, "bins and entries a thread");
#pragma unroll
    for (int i = 0; i < BINS; ++i) f.start[tid * BINS + i] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      bin[i] = ~0u;
      if (in(i, c[i], bin[i])) at[i] = atomicAdd(&f.start[bin[i]], 1u);
    }
    __syncthreads();
    uint32_t n[BINS], own = 0, all;
#pragma unroll
    for (int i = 0; i < BINS; ++i) n[i] = f.start[tid * BINS + i], own += n[i];
    uint32_t before = block_scan(own, sh.scan_n, all);
#pragma unroll
    for (int i = 0; i < BINS; ++i) f.start[tid * BINS + i] = before, before += n[i];
    if (tid == 0) f.start[ROW_SORT_BINS] = all;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (bin[i] != ~0u) f.loose[f.start[bin[i]] + at[i]] = c[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (bin[i] != ~0u) {
        const uint32_t b0 = f.start[bin[i]], b1 = f.start[bin[i] + 1];
        uint32_t r = b0;
        if (b1 - b0 > 1)
#pragma unroll 1
          for (uint32_t k = b0; k < b1; ++k) r += f.loose[k] < c[i];
        f.sorted[r] = c[i];
      }
    __syncthreads();
    return all;
  }

  static __device__ __forceinline__ float value_of(uint64_t e) { return row_unkey((uint32_t)(e >> ROW_IDX_BITS)); }

  // The n entries at `from` in descending order of x into f.sorted.  Bins
  // linear in x over [low, m], or over 42 octaves where that is less.
  __device__ __forceinline__ void order_by_value(RowFinish& f, const uint64_t* from, uint32_t n, float low) {
    float scale = fmaxf((ROW_SORT_BINS - 1) / (m - low), (ROW_SORT_BINS - 1) / ROW_MASS_END * c);
    if (!(scale <= ROW_F32_MAX)) scale = 0.0f;  // all equal
    order(f, [&](int i, uint64_t& e, uint32_t& bin) {
      if (tid + i * NT >= n) return false;
      e = from[tid + i * NT];
      bin = (uint32_t)fminf(__fmul_rn(__fsub_rn(m, value_of(e)), scale), (float)(ROW_SORT_BINS - 1));
      return true;
    });
  }
  // Entry number `nth` (from 1) of the n <= ROW_FEW in sh.pool and the mass up
  // to it, into sh.hi and sh.cut_q; both stay where there is no such entry.
  __device__ __forceinline__ void nth_of_few(uint32_t n, uint32_t nth) {
    uint64_t* const q = sh.pool + ROW_FEW;
    const uint64_t e = tid < n ? sh.pool[tid] : 0;
    if (tid < n) q[tid] = mass(value_of(e));
    __syncthreads();
    uint32_t rank_in = 0;
    uint64_t upto = 0;
#pragma unroll 1
    for (uint32_t i = 0; i < n; ++i)
      if (sh.pool[i] <= e) ++rank_in, upto += q[i];
    if (tid < n && rank_in == nth) sh.hi = e, sh.cut_q = upto;
    __syncthreads();
  }

  // Of the n <= ROW_POOL entries with places f.sorted, all different, and sums
  // f.input: the one at which the running sum in order of place reaches `goal`
  // (~0: none does).  Exact sums by bins leave the
  // entries of one bin, and so on until few enough to be compared with each
  // other are left.  Bins are linear in the place over [lo, hi]; scale >= 0: the first
  // are linear in x, 1 / scale from m down.  Empties f.input of what drops out.
  // One copy of this serves all cuts and draws of a row.
  static __device__ __noinline__ uint64_t reach(RowFinish& f, Shared& sh, uint32_t n, uint64_t goal, uint64_t lo, uint64_t hi, float m,
                                                float scale) {
    constexpr int BINS = ROW_SORT_BINS / NT;
    constexpr uint32_t FEW = 64;
    static_assert(BINS * NT == ROW_SORT_BINS, "bins a thread");
    const uint32_t tid = threadIdx.x;
    uint32_t* const low = reinterpret_cast<uint32_t*>(f.loose);  // a bin's sum: the low 20 bits of each
    uint32_t* const high = low + ROW_SORT_BINS;                  // and the rest
    uint64_t left = goal;
    uint32_t undecided = n;
#pragma unroll 1
    while (undecided > FEW) {
      const int shift = max(0, 64 - __clzll((long long)((hi - lo) | 1)) - 10);
      auto bin_of = [&](uint64_t e) {
        return scale >= 0.0f ? (uint32_t)fminf(__fmul_rn(__fsub_rn(m, value_of(e)), scale), (float)(ROW_SORT_BINS - 1))
                             : (uint32_t)((e - lo) >> shift);
      };
#pragma unroll
      for (int i = 0; i < BINS; ++i) f.start[tid + i * NT] = low[tid + i * NT] = high[tid + i * NT] = 0;
      __syncthreads();
      if (tid == 0) sh.cut_n = ~0u;
#pragma unroll 1
      for (uint32_t i = tid; i < n; i += NT) {
        const uint64_t q = f.input[i];
        if (!q) continue;
        const uint32_t b = bin_of(f.sorted[i]);
        atomicAdd(&f.start[b], 1u);
        atomicAdd(&low[b], (uint32_t)q & 0xfffffu);
        atomicAdd(&high[b], (uint32_t)(q >> 20));
      }
      __syncthreads();
      uint64_t s[BINS], own = 0, all;
#pragma unroll
      for (int i = 0; i < BINS; ++i) {
        const uint32_t b = tid * BINS + i;
        s[i] = ((uint64_t)high[b] << 20) + low[b];
        own += s[i];
      }
      uint64_t run = block_scan(own, sh.scan_q, all);
      if (run < left && left <= run + own) {
#pragma unroll
        for (int i = 0; i < BINS; ++i) {
          if (run < left && left <= run + s[i]) sh.cut_n = tid * BINS + i, sh.cut_q = run, sh.above = f.start[tid * BINS + i];
          run += s[i];
        }
      }
      __syncthreads();
      const uint32_t cut = sh.cut_n;
      if (cut == ~0u) break;
      left -= sh.cut_q;
      undecided = sh.above;
#pragma unroll 1
      for (uint32_t i = tid; i < n; i += NT)
        if (f.input[i] && bin_of(f.sorted[i]) != cut) f.input[i] = 0;
      if (scale < 0.0f) lo += (uint64_t)cut << shift, hi = min(hi, lo + (((uint64_t)1 << shift) - 1));
      scale = -1.0f;
    }
    __syncthreads();
    if (tid == 0) sh.count = 0, sh.cut_c = ~0ull;
    __syncthreads();
    if (undecided <= FEW) {
      uint64_t* const c = f.loose;
      uint64_t* const q = f.loose + FEW;
#pragma unroll 1
      for (uint32_t i = tid; i < n; i += NT)
        if (f.input[i]) {
          const uint32_t at = atomicAdd(&sh.count, 1u);
          c[at] = f.sorted[i], q[at] = f.input[i];
        }
      __syncthreads();
      const uint32_t few = sh.count;
      if (tid < few) {
        const uint64_t own = c[tid];
        uint64_t upto = 0;
#pragma unroll 2
        for (uint32_t i = 0; i < few; ++i) upto += c[i] <= own ? q[i] : 0;
        if (upto >= left && upto - q[tid] < left) sh.cut_c = own;
      }
      __syncthreads();
    }
    return sh.cut_c;
  }

  // The same sums for n <= NT entries and for each of them, by comparing it
  // with all: entry tid / each of `each` neighbouring threads, which share its
  // comparisons.  less(i) says whether entry i comes before it, q its f.input;
  // returns the sum before it, and their number.
  template <typename L> static __device__ __forceinline__ uint64_t before_of(const RowFinish& f, uint32_t n, uint32_t each, uint32_t& number, L less) {
    uint64_t sum = 0;
    number = 0;
#pragma unroll 2
    for (uint32_t i = threadIdx.x & (each - 1); i < n; i += each) {
      const uint64_t q = f.input[i];
      const bool yes = less(f.sorted[i]);
      number += yes;
      sum += yes ? q : 0;
    }
#pragma unroll 1
    for (uint32_t d = 1; d < each; d <<= 1) {
      sum += __shfl_xor_sync(~0u, sum, d);
      number += __shfl_xor_sync(~0u, number, d);
    }
    return sum;
  }
  // finish_listed() for n <= NT / 2 entries.
  template <typename H>
  __device__ __forceinline__ void finish_few(RowFinish& f, uint32_t n, const RowParams& p, uint64_t total, H hit) {
    const uint32_t each = n <= NT / 8 ? 8 : n <= NT / 4 ? 4 : 2, slot = tid / each;
    const bool in = slot < n, works = wid * (32 / each) < n;
    const uint64_t e = in ? f.sorted[slot] : ~0ull;
    const float z = value_of(e), w = in ? weight(z) : 0.0f;
    const uint64_t q = row_q(w);
    if (in) f.input[slot] = q;
    if (tid == 0) sh.cut_q = total, sh.cut_c = ~0ull;
    __syncthreads();
    uint32_t rank_of = 0, number;
    uint64_t before = 0;
    if (works) before = before_of(f, n, each, rank_of, [&](uint64_t other) { return other < e; });
    if (p.by_k) {
      if (in && rank_of == min(p.k, n) - 1) sh.cut_c = e, sh.cut_q = before + q;
      __syncthreads();
    }
    uint64_t last = sh.cut_c, mass = sh.cut_q;
    if (p.by_p) {
      const uint64_t target = row_target(p.p, mass);
      __syncthreads();
      if (in && before < target && target <= before + q) sh.cut_c = e, sh.cut_q = before + q;
      __syncthreads();
      last = sh.cut_c, mass = sh.cut_q;
    }
    const uint64_t own = in && e <= last && w >= p.least_w ? q : 0;
    if (p.by_w) {
      __syncthreads();
      block_scan(tid % each ? 0 : own, sh.scan_q, mass);
    }
    if (__syncthreads_or(own && own == mass)) {  // one entry is left
      if (own && tid % each == 0) hit(z, (int)(e & (ROW_MAX_COLS - 1)));
      return;
    }
    const uint64_t t = row_draw(p.u, mass);
    if (in) f.input[slot] = own;  // kept masses
    __syncthreads();
    if (!works) return;
    const uint32_t j = (uint32_t)e & (ROW_MAX_COLS - 1);
    before = before_of(f, n, each, number, [&](uint64_t other) { return ((uint32_t)other & (ROW_MAX_COLS - 1)) < j; });
    if (tid % each == 0 && own && before <= t && t < before + own) hit(z, (int)j);
  }

  // Cuts the n entries of f.sorted, those above `edge`, to the first k, then to
  // the shortest prefix of at least p of their mass (without k: of the row's,
  // `total`), then to w >= least_w, and draws, in index order.
  template <typename H>
  __device__ __forceinline__ void finish_listed(RowFinish& f, uint32_t n, float edge, const RowParams& q, uint64_t total, H hit) {
    if (n <= (uint32_t)NT / 2) {
      finish_few(f, n, q, total, hit);
      return;
    }
    float scale = fmaxf((ROW_SORT_BINS - 1) / (m - edge), (ROW_SORT_BINS - 1) / ROW_MASS_END * c);
    if (!(scale <= ROW_F32_MAX)) scale = 0.0f;  // all equal
    uint64_t last = ~0ull;
#pragma unroll 1
    for (int step = q.by_k ? 0 : q.by_p ? 1 : 2; step < 3; step += step == 0 && !q.by_p ? 2 : 1) {
      uint64_t own = 0, all;
#pragma unroll 1
      for (uint32_t i = tid; i < n; i += NT) {
        const uint64_t e = f.sorted[i];
        const float w = weight(value_of(e));
        const uint64_t v = e <= last && (step < 2 || w >= q.least_w) ? row_q(w) : 0;
        own += v;
        f.input[i] = step ? v : 1;
        if (step == 2) f.sorted[i] = (e & (ROW_MAX_COLS - 1)) << 32 | e >> ROW_IDX_BITS;
      }
      block_scan(own, sh.scan_q, all);
      const uint64_t goal = step == 0 ? q.k : step == 1 ? row_target(q.p, q.by_k ? all : total) : row_draw(q.u, all) + 1;
      const uint64_t lo = step < 2 ? (uint64_t)row_key(m) << ROW_IDX_BITS : 0;
      const uint64_t hi = step < 2 ? (uint64_t)row_key(edge) << ROW_IDX_BITS | (ROW_MAX_COLS - 1) : (uint64_t)cols << 32;
      const uint64_t r = reach(f, sh, n, goal, lo, hi, m, step < 2 ? scale : -1.0f);
      if (step < 2)
        last = min(last, r);
      else if (tid == 0)
        hit(row_unkey((uint32_t)r), (int)(r >> 32));
    }
  }

  // (key, index) without the bits that no key of 16-bit logits has: neighbouring
  // values are then as near as their entries are, and one round of bins parts
  // both.  A key's low bits are all 1 or, below 0, all 0.
  static __device__ __forceinline__ uint64_t squeezed(uint64_t e) {
    return e >> (ROW_IDX_BITS + E::ZEROS) << ROW_IDX_BITS | (e & (ROW_MAX_COLS - 1));
  }
  static __device__ __forceinline__ uint64_t unsqueezed(uint64_t s) {
    const uint32_t key = (uint32_t)(s >> ROW_IDX_BITS) << E::ZEROS;
    return (uint64_t)(key >> 31 ? key : key | ((1u << E::ZEROS) - 1)) << ROW_IDX_BITS | (s & (ROW_MAX_COLS - 1));
  }
  // Cuts the n entries in sh.pool, those of [sh.lo, sh.hi], where the prefix of
  // `target` of them (by_mass: of mass `target` with what sh.mass holds) ends, and
  // adds the kept ones' masses to their stretches' in sh.part.  Returns the
  // last entry of the cut.
  __device__ __forceinline__ uint64_t finish_pool(RowFinish& f, uint32_t n, bool by_mass, float least_w, uint64_t target) {
#pragma unroll 1
    for (uint32_t i = tid; i < n; i += NT) {
      f.sorted[i] = squeezed(sh.pool[i]);
      f.input[i] = by_mass ? mass(value_of(sh.pool[i])) : 1;
    }
    const uint64_t end = sh.hi, left = by_mass ? target - handed(sh.mass) : target;
    // the interval's ends lie between values, too: of their own index only 32-bit logits can make use
    const uint64_t any = E::ZEROS ? ROW_MAX_COLS - 1 : 0;
    const uint64_t at = reach(f, sh, n, left, squeezed(sh.lo) & ~any, squeezed(end) | any, m, -1.0f);
    const uint64_t last = at == ~0ull ? end : unsqueezed(at);
    // the warps' kept masses: before the interval, and those of its entries
    if (tid < ROW_SUMS) f.part[tid][0] = f.part[tid][1] = 0;
    __syncthreads();
#pragma unroll 1
    for (uint32_t i = tid; i < n; i += NT) {
      const uint64_t e = sh.pool[i];
      const float w = weight(value_of(e));
      if (e > last || w < least_w) continue;
      const uint32_t v = (((uint32_t)e & (ROW_MAX_COLS - 1)) + lead) / N;
      const uint32_t cta = v / part_vecs, p0 = cta * part_vecs, p1 = min(p0 + part_vecs, total_vecs);
      const uint32_t at = cta * WARPS + (v - p0) / ((p1 - p0 + WARPS - 1) / WARPS);
      const uint64_t kept = row_q(w);
      atomicAdd(&f.part[at][0], (uint32_t)kept & 0xfffffu);
      atomicAdd(&f.part[at][1], (uint32_t)(kept >> 20));
    }
    __syncthreads();
    if (tid < CTAS * WARPS) (&sh.part[0][0])[tid] += ((uint64_t)f.part[tid][1] << 20) + f.part[tid][0];
    __syncthreads();
    return last;
  }

  // Writes the first `have` of f.sorted as the row's best.
  __device__ __forceinline__ void put_best(const RowArgs& a, uint32_t row, const RowFinish& f, uint32_t have, float ln) const {
#pragma unroll 1
    for (int i = tid; i < a.n; i += NT) {
      const bool in = i < (int)have;
      const uint64_t e = in ? f.sorted[i] : 0;
      a.best_idx[(int64_t)row * a.n + i] = in ? (int)(e & (ROW_MAX_COLS - 1)) : -1;
      a.best_logprob[(int64_t)row * a.n + i] = in ? (value_of(e) - m) - ln : -INFINITY;
    }
  }
  __device__ __forceinline__ void put_nothing(const RowArgs& a, uint32_t row) const {
#pragma unroll 1
    for (int i = tid; i < a.n; i += NT)
      a.best_idx[(int64_t)row * a.n + i] = -1, a.best_logprob[(int64_t)row * a.n + i] = -INFINITY;
    if (a.lse && tid == 0) a.lse[row] = -INFINITY;
  }

  // ---- over the row in memory, by one CTA ----
  // Draws among the entries of vectors [v0, v1) up to `last` in (key, index)
  // order, with w >= least_w: the one at which the running mass exceeds t.
  template <typename H>
  __device__ __forceinline__ void scan_memory(uint32_t v0, uint32_t v1, uint64_t t, float least_w, uint64_t last, H hit) {
    const float low = last == ~0ull ? -INFINITY : value_of(last);
    const int low_j = (int)(last & (ROW_MAX_COLS - 1));
    auto value = [&](float z, int j) -> uint64_t {
      const float w = weight(z);
      return w >= least_w && (z > low || (z == low && j <= low_j)) ? row_q(w) : 0;
    };
    const bool takes_equals = last != ~0ull && weight(low) >= least_w;
    constexpr int PER = 2;  // vectors a thread, side by side
#pragma unroll 1
    for (uint32_t i0 = v0; i0 < v1; i0 += NT * PER) {
      const uint32_t i = i0 + tid * PER;
      uint4 v[PER];
#pragma unroll
      for (int k = 0; k < PER; ++k) v[k] = i + k < v1 ? from_memory(i + k) : nothing();
      const int j0 = (int)(i * N) - lead;
      Sum sum(m, c);
#pragma unroll
      for (int k = 0; k < PER; ++k) sum.template add<HEAVY>(v[k], low, least_w);
      uint64_t own = sum.mass(), all;
      if (takes_equals) {
#pragma unroll 1
        for (int k = 0; k < PER; ++k) {
          const uint4 of = k ? v[1] : v[0];
          each_of(hits(of, low, low), of, 0, [&](float z, int e) { own += j0 + k * N + e - first <= low_j ? mass(z) : 0; });
        }
      }
      uint64_t run = block_scan(own, sh.scan_q, all);
      if (t < all) {
        // the thread whose vectors hold the draw: its warp takes an entry a lane
        const uint32_t has = __ballot_sync(~0u, t >= run && t < run + own);
        if (has) {
          const int owner = __ffs((int)has) - 1;
          const uint32_t at = __shfl_sync(~0u, i, owner) + lane / N;
          const float z = E::at(lane < PER * N && at < v1 ? from_memory(at) : nothing(), lane % N);
          const int j = (int)(at * N) - lead + lane % N;
          const uint64_t q = lane < PER * N ? value(z, j) : 0, upto = __shfl_sync(~0u, run, owner) + warp_scan(q, lane);
          if (t < upto && t >= upto - q) hit(z, j);
        }
        return;
      }
      t -= all;
      __syncthreads();
    }
  }
  // The same over the cluster's parts, given the sum of each warp's stretch.
  template <typename H>
  __device__ __forceinline__ void scan_parts(const Sums& of, uint64_t t, float least_w, uint64_t last, H hit) {
    // each warp finds the stretch for itself: lanes hold up to four sums each, in order
    constexpr int PER = (CTAS * WARPS + 31) / 32;
    const uint32_t count = ctas * WARPS;
    uint64_t s[PER], own = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const uint32_t i = lane * PER + k;
      s[k] = i < count ? (&of[0][0])[i] : 0;
      own += s[k];
    }
    uint64_t run = warp_scan(own, lane) - own;
    uint32_t which = 0;
    uint64_t left = t;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      if (t >= run && t < run + s[k]) which = lane * PER + k + 1, left = t - run;
      run += s[k];
    }
    const uint32_t has = __ballot_sync(~0u, which != 0);
    if (!has) return;
    const int owner = __ffs((int)has) - 1;
    which = __shfl_sync(~0u, which, owner) - 1;
    left = __shfl_sync(~0u, left, owner);
    uint32_t v0, v1;
    stretch(which / WARPS, which % WARPS, v0, v1);
    scan_memory(v0, v1, left, least_w, last, hit);
  }
};

// ---- sampling ---------------------------------------------------------------------
// Every CTA of the row: the load with the maximum, then a pass that sums the
// weights and, where a cut is asked for, lists its candidates -- the entries
// above a value that at least top_k of them are known to reach, or, for a
// nucleus, above a guess; the first CTA cuts them and draws.  Without a cut it
// draws from the warps' sums and reads the stretch that holds the drawn entry
// again.
//
// A cut that does not end among the candidates (a nucleus beyond the guess,
// a large top_k, many equal values) keeps the cluster to narrow it down.
//
// Measured (B200, device time): 1 x 32768 f32 9.7 us; 16 x 131072 bf16 of mixed
// parameters 14 to 21 us; 256 x 131072 bf16, nuclei, 66 us (a sixth of the rows
// are narrowed down, and one of those among the last to start makes the tail); 200 x
// 100003 f16 without cuts 27 to 29 us (1.4 TB/s); 64 x 131072 f32 with nuclei of tens
// of thousands 54 us; 512 x 131072 f32 of mixed parameters 114 us (2.4 TB/s).
template <typename T, int NT, bool MEM>
__device__ __forceinline__ void row_sample(const RowArgs& a, uint32_t row, typename Row<T, NT, MEM>::Shared& sh, uint4* data) {
  RowFinish& f = *reinterpret_cast<RowFinish*>(data);
  Row<T, NT, MEM> r(sh, data, a, row, MEM ? 0 : cg::this_cluster().block_rank(), MEM ? 1 : cg::this_cluster().num_blocks(), MEM ? 2 : 1);
  const RowParams q(a, row);
  r.load(q.by_k || q.by_p);
  auto store_nothing = [&] {
    if (r.rank == 0 && r.tid == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = -INFINITY;
    }
  };
  if (r.m == -INFINITY) return store_nothing();
  r.c = q.c();
  const uint32_t k = q.k;
  const float least_w = q.least_w;
  uint64_t total = 0;
  auto store = [&](float z, int j) {
    a.tokens[row] = j;
    if (a.logprobs) a.logprobs[row] = row_neg_y(z, r.m, r.c) * ROW_LN2 - logf((float)total * 0x1p-40f);
  };
  const float edge = q.cuts() ? r.edge_for(q) : q.greedy ? r.m : INFINITY;
  const uint64_t own = r.weigh_and_list(edge, q.greedy);
  uint64_t last = ~0ull;  // the last entry of the cut
  if (!q.cuts()) {
    r.template hand<false>(sh.part, own);
    if (!r.last_part()) return;
    total = r.handed(sh.part);
    if (q.greedy) {
      if (r.tid == 0) store(r.m, (int)sh.first);
      return;
    }
  } else {
    // ---- candidates ----
    r.template hand<true>(sh.mass, own);
    if (edge < INFINITY) {
      r.tell_list();
      if (q.by_p && !q.by_k) {
        uint64_t part = 0;
#pragma unroll 1
        for (uint32_t i = r.tid; i < min(sh.count, r.room); i += NT) part += r.mass(r.value_of(sh.list[i]));
        r.template hand<true>(sh.part, part);
      }
    }
    r.cluster.sync();
    uint32_t n = 0;
    bool enough = false;
    if (edge < INFINITY) {
      enough = r.all_listed(n);
      if (q.by_k && enough && r.rank) return;
    }
    total = r.handed(sh.mass);
    if (enough && !q.by_k && q.by_p) enough = r.handed(sh.part) >= row_target(q.p, total);
    if (enough) {
      if (r.rank) return;
      r.each_listed([&](uint32_t i, uint64_t e) { f.sorted[i] = e; });
      __syncthreads();
      r.finish_listed(f, n, edge, q, total, store);
      return;
    }

    // ---- a cut beyond the candidates ----
    if (q.by_k || q.by_p) {
      typename Row<T, NT, MEM>::Left left{0, 0};
      uint32_t above_n = 0;
      uint64_t mass = total, target = k;
      // the top k, then the nucleus in their mass
#pragma unroll 1
      for (int by_mass = q.by_k ? 0 : 1; by_mass <= (q.by_p ? 1 : 0); ++by_mass) {
        if (by_mass) target = row_target(q.p, mass);
        left = r.narrow(by_mass, target, by_mass ? mass - target : 0, least_w, !by_mass && q.by_p ? ROW_FEW : ROW_POOL);
        if (by_mass || !q.by_p) continue;
        if (!r.rank) {  // the mass of the top k
          const uint64_t above = r.handed(sh.mass);
          r.cluster.barrier_arrive();  // the others' entries
          r.cluster.barrier_wait();
          if (r.tid == 0) sh.cut_q = total - above;
          __syncthreads();
          r.nth_of_few(left.n, k - left.above_n);
          if (r.tid < (int)r.ctas) *r.cluster.map_shared_rank(&sh.cut_q, r.tid) = above + sh.cut_q;
        } else {
          r.cluster.sync();
        }
        r.cluster.sync();
        mass = sh.cut_q;
      }
      if (!q.by_p) above_n = left.above_n;
      if (!r.last_part()) return;
      last = r.finish_pool(f, left.n, q.by_p, least_w, target - above_n);
    } else {  // min_p alone
      const uint64_t kept = r.heavy(-INFINITY, least_w);
      r.cluster.sync();  // every CTA has read the sums before the next ones
      r.template hand<false>(sh.part, kept);
      if (!r.last_part()) return;
    }
    __syncthreads();
  }
  const uint64_t mass = r.handed(sh.part);
  if (mass)
    r.scan_parts(sh.part, row_draw(q.u, mass), least_w, last, store);
  else
    store_nothing();
}

// ---- the n best ---------------------------------------------------------------------
// As a sampling row with top_k = n, whose ordered candidates are the answer.
// Measured (B200, device time): n = 5 of 1 x 32768 f32 8.3 us, n = 20 of 128 x
// 131072 bf16 18.0 us (1.9 TB/s), n = 8 of 1024 x 50021 f32 68 us (3.0 TB/s,
// one streaming CTA a row: two passes, of 16 instructions an entry together, with
// 57% of the issue slots taken and 37% of DRAM's rate).
template <typename T, int NT, bool MEM>
__device__ __forceinline__ void row_best(const RowArgs& a, uint32_t row, typename Row<T, NT, MEM>::Shared& sh, uint4* data) {
  RowFinish& f = *reinterpret_cast<RowFinish*>(data);
  Row<T, NT, MEM> r(sh, data, a, row, MEM ? 0 : cg::this_cluster().block_rank(), MEM ? 1 : cg::this_cluster().num_blocks(), MEM ? 2 : 1);
  r.load(true);
  if (r.m == -INFINITY) {
    if (r.rank == 0) r.put_nothing(a, row);
    return;
  }
  r.c = ROW_LOG2E;
  const uint32_t k = (uint32_t)a.n;
  float edge = r.edge_for_best(k);
  r.template hand<true>(sh.mass, r.weigh_and_list(edge, false));
  r.tell_list();
  r.cluster.sync();
  uint32_t n = 0;
  const bool listed = edge < INFINITY && r.all_listed(n);
  if (listed && r.rank) return;
  const float ln = logf((float)r.handed(sh.mass) * 0x1p-40f);
  const uint64_t* from = f.input;
  if (listed) {
    r.each_listed([&](uint32_t i, uint64_t e) { f.input[i] = e; });
    __syncthreads();
  } else {
    // the n-th entry, then the entries up to it
    const auto left = r.narrow(false, k, 0, 0.0f, ROW_FEW);
    r.cluster.sync();
    if (r.rank == 0) {
      r.nth_of_few(left.n, k - left.above_n);
      if (r.tid > 0 && r.tid < (int)r.ctas) *r.cluster.map_shared_rank(&sh.hi, r.tid) = sh.hi;
    }
    if (r.tid == 0) sh.count = 0;
    r.cluster.sync();
    r.between(r.value_of(sh.hi), r.m, [&](float z, int j) {
      const uint64_t e = (uint64_t)row_key(z) << ROW_IDX_BITS | (uint32_t)j;
      if (e > sh.hi) return;
      const uint32_t at = atomicAdd(&sh.count, 1u);
      if (at < ROW_POOL) sh.pool[at] = e;
    });
    r.tell_pool();
    edge = r.value_of(sh.hi);
    r.cluster.sync();
    n = r.pooled(ROW_POOL);
    from = sh.pool;
    if (!r.last_part()) return;
  }
  if (a.lse && r.tid == 0) a.lse[row] = r.m + ln;
  r.order_by_value(f, from, n, edge);
  r.put_best(a, row, f, min(n, k), ln);
}

// One cluster a row: 256 threads and up to 64 KB of the row a CTA, so that three
// CTAs share an SM and one's barriers hide behind the others' work (512 threads
// a CTA, two on an SM: slower in every phase with a barrier).
constexpr int ROW_CLUSTER_THREADS = 256;
template <typename T, bool BEST> __global__ void __launch_bounds__(ROW_CLUSTER_THREADS, 3) k_row_cluster(const RowArgs a) {
  extern __shared__ __align__(16) unsigned char row_smem[];
  using R = Row<T, ROW_CLUSTER_THREADS, false>;
  static_assert(3 * (R::SHARED_BYTES + (64 << 10) + 1024) <= 228 << 10, "three CTAs on an SM");
  typename R::Shared& sh = *reinterpret_cast<typename R::Shared*>(row_smem);
  uint4* const data = reinterpret_cast<uint4*>(row_smem + R::SHARED_BYTES);
  const uint32_t row = blockIdx.x / cg::this_cluster().num_blocks();
  BEST ? row_best<T, ROW_CLUSTER_THREADS, false>(a, row, sh, data) : row_sample<T, ROW_CLUSTER_THREADS, false>(a, row, sh, data);
}

// One CTA a row, two on an SM, each with 64 KB of loads in flight (of 1024
// threads, one on an SM: 107 us against 70 for n = 8 of 1024 x 50021 f32).
constexpr int ROW_SOLO_THREADS = 512;
template <typename T, bool BEST> __global__ void __launch_bounds__(ROW_SOLO_THREADS, 2) k_row_solo(const RowArgs a) {
  extern __shared__ __align__(16) unsigned char row_smem[];
  using R = Row<T, ROW_SOLO_THREADS, true>;
  typename R::Shared& sh = *reinterpret_cast<typename R::Shared*>(row_smem);
  uint4* const data = reinterpret_cast<uint4*>(row_smem + R::SHARED_BYTES);
  BEST ? row_best<T, ROW_SOLO_THREADS, true>(a, blockIdx.x, sh, data) : row_sample<T, ROW_SOLO_THREADS, true>(a, blockIdx.x, sh, data);
}

}  // namespace fs
