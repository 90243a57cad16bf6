// fs_rows.cu -- C entries of the row operators over logits (fs_sample_rows,
// fs_top_logprobs); kernels in fs_rows.cuh.
#include "forgesort.h"
#include "fs_internal.h"
#include "fs_rows.cuh"
#include "fs_rows_stream.cuh"

#include <atomic>

using namespace fs;

namespace {

// Shared-memory bytes of row data a CTA may hold: a row of 2^19 32-bit logits over 16 CTAs.
constexpr uint32_t ROW_PART_MAX = 132u << 10;

#define FS_ROWS_CUDA(s, call)                                        \
  do {                                                               \
    cudaError_t e_ = (call);                                         \
    if (e_ != cudaSuccess) return sorter_cuda_fail((s), e_, #call);  \
  } while (0)

size_t elem_bytes(int dtype) { return dtype == FS_LOGITS_F32 ? 4 : 2; }

// CTAs per row: as many as cut it into parts of PART bytes, of which three fit
// an SM, and more while the batch has fewer CTAs than the GPU has SMs and a
// part keeps PART_MIN bytes.
#ifndef VPART
#define VPART 64
#endif
constexpr uint32_t PART = VPART << 10;
constexpr uint32_t PART_MIN = 16u << 10;
// Large batches go in passes over all rows, in groups of STREAM_ROWS rows
// (of 25 KB of scratch each), cut into parts of STREAM_PART bytes.
#ifndef VSPART
#define VSPART 16
#endif
constexpr uint64_t STREAM_ROWS = 1024;
#ifndef VCTAS
#define VCTAS 5
#endif
constexpr uint32_t STREAM_CTAS = VCTAS;  // CTAs an SM
constexpr uint32_t STREAM_PART = VSPART << 10;

uint32_t row_ctas(uint32_t vecs, uint64_t rows, int sm_count) {
  const uint32_t bytes = vecs * 16;
  uint32_t c = (bytes + PART - 1) / PART;
  while (c < 8 && rows * c * 2 <= (uint64_t)sm_count && bytes / (2 * c) >= PART_MIN) c *= 2;
  return c < ROW_MAX_CLUSTER ? c : ROW_MAX_CLUSTER;
}

// A launch behind the call's previous one (fs_rows_stream.cuh), scheduled
// while that one drains; every such kernel waits for it first.
template <typename Kern, typename... Args>
cudaError_t chained(const SorterView& v, Kern kern, unsigned grid, size_t smem, uint32_t cluster, const Args&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(ROW_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = v.stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = cluster;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

// 16-byte vectors of a row: with the worst lead, unless every row begins at a
// vector.
uint32_t row_vecs(const RowArgs& a, int lanes) {
  const int64_t step = a.rows > 1 ? a.stride : 0;
  const bool aligned = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && step % lanes == 0;
  return (a.cols + (aligned ? lanes - 1 : 2 * lanes - 2)) / lanes;
}
size_t cluster_smem(uint32_t part_vecs) {
  const size_t part = (size_t)part_vecs * 16;
  return ROW_SHARED_BYTES + (part > sizeof(RowFinish) ? part : sizeof(RowFinish));
}
// The passes' shared memory: the copies in flight, which the last CTA's working memory lies over.
constexpr size_t RING_SMEM = ROW_SHARED_BYTES + sizeof(RowRing);
static_assert(sizeof(RowFinish) <= sizeof(RowRing) && sizeof(RowWide) <= sizeof(RowRing) && RING_SMEM <= 48 << 10, "fits");

// Small batches: one cluster a row.
template <typename T, bool BEST> int launch_clusters(fs_sorter* s, const SorterView& v, RowArgs& a, int* launches) {
  const uint32_t vecs = row_vecs(a, RowElem<T>::N), ctas = row_ctas(vecs, a.rows, v.sm_count);
  a.part_vecs = (vecs + ctas - 1) / ctas;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.rows * ctas);
  cfg.blockDim = dim3(ROW_THREADS);
  cfg.dynamicSmemBytes = cluster_smem(a.part_vecs);
  cfg.stream = v.stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ctas;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  FS_ROWS_CUDA(s, cudaLaunchKernelEx(&cfg, k_rows<T, BEST>, static_cast<const RowArgs>(a)));
  *launches += 1;
  return FS_OK;
}

// Large batches: passes over all rows, with scratch from the stream-ordered
// allocator, so that a call keeps nothing and may be captured.
template <typename T, bool BEST> int launch_passes(fs_sorter* s, const SorterView& v, RowArgs& a, int* launches) {
  const uint32_t vecs = row_vecs(a, RowElem<T>::N);
  RowStream st{};
  // as many parts as fill the GPU once, of at least STREAM_PART bytes
  st.parts = (uint32_t)v.sm_count * STREAM_CTAS / a.rows;
  if (st.parts > vecs * 16 / STREAM_PART) st.parts = vecs * 16 / STREAM_PART;
  if (st.parts > ROW_MAX_CLUSTER) st.parts = ROW_MAX_CLUSTER;
  if (st.parts < 1) st.parts = 1;
  a.part_vecs = (vecs + st.parts - 1) / st.parts;
  const bool narrows = !BEST && a.top_p;  // rows may have wide nuclei
  size_t bytes = 0;
  auto take = [&](size_t n) {
    const size_t at = bytes;
    bytes += (n + 255) / 256 * 256;
    return at;
  };
  const size_t R = a.rows;
  const size_t o_rec = take(R * sizeof(RowRecord)), o_counts = take(8), zeroed = bytes;
  const size_t o_tops = take(R * ROW_TOPS * 4), o_mass = take(R * ROW_SUMS * 8), o_list = take(R * ROW_LIST * 8), o_left = take(R * 4);
  const size_t o_wide = take(narrows ? R * 4 : 0), o_part = take(narrows ? R * ROW_SUMS * 8 : 0);
  const size_t o_bins = take(narrows ? R * ROW_BINS * 4 : 0), o_pool = take(narrows ? R * ROW_WIDE_POOL * 8 : 0);
  void* mem = nullptr;
  FS_ROWS_CUDA(s, cudaMallocFromPoolAsync(&mem, bytes, v.pool, v.stream));
  unsigned char* const b = static_cast<unsigned char*>(mem);
  st.rec = reinterpret_cast<RowRecord*>(b + o_rec);
  st.counts = reinterpret_cast<uint32_t*>(b + o_counts);
  st.tops = reinterpret_cast<uint32_t*>(b + o_tops);
  st.mass = reinterpret_cast<uint64_t*>(b + o_mass);
  st.list = reinterpret_cast<uint64_t*>(b + o_list);
  st.left = reinterpret_cast<uint32_t*>(b + o_left);
  st.wide = reinterpret_cast<uint32_t*>(b + o_wide);
  st.part = reinterpret_cast<uint64_t*>(b + o_part);
  st.bins = reinterpret_cast<uint32_t*>(b + o_bins);
  st.pool = reinterpret_cast<uint64_t*>(b + o_pool);
  const RowArgs args = a;
  const unsigned grid = a.rows * st.parts;
  cudaError_t e = cudaMemsetAsync(mem, 0, zeroed, v.stream);
  if (e == cudaSuccess) {
    k_stream_max<T, BEST><<<grid, ROW_THREADS, RING_SMEM, v.stream>>>(args, st);
    e = cudaGetLastError();
  }
  if (e == cudaSuccess) e = chained(v, k_stream_weigh<T, BEST>, grid, RING_SMEM, 0, args, st);
  if constexpr (!BEST) {
    if (narrows) {
      const unsigned most = (unsigned)v.sm_count * 3, few = grid < most ? grid : most;
      if (e == cudaSuccess) e = chained(v, k_stream_bins<T>, few, RING_SMEM, 0, args, st);
      if (e == cudaSuccess) e = chained(v, k_stream_cut<T>, few, RING_SMEM, 0, args, st);
      *launches += 2;
    }
  }
  if (e == cudaSuccess && (BEST || a.top_k || a.top_p || a.min_p)) {
    RowArgs left = a;
    left.only = st.left;
    left.only_n = st.counts + 1;
    const uint32_t ctas = row_ctas(vecs, 1, v.sm_count), most = (uint32_t)v.sm_count / ctas;
    left.part_vecs = (vecs + ctas - 1) / ctas;
    e = chained(v, k_rows<T, BEST>, (a.rows < most ? a.rows : most) * ctas, cluster_smem(left.part_vecs), ctas,
                static_cast<const RowArgs>(left));
    *launches += 1;
  }
  *launches += 2;
  const cudaError_t freed = cudaFreeAsync(mem, v.stream);
  FS_ROWS_CUDA(s, e);
  FS_ROWS_CUDA(s, freed);
  return FS_OK;
}

template <typename T, bool BEST> int launch(fs_sorter* s, const SorterView& v, RowArgs a, int* launches) {
  static std::atomic<bool> configured[SORTER_MAX_DEVICES];
  if (!configured[v.device].load()) {  // idempotent: two threads may both get here
    FS_ROWS_CUDA(s, cudaFuncSetAttribute(k_rows<T, BEST>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)(ROW_SHARED_BYTES + ROW_PART_MAX)));
    FS_ROWS_CUDA(s, cudaFuncSetAttribute(k_rows<T, BEST>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    configured[v.device].store(true);
  }
  const uint64_t total = a.rows;
  if (total * a.cols * sizeof(T) < v.row_pass_min) return launch_clusters<T, BEST>(s, v, a, launches);
  for (uint64_t r = 0; r < total; r += STREAM_ROWS) {
    RowArgs g = a;
    g.rows = (uint32_t)(total - r < STREAM_ROWS ? total - r : STREAM_ROWS);
    g.x = static_cast<const T*>(a.x) + (int64_t)r * a.stride;
    if constexpr (BEST) {
      g.best_idx = a.best_idx + r * a.n;
      g.best_logprob = a.best_logprob + r * a.n;
      g.lse = a.lse ? a.lse + r : nullptr;
    } else {
      g.temperature = a.temperature ? a.temperature + r : nullptr;
      g.top_k = a.top_k ? a.top_k + r : nullptr;
      g.top_p = a.top_p ? a.top_p + r : nullptr;
      g.min_p = a.min_p ? a.min_p + r : nullptr;
      g.uniform = a.uniform + r;
      g.tokens = a.tokens + r;
      g.logprobs = a.logprobs ? a.logprobs + r : nullptr;
    }
    const int rc = launch_passes<T, BEST>(s, v, g, launches);
    if (rc) return rc;
  }
  return FS_OK;
}

template <bool BEST> int launch_rows(fs_sorter* s, const SorterView& v, int dtype, const RowArgs& a, int sync) {
  int launches = 0;
  const int rc = dtype == FS_LOGITS_F32   ? launch<float, BEST>(s, v, a, &launches)
                 : dtype == FS_LOGITS_F16 ? launch<__half, BEST>(s, v, a, &launches)
                                          : launch<__nv_bfloat16, BEST>(s, v, a, &launches);
  return rc ? rc : sorter_finish(s, v, launches, sync);
}

int check_rows(fs_sorter* s, int dtype, const void* logits, uint64_t rows, uint64_t cols, int64_t stride) {
  if (dtype < FS_LOGITS_F32 || dtype > FS_LOGITS_BF16) return sorter_fail(s, FS_E_INVALID, "unknown logits dtype %d", dtype);
  if (cols == 0 || cols > ROW_MAX_COLS)
    return sorter_fail(s, FS_E_INVALID, "cols = %llu outside [1, %u]", (unsigned long long)cols, ROW_MAX_COLS);
  if (rows > (1u << 26)) return sorter_fail(s, FS_E_INVALID, "rows = %llu exceeds 2^26", (unsigned long long)rows);
  if (rows > 1 && stride < 0)
    return sorter_fail(s, FS_E_INVALID, "row stride %lld is negative", (long long)stride);
  if (!logits) return sorter_fail(s, FS_E_INVALID, "logits is NULL");
  if (reinterpret_cast<uintptr_t>(logits) % elem_bytes(dtype))
    return sorter_fail(s, FS_E_INVALID, "logits is not aligned to its elements");
  return FS_OK;
}

}  // namespace

extern "C" {

int fs_sample_rows(fs_sorter* s, int dtype, const void* logits, uint64_t rows, uint64_t cols, int64_t row_stride,
                   const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                   const float* uniform, int32_t* tokens, float* logprobs, int sync, void* stream) {
  if (!s) return FS_E_INVALID;
  if (rows == 0) return FS_OK;
  int rc = check_rows(s, dtype, logits, rows, cols, row_stride);
  if (rc) return rc;
  if (!uniform || !tokens) return sorter_fail(s, FS_E_INVALID, "uniform or tokens is NULL");
  SorterView v;
  if ((rc = sorter_view(s, stream, &v))) return rc;
  const size_t span = ((size_t)(rows - 1) * row_stride + cols) * elem_bytes(dtype);
  const struct { const void* p; size_t bytes; const char* what; } ptrs[] = {
      {logits, span, "logits"},          {uniform, rows * 4, "uniform"}, {tokens, rows * 4, "tokens"},
      {temperature, rows * 4, "temperature"}, {top_k, rows * 4, "top_k"}, {top_p, rows * 4, "top_p"},
      {min_p, rows * 4, "min_p"},        {logprobs, rows * 4, "logprobs"}};
  for (const auto& q : ptrs)
    if (q.p && (rc = sorter_check(s, q.p, q.bytes, q.what))) return rc;
  RowArgs a{};
  a.x = logits;
  a.stride = row_stride;
  a.rows = (uint32_t)rows;
  a.cols = (uint32_t)cols;
  a.temperature = temperature;
  a.top_k = top_k;
  a.top_p = top_p;
  a.min_p = min_p;
  a.uniform = uniform;
  a.tokens = tokens;
  a.logprobs = logprobs;
  return launch_rows<false>(s, v, dtype, a, sync);
}

int fs_top_logprobs(fs_sorter* s, int dtype, const void* logits, uint64_t rows, uint64_t cols, int64_t row_stride,
                    int n, int32_t* indices, float* logprobs, float* lse, int sync, void* stream) {
  if (!s) return FS_E_INVALID;
  if (rows == 0) return FS_OK;
  int rc = check_rows(s, dtype, logits, rows, cols, row_stride);
  if (rc) return rc;
  if (n < 1 || n > ROW_BEST_MAX) return sorter_fail(s, FS_E_INVALID, "n = %d outside [1, %d]", n, ROW_BEST_MAX);
  if (!indices || !logprobs) return sorter_fail(s, FS_E_INVALID, "indices or logprobs is NULL");
  SorterView v;
  if ((rc = sorter_view(s, stream, &v))) return rc;
  const size_t span = ((size_t)(rows - 1) * row_stride + cols) * elem_bytes(dtype);
  if ((rc = sorter_check(s, logits, span, "logits")) || (rc = sorter_check(s, indices, rows * n * 4, "indices")) ||
      (rc = sorter_check(s, logprobs, rows * n * 4, "logprobs")) || (lse && (rc = sorter_check(s, lse, rows * 4, "lse"))))
    return rc;
  RowArgs a{};
  a.x = logits;
  a.stride = row_stride;
  a.rows = (uint32_t)rows;
  a.cols = (uint32_t)cols;
  a.n = n;
  a.best_idx = indices;
  a.best_logprob = logprobs;
  a.lse = lse;
  return launch_rows<true>(s, v, dtype, a, sync);
}

}  // extern "C"
