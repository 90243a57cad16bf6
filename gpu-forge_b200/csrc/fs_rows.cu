// fs_rows.cu -- C entries of the row operators over logits (fs_sample_rows,
// fs_top_logprobs); kernels in fs_rows.cuh.
#include "forgesort.h"
#include "fs_internal.h"
#include "fs_rows.cuh"

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

uint32_t row_ctas(uint32_t vecs, uint64_t rows, int sm_count) {
  const uint32_t bytes = vecs * 16;
  uint32_t c = (bytes + PART - 1) / PART;
  while (c < 8 && rows * c * 2 <= (uint64_t)sm_count && bytes / (2 * c) >= PART_MIN) c *= 2;
  return c < ROW_MAX_CLUSTER ? c : ROW_MAX_CLUSTER;
}

template <typename Kern>
int launch(fs_sorter* s, const SorterView& v, Kern kern, std::atomic<bool>* configured, RowArgs& a, int lanes) {
  if (!configured[v.device].load()) {  // idempotent: two threads may both get here
    FS_ROWS_CUDA(s, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)(ROW_SHARED_BYTES + ROW_PART_MAX)));
    FS_ROWS_CUDA(s, cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    configured[v.device].store(true);
  }
  // vectors of a row: with the worst lead of lanes - 1 elements, unless every row begins at a vector
  const int64_t step = a.rows > 1 ? a.stride : 0;
  const bool aligned = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && step % lanes == 0;
  const uint32_t vecs = (a.cols + (aligned ? lanes - 1 : 2 * lanes - 2)) / lanes;
  const uint32_t ctas = row_ctas(vecs, a.rows, v.sm_count);
  a.part_vecs = (vecs + ctas - 1) / ctas;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.rows * ctas);
  cfg.blockDim = dim3(ROW_THREADS);
  const size_t part = (size_t)a.part_vecs * 16;
  cfg.dynamicSmemBytes = ROW_SHARED_BYTES + (part > sizeof(RowFinish) ? part : sizeof(RowFinish));
  cfg.stream = v.stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ctas;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  FS_ROWS_CUDA(s, cudaLaunchKernelEx(&cfg, kern, static_cast<const RowArgs>(a)));
  return FS_OK;
}

template <typename T> int launch_sample(fs_sorter* s, const SorterView& v, RowArgs& a) {
  static std::atomic<bool> configured[SORTER_MAX_DEVICES];
  return launch(s, v, k_row_sample<T>, configured, a, RowElem<T>::N);
}
template <typename T> int launch_best(fs_sorter* s, const SorterView& v, RowArgs& a) {
  static std::atomic<bool> configured[SORTER_MAX_DEVICES];
  return launch(s, v, k_row_best<T>, configured, a, RowElem<T>::N);
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
  rc = dtype == FS_LOGITS_F32   ? launch_sample<float>(s, v, a)
       : dtype == FS_LOGITS_F16 ? launch_sample<__half>(s, v, a)
                                : launch_sample<__nv_bfloat16>(s, v, a);
  return rc ? rc : sorter_finish(s, v, 1, sync);
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
  rc = dtype == FS_LOGITS_F32   ? launch_best<float>(s, v, a)
       : dtype == FS_LOGITS_F16 ? launch_best<__half>(s, v, a)
                                : launch_best<__nv_bfloat16>(s, v, a);
  return rc ? rc : sorter_finish(s, v, 1, sync);
}

}  // extern "C"
