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
// part keeps PART_MIN bytes.  (16 x 131072 bf16: 8 CTAs a row 30 us, 4 CTAs 41 us;
// 256 x 131072 bf16: 4 CTAs 105 us, 8 CTAs 123 us; 512 x 131072 f32: 8 CTAs 153 us,
// 16 CTAs 241 us, when that was tried.)
constexpr uint32_t PART = 64u << 10;
constexpr uint32_t PART_MIN = 16u << 10;

uint32_t row_ctas(uint32_t bytes, uint64_t rows, int sm_count) {
  uint32_t c = (bytes + PART - 1) / PART;
  while (c < 8 && rows * c * 2 <= (uint64_t)sm_count && bytes / (2 * c) >= PART_MIN) c *= 2;
  return c < ROW_MAX_CLUSTER ? c : ROW_MAX_CLUSTER;
}

// 16-byte vectors of a row: with the worst lead, unless every row begins at a
// vector.
uint32_t row_vecs(const RowArgs& a, int lanes) {
  const int64_t step = a.rows > 1 ? a.stride : 0;
  const bool aligned = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && step % lanes == 0;
  return (a.cols + (aligned ? lanes - 1 : 2 * lanes - 2)) / lanes;
}

// Sets, once per device, what a kernel needs beyond the defaults.
template <typename Kern> cudaError_t configure(std::atomic<bool>& done, Kern kern, size_t smem, bool clusters) {
  if (done.load()) return cudaSuccess;  // idempotent: two threads may both get here
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e == cudaSuccess && clusters) e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) done.store(true);
  return e;
}

// One cluster a row.
template <typename T, bool BEST> int launch_clusters(fs_sorter* s, const SorterView& v, RowArgs& a) {
  using R = Row<T, ROW_CLUSTER_THREADS, false>;
  static std::atomic<bool> configured[SORTER_MAX_DEVICES];
  FS_ROWS_CUDA(s, configure(configured[v.device], k_row_cluster<T, BEST>, R::SHARED_BYTES + ROW_PART_MAX, true));
  const uint32_t vecs = row_vecs(a, RowElem<T>::N), ctas = row_ctas(vecs * 16, a.rows, v.sm_count);
  a.part_vecs = (vecs + ctas - 1) / ctas;
  const size_t part = (size_t)a.part_vecs * 16;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.rows * ctas);
  cfg.blockDim = dim3(ROW_CLUSTER_THREADS);
  cfg.dynamicSmemBytes = R::SHARED_BYTES + (part > sizeof(RowFinish) ? part : sizeof(RowFinish));
  cfg.stream = v.stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ctas;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  FS_ROWS_CUDA(s, cudaLaunchKernelEx(&cfg, k_row_cluster<T, BEST>, static_cast<const RowArgs>(a)));
  return FS_OK;
}

// One CTA a row.
template <typename T, bool BEST> int launch_solo(fs_sorter* s, const SorterView& v, RowArgs& a) {
  using R = Row<T, ROW_SOLO_THREADS, true>;
  static_assert(sizeof(RowFinish) <= R::RING_BYTES, "fits");
  constexpr size_t smem = R::SHARED_BYTES + R::RING_BYTES;
  static std::atomic<bool> configured[SORTER_MAX_DEVICES];
  FS_ROWS_CUDA(s, configure(configured[v.device], k_row_solo<T, BEST>, smem, false));
  a.part_vecs = row_vecs(a, RowElem<T>::N);
  k_row_solo<T, BEST><<<a.rows, ROW_SOLO_THREADS, smem, v.stream>>>(a);
  FS_ROWS_CUDA(s, cudaGetLastError());
  return FS_OK;
}

// A cluster a row, or one CTA that streams it.  While one wave of clusters
// takes the batch, clusters: they read a row once and several CTAs share its
// work (16 rows of 128256 bf16, n = 20: 10.4 us against 17.9; 96 rows: 16.0
// against 18.6).  Beyond, a streaming CTA has no partners to wait for (148 rows:
// 18.6 us against 24.7; 1024 rows: 92 against 111; 1024 x 128256 f32: 151
// against 184), though it loses where its rows fill the SMs one and a bit times
// (160 rows: 28.8 against 25.1; 200 x 100003 f16 without cuts: 26.8 against
// 25.4); not for rows of a single part (512 x 32000 bf16: 26.8 us against
// 21.7).  Nor for nuclei: a row whose cut lies far down takes several times as
// long as the rest of the batch, and less so on several CTAs (256 x 131072 bf16
// peaked rows, a sixth of them such: 66 us by clusters, 104 streaming; 512
// x 131072 f32, a twentieth of them, 112 and 144.  Where all rows are such, clusters
// lose in 32 bits: 256 x 128256 bf16 106 and 115 us, 512 x 128256 f32 279 and
// 242).  Whether there are nuclei is told by top_p being passed: its numbers are
// on the device, so a batch of ones takes clusters, too.
template <typename T, bool BEST> int launch(fs_sorter* s, const SorterView& v, RowArgs& a) {
  const uint32_t ctas = row_ctas(row_vecs(a, RowElem<T>::N) * 16, a.rows, v.sm_count);
  const bool streams = !a.top_p && ctas > 1 && (uint64_t)ctas * a.rows > 3ull * v.sm_count;
  return (v.row_form ? v.row_form == 2 : streams) ? launch_solo<T, BEST>(s, v, a) : launch_clusters<T, BEST>(s, v, a);
}

template <bool BEST> int launch_rows(fs_sorter* s, const SorterView& v, int dtype, RowArgs& a, int sync) {
  const int rc = dtype == FS_LOGITS_F32   ? launch<float, BEST>(s, v, a)
                 : dtype == FS_LOGITS_F16 ? launch<__half, BEST>(s, v, a)
                                          : launch<__nv_bfloat16, BEST>(s, v, a);
  return rc ? rc : sorter_finish(s, v, 1, sync, false);
}

int check_rows(fs_sorter* s, int dtype, const void* logits, uint64_t rows, uint64_t cols, int64_t stride) {
  if (dtype < FS_LOGITS_F32 || dtype > FS_LOGITS_BF16) return sorter_fail(s, FS_E_INVALID, "unknown logits dtype %d", dtype);
  if (cols == 0 || cols > ROW_MAX_COLS)
    return sorter_fail(s, FS_E_INVALID, "cols = %llu outside [1, %u]", (unsigned long long)cols, ROW_MAX_COLS);
  if (rows > (1u << 26)) return sorter_fail(s, FS_E_INVALID, "rows = %llu exceeds 2^26", (unsigned long long)rows);
  if (rows > 1 && stride < 0)
    return sorter_fail(s, FS_E_INVALID, "row stride %lld is negative", (long long)stride);
  if (!logits) return sorter_fail(s, FS_E_INVALID, "logits is NULL");
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
  if ((rc = sorter_check(s, logits, span, elem_bytes(dtype), "logits"))) return rc;
  const struct { const void* p; size_t bytes; const char* what; } ptrs[] = {
      {uniform, rows * 4, "uniform"}, {tokens, rows * 4, "tokens"},
      {temperature, rows * 4, "temperature"}, {top_k, rows * 4, "top_k"}, {top_p, rows * 4, "top_p"},
      {min_p, rows * 4, "min_p"},        {logprobs, rows * 4, "logprobs"}};
  for (const auto& q : ptrs)
    if (q.p && (rc = sorter_check(s, q.p, q.bytes, 4, q.what))) return rc;
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
  if ((rc = sorter_check(s, logits, span, elem_bytes(dtype), "logits")) ||
      (rc = sorter_check(s, indices, rows * n * 4, 4, "indices")) ||
      (rc = sorter_check(s, logprobs, rows * n * 4, 4, "logprobs")) ||
      (lse && (rc = sorter_check(s, lse, rows * 4, 4, "lse"))))
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
