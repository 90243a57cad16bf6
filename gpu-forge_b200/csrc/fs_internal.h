// fs_internal.h -- what the serving operators (fs_rows.cu, fs_slots.cu) use of
// a sorter: its device, stream, error text and device error word.
// Defined in fs_sort.cu; not part of the C ABI.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

#include "forgesort.h"

namespace fs {

struct SorterView {
  int device;
  int sm_count;
  cudaStream_t stream;
  int* host_err;  // device alias of the mapped error word (DEV_ERR_*)
  int row_form;   // FORGESORT_ROW_FORM: 0 by size, 1 a cluster a row, 2 a CTA a row
};

// Makes the sorter's device current and fills *v; stream NULL: the sorter's.
int sorter_view(fs_sorter* s, void* stream, SorterView* v);
// Records a failure's text on the sorter; returns `code`.
int sorter_fail(fs_sorter* s, int code, const char* fmt, ...) __attribute__((format(printf, 3, 4)));
int sorter_cuda_fail(fs_sorter* s, cudaError_t e, const char* what);
// Checks that p is device or managed memory of the sorter's device, as the
// device-resident sorts do, and aligned to its elements of `align` bytes.
int sorter_check(fs_sorter* s, const void* p, size_t bytes, size_t align, const char* what);
// Ends a call that enqueued `launches` kernels on v.stream: waits and reports
// device-side failures when sync != 0.  may_fail: they use v.host_err, so
// fs_synchronize and fs_destroy wait for them.
int sorter_finish(fs_sorter* s, const SorterView& v, int launches, int sync, bool may_fail);

// Device ordinals that per-device caches cover (fs_create refuses more).
constexpr int SORTER_MAX_DEVICES = 64;

}  // namespace fs
