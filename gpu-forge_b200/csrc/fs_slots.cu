// fs_slots.cu -- block tables and slot maps of a batch's step over a paged
// cache, from the requests' lengths (fs_plan_slots).
//
// With ctx_r tokens of request r in the cache, new_r to come and pages of P
// tokens, request r holds have_r = ceil(ctx_r / P) pages and needs
// need_r = ceil((ctx_r + new_r) / P).  Two exclusive sums over the requests
// -- of new_r (where its tokens start in the step) and of need_r - have_r
// (where its pages start in the list of free pages) -- decide everything
// else token by token: token i belongs to the request whose range holds i,
// its position is ctx_r + i - start_r, and its page is an entry of the
// request's row of the block table if it is one of the have_r, else the next
// free page, which the page's first token also writes into the table.
#include "forgesort.h"
#include "fs_device.cuh"
#include "fs_internal.h"

using namespace fs;

namespace {

#define FS_SLOTS_CUDA(s, call)                                       \
  do {                                                               \
    cudaError_t e_ = (call);                                         \
    if (e_ != cudaSuccess) return sorter_cuda_fail((s), e_, #call);  \
  } while (0)

struct SlotArgs {
  const void* ctx;
  const void* neu;
  uint32_t requests;
  uint32_t page;
  uint64_t page_part;  // (2^64 - 1) / page
  int32_t* table;
  uint32_t width;
  int64_t table_stride;
  const int32_t* free_pages;
  uint64_t n_free;
  const int32_t* cursor;
  int32_t* query_start;
  void* seq_lens;
  void* positions;
  int32_t* request_of;
  int64_t* slots;
  uint64_t capacity;
  int32_t* cursor_out;
  int* host_err;
  bool wide;  // positions, request_of and slots begin at 16-byte boundaries
};

template <typename I> __device__ __forceinline__ int64_t length_of(const void* p, uint32_t r) {
  const int64_t v = static_cast<const I*>(p)[r];
  return v > 0 ? v : 0;
}
template <typename I> __device__ __forceinline__ constexpr int64_t longest() {
  return sizeof(I) == 4 ? 0x7fffffffll : 0x7fffffffffffffffll;
}
// tokens / page and what is left: the product with
// the page's reciprocal, which is at most one too small.  (The code of a step
// runs once, from cold: a 64-bit division is an order of magnitude longer.)
__device__ __forceinline__ uint64_t div_page(uint64_t tokens, const SlotArgs& a, uint64_t& left) {
  uint64_t n = __umul64hi(tokens, a.page_part);
  left = tokens - n * a.page;
  if (left >= a.page) ++n, left -= a.page;
  return n;
}
__device__ __forceinline__ int64_t pages_of(int64_t tokens, const SlotArgs& a) {
  uint64_t left;
  const uint64_t n = div_page((uint64_t)tokens, a, left);
  return (int64_t)min(n + (left != 0), (uint64_t)a.width);
}

constexpr int SLOT_THREADS = 512;
constexpr int SLOT_CHUNK = 4 * SLOT_THREADS;  // requests scanned at a time
constexpr int64_t MOST_TOKENS = 0x7fffffff;   // query_start is of 32 bits

// Sums of two numbers over the lanes up to each.
__device__ __forceinline__ void warp_scan(int64_t& x, int64_t& y, int lane) {
#pragma unroll 1
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t ox = __shfl_up_sync(~0u, x, d), oy = __shfl_up_sync(~0u, y, d);
    if (lane >= d) x += ox, y += oy;
  }
}
// Exclusive sums of two numbers over the block.
__device__ __forceinline__ void block_scan(int64_t& x, int64_t& y, int64_t (*warp)[2], int64_t& all_x, int64_t& all_y) {
  constexpr int WARPS = SLOT_THREADS / 32;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int64_t x0 = x, y0 = y;
  warp_scan(x, y, lane);
  if (lane == 31) warp[wid][0] = x, warp[wid][1] = y;
  __syncthreads();
  int64_t wx = lane < WARPS ? warp[lane][0] : 0, wy = lane < WARPS ? warp[lane][1] : 0;
  const int64_t ox = wx, oy = wy;
  warp_scan(wx, wy, lane);
  all_x = __shfl_sync(~0u, wx, 31), all_y = __shfl_sync(~0u, wy, 31);
  x += __shfl_sync(~0u, wx - ox, wid) - x0;
  y += __shfl_sync(~0u, wy - oy, wid) - y0;
}

// Every CTA takes both sums over all requests, SLOT_CHUNK of them at a time,
// and plans the tokens of its own tiles of SLOT_THREADS x TOK tokens that belong to
// the chunk; the first CTA writes what is one per request.  The sums are taken
// again by each CTA (two numbers per request from L2) instead of handed on:
// one launch, no scratch, nobody waits.  A thread plans TOK neighbouring
// tokens: it looks its request up once and writes 16 bytes at a time.  TOK is 4
// in steps of more tokens than an SM has threads for (2^20 tokens: 14.7 us, one
// token a thread 18.5), else 1 (4096 tokens: 10.3 us, four 12.4).
//
// Bound: the writes of a large step (21 MB for 2^20 prompt tokens with 64-bit
// positions, 3.2 us), else the chain load - scan - search - page - store of one CTA.
// Measured (B200, device time): 32 decoding requests 6.2 us, 4096 10.3 us (two
// chunks of requests one after the other), 2^20 tokens of 512 prompts 14.7 us
// (20.5 us with one token a thread and 64-bit divisions).
template <typename I, int TOK> __device__ __forceinline__ void put(I* to, const I (&v)[TOK]) {
  constexpr int PER = 16 / sizeof(I) < TOK ? 16 / sizeof(I) : TOK;
#pragma unroll
  for (int k = 0; k < TOK; k += PER) {
    union { I e[PER]; uint4 v; } u;
#pragma unroll
    for (int e = 0; e < PER; ++e) u.e[e] = v[k + e];
    *reinterpret_cast<uint4*>(to + k) = u.v;
  }
}
template <typename I, int TOK> __global__ void __launch_bounds__(SLOT_THREADS) k_plan_slots(const SlotArgs a) {
  __shared__ int64_t warp[SLOT_THREADS / 32][2];
  __shared__ int32_t start[SLOT_CHUNK + 1];  // of the chunk's requests
  __shared__ int32_t took[SLOT_CHUNK];       // pages of those before, at most 2^31 - 1: there are no more free ones
  const int tid = threadIdx.x;
  const int64_t cursor = a.cursor[0] > 0 ? a.cursor[0] : 0;
  int64_t tokens = 0, pages = 0;  // of the chunks before
  bool missed = false;
  for (uint32_t r0 = 0; r0 < a.requests; r0 += SLOT_CHUNK) {
    const int n = (int)min((uint32_t)SLOT_CHUNK, a.requests - r0);
    constexpr int PER = SLOT_CHUNK / SLOT_THREADS;
    int64_t t = 0, p = 0, neu[PER], more[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int l = tid * PER + k;
      neu[k] = more[k] = 0;
      if (l < n) {
        const int64_t ctx = length_of<I>(a.ctx, r0 + l);
        neu[k] = length_of<I>(a.neu, r0 + l);
        // no length passes its type's largest number, and no sum of 2^24 of them 64 bits
        const uint64_t sum = (uint64_t)ctx + (uint64_t)neu[k];
        const int64_t len = (int64_t)min(sum, (uint64_t)longest<I>());
        if (sum > (uint64_t)longest<I>()) neu[k] = longest<I>() - ctx, missed = true;
        neu[k] = min(neu[k], MOST_TOKENS);
        more[k] = pages_of(len, a) - pages_of(ctx, a);
        if (blockIdx.x == 0) static_cast<I*>(a.seq_lens)[r0 + l] = (I)len;
      }
      t += neu[k], p += more[k];
    }
    int64_t all_t, all_p;
    block_scan(t, p, warp, all_t, all_p);
    t += tokens, p += pages;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int l = tid * PER + k;
      if (l < n) {
        start[l] = (int32_t)min(t, MOST_TOKENS);
        took[l] = (int32_t)min(p, MOST_TOKENS);
        if (blockIdx.x == 0) a.query_start[r0 + l] = start[l];
      }
      t += neu[k], p += more[k];
    }
    const uint32_t from = (uint32_t)min(tokens, MOST_TOKENS), to = (uint32_t)min(tokens + all_t, MOST_TOKENS);
    tokens += all_t, pages += all_p;
    __syncthreads();
    // the first of this CTA's tiles that reaches into [from, to)
    constexpr int TILE = SLOT_THREADS * TOK;
    uint32_t tile = from / TILE;
    const uint32_t at = tile % gridDim.x;
    tile += blockIdx.x >= at ? blockIdx.x - at : gridDim.x - at + blockIdx.x;
#pragma unroll 1
    for (uint32_t i0 = tile * TILE + tid * TOK; i0 - tid * TOK < to; i0 += gridDim.x * TILE) {
      const uint32_t i1 = max(i0, from), i2 = min(i0 + TOK, to);
      if (i1 >= i2) continue;
      int lo = 0, hi = n;  // the chunk's last request that starts at or before i1
#pragma unroll 1
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if ((uint32_t)start[mid] <= i1)
          lo = mid;
        else
          hi = mid;
      }
      int32_t request[TOK];
      I position[TOK];
      int64_t slot[TOK];
      uint64_t pos = 0, nth = 0, off = 0, have = 0;
      int32_t* row = nullptr;
      int32_t id = -1;
      bool look = true;  // the request is a new one
#pragma unroll
      for (int k = 0; k < TOK; ++k) {
        const uint32_t i = i0 + k;
        if (i < i1 || i >= i2) continue;
#pragma unroll 1
        while (lo + 1 < n && (uint32_t)start[lo + 1] <= i) ++lo, look = true;
        bool turn = look;  // the page is another one
        if (look) {
          const int64_t ctx = length_of<I>(a.ctx, r0 + lo);
          pos = (uint64_t)ctx + (i - (uint32_t)start[lo]);
          nth = div_page(pos, a, off);
          have = (uint64_t)pages_of(ctx, a);
          row = a.table + (int64_t)(r0 + lo) * a.table_stride;
          look = false;
        } else {
          ++pos;
          if (++off == a.page) ++nth, off = 0, turn = true;
        }
        if (turn) {
          id = -1;
          if (nth < have) {
            id = row[nth];
          } else if (nth < a.width) {
            const uint64_t f = (uint64_t)cursor + (uint32_t)took[lo] + nth - have;
            if (f < a.n_free) id = a.free_pages[f];
            if (off == 0) row[nth] = id;
          }
        }
        missed |= id < 0 || i >= a.capacity;
        request[k] = (int32_t)(r0 + lo);
        position[k] = (I)pos;
        slot[k] = id < 0 ? -1 : (int64_t)id * a.page + (int64_t)off;
      }
      if (TOK > 1 && a.wide && i2 - i1 == TOK && i2 <= a.capacity) {
        put(a.request_of + i0, request);
        put(static_cast<I*>(a.positions) + i0, position);
        put(a.slots + i0, slot);
      } else {
#pragma unroll
        for (int k = 0; k < TOK; ++k) {
          const uint32_t i = i0 + k;
          if (i < i1 || i >= i2 || i >= a.capacity) continue;
          a.request_of[i] = request[k];
          static_cast<I*>(a.positions)[i] = position[k];
          a.slots[i] = slot[k];
        }
      }
    }
    __syncthreads();
  }
  const int64_t end = min(tokens, MOST_TOKENS);
  for (int64_t i = end + (int64_t)blockIdx.x * SLOT_THREADS + tid; i < (int64_t)a.capacity;
       i += (int64_t)gridDim.x * SLOT_THREADS) {
    a.request_of[i] = -1;
    static_cast<I*>(a.positions)[i] = 0;
    a.slots[i] = -1;
  }
  if (blockIdx.x == 0 && tid == 0) {
    a.query_start[a.requests] = (int32_t)end;
    a.cursor_out[0] = (int32_t)min(cursor + pages, (int64_t)a.n_free);
    if (tokens > end) missed = true;
  }
  if (missed) *a.host_err = DEV_ERR_PAGES;
}

template <typename I, int TOK> int launch_tokens(fs_sorter* s, const SorterView& v, const SlotArgs& a) {
  constexpr uint64_t TILE = SLOT_THREADS * TOK;
  const uint64_t tiles = (a.capacity + TILE - 1) / TILE, cap = (uint64_t)v.sm_count * 2;  // as many as run at a time
  k_plan_slots<I, TOK><<<(unsigned)(tiles < 1 ? 1 : tiles < cap ? tiles : cap), SLOT_THREADS, 0, v.stream>>>(a);
  FS_SLOTS_CUDA(s, cudaGetLastError());
  return FS_OK;
}
template <typename I> int launch_slots(fs_sorter* s, const SorterView& v, const SlotArgs& a) {
  return a.capacity > (uint64_t)v.sm_count * SLOT_THREADS ? launch_tokens<I, 4>(s, v, a) : launch_tokens<I, 1>(s, v, a);
}

}  // namespace

extern "C" int fs_plan_slots(fs_sorter* s, int index_bytes, const void* context_lens, const void* new_lens,
                             uint64_t requests, uint32_t page_size, int32_t* block_table, uint64_t table_width,
                             int64_t table_stride, const int32_t* free_pages, uint64_t n_free, const int32_t* cursor,
                             int32_t* query_start, void* seq_lens, void* positions, int32_t* request_of,
                             int64_t* slots, uint64_t capacity, int32_t* cursor_out, int sync, void* stream) {
  if (!s) return FS_E_INVALID;
  if (index_bytes != 4 && index_bytes != 8)
    return sorter_fail(s, FS_E_INVALID, "lengths must be of 4 or 8 bytes, got %d", index_bytes);
  if (requests > (1u << 24)) return sorter_fail(s, FS_E_INVALID, "requests = %llu exceeds 2^24", (unsigned long long)requests);
  if (page_size == 0 || page_size > (1u << 20)) return sorter_fail(s, FS_E_INVALID, "page size %u outside [1, 2^20]", page_size);
  if ((requests && table_width == 0) || table_width > 0x7fffffffull)
    return sorter_fail(s, FS_E_INVALID, "block table width %llu outside [1, 2^31)", (unsigned long long)table_width);
  if (requests > 1 && table_stride < (int64_t)table_width)
    return sorter_fail(s, FS_E_INVALID, "block table rows overlap: stride %lld, width %llu", (long long)table_stride,
                       (unsigned long long)table_width);
  if (n_free > 0x7fffffffull) return sorter_fail(s, FS_E_INVALID, "more than 2^31 - 1 free pages");
  if (capacity > 0x7fffffffull) return sorter_fail(s, FS_E_INVALID, "more than 2^31 - 1 tokens");
  // without requests: places to fill and a cursor to hand on, but no lengths and no table
  if ((requests && (!context_lens || !new_lens || !block_table || !seq_lens)) || !cursor || !query_start || !cursor_out ||
      (n_free && !free_pages) || (capacity && (!positions || !request_of || !slots)))
    return sorter_fail(s, FS_E_INVALID, "a required pointer is NULL");
  SorterView v;
  int rc = sorter_view(s, stream, &v);
  if (rc) return rc;
  // the outputs first, then what is read, then the table, which is both
  constexpr int OUTPUTS = 6, PLAIN = 10;
  const size_t I = index_bytes;
  const struct { const void* p; size_t bytes, align; const char* what; } ptrs[] = {
      {query_start, (requests + 1) * 4, 4, "query_start"}, {requests ? seq_lens : nullptr, requests * I, I, "seq_lens"},
      {capacity ? positions : nullptr, capacity * I, I, "positions"},
      {capacity ? request_of : nullptr, capacity * 4, 4, "request_of"}, {capacity ? slots : nullptr, capacity * 8, 8, "slots"},
      {cursor_out, 4, 4, "cursor_out"},
      {requests ? context_lens : nullptr, requests * I, I, "context_lens"},
      {requests ? new_lens : nullptr, requests * I, I, "new_lens"},
      {n_free ? free_pages : nullptr, n_free * 4, 4, "free_pages"}, {cursor, 4, 4, "cursor"},
      {requests ? block_table : nullptr, ((size_t)(requests - 1) * table_stride + table_width) * 4, 4, "block_table"}};
  // CTAs read all of the inputs while others write
  for (int i = 0; i < OUTPUTS; ++i)
    for (int j = i + 1; j < PLAIN; ++j) {
      const uintptr_t x = reinterpret_cast<uintptr_t>(ptrs[i].p), y = reinterpret_cast<uintptr_t>(ptrs[j].p);
      if (x && y && x < y + ptrs[j].bytes && y < x + ptrs[i].bytes)
        return sorter_fail(s, FS_E_INVALID, "%s and %s overlap", ptrs[i].what, ptrs[j].what);
    }
  for (const auto& q : ptrs)
    if (q.p && (rc = sorter_check(s, q.p, q.bytes, q.align, q.what))) return rc;
  SlotArgs a{};
  a.ctx = context_lens;
  a.neu = new_lens;
  a.requests = (uint32_t)requests;
  a.page = page_size;
  a.page_part = ~0ull / page_size;
  a.table = block_table;
  a.width = (uint32_t)table_width;
  a.table_stride = table_stride;
  a.free_pages = free_pages;
  a.n_free = n_free;
  a.cursor = cursor;
  a.query_start = query_start;
  a.seq_lens = seq_lens;
  a.positions = positions;
  a.request_of = request_of;
  a.slots = slots;
  a.capacity = capacity;
  a.cursor_out = cursor_out;
  a.host_err = v.host_err;
  a.wide = (reinterpret_cast<uintptr_t>(positions) | reinterpret_cast<uintptr_t>(request_of) | reinterpret_cast<uintptr_t>(slots)) % 16 == 0;
  rc = index_bytes == 4 ? launch_slots<int32_t>(s, v, a) : launch_slots<int64_t>(s, v, a);
  return rc ? rc : sorter_finish(s, v, 1, sync, true);
}
