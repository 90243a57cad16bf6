// fs_rows_stream.cuh -- the row operators over large batches: the same
// definitions and the same whole numbers as fs_rows.cuh, as passes over the
// whole batch instead of one cluster a row.
//
// A cluster that keeps its row in shared memory reads it from HBM once, but
// holds that memory through the row's barriers and its ranking: three CTAs of
// 64 KB on an SM for about 10 us each are 2 TB/s.  Passes hold nothing: any
// number of CTAs stream the batch, and whichever CTA is the last to finish with
// a row (an atomic counter tells) draws the conclusion for it.
//   k_stream_max    the row's maximum and published thread maxima; the last
//                   CTA of a row finds its candidates' edge
//   k_stream_weigh  the sum of the weights, and the candidates; the last CTA
//                   orders, cuts and draws.  Rows in reverse order, so that
//                   what the first pass read last is still in L2
//   k_stream_bins   for rows whose nucleus does not end among the candidates,
//                   weights by bin; the last CTA finds the interval it ends in
//   k_stream_cut    the exact mass before the interval and its entries; the
//                   last CTA cuts and draws
//   k_rows          (fs_rows.cuh) the rows that fit none of these
// Reading twice costs HBM time beyond the size of L2 (126 MB), and is still
// the faster from a few megabytes on.
#pragma once

#include "fs_rows.cuh"

namespace fs {

struct RowRecord {
  float m, c, edge;
  uint32_t dirty;       // the row has NaN or +inf
  uint32_t done[4];     // CTAs that have finished with it, by pass
  uint32_t list_n, pool_n, first, pad;
  uint64_t total, lo, hi, target;
};

struct RowStream {
  RowRecord* rec;       // a record a row, zero before the first pass
  uint32_t* tops;       // ROW_TOPS a row
  uint64_t* mass;       // ROW_SUMS a row: each warp's sum
  uint64_t* part;       // ... of its kept entries
  uint64_t* list;       // ROW_LIST a row
  uint32_t* wide;       // rows whose nucleus is wide,
  uint32_t* left;       // rows left to k_rows,
  uint32_t* counts;     // and their numbers
  uint32_t* bins;       // ROW_BINS for each wide row
  uint64_t* pool;       // ROW_WIDE_POOL for each wide row
  uint32_t parts;       // CTAs a row
};
constexpr int ROW_SUMS = ROW_MAX_CLUSTER * ROW_WARPS;
constexpr int ROW_WIDE_POOL = 4095;  // entries of a wide nucleus's last interval: below 2^12, see RowWide

// The last CTA's working memory for a wide row.
struct RowWide {
  uint32_t sums[1024][2];  // masses by bin of the interval: of their low 20 bits, of the rest (both below 2^32)
  uint32_t part[ROW_SUMS][2];
  uint64_t few[ROW_THREADS], few_q[ROW_THREADS];
};

// Whether this CTA is the last of `parts` to get here; what the others wrote
// is then visible.
__device__ __forceinline__ bool row_last(uint32_t* done, uint32_t parts, uint32_t& flag) {
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) flag = atomicAdd(done, 1u) == parts - 1;
  __syncthreads();
  if (!flag) return false;
  if (threadIdx.x == 0) *done = 0;
  __threadfence();
  return true;
}

// Each thread keeps ROW_AHEAD vectors in flight, in slots of its own in shared
// memory: no registers, and nothing to wait for but its own copies.
constexpr int ROW_AHEAD = 8;
using RowRing = uint4[ROW_AHEAD][ROW_THREADS];

// f(vector, number) for the vectors of warp r.wid's stretch of part r.rank.
template <typename T, typename F> __device__ __forceinline__ void row_stream(const Row<T>& r, RowRing& ring, bool dirty, F f) {
  uint32_t v0, v1;
  r.stretch(r.rank, r.wid, v0, v1);
  const bool head = v0 < v1 && !r.inside(v0), tail = v0 + head < v1 && !r.inside(v1 - 1);
  const uint32_t end = v1 - tail;
  uint32_t i = v0 + head + r.lane, next = i;
  const uint32_t slot = smem_of(&ring[0][r.tid]);
  auto fetch = [&](int s) {
    if (next < end)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slot + s * (uint32_t)sizeof(ring[0])), "l"(r.vecs + next) : "memory");
    asm volatile("cp.async.commit_group;" ::: "memory");
    next += 32;
  };
#pragma unroll
  for (int s = 0; s < ROW_AHEAD; ++s) fetch(s);
  while (i < end) {
#pragma unroll
    for (int s = 0; s < ROW_AHEAD; ++s) {
      asm volatile("cp.async.wait_group %0;" ::"n"(ROW_AHEAD - 1) : "memory");
      if (i < end) {
        const uint4 v = ring[s][r.tid];
        f(dirty ? r.cleaned(v) : v, i);
        i += 32;
      }
      fetch(s);
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (head && r.lane == 0) f(r.cleaned(r.ragged(v0)), v0);
  if (tail && r.lane == 1) f(r.cleaned(r.ragged(v1 - 1)), v1 - 1);
}
// f(x, index) for the entries of a vector that mask names
template <typename T, typename F> __device__ __forceinline__ void row_each(const Row<T>& r, uint32_t mask, const uint4& v, uint32_t i, F f) {
  while (mask) {
    const int e = __ffs((int)mask) - 1;
    mask &= mask - 1;
    f(RowElem<T>::at(v, e), (int)(i * Row<T>::N) - r.lead + e);
  }
}
template <typename V> __device__ __forceinline__ V row_get(const V* p) { return __ldcg(p); }  // written by other CTAs

template <typename T, bool BEST> __global__ void __launch_bounds__(ROW_THREADS, 4) k_stream_max(const RowArgs a, const RowStream s) {
  extern __shared__ __align__(16) unsigned char row_smem[];
  RowShared& sh = *reinterpret_cast<RowShared*>(row_smem);
  RowRing& ring = *reinterpret_cast<RowRing*>(row_smem + ROW_SHARED_BYTES);
  asm volatile("griddepcontrol.launch_dependents;");
  using E = RowElem<T>;
  const uint32_t row = blockIdx.x / s.parts;
  Row<T> r(sh, nullptr, a, row, blockIdx.x % s.parts, s.parts, 2);
  RowRecord& rec = s.rec[row];
  bool tops = true;
  if constexpr (!BEST) {
    const RowParams q(a, row);
    tops = q.by_k || q.by_p;
  }
  // two maxima a thread, of its vectors of even and odd numbers
  typename E::Top top[2] = {E::top0(), E::top0()};
  row_stream(r, ring, false, [&](const uint4& v, uint32_t i) {
    if (i & 32)
      top[1] = E::top(top[1], v);
    else
      top[0] = E::top(top[0], v);
  });
  if (__any_sync(~0u, !(E::value(top[0]) <= ROW_F32_MAX && E::value(top[1]) <= ROW_F32_MAX))) {
    rec.dirty = 1;  // the warp looks through its stretch again
    uint32_t v0, v1;
    r.stretch(r.rank, r.wid, v0, v1);
    top[0] = top[1] = E::top0();
    for (uint32_t i = v0 + r.lane; i < v1; i += 32) top[0] = E::top(top[0], r.from_memory(i));
  }
  const uint32_t per = r.top_count();
  uint32_t* const all = s.tops + (size_t)row * ROW_TOPS;
#pragma unroll
  for (int l = 0; l < 2; ++l) {
    r.mine = E::value(top[l]);
    const uint32_t key = tops ? r.sorted_tops() : __reduce_min_sync(~0u, row_key(r.mine));
    if (r.lane < (int)(tops ? per : 1)) all[((r.rank * ROW_WARPS + r.wid) * 2 + l) * per + r.lane] = key;
  }
  if (!row_last(&rec.done[0], s.parts, sh.found)) return;

  for (uint32_t i = r.tid; i < per * r.lists; i += ROW_THREADS) sh.tops[i] = row_get(all + i);
  __syncthreads();
  r.find_max();
  float edge = INFINITY;
  if (r.m == -INFINITY) {
    if constexpr (BEST) {
      r.put_nothing(a, row);
    } else if (r.tid == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = -INFINITY;
    }
  } else if constexpr (BEST) {
    r.c = ROW_LOG2E;
    edge = r.edge_for_best((uint32_t)a.n);
  } else {
    const RowParams q(a, row);
    r.c = q.c();
    if (q.greedy)
      edge = r.m;
    else if (q.cuts())
      edge = r.edge_for(q);
  }
  if (r.tid == 0) rec.m = r.m, rec.c = r.c, rec.edge = edge, rec.first = ~0u;
}

template <typename T, bool BEST> __global__ void __launch_bounds__(ROW_THREADS, 4) k_stream_weigh(const RowArgs a, const RowStream s) {
  extern __shared__ __align__(16) unsigned char row_smem[];
  RowShared& sh = *reinterpret_cast<RowShared*>(row_smem);
  RowFinish& f = *reinterpret_cast<RowFinish*>(row_smem + ROW_SHARED_BYTES);
  RowRing& ring = *reinterpret_cast<RowRing*>(row_smem + ROW_SHARED_BYTES);  // until the row's last CTA finishes
  const uint32_t row = a.rows - 1 - blockIdx.x / s.parts;
  Row<T> r(sh, nullptr, a, row, blockIdx.x % s.parts, s.parts, 2);
  RowRecord& rec = s.rec[row];
  __syncthreads();
  row_chain_wait();
  r.m = row_get(&rec.m), r.c = row_get(&rec.c);
  if (r.m == -INFINITY) return;
  const float edge = row_get(&rec.edge);
  bool greedy = false;
  if constexpr (!BEST) greedy = a.temperature && !(a.temperature[row] > 0.0f);
  typename Row<T>::Sum sum(r.m, r.c);
  row_stream(r, ring, row_get(&rec.dirty) != 0, [&](const uint4& v, uint32_t i) {
    sum.template add<false>(v, 0.0f);
    if (RowElem<T>::value(RowElem<T>::top(RowElem<T>::top0(), v)) >= edge)
      row_each(r, r.hits(v, edge, INFINITY), v, i, [&](float z, int j) {
        if (greedy) {
          atomicMin(&rec.first, (uint32_t)j);
        } else {
          const uint32_t at = atomicAdd(&sh.count, 1u);
          if (at < ROW_LIST) sh.list[at] = (uint64_t)row_key(z) << ROW_IDX_BITS | (uint32_t)j;
        }
      });
  });
  const uint64_t own = warp_sum_u64(sum.mass());
  uint64_t* const masses = s.mass + (size_t)row * ROW_SUMS;
  uint64_t* const list = s.list + (size_t)row * ROW_LIST;
  if (r.lane == 0) masses[r.rank * ROW_WARPS + r.wid] = own;
  __syncthreads();
  uint32_t n = sh.count;
  if (n) {
    if (r.tid == 0) sh.found = atomicAdd(&rec.list_n, n);
    __syncthreads();
    const uint32_t base = sh.found;
    for (uint32_t i = r.tid; i < min(n, (uint32_t)ROW_LIST) && base + i < ROW_LIST; i += ROW_THREADS) list[base + i] = sh.list[i];
    __syncthreads();
  }
  if (!row_last(&rec.done[1], s.parts, sh.found)) return;

  for (uint32_t i = r.tid; i < s.parts * ROW_WARPS; i += ROW_THREADS) (&sh.mass[0][0])[i] = row_get(masses + i);
  __syncthreads();
  const uint64_t total = r.handed(sh.mass);
  n = row_get(&rec.list_n);
  const bool listed = edge < INFINITY && n <= (uint32_t)ROW_LIST;
  auto leave = [&] {
    if (r.tid == 0) s.left[atomicAdd(&s.counts[1], 1u)] = row;
  };
  if constexpr (BEST) {
    if (!listed) return leave();
    const float ln = logf((float)total * 0x1p-40f);
    if (a.lse && r.tid == 0) a.lse[row] = r.m + ln;
    for (uint32_t i = r.tid; i < n; i += ROW_THREADS) f.input[i] = row_get(list + i);
    __syncthreads();
    r.order_by_value(f, f.input, n, edge);
    r.put_best(a, row, f, min(n, (uint32_t)a.n), ln);
  } else {
    const RowParams q(a, row);
    auto store = [&](float z, int j) {
      a.tokens[row] = j;
      if (a.logprobs) a.logprobs[row] = row_neg_y(z, r.m, r.c) * ROW_LN2 - logf((float)total * 0x1p-40f);
    };
    if (q.greedy) {
      if (r.tid == 0) store(r.m, (int)row_get(&rec.first));
      return;
    }
    if (!q.cuts()) {
      r.scan_parts(sh.mass, row_draw(q.u, total), [&](float z, int) { return r.mass(z); }, store);
      return;
    }
    uint64_t* const to = n <= (uint32_t)ROW_THREADS ? f.loose : f.input;
    uint64_t part = 0, all = 0;
    if (listed)
      for (uint32_t i = r.tid; i < n; i += ROW_THREADS) {
        to[i] = row_get(list + i);
        part += r.mass(r.value_of(to[i]));
      }
    const uint64_t target = row_target(q.p, total);
    if (q.by_p && !q.by_k) {
      r.block_scan(part, sh.scan_q, all);
      if (all < target || !listed) {  // narrow it down
        if (r.tid == 0) sh.found = atomicAdd(&s.counts[0], 1u);
        __syncthreads();
        const uint32_t slot = sh.found;
        for (int b = r.tid; b < ROW_BINS; b += ROW_THREADS) s.bins[(size_t)slot * ROW_BINS + b] = 0;
        if (r.tid == 0) s.wide[slot] = row, rec.total = total, rec.target = target;
        return;
      }
    } else if (!listed) {
      return leave();
    }
    __syncthreads();
    r.finish_listed(f, n, edge, q, total, store);
  }
}

// Wide rows are cut anew, into as many parts as give every CTA one.
__device__ __forceinline__ uint32_t row_wide_parts(RowArgs& a, uint32_t n, uint32_t vecs) {
  const uint32_t parts = max(1u, min(min(gridDim.x / max(n, 1u), (uint32_t)ROW_MAX_CLUSTER), vecs / (2 * ROW_THREADS)));
  a.part_vecs = (vecs + parts - 1) / parts;
  return parts;
}

template <typename T> __global__ void __launch_bounds__(ROW_THREADS, 4) k_stream_bins(const RowArgs args, const RowStream s) {
  extern __shared__ __align__(16) unsigned char row_smem[];
  RowShared& sh = *reinterpret_cast<RowShared*>(row_smem);
  RowRing& ring = *reinterpret_cast<RowRing*>(row_smem + ROW_SHARED_BYTES);
  row_chain_wait();
  RowArgs a = args;
  const uint32_t wide = row_get(&s.counts[0]), parts = row_wide_parts(a, wide, s.parts * args.part_vecs);
  for (uint32_t item = blockIdx.x; item < wide * parts; item += gridDim.x) {
    const uint32_t slot = item / parts, row = row_get(&s.wide[slot]);
    __syncthreads();
    Row<T> r(sh, nullptr, a, row, item % parts, parts, 2);
    RowRecord& rec = s.rec[row];
    r.m = row_get(&rec.m), r.c = row_get(&rec.c);
    const float c42 = fminf(r.c * ROW_BIN_SCALE, ROW_F32_MAX);
    for (int b = r.tid; b < ROW_BINS; b += ROW_THREADS) sh.bins[b] = 0;
    if (r.tid == 0) sh.b1 = sh.b2 = ~0u, sh.last = 0;
    __syncthreads();
    row_stream(r, ring, row_get(&rec.dirty) != 0, [&](const uint4& v, uint32_t) { r.count_bins(v, true, c42); });
    __syncthreads();
    uint32_t* const bins = s.bins + (size_t)slot * ROW_BINS;
    for (int b = r.tid; b < ROW_BINS; b += ROW_THREADS)
      if (const uint32_t v = sh.bins[b]) atomicAdd(&bins[b], v);
    if (!row_last(&rec.done[2], parts, sh.found)) continue;
    for (int b = r.tid; b < ROW_BINS; b += ROW_THREADS) sh.bins[b] = row_get(bins + b);
    __syncthreads();
    r.end_bins(true, true, true, (float)row_get(&rec.target) * 0x1p-28f, 0, 1.0f);
    if (r.tid == 0) {
      // the bins' bounds in x, by more than their rounding; what that adds is only more entries to look at
      const float b1 = (float)min(sh.b1, sh.last), b2 = (float)min(sh.b2, sh.last);
      const float slack = fabsf(r.m) * 0x1p-21f;
      const float up = fminf(r.m - (b1 - 0.5f) / c42 * (1.0f - 0x1p-18f) + slack, r.m);
      const float down = fmaxf(r.m - (b2 + 0.5f) / c42 * (1.0f + 0x1p-18f) - slack, -ROW_F32_MAX);
      rec.lo = (uint64_t)row_key(up) << ROW_IDX_BITS;
      rec.hi = (uint64_t)row_key(down) << ROW_IDX_BITS | (ROW_MAX_COLS - 1);
    }
  }
}

template <typename T> __global__ void __launch_bounds__(ROW_THREADS, 3) k_stream_cut(const RowArgs args, const RowStream s) {
  extern __shared__ __align__(16) unsigned char row_smem[];
  RowShared& sh = *reinterpret_cast<RowShared*>(row_smem);
  RowWide& f = *reinterpret_cast<RowWide*>(row_smem + ROW_SHARED_BYTES);
  RowRing& ring = *reinterpret_cast<RowRing*>(row_smem + ROW_SHARED_BYTES);  // until the row's last CTA finishes
  row_chain_wait();
  RowArgs a = args;
  const uint32_t wide = row_get(&s.counts[0]), parts = row_wide_parts(a, wide, s.parts * args.part_vecs);
  for (uint32_t item = blockIdx.x; item < wide * parts; item += gridDim.x) {
    const uint32_t slot = item / parts, row = row_get(&s.wide[slot]);
    __syncthreads();
    Row<T> r(sh, nullptr, a, row, item % parts, parts, 2);
    RowRecord& rec = s.rec[row];
    const RowParams q(a, row);
    r.m = row_get(&rec.m), r.c = row_get(&rec.c);
    const uint64_t lo = row_get(&rec.lo), hi = row_get(&rec.hi);
    const float over = r.value_of(lo), least = r.value_of(hi);
    __syncthreads();
    typename Row<T>::Sum sum(r.m, r.c);
    uint64_t kept = 0;
    row_stream(r, ring, row_get(&rec.dirty) != 0, [&](const uint4& v, uint32_t i) {
      sum.template add<true>(v, over);
      row_each(r, r.hits(v, least, over), v, i, [&](float z, int j) {
        const uint32_t at = atomicAdd(&sh.count, 1u);
        if (at < ROW_POOL) sh.pool[at] = (uint64_t)row_key(z) << ROW_IDX_BITS | (uint32_t)j;
      });
      if (q.by_w) {
        float z[Row<T>::N];
        RowElem<T>::get(v, z);
#pragma unroll
        for (int e = 0; e < Row<T>::N; ++e) {
          const float w = r.weight(z[e]);
          if (z[e] > over && w >= q.least_w) kept += row_q(w);
        }
      }
    });
    const uint64_t own = warp_sum_u64(sum.mass());
    kept = q.by_w ? warp_sum_u64(kept) : own;
    uint64_t* const masses = s.mass + (size_t)row * ROW_SUMS;
    uint64_t* const kepts = s.part + (size_t)row * ROW_SUMS;
    uint64_t* const pool = s.pool + (size_t)slot * ROW_WIDE_POOL;
    if (r.lane == 0) masses[r.rank * ROW_WARPS + r.wid] = own, kepts[r.rank * ROW_WARPS + r.wid] = kept;
    __syncthreads();
    uint32_t n = sh.count;
    if (r.tid == 0) sh.found = atomicAdd(&rec.pool_n, n <= ROW_POOL ? n : ROW_WIDE_POOL + 1);  // more is too much
    __syncthreads();
    const uint32_t base = sh.found;
    for (uint32_t i = r.tid; i < min(n, (uint32_t)ROW_POOL) && base + i < ROW_WIDE_POOL; i += ROW_THREADS) pool[base + i] = sh.pool[i];
    __syncthreads();
    if (!row_last(&rec.done[3], parts, sh.found)) continue;

    // the entry of the interval at which the mass reaches the target: by bins of the interval, then among a bin's
    n = row_get(&rec.pool_n);
    auto leave = [&] {
      if (r.tid == 0) s.left[atomicAdd(&s.counts[1], 1u)] = row;
    };
    if (n > (uint32_t)ROW_WIDE_POOL) {
      leave();
      continue;
    }
    for (uint32_t i = r.tid; i < parts * ROW_WARPS; i += ROW_THREADS)
      (&sh.mass[0][0])[i] = row_get(masses + i), (&sh.part[0][0])[i] = row_get(kepts + i);
    for (int i = r.tid; i < 1024; i += ROW_THREADS) f.sums[i][0] = f.sums[i][1] = 0;
    if (r.tid < ROW_SUMS) f.part[r.tid][0] = f.part[r.tid][1] = 0;
    if (r.tid == 0) sh.count = 0, sh.cut_c = hi, sh.cut_n = 1024;
    __syncthreads();
    const int shift = max(0, 64 - __clzll((long long)((hi - lo) | 1)) - 10);
    for (uint32_t i = r.tid; i < n; i += ROW_THREADS) {
      const uint64_t e = row_get(pool + i), m = r.mass(r.value_of(e));
      uint32_t* const to = f.sums[(e - lo) >> shift];
      atomicAdd(&to[0], (uint32_t)m & 0xfffffu);
      atomicAdd(&to[1], (uint32_t)(m >> 20));
    }
    __syncthreads();
    uint64_t b[4], t = 0, all;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t* const p = f.sums[4 * r.tid + i];
      b[i] = ((uint64_t)p[1] << 20) + p[0];
      t += b[i];
    }
    const uint64_t target = row_get(&rec.target);
    uint64_t run = r.handed(sh.mass) + r.block_scan(t, sh.scan_q, all);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (run < target && target <= run + b[i]) sh.cut_n = 4 * r.tid + i, sh.cut_q = run;
      run += b[i];
    }
    __syncthreads();
    const uint32_t bin = sh.cut_n;
    auto keep = [&](uint64_t e, uint64_t m) {  // adds to its stretch's kept mass
      if (r.weight(r.value_of(e)) < q.least_w) return;
      const uint32_t v = (((uint32_t)e & (ROW_MAX_COLS - 1)) + r.lead) / Row<T>::N;
      const uint32_t part = v / r.part_vecs, p0 = part * r.part_vecs, p1 = min(p0 + r.part_vecs, r.total_vecs);
      uint32_t* const to = f.part[part * ROW_WARPS + (v - p0) / ((p1 - p0 + ROW_WARPS - 1) / ROW_WARPS)];
      atomicAdd(&to[0], (uint32_t)m & 0xfffffu);
      atomicAdd(&to[1], (uint32_t)(m >> 20));
    };
    for (uint32_t i = r.tid; i < n; i += ROW_THREADS) {
      const uint64_t e = row_get(pool + i), m = r.mass(r.value_of(e));
      const uint32_t at_bin = (uint32_t)((e - lo) >> shift);
      if (at_bin < bin) {
        keep(e, m);
      } else if (at_bin == bin) {
        const uint32_t at = atomicAdd(&sh.count, 1u);
        if (at < ROW_THREADS) f.few[at] = e, f.few_q[at] = m;
      }
    }
    __syncthreads();
    const uint32_t few = sh.count;
    if (few > ROW_THREADS || bin == 1024) {  // the estimate of the interval is never that far off
      leave();
      continue;
    }
    if (r.tid < few) {
      const uint64_t e = f.few[r.tid], m = f.few_q[r.tid];
      uint64_t before = sh.cut_q;
      for (uint32_t i = 0; i < few; ++i) before += f.few[i] < e ? f.few_q[i] : 0;
      if (before < target) keep(e, m);
      if (before < target && target <= before + m) sh.cut_c = e;
    }
    __syncthreads();
    if (r.tid < ROW_SUMS) (&sh.part[0][0])[r.tid] += ((uint64_t)f.part[r.tid][1] << 20) + f.part[r.tid][0];
    const uint64_t last = sh.cut_c, total = row_get(&rec.total);
    __syncthreads();
    r.scan_parts(sh.part, row_draw(q.u, r.handed(sh.part)),
                 [&](float z, int j) -> uint64_t {
                   const float w = r.weight(z);
                   return w >= q.least_w && ((uint64_t)row_key(z) << ROW_IDX_BITS | (uint32_t)j) <= last ? row_q(w) : 0;
                 },
                 [&](float z, int j) {
                   a.tokens[row] = j;
                   if (a.logprobs) a.logprobs[row] = row_neg_y(z, r.m, r.c) * ROW_LN2 - logf((float)total * 0x1p-40f);
                 });
  }
}

}  // namespace fs
