// Page tables and slot maps built on the device from request lengths (no
// reference counterpart: its KvCache holds one sequence, src/model/
// cache.rs:7-13). The rules are those of a paged KvBatch on the host: pages
// of 64 rows taken from the end of a free list in sequence order, returned
// to its end, nothing changed when the list is too short.
//
// Both kernels are bound by latency (a step of 32 sequences touches 2 KB):
// extend and release of 32 sequences take 5.9 us together, of 512 6.8 us.
// Every CTA scans the sequences itself instead of waiting for another CTA's
// prefix sums, so one launch does the step, with no counter and no
// workspace: the inputs a CTA reads (lens, n_free, the free list below
// n_free, table entries below the old page count) are never written by the
// launch, whose results go to lens_out, n_free_out and entries above.
#include <algorithm>

#include "serve.cuh"

namespace ifx {

namespace {

constexpr int kPagesThreads = 256;

// Exclusive sums of two 64-bit values over the CTA, and the totals.
__device__ __forceinline__ void block_scan2(long long &a, long long &b, long long &ta, long long &tb) {
  __shared__ long long wa[kPagesThreads / 32], wb[kPagesThreads / 32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const long long a0 = a, b0 = b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long xa = __shfl_up_sync(0xffffffffu, a, o), xb = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) {
      a += xa;
      b += xb;
    }
  }
  if (lane == 31) {
    wa[w] = a;
    wb[w] = b;
  }
  __syncthreads();
  ta = tb = 0;
  long long pa = 0, pb = 0;
#pragma unroll
  for (int i = 0; i < kPagesThreads / 32; ++i) {
    if (i == w) {
      pa = ta;
      pb = tb;
    }
    ta += wa[i];
    tb += wb[i];
  }
  a += pa - a0;
  b += pb - b0;
}

// Largest i with pre[i] <= x (pre ascending, pre[0] = 0).
__device__ __forceinline__ int owner(const int *pre, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (pre[mid] <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ int pages_of(int rows) { return (rows + kKv4PageRows - 1) / kKv4PageRows; }

__global__ void __launch_bounds__(kPagesThreads) pages_extend_kernel(const __grid_constant__ PagesExtendArgs a) {
  extern __shared__ int sm[];
  const int B = a.n_seqs, tid = threadIdx.x;
  int *qs = sm, *ps = sm + B, *ln = sm + 2 * B;  // first new row, first new page, old length of each sequence
  __shared__ int s_bad;
  if (tid == 0) s_bad = 0;
  const int per = (B + kPagesThreads - 1) / kPagesThreads;
  const int b0 = min(B, tid * per), b1 = min(B, b0 + per);
  const long long cap = (long long)a.max_pages * kKv4PageRows;
  const int n_free = min(max(a.n_free[0], 0), a.n_pages);
  long long tok = 0, pg = 0;
  int bad = 0;
  for (int b = b0; b < b1; ++b) {
    const int len = (int)min((long long)max(a.lens[b], 0), cap), add = max(a.add[b], 0);
    if ((long long)max(a.lens[b], 0) + add > cap) bad = 2;
    ln[b] = len;
    qs[b] = add;
    tok += add;
    pg += pages_of((int)min(cap, (long long)len + add)) - pages_of(len);
  }
  long long tt, tp;
  block_scan2(tok, pg, tt, tp);
  if (bad) s_bad = bad;  // any writer stores the same value
  __syncthreads();
  bad = s_bad ? s_bad : tt > a.max_tokens ? 3 : tp > n_free ? 1 : 0;
  const bool lead = blockIdx.x == 0;
  for (int b = b0; b < b1; ++b) {
    const int len = ln[b], add = qs[b];
    if (lead) {
      a.lens_out[b] = bad ? a.lens[b] : len + add;
      a.q_start[b] = bad ? 0 : (int)tok;
    }
    if (!bad) {
      qs[b] = (int)tok;
      ps[b] = (int)pg;
      tok += add;
      pg += pages_of(len + add) - pages_of(len);
    }
  }
  if (lead && tid == 0) {
    a.q_start[B] = bad ? 0 : (int)tt;
    a.n_free_out[0] = bad ? a.n_free[0] : n_free - (int)tp;
    a.status[0] = bad;
  }
  __syncthreads();
  const int live = bad ? 0 : (int)tt, fresh = bad ? 0 : (int)tp;
  const int64_t step = (int64_t)gridDim.x * kPagesThreads, at = (int64_t)blockIdx.x * kPagesThreads + tid;
  for (int64_t i = at; i < fresh; i += step) {
    const int b = owner(ps, B, (int)i);
    a.table[(size_t)b * a.max_pages + pages_of(ln[b]) + ((int)i - ps[b])] = a.free_pages[n_free - 1 - (int)i];
  }
  for (int64_t i = at; i < a.max_tokens; i += step) {
    int b = -1, pos = -1, slot = -1;
    if (i < live) {
      b = owner(qs, B, (int)i);
      pos = ln[b] + ((int)i - qs[b]);
      const int held = pages_of(ln[b]), j = pos / kKv4PageRows;
      const int page = j < held ? a.table[(size_t)b * a.max_pages + j] : a.free_pages[n_free - 1 - (ps[b] + j - held)];
      slot = (unsigned)page <= INT32_MAX / kKv4PageRows ? page * kKv4PageRows + pos % kKv4PageRows : -1;
    }
    a.slots[i] = slot;
    if (a.positions) a.positions[i] = pos;
    if (a.seqs) a.seqs[i] = b;
  }
}

__global__ void __launch_bounds__(kPagesThreads) pages_release_kernel(const __grid_constant__ PagesReleaseArgs a) {
  extern __shared__ int sm[];
  const int B = a.n_seqs, tid = threadIdx.x;
  const int per = (B + kPagesThreads - 1) / kPagesThreads;
  const int b0 = min(B, tid * per), b1 = min(B, b0 + per);
  const long long cap = (long long)a.max_pages * kKv4PageRows;
  const int n_free = min(max(a.n_free[0], 0), a.n_pages);
  const bool lead = blockIdx.x == 0;
  long long pg = 0, none = 0, tp, tn;
  for (int b = b0; b < b1; ++b) {
    const int n = a.done[b] ? pages_of((int)min((long long)max(a.lens[b], 0), cap)) : 0;
    sm[b] = n;
    pg += n;
    if (lead) a.lens_out[b] = a.done[b] ? 0 : a.lens[b];
  }
  block_scan2(pg, none, tp, tn);
  for (int b = b0; b < b1; ++b) {
    const int n = sm[b];
    sm[b] = (int)min(pg, (long long)INT32_MAX);
    pg += n;
  }
  // a list that would overflow (a page released twice) is cut at its end
  const int total = (int)min(tp, (long long)(a.n_pages - n_free));
  if (lead && tid == 0) a.n_free_out[0] = n_free + total;
  __syncthreads();
  for (int i = blockIdx.x * kPagesThreads + tid; i < total; i += gridDim.x * kPagesThreads) {
    const int b = owner(sm, B, i);
    a.free_pages[n_free + i] = a.table[(size_t)b * a.max_pages + (i - sm[b])];
  }
}

unsigned grid_for(int64_t items) {
  // two items per thread; beyond two CTAs per SM the threads loop
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>((items + 2 * kPagesThreads - 1) / (2 * kPagesThreads), 2 * kNumSMs));
}

}  // namespace

ifx_status op_pages_extend(const PagesExtendArgs &a, cudaStream_t st) {
  const size_t smem = (size_t)a.n_seqs * 3 * sizeof(int);
  static std::atomic<uint64_t> done{0};
  IFX_TRY(raise_smem(pages_extend_kernel, kMaxServeSeqs * 12, done));
  pages_extend_kernel<<<grid_for(a.max_tokens), kPagesThreads, smem, st>>>(a);
  IFX_CUDA(cudaGetLastError());
  return IFX_OK;
}

ifx_status op_pages_release(const PagesReleaseArgs &a, cudaStream_t st) {
  const size_t smem = (size_t)a.n_seqs * sizeof(int);
  pages_release_kernel<<<grid_for(std::min<int64_t>((int64_t)a.n_seqs * a.max_pages, a.n_pages)), kPagesThreads, smem, st>>>(a);
  IFX_CUDA(cudaGetLastError());
  return IFX_OK;
}

}  // namespace ifx
