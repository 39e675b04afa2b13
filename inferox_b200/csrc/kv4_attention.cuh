// What the attention kernels over the cache in 4 bits share: how sequences are
// cut into units of work, and rows and results found.
#pragma once
#include "serve.cuh"

namespace ifx {
namespace kv4 {

// Scratch in global memory: per CTA two partial results and where its range
// of tiles begins.
struct RangeInfo {
  long long begin, end;  // the segment that holds the CTA's first unit
  long long total;       // units of the launch
  int seq, h, ct, live;  // live: CTAs that share them (0: this one has none)
};

// The units dealt out evenly over `live` CTAs.
struct Deal {
  long long each;
  int more, live;  // the first `more` CTAs have one unit more
  __device__ __forceinline__ Deal(long long total, int l) : live(l) {
    each = total >> 32 ? total / l : (uint32_t)total / (uint32_t)l;
    more = (int)(total - each * l);
  }
  __device__ __forceinline__ long long begin(int c) const { return each * c + min(c, more); }
  __device__ __forceinline__ int owner(long long u) const {  // the CTA that has unit u
    const long long cut = (each + 1) * more;
    return u < cut ? (int)(u / (each + 1)) : more + (int)((u - cut) / each);
  }
};

template <int N>
__device__ __forceinline__ void ld_words(const uint8_t *p, uint32_t (&w)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 v = reinterpret_cast<const uint4 *>(p)[i];
      w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const uint2 v = reinterpret_cast<const uint2 *>(p)[i];
      w[2 * i] = v.x, w[2 * i + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const uint32_t *>(p)[i];
  }
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// A sequence's share of the work: every (kv head, column tile) is a segment
// of `units` pages, the first of them page `lo`.
struct Seq {
  int len, ql, q0, lo, units, nct;
};
template <int PAIRS>
__device__ __forceinline__ Seq sequence(const Kv4AttnArgs &a, int b) {
  Seq s;
  s.len = max(__ldg(a.kv_len + b), 0);
  if (s.len / kKv4PageRows >= a.max_pages) s.len = min(s.len, a.max_pages * kKv4PageRows);
  s.q0 = a.q_start ? __ldg(a.q_start + b) : b;
  s.ql = a.q_start ? (int)min(a.rows, (int64_t)max(0, __ldg(a.q_start + b + 1) - s.q0)) : 1;
  s.lo = a.window ? (int)(max((int64_t)0, (int64_t)s.len - s.ql - a.window + 1) / kKv4PageRows) : 0;
  // a sequence without rows still has its zeros to write
  s.units = max(1, (s.len + kKv4PageRows - 1) / kKv4PageRows - s.lo);
  s.nct = (int)(((uint32_t)s.ql * (uint32_t)(a.H / a.G) + PAIRS - 1) / PAIRS);
  return s;
}

struct Segment {
  int seq, h, ct, lo, len, ql, q0;
  long long begin, end;  // in units of the whole launch
};

template <int PAIRS>
__device__ __forceinline__ Segment locate(const Kv4AttnArgs &a, const long long *pre, long long u) {
  int lo = 0, hi = a.n_seqs - 1;  // the last sequence that begins at or before u
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (pre[mid] <= u) lo = mid; else hi = mid - 1;
  }
  const Seq s = sequence<PAIRS>(a, lo);
  const long long d = u - pre[lo];
  const long long i = d >> 32 ? d / s.units : (uint32_t)d / (uint32_t)s.units;
  Segment g;
  g.seq = lo;
  g.h = i >> 32 ? (int)(i / s.nct) : (int)((uint32_t)i / (uint32_t)s.nct);
  g.ct = (int)(i - (long long)g.h * s.nct);
  g.lo = s.lo;
  g.len = s.len;
  g.ql = s.ql;
  g.q0 = s.q0;
  g.begin = pre[lo] + i * s.units;
  g.end = g.begin + s.units;
  return g;
}

__device__ __forceinline__ void write4(const Kv4AttnArgs &a, long long row, int col, float4 o) {
  if (a.type == IFX_TYPE_F16) {
    const __half2 x = __floats2half2_rn(o.x, o.y), y = __floats2half2_rn(o.z, o.w);
    *reinterpret_cast<uint2 *>(static_cast<__half *>(a.out) + row * a.out_stride + col) =
        make_uint2(*reinterpret_cast<const uint32_t *>(&x), *reinterpret_cast<const uint32_t *>(&y));
  } else {
    *reinterpret_cast<float4 *>(static_cast<float *>(a.out) + row * a.out_stride + col) = o;
  }
}

// Zeros into the rows of no sequence, shared out over the grid; by one warp of
// every CTA, whose reads of q_start overlap the others' work.
__device__ __forceinline__ void zero_rest(const Kv4AttnArgs &a) {
  const int lane = threadIdx.x & 31, vals = a.H * a.hd;
  const auto zeros = [&](int64_t begin, int64_t end) {
    for (int64_t row = begin + blockIdx.x; row < end; row += gridDim.x)
      for (int c = 4 * lane; c < vals; c += 128) write4(a, row, c, make_float4(0.f, 0.f, 0.f, 0.f));
  };
  zeros(0, min(a.rows, (int64_t)__ldg(a.q_start)));
  zeros(max(0, __ldg(a.q_start + a.n_seqs)), a.rows);
}

// Row of q and out of column pair `p` of a segment, or -1.
template <int PAIRS>
__device__ __forceinline__ long long pair_row(const Kv4AttnArgs &a, int q0, int ql, int ct, int p, int *head) {
  const int grp = a.H / a.G;
  const uint32_t e = (uint32_t)ct * PAIRS + p;  // below rows * grp, which the entry point bounds
  const int tok = (int)(e / (uint32_t)grp);
  *head = (int)(e - (uint32_t)tok * grp);
  const long long row = (long long)q0 + tok;
  return tok < ql && row >= 0 && row < a.rows ? row : -1;
}

}  // namespace kv4

// Query rows per kv head of a sequence (heads times rows), on average: the
// lengths themselves are on the device.
inline int64_t kv4_columns(const Kv4AttnArgs &a) { return (a.rows * (a.H / a.G) + a.n_seqs - 1) / a.n_seqs; }

// Attention of many query rows per kv head: whether its kernels take a call,
// and the scratch they need.
bool kv4_chunks_take(const Kv4AttnArgs &a);
ifx_status kv4_attention_chunks(const Kv4AttnArgs &a, cudaStream_t st);
size_t kv4_chunks_ws(int hd);

}  // namespace ifx
