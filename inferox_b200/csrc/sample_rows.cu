// Row-wise sampling: temperature, top-k, top-p and min-p from given random
// numbers. The rule of Sampler::sample (src/sampler.rs:28-73), for every row
// of a batch with its own settings, and min-p beside its filters.
#include <algorithm>

#include "serve.cuh"

namespace ifx {

namespace {

constexpr int kThreads = 1024;

// A NaN counts as a masked token; -0 and +0 are one value.
__device__ __forceinline__ float clean(float z) { return z != z ? -INFINITY : z + 0.f; }

__device__ __forceinline__ uint32_t ordered(float f) {
  const uint32_t b = __float_as_uint(f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

struct Row {
  const float *z;
  int n;
  float zmax;
  double inv_t, unit;  // unit: the fixed-point mass of weight 1
  float min_p;
};

__device__ __forceinline__ double weight(const Row &r, float z) {
  // (z - zmax) is -inf for a masked token, and inv_t is never 0
  return z == r.zmax ? 1.0 : exp(((double)z - (double)r.zmax) * r.inv_t);
}
__device__ __forceinline__ unsigned long long mass(const Row &r, float z) {
  return __double2ull_rn(weight(r, z) * r.unit);
}

// The last element that a filter keeps, in the order of falling values and,
// among equal ones, rising indices.
struct Bound {
  uint32_t key = 0;
  int idx = INT32_MAX;
};
__device__ __forceinline__ bool kept(const Row &r, float z, int i, const Bound &c) {
  const uint32_t k = ordered(z);
  if (k < c.key || (k == c.key && i > c.idx)) return false;
  return !(r.min_p > 0.f) || weight(r, z) >= (double)r.min_p;
}

__device__ unsigned long long block_sum(unsigned long long v, unsigned long long *red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  unsigned long long t = 0;
  for (int i = 0; i < kThreads / 32; ++i) t += red[i];
  __syncthreads();
  return t;
}

// First kept element, in sorted order, at which the running sum (of ones or
// of masses) reaches `target` (>=) or passes it (>). Sums are of integers:
// they do not depend on the order of the atomics.
__device__ bool find(const Row &r, const Bound &c, bool by_count, unsigned long long target, bool reach,
                     Bound *out, unsigned long long *hist, unsigned long long *scan) {
  const int tid = threadIdx.x;
  uint32_t prefix = 0, mask = 0;
  unsigned long long above = 0;
  for (int b = 24; b >= 0; b -= 8) {
    for (int j = tid; j < 256; j += kThreads) hist[j] = 0;
    __syncthreads();
    for (int i = tid; i < r.n; i += kThreads) {
      const float z = clean(r.z[i]);
      const uint32_t k = ordered(z);
      if ((k & mask) != prefix || !kept(r, z, i, c)) continue;
      atomicAdd(&hist[k >> b & 255u], by_count ? 1ull : mass(r, z));
    }
    __syncthreads();
    if (tid == 0) {
      int sel = -1;
      for (int j = 255; j >= 0 && sel < 0; --j) {
        if (reach ? above + hist[j] >= target : above + hist[j] > target) sel = j;
        else above += hist[j];
      }
      scan[0] = (unsigned long long)(long long)sel;
      scan[1] = above;
    }
    __syncthreads();
    const int sel = (int)(long long)scan[0];
    above = scan[1];
    __syncthreads();
    if (sel < 0) return false;
    prefix |= (uint32_t)sel << b;
    mask |= 255u << b;
  }
  // equal values, by index: each thread a run of them
  const int per = (r.n + kThreads - 1) / kThreads, lo = min(r.n, tid * per), hi = min(r.n, lo + per);
  unsigned long long mine = 0;
  for (int i = lo; i < hi; ++i) {
    const float z = clean(r.z[i]);
    if (ordered(z) == prefix && kept(r, z, i, c)) mine += by_count ? 1ull : mass(r, z);
  }
  scan[2 + tid] = mine;
  __syncthreads();
  if (tid == 0) {
    unsigned long long run = above;
    for (int t = 0; t < kThreads; ++t) {
      const unsigned long long v = scan[2 + t];
      scan[2 + t] = run;
      run += v;
    }
    scan[0] = INT32_MAX;
  }
  __syncthreads();
  unsigned long long run = scan[2 + tid];
  for (int i = lo; i < hi; ++i) {
    const float z = clean(r.z[i]);
    if (ordered(z) != prefix || !kept(r, z, i, c)) continue;
    run += by_count ? 1ull : mass(r, z);
    if (reach ? run >= target : run > target) {
      atomicMin(&scan[0], (unsigned long long)i);
      break;
    }
  }
  __syncthreads();
  out->key = prefix;
  out->idx = (int)scan[0];
  __syncthreads();
  return true;
}

__global__ void __launch_bounds__(kThreads) sample_rows_kernel(const __grid_constant__ SampleRowsArgs a) {
  __shared__ unsigned long long hist[256], scan[2 + kThreads], red[kThreads / 32];
  __shared__ unsigned long long s_key;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  Row r;
  r.z = a.logits + row * a.stride;
  r.n = (int)a.n;
  if (tid == 0) s_key = 0;
  __syncthreads();
  unsigned long long best = 0;  // largest value, last index among equal ones
  for (int i = tid; i < r.n; i += kThreads)
    best = max(best, (unsigned long long)ordered(clean(r.z[i])) << 32 | (uint32_t)i);
  atomicMax(&s_key, best);
  __syncthreads();
  const int last = (int)(uint32_t)s_key;
  r.zmax = clean(r.z[last]);
  const float T = a.temperature ? a.temperature[row] : 1.f;
  if (r.zmax == -INFINITY || !(T > 0.f)) {
    if (tid == 0) {
      a.token[row] = r.zmax == -INFINITY ? -1 : last;
      if (a.logprob) a.logprob[row] = r.zmax == -INFINITY ? -INFINITY : 0.f;
    }
    return;
  }
  r.inv_t = fmax(1.0 / (double)T, 1e-300);  // an infinite T: weight 1 for every unmasked token
  r.unit = exp2((double)(62 - (32 - __clz(r.n))));
  const int top_k = a.top_k ? a.top_k[row] : 0;
  const float top_p = a.top_p ? a.top_p[row] : 1.f;
  r.min_p = a.min_p ? fminf(a.min_p[row], 1.f) : 0.f;
  const double u = fmin(fmax((double)a.u[row], 0.0), 1.0);
  const bool filtered = top_k > 0 || top_p < 1.f || r.min_p > 0.f;
  Bound c;
  unsigned long long m = 0;
  for (int i = tid; i < r.n; i += kThreads) m += mass(r, clean(r.z[i]));
  const unsigned long long M = block_sum(m, red);
  if (filtered) {
    const float keep_p = r.min_p;
    r.min_p = 0.f;  // top-k and top-p are of the whole distribution
    Bound k, p;
    if (top_k > 0 && top_k < r.n) find(r, c, true, (unsigned long long)top_k, true, &k, hist, scan);
    if (top_p < 1.f) {  // at least the first element, whose mass is not 0
      const unsigned long long want = (unsigned long long)ceil(fmax((double)top_p, 0.0) * (double)M);
      find(r, c, false, max(want, 1ull), true, &p, hist, scan);
    }
    c = k.key > p.key || (k.key == p.key && k.idx < p.idx) ? k : p;
    r.min_p = keep_p;
  }
  m = 0;
  for (int i = tid; i < r.n; i += kThreads) {
    const float z = clean(r.z[i]);
    if (kept(r, z, i, c)) m += mass(r, z);
  }
  const unsigned long long S = block_sum(m, red);
  const unsigned long long target = min((unsigned long long)(u * (double)S), S - 1);
  int token = last;
  if (filtered) {
    Bound pick;
    if (find(r, c, false, target, false, &pick, hist, scan)) token = pick.idx;
  } else {
    const int per = (r.n + kThreads - 1) / kThreads, lo = min(r.n, tid * per), hi = min(r.n, lo + per);
    unsigned long long mine = 0;
    for (int i = lo; i < hi; ++i) mine += mass(r, clean(r.z[i]));
    scan[2 + tid] = mine;
    __syncthreads();
    if (tid == 0) {
      unsigned long long run = 0;
      for (int t = 0; t < kThreads; ++t) {
        const unsigned long long v = scan[2 + t];
        scan[2 + t] = run;
        run += v;
      }
    }
    __syncthreads();
    unsigned long long run = scan[2 + tid];
    if (run <= target && target < run + mine)
      for (int i = lo; i < hi; ++i) {
        run += mass(r, clean(r.z[i]));
        if (run > target) {
          scan[0] = (unsigned long long)i;
          break;
        }
      }
    __syncthreads();
    token = (int)scan[0];
  }
  token = min(max(token, 0), r.n - 1);
  if (tid == 0) {
    a.token[row] = token;
    if (a.logprob) {
      const float z = clean(r.z[token]);
      a.logprob[row] = (float)((z == r.zmax ? 0.0 : ((double)z - (double)r.zmax) * r.inv_t) - log((double)S / r.unit));
    }
  }
}

}  // namespace

ifx_status op_sample_rows(const SampleRowsArgs &a, cudaStream_t st) {
  if (!a.rows) return IFX_OK;
  sample_rows_kernel<<<(unsigned)a.rows, kThreads, 0, st>>>(a);
  IFX_CUDA(cudaGetLastError());
  return IFX_OK;
}

}  // namespace ifx
