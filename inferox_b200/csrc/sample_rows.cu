// Row-wise sampling: temperature, top-k, top-p and min-p from given random
// numbers. The rule of Sampler::sample (src/sampler.rs:28-73), for every row
// of a batch with its own settings, and min-p beside its filters.
//
// Mathematics. Weights w_i = exp((z_i - max) / T) are held as 64-bit integers
// w_i 2^s (s = 62 - bits of n, at most 50), so sums do not depend on the
// order of additions and a draw is the same in every layout. Nothing is
// sorted as a whole: in the order of falling z the kept tokens are a prefix,
// and the cut and the draw are each a place where a running count or mass
// passes a target. Such a place is found by a histogram over 2048 buckets of
// equal width in z (the last one takes all tokens whose weight rounds to 0),
// a gather of the bucket (or, when they are few, of all buckets up to it)
// and a sort of what was gathered.
//
// What bounds it. A row is read once (4 n bytes) into the shared memory of a
// cluster of CTAs, which keeps it for the passes that follow; the weights
// cost about 20 instructions in 64-bit floating point each, which overlap
// the reads of other rows. One row alone is bound by latency: five to seven
// cluster barriers.
#include <cooperative_groups.h>

#include <algorithm>

#include "serve.cuh"

namespace cg = cooperative_groups;

namespace ifx {

namespace {

using u64 = unsigned long long;

constexpr int kThreads = 512;
constexpr int kBuckets = 2048;
constexpr int kList = 2048;      // elements a gather can hold
constexpr int kMaxCluster = 8;
constexpr int kMaxChunk = 36864; // elements of a row that one CTA keeps in shared memory

// A NaN counts as a masked token; -0 and +0 are one value.
__device__ __forceinline__ float clean(float z) { return z != z ? -INFINITY : z + 0.f; }

__device__ __forceinline__ uint32_t ordered(float f) {
  const uint32_t b = __float_as_uint(f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k); }

struct Row {
  float zmax;
  double cut;        // this far below the maximum a weight rounds to 0
  double c, unit;    // 32 log2(e) / T; 2^s
  int s;
  const double *pow2;  // 2^(j / 32), in shared memory
};

// exp((z - zmax) / T) by table and polynomial: with x = (z - zmax) 32 log2(e)
// / T = 32 n + j + f, |f| <= 1/2, it is 2^n 2^(j/32) e^y, y = f ln2 / 32. Five
// terms of the series leave y^6 / 720 < 2^-48.
__device__ __forceinline__ double weight(const Row &r, float z) {
  if (z == r.zmax) return 1.0;
  const double d = (double)z - (double)r.zmax;
  if (!(-d < r.cut)) return 0.0;
  const double x = d * r.c;
  constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer
  const double k = x + kRound, f = x - (k - kRound);
  constexpr double y1 = 0.021660849392498290, y2 = y1 * y1 / 2, y3 = y2 * y1 / 3, y4 = y3 * y1 / 4, y5 = y4 * y1 / 5;
  const double e = fma(f, fma(f, fma(f, fma(f, fma(f, y5, y4), y3), y2), y1), 1.0);
  const int i = __double2loint(k);
  const double t = r.pow2[i & 31] * e;
  return __hiloint2double(__double2hiint(t) + (i >> 5) * (1 << 20), __double2loint(t));
}
__device__ __forceinline__ u64 to_mass(const Row &r, double w) {
  // w 2^s <= 2^50: adding 2^52 leaves the rounded integer in the low bits
  return (u64)__double_as_longlong(fma(w, r.unit, 4503599627370496.0)) - 0x4330000000000000ull;
}

// ------------------------------------------------ block-wide sums and scans
struct Shared {
  double pow2[32];
  u64 red[kThreads / 32];
  u64 best;            // this CTA's largest value and its last index
  u64 mass;            // this CTA's total mass
  u64 pick;
  int count, listed;   // tokens with w >= min_p; length of the list
  float zmax;
  int last;
  // the leader's orders to the cluster
  int cmd, level, b0, lo, hi;
};
enum { kDone, kHist, kGather };

__device__ __forceinline__ u64 block_sum(u64 v, Shared &sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.red[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 t = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) t += sh.red[i];
  return t;
}
// Sum of the lower threads' values.
__device__ __forceinline__ u64 block_before(u64 v, Shared &sh) {
  u64 inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 x = __shfl_up_sync(0xffffffffu, inc, o);
    if ((threadIdx.x & 31) >= o) inc += x;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 31) sh.red[threadIdx.x >> 5] = inc;
  __syncthreads();
  u64 base = inc - v;
  for (int i = 0; i < (int)(threadIdx.x >> 5); ++i) base += sh.red[i];
  return base;
}

// ------------------------------------------------------- the long way round
// For the leader alone, when more than kList tokens of one row share (nearly)
// one value: a radix search over the ordered bits of z, then the equal ones
// by index. Every pass reads the whole row again.
struct Bound {
  uint32_t key = 0;
  int idx = INT32_MAX;
};
__device__ bool within(const Bound &c, uint32_t k, int i) { return k > c.key || (k == c.key && i <= c.idx); }

// First token within c, in sorted order, at which the running count or mass
// reaches `target`; c is cut there. `sum` receives the running mass or count
// before that token. hist: 256 entries.
__device__ bool search(const Row &r, const float *z, int n, Bound &c, bool by_count, u64 target, u64 *hist, Shared &sh) {
  const int tid = threadIdx.x;
  uint32_t prefix = 0, mask = 0;
  u64 above = 0;
  const Bound c0 = c;
  for (int b = 24; b >= 0; b -= 8) {
    for (int j = tid; j < 256; j += kThreads) hist[j] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kThreads) {
      const float v = clean(z[i]);
      const uint32_t k = ordered(v);
      if ((k & mask) == prefix && within(c0, k, i)) atomicAdd(&hist[k >> b & 255u], by_count ? 1ull : to_mass(r, weight(r, v)));
    }
    __syncthreads();
    int sel = -1;
    for (int j = 255; j >= 0; --j) {
      if (above + hist[j] >= target) {
        sel = j;
        break;
      }
      above += hist[j];
    }
    __syncthreads();
    if (sel < 0) return false;
    prefix |= (uint32_t)sel << b;
    mask |= 255u << b;
  }
  const int per = (n + kThreads - 1) / kThreads, lo = min(n, tid * per), hi = min(n, lo + per);
  u64 mine = 0;
  for (int i = lo; i < hi; ++i) {
    const float v = clean(z[i]);
    if (ordered(v) == prefix && within(c0, prefix, i)) mine += by_count ? 1ull : to_mass(r, weight(r, v));
  }
  u64 run = above + block_before(mine, sh);
  if (tid == 0) sh.pick = (u64)INT32_MAX;
  __syncthreads();
  if (run < target && run + mine >= target)
    for (int i = lo; i < hi; ++i) {
      const float v = clean(z[i]);
      if (ordered(v) != prefix || !within(c0, prefix, i)) continue;
      run += by_count ? 1ull : to_mass(r, weight(r, v));
      if (run >= target) {
        sh.pick = (u64)i;
        break;
      }
    }
  __syncthreads();
  c.key = prefix;
  c.idx = (int)sh.pick;
  __syncthreads();
  return true;
}

__device__ int long_way(const Row &r, const float *z, int n, u64 k_eff, u64 p_mass, double u, u64 *hist, Shared &sh, u64 *kept) {
  const Bound all;
  Bound a = all, b = all;
  if (k_eff < (u64)n) search(r, z, n, a, true, k_eff, hist, sh);
  if (p_mass) search(r, z, n, b, false, p_mass, hist, sh);
  Bound c = a.key > b.key || (a.key == b.key && a.idx < b.idx) ? a : b;
  u64 m = 0;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const float v = clean(z[i]);
    if (within(c, ordered(v), i)) m += to_mass(r, weight(r, v));
  }
  *kept = block_sum(m, sh);
  const u64 target = min((u64)(u * (double)*kept), *kept - 1);
  search(r, z, n, c, false, target + 1, hist, sh);
  return c.idx;
}

// --------------------------------------------------------------- the kernel
// A cluster of gridDim.x CTAs per row. IN_SMEM: each CTA's share of the row
// stays in its shared memory; otherwise every pass reads it from global
// memory (rows beyond 8 * kMaxChunk tokens).
template <bool IN_SMEM>
__global__ void __launch_bounds__(kThreads) sample_rows_kernel(const __grid_constant__ SampleRowsArgs a) {
  extern __shared__ __align__(16) uint8_t sm[];
  __shared__ Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.y;
  const int n = (int)a.n, per = ((n + C - 1) / C + 3) & ~3, lo = min(n, rank * per), len = min(n, lo + per) - lo;
  const float *zrow = a.logits + row * a.stride;
  u64 *hmass = reinterpret_cast<u64 *>(sm);                       // [kBuckets]
  int *hcount = reinterpret_cast<int *>(hmass + kBuckets);        // [kBuckets]
  u64 *list = reinterpret_cast<u64 *>(hcount + kBuckets);         // [kList], the leader's
  float *zs = reinterpret_cast<float *>(list + kList);            // [per]
  auto value = [&](int i) { return IN_SMEM ? zs[i] : clean(zrow[lo + i]); };

  // ---- read the row; its largest value and the last index that has it
  float top = -INFINITY;
  int at = -1;
  auto see = [&](float z, int i) {
    if (z >= top) {
      top = z;
      at = i;
    }
  };
  if ((reinterpret_cast<uintptr_t>(zrow) & 15) == 0) {
    const float4 *src = reinterpret_cast<const float4 *>(zrow + lo);
    for (int i = tid; i < len / 4; i += kThreads) {
      float4 v = __ldcs(src + i);
      v = make_float4(clean(v.x), clean(v.y), clean(v.z), clean(v.w));
      if (IN_SMEM) reinterpret_cast<float4 *>(zs)[i] = v;
      see(v.x, 4 * i), see(v.y, 4 * i + 1), see(v.z, 4 * i + 2), see(v.w, 4 * i + 3);
    }
    for (int i = (len & ~3) + tid; i < len; i += kThreads) {
      const float z = clean(zrow[lo + i]);
      if (IN_SMEM) zs[i] = z;
      see(z, i);
    }
  } else {
    for (int i = tid; i < len; i += kThreads) {
      const float z = clean(zrow[lo + i]);
      if (IN_SMEM) zs[i] = z;
      see(z, i);
    }
  }
  u64 best = at < 0 ? 0 : (u64)ordered(top) << 32 | (uint32_t)(lo + at);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if (lane == 0) sh.red[warp] = best;
  if (tid < 32) sh.pow2[tid] = exp2((double)tid * 0.03125);
  for (int i = tid; i < kBuckets; i += kThreads) hmass[i] = 0, hcount[i] = 0;
  __syncthreads();
  if (tid == 0) {
    for (int i = 0; i < kThreads / 32; ++i) best = max(best, sh.red[i]);
    sh.best = best;
    sh.count = 0;
    sh.listed = 0;
  }
  cluster.sync();
  if (warp == 0) {
    best = lane < C ? cluster.map_shared_rank(&sh, lane)->best : 0;
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) {
      sh.last = (int)(uint32_t)best;
      sh.zmax = unordered((uint32_t)(best >> 32));
    }
  }
  __syncthreads();
  const float T = a.temperature ? a.temperature[row] : 1.f;
  Row r;
  r.zmax = sh.zmax;
  const int last = sh.last;
  const bool none = r.zmax == -INFINITY;
  if (none || !(T > 0.f)) {
    if (rank == 0 && tid == 0) {
      a.token[row] = none ? -1 : last;
      if (a.logprob) a.logprob[row] = none ? -INFINITY : 0.f;
    }
    cluster.sync();  // others may still read this CTA's maximum
    return;
  }
  r.s = min(50, 62 - (32 - __clz(n)));
  r.unit = __hiloint2double((1023 + r.s) << 20, 0);
  r.c = fmax(46.166241308446828 / (double)T, 1e-300);  // 32 log2(e) / T
  r.pow2 = sh.pow2;
  // below 2^-(s+2) of the maximum nothing counts
  r.cut = (r.s + 2) * 0.6931471805599453 * (double)T;
  const float scale = (float)(kBuckets - 1) / (float)r.cut;
  const int top_k = a.top_k ? a.top_k[row] : 0;
  const float top_p = a.top_p ? a.top_p[row] : 1.f, min_p = a.min_p ? fminf(a.min_p[row], 1.f) : 0.f;
  const double u = fmin(fmax((double)a.u[row], 0.0), 1.0);
  auto finish = [&](int token, u64 kept) {  // one thread of the leader
    a.token[row] = token;
    if (a.logprob) {
      const float z = clean(zrow[token]);
      const double t = z == r.zmax ? 0.0 : ((double)z - (double)r.zmax) * fmax(1.0 / (double)T, 1e-300);
      a.logprob[row] = (float)(t - log((double)kept / r.unit));
    }
  };

  if (top_k <= 0 && !(top_p < 1.f) && !(min_p > 0.f)) {
    // ---- no filter: the draw is in index order. Every warp sums a run of
    // its CTA's share; the one that holds the target walks its run again
    const int run = ((len + kThreads / 32 - 1) / (kThreads / 32) + 31) & ~31, w0 = min(len, warp * run), w1 = min(len, w0 + run);
    u64 m = 0;
    for (int i = w0 + lane; i < w1; i += 32) m += to_mass(r, weight(r, value(i)));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
    if (lane == 0) sh.red[warp] = m;
    __syncthreads();
    if (tid == 0) {
      u64 t = 0;
      for (int i = 0; i < kThreads / 32; ++i) t += sh.red[i];
      sh.mass = t;
    }
    cluster.sync();
    u64 total = 0, before = 0;
    for (int i = 0; i < C; ++i) {
      const u64 x = cluster.map_shared_rank(&sh, i)->mass;
      if (i < rank) before += x;
      total += x;
    }
    const u64 target = min((u64)(u * (double)total), total - 1);
    for (int i = 0; i < warp; ++i) before += sh.red[i];
    if (before <= target && target < before + m) {
      for (int i0 = w0; i0 < w1; i0 += 32) {
        const u64 x = i0 + lane < w1 ? to_mass(r, weight(r, value(i0 + lane))) : 0;
        u64 inc = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const u64 y = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += y;
        }
        const uint32_t over = __ballot_sync(0xffffffffu, before + inc > target);
        if (over) {
          if (lane == 0) finish(lo + i0 + __ffs(over) - 1, total);
          break;
        }
        before += __shfl_sync(0xffffffffu, inc, 31);
      }
    }
    cluster.sync();  // others may still read this CTA's mass
    return;
  }

  // ---- filters
  Shared *boss = cluster.map_shared_rank(&sh, 0);
  u64 *boss_list = cluster.map_shared_rank(list, 0);
  auto bucket = [&](float z) {
    const float d = z == r.zmax ? 0.f : r.zmax - z;
    return min(kBuckets - 1, (int)(d * scale));
  };
  auto within_bucket = [&](float z, int b) {  // a bucket's own buckets
    const float d = z == r.zmax ? 0.f : r.zmax - z;
    return min(kBuckets - 1, max(0, (int)(fmaf(d, scale, -(float)b) * kBuckets)));
  };
  // masses are needed for top-p, and where the cut may leave more than a list
  bool masses = top_p < 1.f || top_k <= 0 || top_k > kList / 2;
  // the leader's bookkeeping, the same in all its threads
  u64 total = 0, k_eff = 0, p_mass = 0, kept = 0, target = 0, cbase = 0, mbase = 0;
  bool drawing = false, first = true;
  int level = 0, b0 = 0, cmd = kHist, glo = 0, ghi = 0;
  for (;;) {
    if (cmd == kHist) {
      if (!first) {
        for (int i = tid; i < kBuckets; i += kThreads) hmass[i] = 0, hcount[i] = 0;
        __syncthreads();
      }
      int above = 0;
      for (int i = tid; i < len; i += kThreads) {
        const float z = value(i);
        int b = bucket(z);
        if (level) {
          if (b != b0) continue;
          b = within_bucket(z, b0);
        }
        atomicAdd(&hcount[b], 1);
        if (masses || (first && min_p > 0.f)) {
          const double w = weight(r, z);
          if (masses) {
            const u64 m = to_mass(r, w);
            if (m) atomicAdd(&hmass[b], m);
          }
          above += w >= (double)min_p;
        }
      }
      if (first && min_p > 0.f) {
        for (int o = 16; o > 0; o >>= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
        if (lane == 0) atomicAdd(&sh.count, above);
      }
    } else {  // kGather
      for (int i = tid; i < len; i += kThreads) {
        const float z = value(i);
        int b = bucket(z);
        if (level) {
          if (b != b0) continue;
          b = within_bucket(z, b0);
        }
        if (b >= glo && b <= ghi) {
          const int p = atomicAdd(&boss->listed, 1);
          if (p < kList) boss_list[p] = (u64)ordered(z) << 32 | (0xffffffffu - (uint32_t)(lo + i));
        }
      }
    }
    cluster.sync();
    if (rank == 0) {
      int next = -1, bc = -1;
      if (cmd == kHist) {
        // the cluster's histogram, then its running sums in place
        constexpr int kPer = kBuckets / kThreads;
        u64 c[kPer], m[kPer], cs = 0, ms = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) c[j] = m[j] = 0;
        for (int k = 0; k < C; ++k) {
          const int *rc = cluster.map_shared_rank(hcount, k) + tid * kPer;
          const u64 *rm = cluster.map_shared_rank(hmass, k) + tid * kPer;
#pragma unroll
          for (int j = 0; j < kPer; ++j) {
            c[j] += rc[j];
            if (masses) m[j] += rm[j];
          }
        }
#pragma unroll
        for (int j = 0; j < kPer; ++j) cs += c[j], ms += m[j];
        u64 cb = block_before(cs, sh), mb = masses ? block_before(ms, sh) : 0;
        // hcount / hmass: sums up to and with a bucket, within this level
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          cb += c[j], mb += m[j];
          hcount[tid * kPer + j] = (int)cb;
          hmass[tid * kPer + j] = mb;
        }
        __syncthreads();
        if (level == 0) {
          total = hmass[kBuckets - 1];
          cbase = mbase = 0;
        }
        if (first) {
          k_eff = top_k > 0 ? min(top_k, n) : n;
          if (min_p > 0.f) {
            u64 k = 0;
            for (int i = 0; i < C; ++i) k += cluster.map_shared_rank(&sh, i)->count;
            k_eff = min(k_eff, max(k, 1ull));
          }
        }
        if (top_p < 1.f && !p_mass) p_mass = max((u64)ceil(fmax((double)top_p, 0.0) * (double)total), 1ull);
      }
      const bool had_hist = cmd == kHist;
      if (had_hist) {
        // ---- the bucket in which the count reaches k_eff, or the mass p_mass
        // (the cut), or in which the mass passes the draw's target
        int mine = kBuckets;
        for (int i = tid; i < kBuckets; i += kThreads) {
          const u64 cc = cbase + (u64)hcount[i], mm = mbase + hmass[i];
          const bool hit = drawing ? mm > target : cc >= k_eff || (p_mass && mm >= p_mass);
          if (hit) {
            mine = i;
            break;
          }
        }
        for (int o = 16; o > 0; o >>= 1) mine = min(mine, __shfl_xor_sync(0xffffffffu, mine, o));
        __syncthreads();
        if (lane == 0) sh.red[warp] = mine;
        __syncthreads();
        bc = kBuckets;
        for (int i = 0; i < kThreads / 32; ++i) bc = min(bc, (int)sh.red[i]);
        if (!drawing && level == 0 && bc >= kBuckets - 1) {
          // no cut among the tokens that count
          if (!masses) {
            masses = true;
            next = kHist;
          } else {
            kept = total;
            target = min((u64)(u * (double)kept), kept - 1);
            drawing = true;
            mine = kBuckets;
            for (int i = tid; i < kBuckets; i += kThreads)
              if (hmass[i] > target) {
                mine = i;
                break;
              }
            for (int o = 16; o > 0; o >>= 1) mine = min(mine, __shfl_xor_sync(0xffffffffu, mine, o));
            __syncthreads();
            if (lane == 0) sh.red[warp] = mine;
            __syncthreads();
            bc = kBuckets;
            for (int i = 0; i < kThreads / 32; ++i) bc = min(bc, (int)sh.red[i]);
          }
        }
        if (next < 0) {
          bc = min(bc, kBuckets - 1);
          const int upto = hcount[bc], alone = upto - (bc ? hcount[bc - 1] : 0);
          if (!drawing && level == 0 && upto <= kList) {
            next = kGather;
            glo = 0;
            ghi = bc;
            cbase = mbase = 0;
          } else if (!masses) {
            masses = true;  // what lies before the bucket is needed
            next = kHist;
          } else if (alone <= kList || level == 0) {
            if (bc) cbase += (u64)hcount[bc - 1], mbase += hmass[bc - 1];
            if (alone <= kList) {
              next = kGather;
              glo = ghi = bc;
            } else {
              next = kHist;
              level = 1;
              b0 = bc;
            }
          } else {
            const int token = long_way(r, zrow, n, k_eff, p_mass, u, hmass, sh, &kept);
            if (tid == 0) finish(min(max(token, 0), n - 1), kept);
            next = kDone;
          }
        }
      } else {
        // ---- sort what was gathered (falling value, rising index), running masses
        const int cnt = min(sh.listed, kList);
        int size = 2;
        while (size < cnt) size <<= 1;
        for (int i = cnt + tid; i < size; i += kThreads) list[i] = 0;
        __syncthreads();
        for (int k = 2; k <= size; k <<= 1)
          for (int j = k >> 1; j > 0; j >>= 1) {
            for (int e = tid; e < size / 2; e += kThreads) {
              const int x = 2 * e - (e & (j - 1)), y = x + j;
              const u64 p = list[x], q = list[y];
              if ((p < q) == ((x & k) == 0)) list[x] = q, list[y] = p;
            }
            __syncthreads();
          }
        constexpr int kPer = kList / kThreads;
        u64 m[kPer], ms = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const int i = tid * kPer + j;
          m[j] = i < cnt ? to_mass(r, weight(r, unordered((uint32_t)(list[i] >> 32)))) : 0;
          ms += m[j];
        }
        const u64 before = mbase + block_before(ms, sh);
        if (!drawing) {
          // how many are kept, and their mass
          u64 keep = k_eff - min(k_eff, cbase), run = before;
          if (tid == 0) sh.pick = min(keep, (u64)cnt);
          __syncthreads();
          if (p_mass) {
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
              if (run < p_mass && run + m[j] >= p_mass) atomicMin(&sh.pick, (u64)(tid * kPer + j + 1));
              run += m[j];
            }
          }
          __syncthreads();
          keep = sh.pick;
          u64 inside = 0;
#pragma unroll
          for (int j = 0; j < kPer; ++j)
            if ((u64)(tid * kPer + j) < keep) inside += m[j];
          kept = mbase + block_sum(inside, sh);
          target = min((u64)(u * (double)kept), kept - 1);
          drawing = true;
        }
        if (target >= mbase) {
          u64 run = before;
#pragma unroll
          for (int j = 0; j < kPer; ++j) {
            if (run <= target && target < run + m[j])
              finish((int)(0xffffffffu - (uint32_t)list[tid * kPer + j]), kept);
            run += m[j];
          }
          next = kDone;
        } else {
          // the draw falls before the cut's bucket: find its own
          next = kHist;
          level = 0;
        }
      }
      __syncthreads();
      if (tid == 0) {
        sh.cmd = next;
        sh.level = level;
        sh.b0 = b0;
        sh.lo = glo;
        sh.hi = ghi;
        sh.listed = 0;
        sh.count = masses;
      }
    }
    cluster.sync();
    cmd = boss->cmd;
    level = boss->level;
    b0 = boss->b0;
    glo = boss->lo;
    ghi = boss->hi;
    masses = boss->count;
    first = false;
    if (cmd == kDone) break;
    cluster.sync();  // the orders are read before the leader gives new ones
  }
  cluster.sync();  // the leader's orders are read before it leaves
}

template <bool IN_SMEM>
ifx_status run(const SampleRowsArgs &a, int cluster, size_t smem, cudaStream_t st) {
  auto kernel = sample_rows_kernel<IN_SMEM>;
  if (smem > 48 * 1024) IFX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024));
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  SampleRowsArgs part = a;
  for (int64_t at = 0; at < a.rows; at += 65535) {  // grid.y
    part.rows = std::min<int64_t>(65535, a.rows - at);
    part.logits = a.logits + at * a.stride;
    part.u = a.u + at;
    part.temperature = a.temperature ? a.temperature + at : nullptr;
    part.top_k = a.top_k ? a.top_k + at : nullptr;
    part.top_p = a.top_p ? a.top_p + at : nullptr;
    part.min_p = a.min_p ? a.min_p + at : nullptr;
    part.token = a.token + at;
    part.logprob = a.logprob ? a.logprob + at : nullptr;
    cfg.gridDim = dim3((unsigned)cluster, (unsigned)part.rows);
    IFX_CUDA(cudaLaunchKernelEx(&cfg, kernel, part));
  }
  return IFX_OK;
}

}  // namespace

ifx_status op_sample_rows(const SampleRowsArgs &a, cudaStream_t st) {
  if (!a.rows) return IFX_OK;
  // the CTAs of a row: eight while a CTA then has 2048 tokens or more
  int cluster = 1;
  while (cluster < kMaxCluster && a.n > (int64_t)cluster * 2048) cluster *= 2;
  const int64_t per = ((a.n + cluster - 1) / cluster + 3) & ~(int64_t)3;
  const size_t base = kBuckets * (sizeof(u64) + sizeof(int)) + kList * sizeof(u64);
  if (per <= kMaxChunk) return run<true>(a, cluster, base + (size_t)per * sizeof(float), st);
  return run<false>(a, cluster, base, st);
}

}  // namespace ifx
