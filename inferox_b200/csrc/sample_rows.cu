// Row-wise sampling: temperature, top-k, top-p and min-p from given random
// numbers. The rule of Sampler::sample (src/sampler.rs:28-73), for every row
// of a batch with its own settings, and min-p beside its filters.
//
// Mathematics. Weights w_i = exp((z_i - max) / T) are held as 64-bit integers
// w_i 2^s (s = 62 - bits of n, at most 50), so sums do not depend on the
// order of additions and a draw is the same in every layout. Nothing is
// sorted as a whole: in the order of falling z the kept tokens are a prefix,
// and the cut and the draw are each a place where a running count or mass
// passes a target. Tokens are counted in 2048 buckets of equal width in z
// (the last one takes all whose weight rounds to 0). A bucket is so narrow
// that its count times the weight of its middle is its mass to 1%: that
// guesses the place, and one pass that sums the masses before a window of 16
// buckets and of each bucket in it makes it exact. The bucket (or, when they
// are few, all up to it) is gathered and sorted.
//
// What bounds it. A row is read once (4 n bytes) into the shared memory of a
// cluster of CTAs, which keeps it for the passes that follow; the weights
// cost about 20 instructions each, 11 of them in 64-bit floating point (an
// SM does two warps' worth a clock), which overlap the reads of other rows.
// One row alone is bound by latency: a cluster barrier takes 1 us. Measured:
// one row of 32000 16 us; 64 rows of 128256 with all filters 94 us (0.35
// TB/s of logits); 256 rows without a filter 103 us (1.28 TB/s).
#include <cooperative_groups.h>

#include <algorithm>
#include <utility>

#include "serve.cuh"

namespace cg = cooperative_groups;

namespace ifx {

namespace {

using u64 = unsigned long long;

constexpr int kThreads = 512;
constexpr int kBuckets = 2048;
constexpr int kList = 2048;      // elements a gather can hold
constexpr int kWindow = 16;      // buckets whose masses one pass makes exact
constexpr int kMaxCluster = 8;
constexpr int kMaxChunk = 36864; // elements of a row that one CTA keeps in shared memory

// A NaN counts as a masked token; -0 and +0 are one value.
__device__ __forceinline__ float clean(float z) { return z != z ? -INFINITY : z + 0.f; }

__device__ __forceinline__ uint32_t ordered(float f) {
  const uint32_t b = __float_as_uint(f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k); }

constexpr uint32_t kLost = 0xffffffffu;  // in place of a largest value's bits (a NaN's, which no maximum has)

__device__ const double kPow2[32] = {  // 2^(j / 32)
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237,
    1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228,
    1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.6457554781539649,
    1.681792830507429, 1.7186192981224779, 1.7562521603732995, 1.7947090750031072,
    1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002};
__device__ const double kPow2Fine[4] = {1.0, 1.0054299011128027, 1.0108892860517005, 1.016378314910953};  // 2^(j / 128)

struct Row {
  float zmax;
  double cut;        // this far below the maximum a weight rounds to 0
  float zcut;        // a value from which on below nothing counts
  double c, unit;    // 128 log2(e) / T; 2^s
  int s;
  const double *pow2;  // 2^(j / 128), in shared memory
};

// exp((z - zmax) / T) by table and polynomial: with x = (z - zmax) 128 log2(e)
// / T = 128 n + j + f, |f| <= 1/2, it is 2^n 2^(j/128) e^y, y = f ln2 / 128.
// Four terms of the series leave y^5 / 120 < 2^-49.
__device__ __forceinline__ double weight(const Row &r, float z) {
  const double d = (double)z - (double)r.zmax;
  const double x = d * r.c;
  constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer
  const double k = x + kRound, f = x - (k - kRound);
  constexpr double y1 = 0.0054152123481245725, y2 = y1 * y1 / 2, y3 = y2 * y1 / 3, y4 = y3 * y1 / 4;
  const double e = fma(f, fma(f, fma(f, fma(f, y4, y3), y2), y1), 1.0);
  const int i = __double2loint(k);
  const double t = r.pow2[i & 127] * e;
  const double w = __hiloint2double(__double2hiint(t) + (i >> 7) * (1 << 20), __double2loint(t));
  return z == r.zmax ? 1.0 : z >= r.zcut ? w : 0.0;
}
__device__ __forceinline__ u64 to_mass(const Row &r, double w) {
  // w 2^s <= 2^50: adding 2^52 leaves the rounded integer in the low bits
  return (u64)__double_as_longlong(fma(w, r.unit, 4503599627370496.0)) - 0x4330000000000000ull;
}

// ------------------------------------------------ block-wide sums and scans
// What the leader CTA knows, kept in shared memory between its turns.
struct Book {
  u64 total = 0, gtotal = 0;   // the row's mass, exact and guessed
  u64 k_eff = 0, p_mass = 0;   // the count and the mass that are kept (0: no top-p)
  u64 kept = 0, target = 0;    // kept mass, and the draw's place in it
  u64 cbase = 0, mbase = 0;    // count and mass before what is gathered
  u64 cup = 0, mup = 0;        // ... before the bucket that level 1 splits
  int drawing = 0, whole_list = 0, tries = 0;
};

// One row's task: the logits, the settings, where the answer goes.
struct Task {
  Row row;
  const float *z;
  int *token;
  float *logprob;
  double u, inv_t;
  float top_p, min_p;
  int n, top_k;
};

struct Shared {
  Task task;
  Book book;
  double pow2[128];
  u64 red[kThreads / 32];
  u64 best;            // this CTA's largest value (ordered bits)
  u64 mass;            // this CTA's mass: of all its tokens, or before the window
  u64 window[kWindow]; // ... and of each bucket in it
  u64 parts[kThreads / 32][kWindow];  // the same by warp
  u64 pick;
  int count, listed;   // tokens with w >= min_p; length of the list
  int place;
  int last;            // greedy rows: the last index of the largest value
  // the leader's orders to the cluster
  int cmd, level, b0, lo, hi, masses, first;
};
enum { kDone, kHist, kMass, kGather };

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
  const int lane = threadIdx.x & 31;
  u64 inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 x = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += x;
  }
  __syncthreads();
  if (lane == 31) sh.red[threadIdx.x >> 5] = inc;
  __syncthreads();
  u64 base = inc - v;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) base += i < (int)(threadIdx.x >> 5) ? sh.red[i] : 0;
  return base;
}
__device__ __forceinline__ int block_min(int v, Shared &sh) {
  v = __reduce_min_sync(0xffffffffu, v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.red[threadIdx.x >> 5] = (u64)v;
  __syncthreads();
  int m = (int)sh.red[0];
#pragma unroll
  for (int i = 1; i < kThreads / 32; ++i) m = min(m, (int)sh.red[i]);
  return m;
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

// ------------------------------------------------------- the leader's turn
// Between two passes of the cluster the leader CTA reads what the pass found
// and gives the next orders. A function of its own, so that its registers
// are not held during the passes.
__device__ __forceinline__ void finish(const Task &t, int token, u64 kept) {  // one thread
  *t.token = token;
  if (t.logprob) {
    const float z = clean(t.z[token]);
    const double x = z == t.row.zmax ? 0.0 : ((double)z - (double)t.row.zmax) * t.inv_t;
    *t.logprob = (float)(x - log((double)kept / t.row.unit));
  }
}

__device__ __noinline__ void leader_turn(Shared &sh, u64 *list, u64 *guess, int *hcount) {
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), tid = threadIdx.x;
  const Task &t = sh.task;
  const Row &r = t.row;
  const int n = t.n, cmd = sh.cmd;
  int level = sh.level, b0 = sh.b0, glo = sh.lo, ghi = sh.hi;
  bool masses = sh.masses;
  const bool first = sh.first;
  Book k = sh.book;
  int next = -1;
  constexpr int kPer = kBuckets / kThreads;
  // the sum over the cluster's CTAs of what `get` reads
  auto over = [&](auto get) {
    const int lane = tid & 31;
    u64 v = lane < C ? get(cluster.map_shared_rank(&sh, lane)) : 0;
#pragma unroll
    for (int o = kMaxCluster / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return __shfl_sync(0xffffffffu, v, 0);
  };
  // first bucket that fulfils a condition that, once met, stays met
  auto find = [&](auto cond) {
    int mine = kBuckets;
#pragma unroll
    for (int j = kPer - 1; j >= 0; --j)
      if (cond(tid * kPer + j)) mine = tid * kPer + j;
    return block_min(mine, sh);
  };
  auto before_bucket = [&](int b) { return b > 0 ? (u64)hcount[b - 1] : 0ull; };
  // a window around the bucket where the guessed masses reach `want`
  // beyond bucket `from`, whose mass in front is `have`
  auto aim = [&](u64 want, int from, u64 have, int most) {
    const double f = k.total ? (double)k.gtotal / (double)k.total : 1.0, g0 = from > 0 ? (double)guess[from - 1] : 0.0;
    const double x = g0 + ((double)want - (double)have) * (level ? 1.0 : f);
    const int b = min(find([&](int i) { return (double)guess[i] >= x; }), most);
    glo = max(0, min(b, kBuckets - 1) - kWindow / 2);
    next = kMass;
  };
  int bk = kBuckets;  // the bucket in which the count reaches k_eff
  if (cmd == kHist) {
    // the cluster's counts, running sums in place, and the guessed masses
    // (loads from another CTA take a microsecond: all of them at once)
    int c[kPer] = {};
    static_assert(kPer == 4, "");
    int4 x[kMaxCluster];
#pragma unroll
    for (int q = 0; q < kMaxCluster; ++q) x[q] = reinterpret_cast<const int4 *>(cluster.map_shared_rank(hcount, min(q, C - 1)))[tid];
#pragma unroll
    for (int q = 0; q < kMaxCluster; ++q)
      if (q < C) c[0] += x[q].x, c[1] += x[q].y, c[2] += x[q].z, c[3] += x[q].w;
    if (level == 0 && masses) k.total = over([](const Shared *p) { return p->mass; });
    if (first) {
      k.k_eff = t.top_k > 0 ? min(t.top_k, n) : n;
      if (t.min_p > 0.f) {
        const u64 above = over([](const Shared *p) { return (u64)p->count; });
        k.k_eff = min(k.k_eff, max(above, 1ull));
      }
    }
    if (t.top_p < 1.f) k.p_mass = max((u64)ceil(fmax((double)t.top_p, 0.0) * (double)k.total), 1ull);
    u64 g[kPer], cs = 0, gs = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      // level 1: parts of one bucket weigh the same
      const float mid = level ? (float)b0 + 0.5f : (float)(tid * kPer + j) + 0.5f;
      const float w = exp2f(-mid * ((float)(r.s + 2) / (float)(kBuckets - 1)));
      g[j] = (u64)((double)c[j] * (double)w * r.unit);
      cs += (u64)c[j];
      gs += g[j];
    }
    u64 cb = block_before(cs, sh), gb = block_before(gs, sh);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      cb += (u64)c[j], gb += g[j];
      hcount[tid * kPer + j] = (int)cb;
      guess[tid * kPer + j] = gb;
    }
    __syncthreads();
    k.gtotal = guess[kBuckets - 1];
    if (level == 0) k.cup = k.mup = 0;
    k.tries = 0;
  }
  if (cmd != kGather && !k.drawing) {
    bk = find([&](int i) { return k.cup + (u64)hcount[i] >= k.k_eff; });
    if (level == 0 && bk == kBuckets - 1) bk = kBuckets;  // cuts off nothing that counts
  }
  if (cmd == kHist) {
    if (k.drawing) {
      aim(k.target + 1, 0, k.mup, kBuckets - 1);
    } else if (level == 0 && bk == kBuckets && !k.p_mass) {
      if (!masses) {  // fewer tokens than top_k: all masses are needed after all
        masses = true;
        next = kHist;
      } else {
        k.kept = k.total;
        k.target = min((u64)(t.u * (double)k.kept), k.kept - 1);
        k.drawing = true;
        aim(k.target + 1, 0, 0, kBuckets - 1);
      }
    } else {
      // when few: all of them, up to the cut (for top-p a little beyond its guess)
      int upto = bk;
      if (level == 0 && k.p_mass) {
        const double x = (double)k.p_mass * 1.03 * ((double)k.gtotal / (double)k.total);
        upto = min(upto, find([&](int i) { return (double)guess[i] >= x; }));
      }
      upto = min(upto, kBuckets - 2);
      if (level == 0 && hcount[upto] <= kList) {
        next = kGather;
        glo = 0;
        ghi = upto;
        k.cbase = k.mbase = 0;
        k.whole_list = true;
      } else if (!masses) {
        masses = true;  // what lies before the cut's bucket is needed
        next = kHist;
      } else if (k.p_mass) {
        aim(k.p_mass, 0, k.mup, bk);
      } else {
        glo = max(0, bk - kWindow / 2);
        next = kMass;
      }
    }
  } else if (cmd == kMass) {
    // ---- exact masses around the guess
    const u64 e = k.mup + over([](const Shared *p) { return p->mass; });
    u64 mine = 0;
    if (tid < kWindow) {
      u64 x[kMaxCluster];
#pragma unroll
      for (int q = 0; q < kMaxCluster; ++q) x[q] = cluster.map_shared_rank(&sh, min(q, C - 1))->window[tid];
#pragma unroll
      for (int q = 0; q < kMaxCluster; ++q) mine += q < C ? x[q] : 0;
    }
    const u64 front = e + block_before(mine, sh), back = front + mine;
    const u64 want = k.drawing ? k.target + 1 : k.p_mass;
    int hit = kBuckets;
    if (tid < kWindow && glo + tid < kBuckets && want && back >= want) hit = glo + tid;
    hit = block_min(hit, sh);
    const int end = min(kBuckets, glo + kWindow);
    int b = kBuckets;
    if (want && e >= want) {
      b = -1;  // before the window
    } else {
      b = min(hit, k.drawing ? kBuckets : bk);
      if (b >= end) b = kBuckets;  // behind it
    }
    if (b >= 0 && b < kBuckets) {
      __syncthreads();
      if (tid == b - glo) sh.pick = front;
      __syncthreads();
      const u64 alone = (u64)hcount[b] - before_bucket(b);
      k.cbase = k.cup + before_bucket(b);
      k.mbase = sh.pick;
      if (alone <= kList) {
        next = kGather;
        glo = ghi = b;
        k.whole_list = false;
      } else if (level == 0) {
        next = kHist;
        level = 1;
        b0 = b;
        k.cup = k.cbase, k.mup = k.mbase;
      }
    } else if (++k.tries < 32) {
      // aim again from this window's exact edge
      __syncthreads();
      if (tid == kWindow - 1) sh.pick = back;
      __syncthreads();
      const u64 edge = sh.pick;
      const int was = glo;
      if (b < 0) {
        aim(want, was, e, kBuckets - 1);
        glo = max(0, min(glo, was - kWindow));
      } else {
        aim(want ? want : edge, end, edge, k.drawing ? kBuckets - 1 : bk);
        glo = max(glo, min(end, kBuckets - 1));
      }
    }
  } else {
    // ---- sort what was gathered (falling value, rising index), running masses
    const int cnt = min(sh.listed, kList);
    u64 *sorted = list;
    if (cnt <= kThreads) {
      // each thread counts the elements before its own, two a load (at 512
      // elements as long as the sort, and four times for twice as many)
      sorted = list + kList / 2;
      if (tid == 0 && (cnt & 1)) list[cnt] = 0;
      __syncthreads();
      if ((tid & ~31) < cnt) {
        const u64 x = tid < cnt ? list[tid] : 0;
        int px = 0;
#pragma unroll 4
        for (int i = 0; i < cnt; i += 2) {
          const ulonglong2 q = *reinterpret_cast<const ulonglong2 *>(list + i);
          px += (q.x > x) + (q.y > x);
        }
        if (tid < cnt) sorted[px] = x;
      }
      __syncthreads();
    } else {
      int size = 2 * kThreads;
      while (size < cnt) size <<= 1;
      for (int i = cnt + tid; i < size; i += kThreads) list[i] = 0;
      __syncthreads();
      for (int half = 2; half <= size; half <<= 1)
        for (int j = half >> 1; j > 0; j >>= 1) {
          for (int e = tid; e < size / 2; e += kThreads) {
            const int x = 2 * e - (e & (j - 1)), y = x + j;
            const u64 p = list[x], q = list[y];
            if ((p < q) == ((x & half) == 0)) list[x] = q, list[y] = p;
          }
          __syncthreads();
        }
    }
    const int each = cnt <= kThreads ? 1 : cnt <= 2 * kThreads ? 2 : kList / kThreads;
    u64 m[kList / kThreads], ms = 0;
#pragma unroll
    for (int j = 0; j < kList / kThreads; ++j) {
      const int i = tid * each + j;
      m[j] = j < each && i < cnt ? to_mass(r, weight(r, unordered((uint32_t)(sorted[i] >> 32)))) : 0;
      ms += m[j];
    }
    const u64 before = k.mbase + block_before(ms, sh);
    bool cut = true;
    if (!k.drawing) {
      // how many are kept, and their mass
      const u64 room = k.k_eff - min(k.k_eff, k.cbase);
      u64 keep = min(room, (u64)cnt), run = before;
      if (tid == 0) sh.pick = kList + 1;
      __syncthreads();
      if (k.p_mass) {
#pragma unroll
        for (int j = 0; j < kList / kThreads; ++j) {
          if (run < k.p_mass && run + m[j] >= k.p_mass) sh.pick = (u64)(tid * each + j + 1);
          run += m[j];
        }
      }
      __syncthreads();
      const u64 by_mass = sh.pick;
      cut = !k.whole_list || by_mass <= kList || room <= (u64)cnt;
      keep = min(keep, by_mass);
      u64 inside = 0;
#pragma unroll
      for (int j = 0; j < kList / kThreads; ++j)
        if ((u64)(tid * each + j) < keep) inside += m[j];
      k.kept = k.mbase + block_sum(inside, sh);
      k.target = min((u64)(t.u * (double)k.kept), k.kept - 1);
    }
    if (!cut) {
      // the mass was not reached: where it is needs exact sums
      bk = find([&](int i) { return k.cup + (u64)hcount[i] >= k.k_eff; });
      aim(k.p_mass, 0, 0, bk);
    } else {
      k.drawing = true;
      if (k.target >= k.mbase) {
        u64 run = before;
#pragma unroll
        for (int j = 0; j < kList / kThreads; ++j) {
          if (run <= k.target && k.target < run + m[j])
            finish(t, (int)(0xffffffffu - (uint32_t)sorted[tid * each + j]), k.kept);
          run += m[j];
        }
        next = kDone;
      } else if (level == 0) {
        k.tries = 0;
        k.mup = k.cup = 0;
        aim(k.target + 1, 0, 0, kBuckets - 1);
      } else {
        next = kHist;  // the draw falls before the bucket that was split
        level = 0;
      }
    }
  }
  if (next < 0) {
    const int token = long_way(r, t.z, n, k.k_eff, k.p_mass, t.u, guess, sh, &k.kept);
    if (tid == 0) finish(t, min(max(token, 0), n - 1), k.kept);
    next = kDone;
  }
  __syncthreads();
  if (tid == 0) {
    sh.book = k;
    sh.cmd = next;
    sh.level = level;
    sh.b0 = b0;
    sh.lo = glo;
    sh.hi = ghi;
    sh.masses = masses;
    sh.first = 0;
    sh.listed = 0;
  }
}

// --------------------------------------------------------------- the kernel
// A cluster of gridDim.x CTAs per row. IN_SMEM: each CTA's share of the row
// stays in its shared memory; otherwise every pass reads it from global
// memory (rows beyond 8 * kMaxChunk tokens).
template <bool IN_SMEM, int PER_SM>
__global__ void __launch_bounds__(kThreads, PER_SM) sample_rows_kernel(const __grid_constant__ SampleRowsArgs a) {
  extern __shared__ __align__(16) uint8_t sm[];
  __shared__ Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.y;
  const int n = (int)a.n, per = ((n + C - 1) / C + 3) & ~3, lo = min(n, rank * per), len = min(n, lo + per) - lo;
  const float *zrow = a.logits + row * a.stride;
  u64 *list = reinterpret_cast<u64 *>(sm);                        // [kList], the leader's
  u64 *guess = list + kList;                                      // [kBuckets], the leader's
  int *hcount = reinterpret_cast<int *>(guess + kBuckets);        // [kBuckets]
  float *zs = reinterpret_cast<float *>(hcount + kBuckets);       // [per]
  auto value = [&](int i) { return IN_SMEM ? zs[i] : clean(zrow[lo + i]); };
  auto four = [&](int i) {  // values i .. i + 3 (i a multiple of 4), NaN behind the last
    float4 v;
    if (IN_SMEM) {
      v = *reinterpret_cast<const float4 *>(zs + i);
    } else {
      v.x = value(i);
      v.y = i + 1 < len ? value(i + 1) : 0.f;
      v.z = i + 2 < len ? value(i + 2) : 0.f;
      v.w = i + 3 < len ? value(i + 3) : 0.f;
    }
    const float none = __uint_as_float(0x7fc00000u);
    if (i + 4 > len) {
      if (i + 1 >= len) v.y = none;
      if (i + 2 >= len) v.z = none;
      if (i + 3 >= len) v.w = none;
    }
    return v;
  };

  const float T = a.temperature ? a.temperature[row] : 1.f, top_p = a.top_p ? a.top_p[row] : 1.f;
  const float want_p = a.min_p ? a.min_p[row] : 0.f, min_p = want_p > 0.f ? fminf(want_p, 1.f) : 0.f, u_row = a.u[row];
  const int top_k = a.top_k ? a.top_k[row] : 0;
  // ---- read the row (by bulk copies where it is kept); its largest value
  const bool wide = (reinterpret_cast<uintptr_t>(zrow) & 15) == 0;
  __shared__ __align__(8) uint64_t bar;
  if (tid == 0) {
    sh.best = 0;
    if (IN_SMEM && wide) {
      mbar_init(&bar, 1);
      fence_mbar_init();
      const uint32_t bytes = (uint32_t)len / 4 * 16;
      if (bytes) {
        mbar_arrive_expect_tx(&bar, bytes);
        for (uint32_t at = 0; at < bytes; at += 16384)
          bulk_g2s(reinterpret_cast<uint8_t *>(zs) + at, reinterpret_cast<const uint8_t *>(zrow + lo) + at, min(16384u, bytes - at), &bar);
      } else {
        mbar_arrive(&bar);
      }
    }
  }
  if (tid < 128) sh.pow2[tid] = kPow2[tid / 4] * kPow2Fine[tid % 4];
  __syncthreads();
  float top = -INFINITY;
  if (IN_SMEM && wide) {
    // kept as it is: a NaN is in no bucket and has no weight, -0 equals +0
    // until the sort
    if (!mbar_wait(&bar, 0, a.err, kErrSample)) atomicMax(&sh.best, (u64)kLost);
#pragma unroll 4
    for (int i = tid; i < len / 4; i += kThreads) {
      const float4 v = reinterpret_cast<const float4 *>(zs)[i];
      top = fmaxf(top, fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)));
    }
    for (int i = (len & ~3) + tid; i < len; i += kThreads) {
      const float z = zrow[lo + i];
      zs[i] = z;
      top = fmaxf(top, z);
    }
    top += 0.f;
  } else if (wide) {
    const float4 *src = reinterpret_cast<const float4 *>(zrow + lo);
#pragma unroll 4
    for (int i = tid; i < len / 4; i += kThreads) {
      float4 v = __ldcs(src + i);
      v = make_float4(clean(v.x), clean(v.y), clean(v.z), clean(v.w));
      if (IN_SMEM) reinterpret_cast<float4 *>(zs)[i] = v;
      top = fmaxf(top, fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)));
    }
    for (int i = (len & ~3) + tid; i < len; i += kThreads) {
      const float z = clean(zrow[lo + i]);
      if (IN_SMEM) zs[i] = z;
      top = fmaxf(top, z);
    }
  } else {
    for (int i = tid; i < len; i += kThreads) {
      const float z = clean(zrow[lo + i]);
      if (IN_SMEM) zs[i] = z;
      top = fmaxf(top, z);
    }
  }
  const uint32_t mine = __reduce_max_sync(0xffffffffu, ordered(top));
  if (lane == 0) atomicMax(&sh.best, (u64)mine);
  for (int i = tid; i < kBuckets; i += kThreads) hcount[i] = 0;
  if (tid == 0) {
    sh.count = 0;
    sh.listed = 0;
  }
  Row r;
  r.s = min(50, 62 - (32 - __clz(n)));
  r.unit = __hiloint2double((1023 + r.s) << 20, 0);
  r.c = fmax(184.6649652337873 / (double)T, 1e-300);  // 128 log2(e) / T
  r.pow2 = sh.pow2;
  // below 2^-(s+2) of the maximum nothing counts
  r.cut = (r.s + 2) * 0.6931471805599453 * (double)T;
  const float scale = (float)(kBuckets - 1) / (float)r.cut;
  const double u = fmin(fmax((double)u_row, 0.0), 1.0);
  cluster.sync();
  const uint32_t most = __reduce_max_sync(0xffffffffu, lane < C ? (uint32_t)cluster.map_shared_rank(&sh, lane)->best : 0u);
  if (most == kLost) {
    // a copy did not come: no token, and no CTA leaves before its copy is over
    // and the others have read that
    if (IN_SMEM && wide) mbar_wait(&bar, 0, nullptr, 0);
    if (rank == 0 && tid == 0) {
      a.token[row] = -1;
      if (a.logprob) a.logprob[row] = __uint_as_float(0x7fc00000u);
    }
    cluster.sync();
    return;
  }
  r.zmax = unordered(most);
  // (no infinity counts but as the maximum)
  r.zcut = r.zmax == INFINITY ? INFINITY : fmaxf((float)((double)r.zmax - 1.01 * r.cut), -3.402823466e38f);
  const bool none = r.zmax == -INFINITY;
  if (none || !(T > 0.f)) {
    // nothing to draw, or the largest value: its last index
    int at = -1;
    if (!none)
      for (int i = tid; i < len; i += kThreads)
        if (value(i) == r.zmax) at = lo + i;
    at = __reduce_max_sync(0xffffffffu, at);
    __syncthreads();
    if (tid == 0) sh.last = -1;
    __syncthreads();
    if (lane == 0) atomicMax(&sh.last, at);
    cluster.sync();
    if (rank == 0 && tid == 0) {
      for (int i = 0; i < C; ++i) at = max(at, cluster.map_shared_rank(&sh, i)->last);
      a.token[row] = at;
      if (a.logprob) a.logprob[row] = none ? -INFINITY : 0.f;
    }
    cluster.sync();  // others' indices are read before they leave
    return;
  }
  if (tid == 0)
    sh.task = Task{r,     zrow,  a.token + row, a.logprob ? a.logprob + row : nullptr, u, fmax(1.0 / (double)T, 1e-300),
                   top_p, min_p, n,             top_k};
  if (top_k <= 0 && !(top_p < 1.f) && !(min_p > 0.f)) {
    // ---- no filter: the draw is in index order. Every warp sums a run of
    // its CTA's share; the one that holds the target walks its run again
    const int run = ((len + kThreads / 32 - 1) / (kThreads / 32) + 127) & ~127, w0 = min(len, warp * run), w1 = min(len, w0 + run);
    u64 m = 0;
    for (int i = w0 + 4 * lane; i < w1; i += 128) {
      const float4 v = four(i);
      m += to_mass(r, weight(r, v.x)) + to_mass(r, weight(r, v.y)) + to_mass(r, weight(r, v.z)) + to_mass(r, weight(r, v.w));
    }
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
    // the CTAs' masses: all of them, and those of the CTAs before this one
    u64 total = lane < C ? cluster.map_shared_rank(&sh, lane)->mass : 0, before = lane < rank ? total : 0;
#pragma unroll
    for (int o = kMaxCluster / 2; o > 0; o >>= 1) {
      total += __shfl_xor_sync(0xffffffffu, total, o);
      before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    total = __shfl_sync(0xffffffffu, total, 0);
    before = __shfl_sync(0xffffffffu, before, 0);
    // the masses are read: the CTAs without the target leave while its one
    // goes on
    auto read = cluster.barrier_arrive();
    const u64 target = min((u64)(u * (double)total), total - 1);
    if (before <= target && target < before + sh.mass) {
      // this CTA: the warp's run that holds the target, two tokens a thread
      int w = 0;
      while (w < kThreads / 32 - 1 && before + sh.red[w] <= target) before += sh.red[w++];
      const int r0 = min(len, w * run), r1 = min(len, r0 + run), each = (r1 - r0 + kThreads - 1) / kThreads;
      const int e0 = min(r1, r0 + tid * each), e1 = min(r1, e0 + each);
      u64 mine = 0;
      for (int i = e0; i < e1; ++i) mine += to_mass(r, weight(r, value(i)));
      before += block_before(mine, sh);
      if (before <= target && target < before + mine)
        for (int i = e0; i < e1; ++i) {
          before += to_mass(r, weight(r, value(i)));
          if (before > target) {
            finish(sh.task, lo + i, total);
            break;
          }
        }
    }
    cluster.barrier_wait(std::move(read));  // others may still read this CTA's mass
    return;
  }

  // ---- filters
  Shared *boss = cluster.map_shared_rank(&sh, 0);
  u64 *boss_list = cluster.map_shared_rank(list, 0);
  auto depth = [&](float z) { return z == r.zmax ? 0.f : r.zmax - z; };
  // the bucket of z, or (level 1) its place among the 2048 parts of bucket
  // b0; -1: not there (nor is a NaN). Both rise with falling z.
  auto bucket = [&](float z, int level, int b0) {
    if (z != z) return -1;
    const float d = depth(z);
    const int b = min(kBuckets - 1, (int)(d * scale));
    if (level == 0) return b;
    return b == b0 ? min(kBuckets - 1, max(0, (int)(fmaf(d, scale, -(float)b0) * kBuckets))) : -1;
  };
  // a value below which no token of the buckets before `end` lies, with room
  // for the roundings above
  auto edge = [&](int level, int b0, int end) {
    const float e = level ? (float)b0 + (float)end / kBuckets : (float)end;
    if (!level && end >= kBuckets) return -INFINITY;
    const float d = (e + 0.01f) * 1.001f / scale;
    const float x = r.zmax - d - fabsf(r.zmax) * 1e-5f;
    return x == x ? x : -INFINITY;  // (an infinite maximum)
  };
  // f(index of the first, values) for every four neighbouring tokens of a
  // thread, loaded together, ahead of what f writes; behind the last token
  // the value is NaN, which no bucket and no sum takes
  auto fours = [&](auto f) {
    for (int i = 4 * tid; i < len; i += 4 * kThreads) f(i, four(i));
  };
  int cmd = kHist, level = 0, b0 = 0, glo = 0, ghi = 0;
  bool masses = top_p < 1.f || top_k <= 0 || top_k > kList / 2 || min_p > 0.f;  // the first pass sums them all
  bool first = true;
  if (tid == 0) {
    sh.book = Book{};
    sh.cmd = cmd, sh.level = 0, sh.b0 = 0, sh.lo = sh.hi = 0, sh.masses = masses, sh.first = 1;
  }
  for (;;) {
    if (cmd == kHist) {
      if (!first) {
        for (int i = tid; i < kBuckets; i += kThreads) hcount[i] = 0;
        __syncthreads();
      }
      u64 m = 0;
      int above = 0;
      const bool sums = masses && level == 0;
      fours([&](int, float4 v) {
        const float z[4] = {v.x, v.y, v.z, v.w};
        int b[4];
        double w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          b[j] = bucket(z[j], level, b0);
          if (sums) w[j] = weight(r, z[j]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (sums) {
            m += to_mass(r, w[j]);
            above += w[j] >= (double)min_p;  // (counted only where min_p > 0)
          }
          if (b[j] >= 0) atomicAdd(&hcount[b[j]], 1);
        }
      });
      if (sums) {
        m = block_sum(m, sh);
        above = __reduce_add_sync(0xffffffffu, above);
        if (tid == 0) sh.mass = m;
        if (lane == 0 && first) atomicAdd(&sh.count, above);
      }
    } else if (cmd == kMass) {
      if (lane < kWindow) sh.parts[warp][lane] = 0;
      __syncwarp();
      u64 m = 0;
      const float low = edge(level, b0, glo + kWindow);
      fours([&](int, float4 v) {
        if (!(v.x >= low || v.y >= low || v.z >= low || v.w >= low)) return;
        const float z[4] = {v.x, v.y, v.z, v.w};
        u64 x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = to_mass(r, weight(r, z[j]));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          int b = bucket(z[j], level, b0);
          b = b < 0 ? kWindow : b - glo;
          if (b < 0) m += x[j]; else if (b < kWindow && x[j]) atomicAdd(&sh.parts[warp][b], x[j]);
        }
      });
      m = block_sum(m, sh);
      if (tid == 0) sh.mass = m;
      if (tid < kWindow) {
        u64 t = 0;
        for (int i = 0; i < kThreads / 32; ++i) t += sh.parts[i][tid];
        sh.window[tid] = t;
      }
    } else {  // kGather: count, take places in the leader's list, write
      const float low = edge(level, b0, ghi + 1);
      auto in = [&](float z) {
        if (!(z >= low)) return false;
        const int b = bucket(z, level, b0);
        return b >= glo && b <= ghi;
      };
      int hits = 0;
      fours([&](int, float4 v) { hits += in(v.x) + in(v.y) + in(v.z) + in(v.w); });
      int p = (int)block_before((u64)hits, sh);
      if (tid == kThreads - 1) sh.place = p + hits ? atomicAdd(&boss->listed, p + hits) : 0;
      __syncthreads();
      p += sh.place;
      if (hits)
        fours([&](int i, float4 v) {
          const float z[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (in(z[j])) {
              if (p < kList) boss_list[p] = (u64)ordered(z[j] + 0.f) << 32 | (0xffffffffu - (uint32_t)(lo + i + j));
              ++p;
            }
        });
    }
    cluster.sync();
    if (rank == 0) leader_turn(sh, list, guess, hcount);
    cluster.sync();
    // read before the next barrier, behind which the leader gives new orders
    cmd = boss->cmd;
    level = boss->level;
    b0 = boss->b0;
    glo = boss->lo;
    ghi = boss->hi;
    masses = boss->masses;
    first = false;
    if (cmd == kDone) break;
  }
  cluster.sync();  // the leader's orders are read before it leaves
}

template <bool IN_SMEM, int PER_SM>
ifx_status run(const SampleRowsArgs &a, int cluster, size_t smem, cudaStream_t st) {
  auto kernel = sample_rows_kernel<IN_SMEM, PER_SM>;
  static std::atomic<uint64_t> done{0};
  IFX_TRY(raise_smem(kernel, 216 * 1024, done));
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
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, part);
    if (e != cudaSuccess) {
      cudaGetLastError();  // reported here, not to the next call
      return cuda_fail(e, "sample_rows");
    }
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
  const size_t smem = per <= kMaxChunk ? base + (size_t)per * sizeof(float) : base;
  // few rows: more registers for a CTA that has its SM to itself; many: two
  // CTAs an SM, one of which computes while the other waits
  if (a.rows * cluster <= kNumSMs)
    return per <= kMaxChunk ? run<true, 1>(a, cluster, smem, st) : run<false, 1>(a, cluster, smem, st);
  return per <= kMaxChunk ? run<true, 2>(a, cluster, smem, st) : run<false, 2>(a, cluster, smem, st);
}

}  // namespace ifx
