// Attention over the key/value cache in 4 bits, many query rows per kv head (a
// prompt in chunks, long drafts): softmax(scale q k) v as in kv4_attention.cu,
// on the fifth generation's tensor cores.
//
// Mathematics. A tile is 128 query rows of one kv head (its query heads times
// the new rows) and meets page after page of 64 cached rows:
//   scores: S = q_lo k_hi + q_hi k_lo + q_hi k_hi   (128 x 64 x head_dim)
//   output: O = p_lo v_hi + p_hi v_lo + p_hi v_hi   (128 x head_dim x 64)
// with a running maximum and sum per query row. All operands are f16 planes: a
// value's rounding to f16 and the rounded remainder, 22 bits together (of a
// probability down to 2^-35 of the row's largest so far); keys and values, four
// bits times a scale of 11, are exact in two down to 2^-19 of their page's
// largest. O goes over to every page's exponent, by powers of two in f32. S and O are f32
// in tensor memory and start from zero for every page; O is read back and
// added in f32, since the tensor cores cut their sums off instead of rounding
// them (40 pages summed there came out 4.8e-6 off, this way 4e-7).
//
// Layout. Queries and probabilities are the products' A operand and live in
// tensor memory, where the threads that make them write them: only the keys
// and values pass through shared memory, unpacked into K-major core matrices
// of 8 rows x 16 bytes without a swizzle. A value word holds pairs of rows, so
// the transposed values come out of it as the product wants them. Each of 256
// threads has one query row (a lane of tensor memory) and half the columns of
// S, P and O. While the products of a page run, the threads unpack the keys of
// the next; heads of up to 64 need half the tensor memory, so that two CTAs
// share an SM and fill each other's waits.
//
// What bounds it. Instructions: 760 per warp and page at heads of 64 (softmax
// and its planes 230, unpacking 200, output 32), issued at 57% of the rate;
// the tensor cores are busy 24% of the time (twelve 128 x 64 x 16 products each
// way, at full rate). 128 rows of 4 sequences, 32 heads on 8, 2600 keys: heads
// of 64 76 us (140 TFLOP/s of the two plain products), of 128 122 us, of 256
// 209 us; the same with m16n8k16 products on 64 rows took 122, 226 and 659.
#include <algorithm>

#include "kv4_attention.cuh"

namespace ifx {

using namespace kv4;

namespace {

__device__ __forceinline__ uint32_t h2(__half2 x) { return *reinterpret_cast<const uint32_t *>(&x); }
__device__ __forceinline__ __half2 as_h2(uint32_t x) { return *reinterpret_cast<const __half2 *>(&x); }

// The pair (n, n') of f16 subnormals n * 2^-24 as n - 8, n' - 8: one fused
// multiply-add in f16, exact (in steps of 2^-9, to keep the factor in range;
// nibbles at bits 4..7 come 16 times larger).
__device__ __forceinline__ __half2 nibble_pair(uint32_t w, bool high) {
  const uint32_t m = high ? w & 0x00f000f0u : w & 0x000f000fu;
  return __hfma2(as_h2(m), __float2half2_rn(high ? 2048.f : 32768.f), __float2half2_rn(-8.f / 512.f));
}

constexpr int kTcRows = 128, kTcThreads = 256;

template <int NB>
struct TcShape {
  static constexpr int HD = 32 * NB, kTile = Kv4Layout::tile_bytes(NB), kRaw = 4 * kTile;
  static constexpr int kKStep = 64 * 16 + 32;  // 8 dimensions of 64 keys; 32 bytes keep four steps on different banks
  static constexpr int kVStep = HD * 16;       // 8 rows of all dimensions
  static constexpr int kKPlane = 4 * NB * kKStep, kVPlane = 8 * kVStep;
  static constexpr int kK = 2 * kRaw, kV = kK + 2 * kKPlane, kBytes = kV + 2 * kVPlane;
  static constexpr int kPart = kTcRows * (HD + 2) * 4;
  // columns of tensor memory
  static constexpr int kS = 0, kPh = 64, kPl = 96, kQh = 128, kQl = kQh + 16 * NB, kO = kQl + 16 * NB;
  // heads above 192: the output's columns in two turns, half of them at a time
  static constexpr bool kTwice = NB > 6;
  static constexpr int kWidth = kTwice ? HD / 2 : HD, kCols = kO + kWidth <= 256 ? 256 : 512, kPerSm = 512 / kCols;
  static_assert(kO + kWidth <= kCols && (kBytes + (kMaxAttnSeqs + 1) * 8 + 4096) * kPerSm <= 227 * 1024, "one SM's memories");
};

// K-major operand without a swizzle: `step` bytes between 8 values of K, 128
// between 8 rows.
__device__ __forceinline__ uint64_t core_desc(uint32_t saddr, uint32_t step) {
  return (uint64_t)((saddr & 0x3ffffu) >> 4) | ((uint64_t)(step >> 4) << 16) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}
// f16 operands, both K-major, f32 sums, M = 128, N = n.
__device__ constexpr uint32_t tc_idesc(int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTcRows >> 4) << 24); }
__device__ __forceinline__ void tc_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tc_commit(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Sixteen columns of this thread's lane; the values are there after tc_wait_ld.
__device__ __forceinline__ void tc_ld16(uint32_t at, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at));
}
template <int N>
__device__ __forceinline__ void tc_wait_ld(uint32_t (&r)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));  // no use moves above the wait
}
__device__ __forceinline__ void tc_st8(uint32_t at, const uint32_t *r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(at)
               : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t at, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(at)
      : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A page's exponents, of its keys and of its values: the largest scale times
// 2^k lies in [2^14, 2^15), or k is 30 (scales below 2^-15 keep all their bits
// with less); 1000 for a page of zeros. Computed by every warp.
template <int NB>
__device__ __forceinline__ int2 page_exponents(const uint8_t *raw, int rows_here) {
  const int lane = threadIdx.x & 31;
  // a lane's NB words are rows 2 (lane % 8) and the next of tile lane / 8
  const uint8_t *at = raw + lane / 8 * TcShape<NB>::kTile + lane % 8 * NB * 4;
  uint32_t w[2][NB], top[2];
  ld_words<NB>(at + Kv4Layout::k_scales(NB), w[0]);
  ld_words<NB>(at + Kv4Layout::v_scales(NB), w[1]);
  if (rows_here < 64) {
    const int r = lane / 8 * 16 + lane % 8 * 2;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const uint32_t keep = (r + 2 * i / NB < rows_here ? 0x0000ffffu : 0u) | (r + (2 * i + 1) / NB < rows_here ? 0xffff0000u : 0u);
      w[0][i] &= keep;
      w[1][i] &= keep;
    }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    top[k] = w[k][0] & 0x7fff7fffu;
#pragma unroll
    for (int i = 1; i < NB; ++i) top[k] = __vmaxu2(top[k], w[k][i] & 0x7fff7fffu);
  }
  int k[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t most = __reduce_max_sync(0xffffffffu, max(top[i] & 0xffffu, top[i] >> 16));
    k[i] = most ? min(30, 14 + 127 - (int)(__float_as_uint(h2f((uint16_t)min(most, 0x7bffu))) >> 23)) : 1000;
  }
  return make_int2(k[0], k[1]);
}

// Two scales times 2^k, in two steps that f16 can hold.
__device__ __forceinline__ __half2 scaled(uint32_t d2, __half2 f0, __half2 f1) { return __hmul2(__hmul2(as_h2(d2), f0), f1); }
__device__ __forceinline__ __half2 power_pair(int k) { return as_h2((uint32_t)(k + 15) * 0x04000400u); }  // 2^k, -14 <= k <= 15

// Keys of a page into their planes: a thread has one row and the eighth t of
// every block.
template <int NB>
__device__ __forceinline__ void unpack_keys(uint8_t *sm, const uint8_t *raw, int rows_here, int k) {
  using L = TcShape<NB>;
  const int r = threadIdx.x >> 2, t = threadIdx.x & 3;
  const uint8_t *tb = raw + r / 16 * L::kTile;
  const __half2 f0 = power_pair(k == 1000 ? 0 : min(k, 15)), f1 = power_pair(k == 1000 ? 0 : max(k - 15, 0));
  uint32_t w[NB];
  ld_words<NB>(tb + (r % 16 * 4 + t) * NB * 4, w);
  const uint16_t *sc = reinterpret_cast<const uint16_t *>(tb + Kv4Layout::k_scales(NB)) + r % 16 * NB;
  uint8_t *at = sm + L::kK + t * L::kKStep + r * 16;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const __half2 d = scaled(r < rows_here ? sc[b] * 0x10001u : 0u, f0, f1);
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 x = nibble_pair(i < 2 ? w[b] : w[b] >> 8, i & 1);
      const __half2 p = __hmul2(x, d);
      hi[i] = h2(p);
      lo[i] = h2(__hfma2(x, d, __hneg2(p)));
    }
    *reinterpret_cast<uint4 *>(at + 4 * b * L::kKStep) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    *reinterpret_cast<uint4 *>(at + 4 * b * L::kKStep + L::kKPlane) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
}

// Values of a page, transposed: column 8 NB j + 8 b + g is dimension 32 b + 4 g
// + j. A thread has eight rows of dimensions j = 2 jh and 2 jh + 1.
template <int NB>
__device__ __forceinline__ void unpack_values(uint8_t *sm, const uint8_t *raw, int rows_here, int k) {
  using L = TcShape<NB>;
  const __half2 f0 = power_pair(k == 1000 ? 0 : min(k, 15)), f1 = power_pair(k == 1000 ? 0 : max(k - 15, 0));
#pragma unroll
  for (int e = threadIdx.x; e < 128 * NB; e += kTcThreads) {
    const int g = e % 8, b = e / 8 % NB, o = e / (8 * NB) % 8, jh = e / (64 * NB);
    const uint8_t *tb = raw + o / 2 * L::kTile;
    const uint32_t *words = reinterpret_cast<const uint32_t *>(tb + Kv4Layout::v_words(NB)) + (o % 2 * 32 + g) * NB + b;
    const uint16_t *sc = reinterpret_cast<const uint16_t *>(tb + Kv4Layout::v_scales(NB)) + o % 2 * 8 * NB + b;
    uint32_t hi[2][4], lo[2][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t d2 = (uint32_t)sc[2 * i * NB] | (uint32_t)sc[(2 * i + 1) * NB] << 16;
      if (rows_here < 64) {
        if (8 * o + 2 * i >= rows_here) d2 = 0;
        else if (8 * o + 2 * i + 1 >= rows_here) d2 &= 0xffffu;
      }
      const __half2 d = scaled(d2, f0, f1);
      const uint32_t w = words[8 * i * NB] >> (8 * jh);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const __half2 x = nibble_pair(w, j), p = __hmul2(x, d);
        hi[j][i] = h2(p);
        lo[j][i] = h2(__hfma2(x, d, __hneg2(p)));
      }
    }
    uint8_t *at = sm + L::kV + o * L::kVStep + (2 * jh * 8 * NB + 8 * b + g) * 16;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      *reinterpret_cast<uint4 *>(at + j * 128 * NB) = make_uint4(hi[j][0], hi[j][1], hi[j][2], hi[j][3]);
      *reinterpret_cast<uint4 *>(at + j * 128 * NB + L::kVPlane) = make_uint4(lo[j][0], lo[j][1], lo[j][2], lo[j][3]);
    }
  }
}

// The units of a segment whose page a row of the tile sees.
__device__ __forceinline__ void seen_units(const Kv4AttnArgs &a, const Segment &s, long long *first, long long *stop) {
  const int grp = a.H / a.G, tok0 = (int)((uint32_t)s.ct * kTcRows / (uint32_t)grp);
  const int tok1 = (int)min((uint32_t)s.ql - 1u, ((uint32_t)s.ct * kTcRows + kTcRows - 1) / (uint32_t)grp);
  const int hi = s.len - s.ql + tok1, lo = a.window ? max(0, s.len - s.ql + tok0 - a.window + 1) : 0;
  *first = s.begin + max(0, lo / kKv4PageRows - s.lo);
  *stop = hi < 0 ? *first : min(s.end, s.begin + hi / kKv4PageRows + 1 - s.lo);
}

template <int NB>
__global__ void __launch_bounds__(kTcThreads, TcShape<NB>::kPerSm) kv4_attn_tc_kernel(const __grid_constant__ Kv4AttnArgs a) {
  using L = TcShape<NB>;
  constexpr int HD = L::HD, ROWS = kTcRows, HALF = 16 * NB;
  extern __shared__ __align__(128) uint8_t sm[];
  long long *pre = reinterpret_cast<long long *>(sm + L::kBytes);
  __shared__ __align__(8) uint64_t raw_bar[2], s_bar, o_bar, end_bar[2];
  __shared__ int s_sent;  // copies asked for
  __shared__ uint32_t tmem_slot;
  __shared__ long long s_scan[kTcThreads / 32], s_tiles[kTcThreads / 32];
  __shared__ float s_both[2][ROWS], s_sum[2][ROWS];  // what the two threads of a row exchange: largest values, sums
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row = tid & (ROWS - 1), half = tid / ROWS;
  if (tid == 0) {
    mbar_init(&raw_bar[0], 1);
    mbar_init(&raw_bar[1], 1);
    mbar_init(&s_bar, 1);
    mbar_init(&o_bar, 1);
    mbar_init(&end_bar[0], 1);
    mbar_init(&end_bar[1], 1);
    s_sent = 0;
    fence_mbar_init();
  }
  pdl_launch();
  if (a.zero_rest && warp == 1) zero_rest(a);
  {
    const int n = a.n_seqs, per = (n + kTcThreads - 1) / kTcThreads, b0 = min(n, tid * per), b1 = min(n, b0 + per);
    long long mine = 0, tiles = 0;
    for (int b = b0; b < b1; ++b) {
      const Seq s = sequence<ROWS>(a, b);
      pre[b] = mine;
      mine += (long long)s.units * s.nct * a.G;
      tiles += (long long)s.nct * a.G;
    }
    long long inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, inc, o), y = __shfl_xor_sync(0xffffffffu, tiles, o);
      if (lane >= o) inc += x;
      tiles += y;
    }
    if (lane == 31) {
      s_scan[warp] = inc;
      s_tiles[warp] = tiles;
    }
    __syncthreads();
    long long base = inc - mine;
    for (int i = 0; i < warp; ++i) base += s_scan[i];
    for (int b = b0; b < b1; ++b) pre[b] += base;
    if (tid == kTcThreads - 1) pre[n] = base + mine;
    __syncthreads();
  }
  const long long total = pre[a.n_seqs];
  // a CTA takes four pages or more, for few partials, or a tile of fewer
  long long tiles = 0;
  for (int i = 0; i < kTcThreads / 32; ++i) tiles += s_tiles[i];
  const int live = (int)min((long long)gridDim.x, max(tiles, (total + 3) / 4));
  RangeInfo *info = static_cast<RangeInfo *>(a.ws);
  if ((int)blockIdx.x >= live) {
    if (tid == 0) info[blockIdx.x].live = 0;
    return;
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(L::kCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = tmem_slot, mine = tmem + ((uint32_t)(32 * (warp & 3)) << 16);  // this thread's lane
  const Deal deal(total, live);
  const long long u0 = deal.begin(blockIdx.x), u1 = deal.begin(blockIdx.x + 1);
  const int grp = a.H / a.G;
  Segment s = locate<ROWS>(a, pre, u0);
  if (tid == 0) info[blockIdx.x] = RangeInfo{s.begin, s.end, total, s.seq, s.h, s.ct, live};

  // thread 64: the copies, up to two pages ahead of the products; the page's
  // number is read one copy ahead, so that its latency is not waited for
  Segment fs = s;
  long long fu, fstop;
  int fpage = -1;
  seen_units(a, fs, &fu, &fstop);
  fu = max(fu, u0);
  fstop = min(fstop, u1);
  auto look = [&]() {
    while (fu >= fstop) {
      if (fs.end >= u1) return;
      fs = locate<ROWS>(a, pre, fs.end);
      seen_units(a, fs, &fu, &fstop);
      fstop = min(fstop, u1);
    }
    const int j = fs.lo + (int)(fu - fs.begin);
    fpage = j < a.max_pages ? __ldg(a.table + (size_t)fs.seq * a.max_pages + j) : -1;
  };
  auto fetch = [&](int st) {
    if (fu >= fstop) return;
    const int j = fs.lo + (int)(fu - fs.begin), tiles = min(4, (fs.len - j * kKv4PageRows + kKv4TileRows - 1) / kKv4TileRows);
    if ((unsigned)fpage < (unsigned)a.n_pages && tiles > 0) {
      mbar_arrive_expect_tx(&raw_bar[st], (uint32_t)(tiles * L::kTile));
      bulk_g2s(sm + st * L::kRaw, a.pages + ((int64_t)fpage * a.G + fs.h) * L::kRaw, (uint32_t)(tiles * L::kTile), &raw_bar[st]);
    } else {
      mbar_arrive(&raw_bar[st]);
    }
    ++s_sent;
    ++fu;
    look();
  };
  if (tid == 64) {
    look();
    fetch(0);
    fetch(1);
  }
  // (an address counts in 16 bytes in the lowest bits)
  const uint64_t keys = core_desc(smem_u32(sm + L::kK), L::kKStep), vals = core_desc(smem_u32(sm + L::kV), L::kVStep);
  auto issue_scores = [&]() {
    tc_after();
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) {
      tc_mma(tmem + L::kS, tmem + L::kQl + 8 * i, keys + 2 * i * L::kKStep / 16, tc_idesc(64), i > 0);
      tc_mma(tmem + L::kS, tmem + L::kQh + 8 * i, keys + (L::kKPlane + 2 * i * L::kKStep) / 16, tc_idesc(64), 1);
    }
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) tc_mma(tmem + L::kS, tmem + L::kQh + 8 * i, keys + 2 * i * L::kKStep / 16, tc_idesc(64), 1);
    tc_commit(&s_bar);
  };
  auto issue_output = [&](int turn) {
    tc_after();
    const uint64_t v = vals + turn * L::kWidth;  // 16 bytes a column
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      tc_mma(tmem + L::kO, tmem + L::kPl + 8 * i, v + 2 * i * L::kVStep / 16, tc_idesc(L::kWidth), i > 0);
      tc_mma(tmem + L::kO, tmem + L::kPh + 8 * i, v + (L::kVPlane + 2 * i * L::kVStep) / 16, tc_idesc(L::kWidth), 1);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) tc_mma(tmem + L::kO, tmem + L::kPh + 8 * i, v + 2 * i * L::kVStep / 16, tc_idesc(L::kWidth), 1);
    tc_commit(&o_bar);
  };

  int st = 0;
  uint32_t phase = 0, s_phase = 0, o_phase = 0;
  long long u = u0;
  // a wait gave up: in this thread, which waits for nothing more then (and
  // thread 64 asks for nothing), and, from a segment's end on, in any of the
  // CTA: that segment and the ones behind it get NaN
  bool ok = true, lost = false;
  while (u < u1) {
    int head;
    const long long prow = pair_row<ROWS>(a, s.q0, s.ql, s.ct, row, &head);
    float qs = 0.f;
    if (!lost) {
      // ---- half of the thread's query row, two f16 planes, scaled by a power
      // of two that puts the row's largest magnitude into [2^10, 2^11)
      float x[HALF];
      float big = 0.f;
#pragma unroll
      for (int i = 0; i < HALF; i += 8) {
        if (prow < 0) {
#pragma unroll
          for (int k = 0; k < 8; ++k) x[i + k] = 0.f;
          continue;
        }
        const int64_t at = prow * a.q_stride + (int64_t)(s.h * grp + head) * HD + half * HALF + i;
        if (a.type == IFX_TYPE_F16) {
          const uint4 v = *reinterpret_cast<const uint4 *>(static_cast<const __half *>(a.q) + at);
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 f = __half22float2(as_h2(w[k]));
            x[i + 2 * k] = f.x;
            x[i + 2 * k + 1] = f.y;
          }
        } else {
          const float4 *v = reinterpret_cast<const float4 *>(static_cast<const float *>(a.q) + at);
          const float4 y = v[0], z = v[1];
          x[i] = y.x, x[i + 1] = y.y, x[i + 2] = y.z, x[i + 3] = y.w;
          x[i + 4] = z.x, x[i + 5] = z.y, x[i + 6] = z.z, x[i + 7] = z.w;
        }
      }
#pragma unroll
      for (int i = 0; i < HALF; ++i) big = fabsf(x[i]) < INFINITY ? fmaxf(big, fabsf(x[i])) : INFINITY;
      s_both[half][row] = big;
      __syncthreads();
      big = fmaxf(s_both[0][row], s_both[1][row]);
      const int e = big > 0.f ? min(100, max(-117, 10 + 127 - (int)(__float_as_uint(big) >> 23))) : 0;
      // the scale's sign goes into the query, so that the factor of the scores
      // is positive and the largest product is the largest score; a scale of 0
      // makes the query 0
      const float up = a.scale == 0.f ? 0.f : copysignf(__uint_as_float((uint32_t)(127 + e) << 23), a.scale);
#pragma unroll
      for (int i = 0; i < HALF; i += 16) {  // dimensions of eight in the order 0 4 1 5 2 6 3 7
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float v = x[i + k / 4 * 8 + k % 4] * up, w = x[i + k / 4 * 8 + k % 4 + 4] * up;
          const __half2 p = __floats2half2_rn(v, w);
          const float2 back = __half22float2(p);
          hi[k] = h2(p);
          lo[k] = h2(__floats2half2_rn(v - back.x, w - back.y));
        }
        tc_st8(mine + L::kQh + half * 8 * NB + i / 2, hi);
        tc_st8(mine + L::kQl + half * 8 * NB + i / 2, lo);
      }
      tc_wait_st();
      // nibble pairs come in steps of 2^-9; a query that is not finite has
      // scores NaN
      const float f = a.scale == 0.f ? 1.f : fabsf(a.scale) * 1.4426950408889634f * 512.f * __uint_as_float((uint32_t)(127 - e) << 23);
      qs = big < INFINITY ? fmaxf(f, 1e-27f) : __uint_as_float(0x7fc00000u);
    }
    const int pos = s.len - s.ql + (int)(prow - s.q0);
    const int jmax = prow >= 0 ? pos : INT32_MAX, jmin = prow >= 0 && a.window ? max(0, pos - a.window + 1) : 0;
    const int see_lo = __reduce_max_sync(0xffffffffu, jmin), see_hi = __reduce_min_sync(0xffffffffu, jmax);
    float m = -INFINITY, l = 0.f, alpha = 0.f;
    float o[HALF];
#pragma unroll
    for (int i = 0; i < HALF; ++i) o[i] = 0.f;
    int kref = 1000;  // o counts in 2^-(1 + kref) (p times 2^10, nibbles in 2^-9): the exponent of the last page with values
    auto add_output = [&](int turn) {  // o = o alpha + the page's sums
      ok = ok && mbar_wait(&o_bar, o_phase, nullptr, 0);
      o_phase ^= 1;
      tc_after();
      if (L::kTwice && half != turn) return;
      const uint32_t at = mine + L::kO + (L::kTwice ? 0 : half * HALF);
#pragma unroll
      for (int i = 0; i < HALF; i += 16) {
        uint32_t r[16];
        tc_ld16(at + i, r);
        tc_wait_ld(r);
#pragma unroll
        for (int k = 0; k < 16; ++k) o[i + k] = fmaf(o[i + k], alpha, __uint_as_float(r[k]));
      }
    };
    auto page_at = [&](int j) { return j < a.max_pages ? __ldg(a.table + (size_t)s.seq * a.max_pages + j) : -1; };
    auto rows_of = [&](int page, int j) {  // a missing page hides its rows
      return (unsigned)page < (unsigned)a.n_pages ? min(kKv4PageRows, max(0, s.len - j * kKv4PageRows)) : 0;
    };
    long long first, stop;
    seen_units(a, s, &first, &stop);
    first = max(first, u);
    stop = min(stop, u1);
    if (first < stop && !lost) {
      int j = s.lo + (int)(first - s.begin);
      const int j0 = j, j1 = j + (int)(stop - first);
      int rows_here = rows_of(page_at(j), j), coming = j + 1 < j1 ? page_at(j + 1) : -1;
      ok = ok && mbar_wait(&raw_bar[st], phase, nullptr, 0);
      int2 ks = page_exponents<NB>(sm + st * L::kRaw, rows_here);
      unpack_keys<NB>(sm, sm + st * L::kRaw, rows_here, ks.x);
      fence_async();
      tc_before();
      __syncthreads();
      if (tid == 0) issue_scores();
      for (; j < j1; ++j) {
        const uint8_t *raw = sm + st * L::kRaw;
        const bool next = j + 1 < j1;
        const int row0 = j * kKv4PageRows + 32 * half;  // this thread's 32 keys
        ok = ok && mbar_wait(&s_bar, s_phase, nullptr, 0);
        s_phase ^= 1;
        tc_after();
        uint32_t sr[32];
        tc_ld16(mine + L::kS + 32 * half, sr);
        tc_ld16(mine + L::kS + 32 * half + 16, sr + 16);
        const int kval = ks.y;
        int rows_next = 0;
        int2 ks_next = make_int2(1000, 1000);
        if (next) {
          rows_next = rows_of(coming, j + 1);
          if (j + 2 < j1) coming = page_at(j + 2);
          ok = ok && mbar_wait(&raw_bar[st ^ 1], phase ^ (uint32_t)st, nullptr, 0);
          ks_next = page_exponents<NB>(sm + (st ^ 1) * L::kRaw, rows_next);
          unpack_keys<NB>(sm, sm + (st ^ 1) * L::kRaw, rows_next, ks_next.x);
        }
        tc_wait_ld(sr);
        // ---- running maximum; the page's exponents
        const float f = qs * (ks.x == 1000 ? 1.f : __uint_as_float((uint32_t)(127 - ks.x) << 23));
        const int last = min(kKv4PageRows * j + rows_here - 1, see_hi);  // seen by every row of the warp
        if (row0 < see_lo || last - row0 < 31) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (row0 + i < jmin || row0 + i > jmax || row0 + i >= kKv4PageRows * j + rows_here) sr[i] = 0xff800000u;
        }
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 32; ++i) top[i % 4] = fmaxf(top[i % 4], __uint_as_float(sr[i]));
        float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        s_both[half][row] = mx;
        if (L::kTwice && j > j0) add_output(0);
        fence_async();
        tc_before();
        __syncthreads();  // keys are unpacked, scores read, maxima known
        if (L::kTwice && j > j0 && tid == ROWS) issue_output(1);
        if (next && tid == 0) issue_scores();
        mx = fmaxf(mx, s_both[half ^ 1][row]);
        const float m2 = fmaxf(m, mx == -INFINITY ? -INFINITY : mx * f);
        const float base = m2 == -INFINITY ? 0.f : m2;
        const float shrink = ex2(m - base);
        m = m2;
        // o goes over to what this page's sums count in, in f32 and by powers of
        // two, so that no page costs another's bits (|o| stays below 2^90)
        float scale_o = shrink;
        if (kval != 1000) {
          if (kref != 1000) scale_o *= __uint_as_float((uint32_t)(127 + kval - kref) << 23);
          kref = kval;
        }
        // p enters times 2^10 = exp2(x f - (base - 10)); its sum is divided by that again
        const float down = base - 10.f;
        float sum[2] = {0.f, 0.f};
        uint32_t ph[16], pl[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const float x0 = ex2(fmaf(__uint_as_float(sr[2 * k]), f, -down));
          const float x1 = ex2(fmaf(__uint_as_float(sr[2 * k + 1]), f, -down));
          sum[k & 1] += x0 + x1;
          const float h0 = __uint_as_float(__float_as_uint(x0) & 0xffffe000u), h1 = __uint_as_float(__float_as_uint(x1) & 0xffffe000u);
          ph[k] = h2(__floats2half2_rn(h0, h1));  // the first 11 bits, exactly
          pl[k] = h2(__floats2half2_rn(x0 - h0, x1 - h1));
        }
        l = fmaf(l, shrink, (sum[0] + sum[1]) * 0x1p-10f);
        if (j > j0) add_output(1);
        alpha = scale_o;
        tc_st16(mine + L::kPh + 16 * half, ph);
        tc_st16(mine + L::kPl + 16 * half, pl);
        unpack_values<NB>(sm, raw, rows_here, kval);
        tc_wait_st();
        fence_async();
        tc_before();
        __syncthreads();  // probabilities and values are in place, the page is read
        if (tid == ROWS) issue_output(0);
        if (tid == 64 && ok) fetch(st);
        rows_here = rows_next;
        ks = ks_next;
        phase ^= (uint32_t)st;
        st ^= 1;
      }
      if (L::kTwice) {
        add_output(0);
        tc_before();
        __syncthreads();
        if (tid == ROWS) issue_output(1);
      }
      add_output(1);
    }
    // ---- the segment's end, or the range's: the result, or a partial
    s_sum[half][row] = l;
    lost = __syncthreads_or(!ok);
    const float sum = lost ? __uint_as_float(0x7fc00000u) : s_sum[0][row] + s_sum[1][row];
    const bool whole = s.begin >= u0 && s.end <= u1;
    const float unit = kref == 1000 ? 0.f : __uint_as_float((uint32_t)max(0, 127 - 1 - kref) << 23);
    const float f = !whole ? unit : sum == 0.f ? 0.f : unit / sum;
    if (!whole) {
      // [column / 4][row][column % 4], then the maxima and the sums
      float *part = reinterpret_cast<float *>(static_cast<uint8_t *>(a.ws) + gridDim.x * sizeof(RangeInfo)) +
                    (size_t)(2 * blockIdx.x + (s.begin <= u0 ? 0 : 1)) * (L::kPart / 4);
#pragma unroll
      for (int i = 0; i < HALF; i += 4)
        *reinterpret_cast<float4 *>(part + ((half * HALF + i) / 4 * ROWS + row) * 4) =
            make_float4(o[i] * f, o[i + 1] * f, o[i + 2] * f, o[i + 3] * f);
      part[ROWS * (HD + half) + row] = half ? sum : m;
    } else if (prow >= 0) {
      const int64_t at = prow * a.out_stride + (int64_t)(s.h * grp + head) * HD + 2 * half;
#pragma unroll
      for (int i = 0; i < 8 * NB; ++i) {  // columns i and 8 NB + i: dimensions 2 half and the next of four
        const float x = o[i] * f, y = o[8 * NB + i] * f;
        if (a.type == IFX_TYPE_F16) *reinterpret_cast<__half2 *>(static_cast<__half *>(a.out) + at + 4 * i) = __floats2half2_rn(x, y);
        else *reinterpret_cast<float2 *>(static_cast<float *>(a.out) + at + 4 * i) = make_float2(x, y);
      }
    }
    u = s.end;
    if (u < u1) {
      __syncthreads();  // the sums are read
      s = locate<ROWS>(a, pre, u);
    }
  }
  if (lost) {  // products and copies on their way use this CTA's memories
    if (tid == 0 && a.err) atomicExch(a.err, kErrKv4Chunk);
    if (tid == 0 || tid == ROWS) {  // (the two threads that issue products)
      tc_commit(&end_bar[tid / ROWS]);
      mbar_wait(&end_bar[tid / ROWS], 0, nullptr, 0);
    }
    if (tid == 64)
      for (int i = max(0, s_sent - 2); i < s_sent; ++i) mbar_wait(&raw_bar[i & 1], (uint32_t)(i >> 1) & 1u, nullptr, 0);
  }
  tc_before();
  __syncthreads();
  if (warp == 0) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::kCols) : "memory");
  }
}

// Joins its partials: block c as in kv4_attn_join_kernel, a thread per query
// row and 16 dimensions (block b, four values of g).
template <int NB>
__global__ void __launch_bounds__(256) kv4_attn_tc_join_kernel(const __grid_constant__ Kv4AttnArgs a) {
  pdl_wait();
  constexpr int ROWS = kTcRows, HD = 32 * NB, PART = ROWS * (HD + 2);
  const RangeInfo *info = static_cast<const RangeInfo *>(a.ws);
  const int c = blockIdx.x + 1, grp = a.H / a.G;
  const RangeInfo r = info[c];
  if (!r.live) return;
  const Deal deal(r.total, r.live);
  const long long mine = deal.begin(c), prev = deal.begin(c - 1);
  if (r.begin >= mine || r.begin < prev) return;
  const float *parts = reinterpret_cast<const float *>(static_cast<const uint8_t *>(a.ws) + (gridDim.x + 1) * sizeof(RangeInfo));
  auto at = [&](int k) { return parts + (size_t)(2 * (c - 1 + k) + (k == 0 && r.begin > prev ? 1 : 0)) * PART; };
  const int n = deal.owner(r.end - 1) - c + 2;
  const Seq sq = sequence<ROWS>(a, r.seq);
  const int p = threadIdx.x & (ROWS - 1), cg = blockIdx.y * 2 + threadIdx.x / ROWS;
  int head;
  const long long row = pair_row<ROWS>(a, sq.q0, sq.ql, r.ct, p, &head);
  if (row < 0) return;
  float M = -INFINITY, S = 0.f;
#pragma unroll 4
  for (int k = 0; k < n; ++k) M = fmaxf(M, at(k)[ROWS * HD + p]);
  const float base = M == -INFINITY ? 0.f : M;
  float v[4][4] = {};  // [j][g % 4]
#pragma unroll 4
  for (int k = 0; k < n; ++k) {
    const float *pt = at(k);
    const float w = ex2(pt[ROWS * HD + p] - base);
    S = fmaf(w, pt[ROWS * (HD + 1) + p], S);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4 x = *reinterpret_cast<const float4 *>(pt + ((j * 2 * NB + cg) * ROWS + p) * 4);
      v[j][0] = fmaf(w, x.x, v[j][0]), v[j][1] = fmaf(w, x.y, v[j][1]), v[j][2] = fmaf(w, x.z, v[j][2]), v[j][3] = fmaf(w, x.w, v[j][3]);
    }
  }
  const float f = S == 0.f ? 0.f : 1.f / S;
#pragma unroll
  for (int g = 0; g < 4; ++g)
    write4(a, row, (r.h * grp + head) * HD + 16 * cg + 4 * g, make_float4(v[0][g] * f, v[1][g] * f, v[2][g] * f, v[3][g] * f));
}

template <int NB>
ifx_status run_tc(const Kv4AttnArgs &a, cudaStream_t st) {
  using L = TcShape<NB>;
  auto kernel = kv4_attn_tc_kernel<NB>;
  static std::atomic<uint64_t> done{0};
  IFX_TRY(raise_smem(kernel, L::kBytes + (kMaxAttnSeqs + 1) * 8, done));
  const int grid = kNumSMs * L::kPerSm;
  kernel<<<grid, kTcThreads, L::kBytes + ((size_t)a.n_seqs + 1) * sizeof(long long), st>>>(a);
  IFX_CUDA(cudaGetLastError());
  IFX_CUDA(launch(kv4_attn_tc_join_kernel<NB>, dim3(grid - 1, NB), dim3(256), 0, st, true, a));
  return IFX_OK;
}

}  // namespace

// 128 query rows a tile pay from 64 columns (query rows of a kv head) on, where
// there is work enough for the longer way to the first product. 16 sequences,
// 2600 keys, heads of 64 and 128: 48 columns 73 and 119 us against 73 and 112 of
// kv4_attention.cu, 64 columns 73 and 120 against 90 and 141, 96 columns 75 and
// 122 against 128 and 200. One sequence, 8 kv heads: 256 columns of 64 37 us
// against 36, of 128 41 against 50; 512 columns of 64 39 against 54, over 128
// keys 15 against 17.
bool kv4_chunks_take(const Kv4AttnArgs &a) {
  const int64_t columns = kv4_columns(a);
  return columns >= 64 && columns * a.n_seqs * a.G * a.hd >= 1 << 18;
}

ifx_status kv4_attention_chunks(const Kv4AttnArgs &a, cudaStream_t st) {
  switch (a.hd / 32) {
    case 1: return run_tc<1>(a, st);
    case 2: return run_tc<2>(a, st);
    case 3: return run_tc<3>(a, st);
    case 4: return run_tc<4>(a, st);
    case 5: return run_tc<5>(a, st);
    case 6: return run_tc<6>(a, st);
    case 7: return run_tc<7>(a, st);
    default: return run_tc<8>(a, st);
  }
}

size_t kv4_chunks_ws(int hd) {
  // per CTA two partials
  const size_t ctas = hd <= 64 ? 2 * kNumSMs : kNumSMs;
  return ctas * (sizeof(RangeInfo) + 2 * kTcRows * (size_t)(hd + 2) * sizeof(float));
}

}  // namespace ifx
