// Attention over the key/value cache in 4 bits.
//
// Mathematics. For a query row q and cached rows j (nibbles n, scales d per
// block b of 32): s_j = scale * sum_b dK_jb sum_{i in b} q_i (nK_ji - 8),
// p_j = exp(s_j - max), o_i = sum_j p_j dV_jb (nV_ji - 8) / sum_j p_j, in one
// pass with a running maximum and sum per query row.
//
// What bounds it. 4.5 bits per cached value are read once; at HBM's rate an
// SM has to take in about 40 values per clock, so the instructions per value
// decide. Both products therefore run as integer tensor-core products
// (mma.m16n8k32, s8 in, s32 out, the rate of the f16 m16n8k16 with twice the
// depth: 1.07 ns per MMA and SM against 1.10) on nibbles that need no
// conversion: `(w & 0xf0f0f0f0) ^ 0x80808080` is four signed bytes 16 (n - 8). A block of
// 32 values is exactly one MMA deep. (A form with f16 products, the masked
// nibbles read as f16 subnormals, took as many instructions and was 8 times
// less exact: the adder aligns subnormals by their nominal exponent.)
//
// Precision. The other operand enters as fixed point of 23 bits in three
// byte planes: a query head scaled so that its largest magnitude is 4.1e6,
// and p dV, with p relative to its page's own maximum, scaled
// so that 1 * the page's largest dV is 4.1e6. Where a page's dV differ by more
// than a factor of 8 that would cost the small ones their bits, to a row that
// is hidden, weighs nothing or is large in other dimensions: there every
// query's own largest p dV of a block takes the range, by a power of two (where
// every page is uneven, 64 sequences of 4500 keys take 149 us in place of 125,
// one of 128k 58 in place of 53). A step is at most 2^-19 of that largest term. Products
// and their sums over a block (keys) or a page (values) are exact integers;
// block scales, scores, maxima, sums and outputs are f32.
//
// Shape. Cached rows are the MMA's 16 rows (key product) or its depth (value
// product), the query rows its 8 columns: columns 2 t and 2 t + 1 are planes
// 1 and 0 of query t, plane 2 sits in a tile of its own, so a lane joins
// planes in registers. Four queries (the group of a kv head, times the new
// rows) share every unpacked nibble, or eight with three column tiles. The
// probabilities reach the value product's layout by movmatrix, two rows'
// bytes to a 16-bit element.
//
// Measured (heads of 128): 64 sequences of up to 8k keys, 64 heads on 8, 123 us
// (2.8 TB/s of pages), one of 128k, 32 on 8, 53 us (2.9 TB/s); one of 1k 13 us,
// latency.
#include <algorithm>

#include "kv4_attention.cuh"

namespace ifx {

using namespace kv4;

namespace {

template <int N>
__device__ __forceinline__ void ld_scales(const uint8_t *p, float (&d)[N]) {
  if constexpr (N % 2 == 0) {
    uint32_t w[N / 2];
    ld_words<N / 2>(p, w);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
      d[2 * i] = f.x;
      d[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) d[i] = __half2float(reinterpret_cast<const __half *>(p)[i]);
  }
}

__device__ __forceinline__ uint32_t movm_trans(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// D = A (16x32 s8, row) * B (32x8, col) + C (s32); B of signed bytes, or of
// unsigned ones.
__device__ __forceinline__ void mma_ss(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const int (&c)[4]) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
}
__device__ __forceinline__ void mma_su(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const int (&c)[4]) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
}

constexpr uint32_t kHigh = 0xf0f0f0f0u, kSign = 0x80808080u;

// x + kMagic, |x| <= kTop, has the bits 0x4b400000 + rint(x): byte 0 and byte
// 1 are the integer's low digits (unsigned, to base 256), byte 2 is 64 + its
// signed top digit.
constexpr float kMagic = 12582912.f;
constexpr float kTop = 4.1e6f;
constexpr float kUneven = 8.f;  // ratio of a page's value scales from which on every block has a range of its own
constexpr int kMaxLift = 60;    // (f16 scales are at most 2^40 apart; p dV 2^60 stays far below f32's end)

// 65536 top + 256 mid + low of the three planes' sums; top comes doubled.
__device__ __forceinline__ float planes(int top2, int mid, int low) {
  return fmaf((float)((top2 << 7) + mid), 256.f, (float)low);
}

__device__ __forceinline__ float quad_rows_sum(float v) {  // over the lanes of one column pair
  v += __shfl_xor_sync(0xffffffffu, v, 4);
  v += __shfl_xor_sync(0xffffffffu, v, 8);
  return v + __shfl_xor_sync(0xffffffffu, v, 16);
}
__device__ __forceinline__ float quad_rows_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}

template <int NB, int NT, int NW>
struct Smem {
  static constexpr int kPairs = 4 * NT, kHd = 32 * NB;
  static constexpr int kHalf = Kv4Layout::tile_bytes(NB) / 2;  // a tile's keys, or its values
  static constexpr int kPage = 8 * kHalf;
  static constexpr int kPart = kPairs * (kHd + 2) * 4;  // outputs, maxima, sums
  static_assert(kPart <= kPage && Kv4Layout::v_words(NB) == kHalf, "");
  static constexpr int kParts = NW * kPage;
  static constexpr int kBars = kParts + NW * kPart;
  static constexpr int kBytes = kBars + NW * 16;
  static_assert(kBytes + (kMaxAttnSeqs + 1) * 8 <= 227 * 1024, "shared memory of one CTA");
  // a warp's first partial has a place of its own, its second takes the page
  // buffer once the last copy is consumed
  static __device__ __forceinline__ float *part(uint8_t *sm, int slot) {
    return reinterpret_cast<float *>(sm + ((slot & 1) ? (slot >> 1) * kPage : kParts + (slot >> 1) * kPart));
  }
};

// A launch's units (a page of one kv head of one sequence, for one column
// tile) are numbered along sequences, kv heads, column tiles and pages, and
// dealt out evenly: each live CTA takes a contiguous range, each of its warps
// a part of that, so uneven lengths leave no SM idle. A warp walks its pages
// alone, with no CTA-wide barrier: it bulk-copies the next page's keys while
// it works on this one's values, and the next values during the next keys.
// A segment that lies within its range is finished in registers; others
// leave a partial (maximum, sum, output) in shared memory, which the CTA
// joins, and what reaches beyond the CTA goes to global memory for
// kv4_attn_join_kernel.
template <int NB, int NT, int NW, int MINB>
__global__ void __launch_bounds__(NW * 32, MINB) kv4_attn_kernel(const __grid_constant__ Kv4AttnArgs a) {
  using L = Smem<NB, NT, NW>;
  constexpr int PAIRS = L::kPairs, HD = L::kHd, TT = (NT + 1) / 2, TB = Kv4Layout::tile_bytes(NB), HB = L::kHalf;
  constexpr int SC = 256 * NB;  // the scales behind a half tile's words
  extern __shared__ __align__(128) uint8_t sm[];
  long long *pre = reinterpret_cast<long long *>(sm + L::kBytes);  // [n_seqs + 1]
  __shared__ long long s_scan[NW];
  // what a warp needs between segments only: kept out of its registers
  __shared__ Segment s_now[NW];
  __shared__ int s_next[NW];  // the sequence of the copies
  __shared__ long long s_range[NW][2], s_cta[2];  // units of the warp, of the CTA
  __shared__ int s_seq[2 * NW][3], s_whole[2 * NW], s_join[2 * NW];
  // the warp index by shuffle: the compiler keeps what follows from it in
  // uniform registers
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, g = lane >> 2, t = lane & 3;
  uint64_t *bar = reinterpret_cast<uint64_t *>(sm + L::kBars) + warp * 2;
  if (lane == 0) {
    mbar_init(&bar[0], 1);
    mbar_init(&bar[1], 1);
    fence_mbar_init();
  }
  pdl_launch();
  if (a.zero_rest && warp == 1) zero_rest(a);
  if (tid < 2 * NW) s_seq[tid][0] = -1;
  // units of every sequence, summed
  if (!a.alone) {
    const int n = a.n_seqs, per = (n + NW * 32 - 1) / (NW * 32), b0 = min(n, tid * per), b1 = min(n, b0 + per);
    long long mine = 0;
    for (int b = b0; b < b1; ++b) {
      const Seq s = sequence<PAIRS>(a, b);
      pre[b] = mine;
      mine += (long long)s.units * s.nct * a.G;
    }
    long long inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += x;
    }
    if (lane == 31) s_scan[warp] = inc;
    __syncthreads();
    long long base = inc - mine;
    for (int i = 0; i < warp; ++i) base += s_scan[i];
    for (int b = b0; b < b1; ++b) pre[b] += base;
    if (tid == NW * 32 - 1) pre[n] = base + mine;
    __syncthreads();
  }
  const int grp = a.H / a.G;
  long long c0, c1;  // the CTA's units
  Segment s;
  if (a.alone) {
    // one row per sequence: CTA c takes segment c
    const int nct = (grp + PAIRS - 1) / PAIRS, per_seq = a.G * nct;
    s.seq = blockIdx.x / per_seq;
    const int i = blockIdx.x - s.seq * per_seq;
    s.h = i / nct;
    s.ct = i - s.h * nct;
    const Seq q = sequence<PAIRS>(a, s.seq);
    s.lo = q.lo, s.len = q.len, s.ql = q.ql, s.q0 = q.q0;
    s.begin = c0 = 0;
    s.end = c1 = q.units;
  } else {
    const long long total = pre[a.n_seqs];
    const int live = (int)min((long long)gridDim.x, (total + NW - 1) / NW);
    RangeInfo *info = static_cast<RangeInfo *>(a.ws);
    if ((int)blockIdx.x >= live) {
      if (tid == 0) info[blockIdx.x].live = 0;
      return;
    }
    const Deal deal(total, live);
    c0 = deal.begin(blockIdx.x), c1 = deal.begin(blockIdx.x + 1);
    if (tid == 0) {
      s = locate<PAIRS>(a, pre, c0);
      info[blockIdx.x] = RangeInfo{s.begin, s.end, total, s.seq, s.h, s.ct, live};
    }
  }
  if (tid == 0) s_cta[0] = c0, s_cta[1] = c1;
  __syncthreads();
  const int share = (int)(c1 - c0);
  const long long u0 = c0 + (int64_t)share * warp / NW, u1 = c0 + (int64_t)share * (warp + 1) / NW;

  // ---- the warp's pages
  if (u0 < u1) {
    if (!a.alone) s = locate<PAIRS>(a, pre, u0);
    if (lane == 0) {
      s_now[warp] = s;
      s_next[warp] = s.seq;
      s_range[warp][0] = u0;
      s_range[warp][1] = u1;
    }
    __syncwarp();
    uint8_t *kbuf = sm + warp * L::kPage, *vbuf = kbuf + 4 * HB;
    // cursor of the copies, one page ahead
    int fj = s.lo + (int)(u0 - s.begin), frem = (int)(s.end - u0), fleft = (int)(u1 - u0), fh = s.h, flen = s.len;
    auto page_at = [&]() { return fj < a.max_pages ? __ldg(a.table + (size_t)s_next[warp] * a.max_pages + fj) : -1; };
    int fpage = page_at();
    auto copy = [&](int half, bool more) {  // keys (0) or values (1) of the page at the cursor
      if (!more) return;
      const bool ok = (unsigned)fpage < (unsigned)a.n_pages;
      const int tiles = ok ? min(4, (flen - fj * kKv4PageRows + kKv4TileRows - 1) / kKv4TileRows) : 0;
      if (lane == 0) {
        if (tiles > 0) mbar_arrive_expect_tx(&bar[half], (uint32_t)(tiles * HB));
        else mbar_arrive(&bar[half]);
      }
      __syncwarp();
      if (lane < tiles)
        bulk_g2s((half ? vbuf : kbuf) + lane * HB,
                 a.pages + ((int64_t)fpage * a.G + fh) * (4 * TB) + lane * TB + half * HB, HB, &bar[half]);
    };
    bool ok = (unsigned)fpage < (unsigned)a.n_pages;
    copy(0, fleft > 0);
    copy(1, fleft > 0);

    int left = (int)(u1 - u0);
    uint32_t phase = 0;
    // a copy did not come: seen by this lane, and (from the next vote on) by the
    // warp; then nothing more is asked for, and what is open gets NaN
    bool came = true, lost = false;
    const int czero[4] = {0, 0, 0, 0};
    while (left > 0) {
      // ---- query columns of this segment: lane (g, t) holds column g, that
      // is plane 1 (g even) or 0 (g odd) of pair g >> 1, at dimensions 8 t ..
      // 8 t + 7 of every block (even ones in the first word, as in a key word)
      uint32_t q[NT][NB][2], qt[TT][NB][2];
      int jmax[NT], jmin[NT];
      float qscale[NT];
      const Segment &s = s_now[warp];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        int head;
        const long long row = pair_row<PAIRS>(a, s.q0, s.ql, s.ct, 4 * nt + (g >> 1), &head);
        float x[NB][8];
        uint32_t top = 0;  // bits of the largest magnitude
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[b][i] = 0.f;
          if (row >= 0) {
            const int64_t at = row * a.q_stride + (s.h * grp + head) * HD + 32 * b + 8 * t;
            if (a.type == IFX_TYPE_F16) {
              const uint4 v = *reinterpret_cast<const uint4 *>(static_cast<const __half *>(a.q) + at);
              const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                x[b][2 * i] = f.x;
                x[b][2 * i + 1] = f.y;
              }
            } else {
              const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(a.q) + at);
              const float4 v = p[0], w = p[1];
              x[b][0] = v.x, x[b][1] = v.y, x[b][2] = v.z, x[b][3] = v.w;
              x[b][4] = w.x, x[b][5] = w.y, x[b][6] = w.z, x[b][7] = w.w;
            }
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[b][i]) & 0x7fffffffu);
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float big = fmaxf(__uint_as_float(top), 1e-30f), up = kTop / big;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          uint32_t y[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = __float_as_uint(fmaf(x[b][i], up, kMagic));
          const uint32_t sel = (g & 1) ? 0x0040u : 0x0051u;  // bytes 0 or 1 of two words
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            q[nt][b][i] = prmt(prmt(y[i], y[i + 2], sel), prmt(y[i + 4], y[i + 6], sel), 0x5410u);
            // plane 2: column 2 t is pair t, column 2 t + 1 pair t + 4 (idle when there are four)
            const uint32_t z = prmt(prmt(y[i], y[i + 2], 0x0062u), prmt(y[i + 4], y[i + 6], 0x0062u), 0x5410u);
            if (NT == 1 || (g & 1) == (nt & 1)) qt[nt / 2][b][i] = (z << 1) ^ kSign;
          }
        }
        // lane (g, t) now turns to the scores of pair t; a query that is not
        // finite has scores NaN
        const uint32_t tops = __shfl_sync(0xffffffffu, top, 8 * t);
        const float bigs = fmaxf(__uint_as_float(tops), 1e-30f);
        qscale[nt] = tops >= 0x7f800000u ? __uint_as_float(0x7fc00000u)
                                         : a.scale * (1.4426950408889634f / 16.f) * (bigs / kTop);
        int tok;
        const long long prow = pair_row<PAIRS>(a, s.q0, s.ql, s.ct, 4 * nt + t, &tok);
        // rows jmin .. jmax are seen (a column without a query, whose result is
        // not written, sees whatever is there)
        const int pos = s.len - s.ql + (int)(prow - s.q0);
        jmax[nt] = prow >= 0 ? pos : INT32_MAX;
        jmin[nt] = prow >= 0 && a.window ? max(0, pos - a.window + 1) : 0;
      }
      int see_lo = 0, see_hi = INT32_MAX;  // rows that every column sees
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        see_lo = max(see_lo, jmin[nt]);
        see_hi = min(see_hi, jmax[nt]);
      }
      see_lo = __reduce_max_sync(0xffffffffu, see_lo);
      see_hi = __reduce_min_sync(0xffffffffu, see_hi);
      float o[NT][NB][4], m[NT], l[NT];  // of pair t: dimensions 4 g .. 4 g + 3 of every block
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        m[nt] = -INFINITY;
        l[nt] = 0.f;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[nt][b][i] = 0.f;
      }

      const int len = s.len;
      const long long at = s_range[warp][1] - left;
      int row0 = (s.lo + (int)(at - s.begin)) * kKv4PageRows;
      int todo = min(left, (int)(s.end - at));
      left -= todo;
      for (; todo > 0 && !lost; --todo, row0 += kKv4PageRows) {
        // the cursor moves to the next page (its table entry is on its way
        // while this page's keys are multiplied)
        const bool here = ok;
        --fleft;
        --frem;
        ++fj;
        const bool more = fleft > 0;
        if (more) {
          if (frem == 0) {
            const Segment n = locate<PAIRS>(a, pre, s_range[warp][1] - fleft);
            fj = n.lo, frem = (int)(n.end - n.begin), fh = n.h, flen = n.len;
            __syncwarp();
            if (lane == 0) s_next[warp] = n.seq;
            __syncwarp();
          }
          fpage = page_at();
        }
        // rows that hold nothing (behind the last one, or of a page that does
        // not exist) get scale 0, whatever bytes are there; as values that of the
        // page's first row, since a small one would make the page uneven
        const int live_rows = here ? len - row0 : 0;
        const bool clear = live_rows < kKv4PageRows;
        auto wipe = [&](uint8_t *buf, bool first) {
          for (int r = max(0, live_rows) + lane; r < kKv4PageRows; r += 32)
#pragma unroll
            for (int b = 0; b < NB; ++b)
              reinterpret_cast<uint16_t *>(buf + r / kKv4TileRows * HB + SC)[r % kKv4TileRows * NB + b] =
                  first && live_rows > 0 ? reinterpret_cast<const uint16_t *>(buf + SC)[b] : 0;
          __syncwarp();
        };
        // ---- scores
        came = mbar_wait(&bar[0], phase, nullptr, 0);
        if (clear) wipe(kbuf, false);
        float sc[4][NT][2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint8_t *tb = kbuf + i * HB;
          uint32_t k0[NB], k1[NB];
          ld_words<NB>(tb + (g * 4 + t) * 4 * NB, k0);
          ld_words<NB>(tb + ((g + 8) * 4 + t) * 4 * NB, k1);
          float d0[NB], d1[NB];
          ld_scales<NB>(tb + SC + g * 2 * NB, d0);
          ld_scales<NB>(tb + SC + (g + 8) * 2 * NB, d1);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) sc[i][nt][0] = sc[i][nt][1] = 0.f;
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            const uint32_t w[4] = {(k0[b] << 4 & kHigh) ^ kSign, (k1[b] << 4 & kHigh) ^ kSign, (k0[b] & kHigh) ^ kSign,
                                   (k1[b] & kHigh) ^ kSign};
            int top[TT][4];
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) mma_ss(top[tt], w, qt[tt][b][0], qt[tt][b][1], czero);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              int acc[4];
              mma_su(acc, w, q[nt][b][0], q[nt][b][1], czero);
              sc[i][nt][0] = fmaf(d0[b], planes(top[nt / 2][nt & 1], acc[0], acc[1]), sc[i][nt][0]);
              sc[i][nt][1] = fmaf(d1[b], planes(top[nt / 2][2 + (nt & 1)], acc[2], acc[3]), sc[i][nt][1]);
            }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            sc[i][nt][0] *= qscale[nt];
            sc[i][nt][1] *= qscale[nt];
          }
        }
        if (clear) fence_proxy_async_smem();  // the scales written above, before the next copy
        lost = !__all_sync(0xffffffffu, came);
        if (lost) {  // (copies on their way write this CTA's memory)
          mbar_wait(&bar[0], phase, nullptr, 0);
          mbar_wait(&bar[1], phase, nullptr, 0);
          break;
        }
        copy(0, more);
        if (!here || row0 < see_lo || row0 + kKv4PageRows - 1 > see_hi) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = row0 + i * kKv4TileRows + g;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if (!here || j < jmin[nt] || j > jmax[nt]) sc[i][nt][0] = -INFINITY;
              if (!here || j + 8 < jmin[nt] || j + 8 > jmax[nt]) sc[i][nt][1] = -INFINITY;
            }
          }
        }
        // ---- the page's maxima of value scales and scores, the running maximum
        came = mbar_wait(&bar[1], phase, nullptr, 0);
        phase ^= 1;
        if (clear) wipe(vbuf, true);
        uint32_t top = 0, low = 0x7fff7fffu;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 8 * NB; e += 32)
            if (8 * NB % 32 == 0 || e + lane < 8 * NB) {
              const uint32_t w = reinterpret_cast<const uint32_t *>(vbuf + i * HB + SC)[e + lane] & 0x7fff7fffu;
              top = __vmaxu2(top, w);
              low = __vminu2(low, w);
            }
        top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
        low = __reduce_min_sync(0xffffffffu, min(low & 0xffffu, low >> 16));
        const float dmax = __half2float(__ushort_as_half((uint16_t)min(top, 0x7bffu)));
        const float ps = top ? kTop / dmax : 0.f;
        const bool uneven = kUneven * __half2float(__ushort_as_half((uint16_t)min(low, 0x7bffu))) < dmax;
        float beta[NT], share[NT], base[NT];  // of this page's p dV and p in the running sums
        bool moved = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float loc = -INFINITY;
#pragma unroll
          for (int i = 0; i < 4; ++i) loc = fmaxf(loc, fmaxf(sc[i][nt][0], sc[i][nt][1]));
          loc = quad_rows_max(loc);
          base[nt] = loc == -INFINITY ? 0.f : loc;  // nothing seen here: exp2(-inf - 0) = 0
          share[nt] = 1.f;
          beta[nt] = 1.f;
          if (loc > m[nt]) {
            beta[nt] = ex2(m[nt] - loc);
            m[nt] = loc;
            l[nt] *= beta[nt];
            moved = true;
          } else {
            share[nt] = loc == -INFINITY ? 0.f : ex2(loc - m[nt]);
          }
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
              for (int i = 0; i < 4; ++i) o[nt][b][i] *= beta[nt];
        }
        // ---- probabilities
        uint32_t lifts = 0;  // a byte per column tile: sc counts in 2^lift times ps, beta in its reciprocal
        auto power = [](int e) { return __uint_as_float((uint32_t)(127 + e) << 23); };
        // how far a block's largest term of every query lies below the range
        auto room = [&](int b, int (&by)[NT], auto term) {
          float most[NT] = {};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint16_t *eb = reinterpret_cast<const uint16_t *>(vbuf + i * HB + SC) + g * NB + b;
            const float ea = fabsf(h2f(eb[0])), ec = fabsf(h2f(eb[8 * NB]));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) most[nt] = fmaxf(most[nt], fmaxf(term(i, nt, 0) * ea, term(i, nt, 1) * ec));
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const float x = quad_rows_max(most[nt]);
            const int was = (int)(lifts >> (8 * nt) & 255u);
            by[nt] = x > 0.f ? max(0, min(kMaxLift, was + (int)(__float_as_uint(__fdividef(kTop, x)) >> 23) - 127)) - was : 0;
            lifts += (uint32_t)by[nt] << (8 * nt);
          }
        };
        int first[NT] = {};
        if (uneven) room(0, first, [&](int i, int nt, int r) { return ex2(sc[i][nt][r] - base[nt]) * ps; });
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          beta[nt] = share[nt] * dmax * (1.f / (16.f * kTop)) * power(-first[nt]);
          const float pl = ps * power(first[nt]);
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const float p = ex2(sc[i][nt][r] - base[nt]);
              sum += p;
              sc[i][nt][r] = p * pl;
            }
          l[nt] = fmaf(share[nt], sum, l[nt]);
        }
        // ---- the value product
        uint32_t v0[4][NB], v1[4][NB];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          ld_words<NB>(vbuf + i * HB + (t * 8 + g) * 4 * NB, v0[i]);
          ld_words<NB>(vbuf + i * HB + ((t + 4) * 8 + g) * 4 * NB, v1[i]);
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          if (b > 0 && uneven) {
            int by[NT];
            room(b, by, [&](int i, int nt, int r) { return sc[i][nt][r]; });
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              beta[nt] *= power(-by[nt]);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                sc[i][nt][0] *= power(by[nt]);
                sc[i][nt][1] *= power(by[nt]);
              }
            }
          }
          uint32_t lo[NT][4], hi[TT][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint16_t *eb = reinterpret_cast<const uint16_t *>(vbuf + i * HB + SC) + g * NB + b;
            const float ea = h2f(eb[0]), ec = h2f(eb[8 * NB]);
            uint32_t xa[NT], xb[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              xa[nt] = __float_as_uint(fmaf(sc[i][nt][0], ea, kMagic));
              xb[nt] = __float_as_uint(fmaf(sc[i][nt][1], ec, kMagic));
              // element 2 t: bytes 1 of rows g and g + 8, element 2 t + 1: bytes 0
              lo[nt][i] = movm_trans(prmt(xa[nt], xb[nt], 0x4051u));
            }
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) {
              uint32_t w = prmt(xa[2 * tt], xb[2 * tt], 0x0062u);
              if (NT > 1) w = prmt(w, prmt(xa[NT > 1 ? 2 * tt + 1 : 0], xb[NT > 1 ? 2 * tt + 1 : 0], 0x0062u), 0x5410u);
              hi[tt][i] = movm_trans((w << 1) ^ kSign);  // 64 + digit, doubled: 128 + 2 digit
            }
          }
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
            // dimensions 4 g + 2 mt (low nibbles) and + 1 (high), rows 2 t, 2 t + 8, 2 t + 1, 2 t + 9 of two tiles
            const uint32_t sel = mt ? 0x7351u : 0x6240u;
            int top2[TT][4], acc[NT][4];
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              const uint32_t c0 = prmt(v0[i][b], v1[i][b], sel), c1 = prmt(v0[i + 1][b], v1[i + 1][b], sel);
              const uint32_t w[4] = {(c0 << 4 & kHigh) ^ kSign, (c0 & kHigh) ^ kSign, (c1 << 4 & kHigh) ^ kSign, (c1 & kHigh) ^ kSign};
#pragma unroll
              for (int tt = 0; tt < TT; ++tt) {
                if (i) mma_ss(top2[tt], w, hi[tt][i], hi[tt][i + 1], top2[tt]);
                else mma_ss(top2[tt], w, hi[tt][i], hi[tt][i + 1], czero);
              }
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                if (i) mma_su(acc[nt], w, lo[nt][i], lo[nt][i + 1], acc[nt]);
                else mma_su(acc[nt], w, lo[nt][i], lo[nt][i + 1], czero);
              }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int r = 0; r < 2; ++r)
                o[nt][b][2 * mt + r] = fmaf(beta[nt], planes(top2[nt / 2][2 * r + (nt & 1)], acc[nt][2 * r], acc[nt][2 * r + 1]),
                                            o[nt][b][2 * mt + r]);
          }
        }
        if (clear) fence_proxy_async_smem();
        lost = !__all_sync(0xffffffffu, came);
        if (lost) {
          mbar_wait(&bar[1], phase ^ 1, nullptr, 0);
          if (more) mbar_wait(&bar[0], phase, nullptr, 0);
          break;
        }
        copy(1, more);
        ok = (unsigned)fpage < (unsigned)a.n_pages;
      }

      // ---- the segment's end, or the range's
      const long long from = s_range[warp][0], to = s_range[warp][1];
      const bool whole = s.begin >= from && s.end <= to;
      const int slot = 2 * warp + (s.begin > from ? 1 : 0);
      float *part = L::part(sm, slot);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float sum = lost ? __uint_as_float(0x7fc00000u) : quad_rows_sum(l[nt]);
        int head;
        const long long row = pair_row<PAIRS>(a, s.q0, s.ql, s.ct, 4 * nt + t, &head);
        const float f = !whole ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const float4 v = make_float4(f * o[nt][b][0], f * o[nt][b][1], f * o[nt][b][2], f * o[nt][b][3]);
          if (!whole)
            *reinterpret_cast<float4 *>(part + (4 * nt + t) * HD + 32 * b + 4 * g) = v;
          else if (row >= 0)
            write4(a, row, (s.h * grp + head) * HD + 32 * b + 4 * g, v);
        }
        if (!whole && g == 0) {
          part[PAIRS * HD + 4 * nt + t] = m[nt];
          part[PAIRS * (HD + 1) + 4 * nt + t] = sum;
        }
      }
      if (!whole && lane == 0) {
        s_seq[slot][0] = s.seq;
        s_seq[slot][1] = s.h;
        s_seq[slot][2] = s.ct;
        s_whole[slot] = s.begin >= s_cta[0] && s.end <= s_cta[1];
        s_join[slot] = s.begin <= s_cta[0] ? 0 : 1;
      }
      if (left > 0) {
        const Segment n = locate<PAIRS>(a, pre, to - left);
        __syncwarp();
        if (lane == 0) s_now[warp] = n;
        __syncwarp();
      }
    }
    if (lost && lane == 0 && a.err) atomicExch(a.err, kErrKv4);
  }
  __syncthreads();

  // ---- join the CTA's partials of one segment (slots that follow one
  // another): every warp finds the runs of slots for itself
  static_assert(2 * NW <= 32, "");
  const int mine0 = lane < 2 * NW ? s_seq[lane][0] : -1;
  const uint32_t used = __ballot_sync(0xffffffffu, mine0 >= 0);
  const int mine1 = mine0 >= 0 ? s_seq[lane][1] : 0, mine2 = mine0 >= 0 ? s_seq[lane][2] : 0;
  const uint32_t lower = used & ((1u << lane) - 1);
  const int from = lower ? 31 - __clz(lower) : lane;
  const int prev0 = __shfl_sync(0xffffffffu, mine0, from), prev1 = __shfl_sync(0xffffffffu, mine1, from),
            prev2 = __shfl_sync(0xffffffffu, mine2, from);
  const bool follows = lower != 0 && prev0 == mine0 && prev1 == mine1 && prev2 == mine2;
  uint32_t starts = __ballot_sync(0xffffffffu, mine0 >= 0 && !follows);
  float *out_parts = reinterpret_cast<float *>(static_cast<uint8_t *>(a.ws) + gridDim.x * sizeof(RangeInfo)) +
                     (size_t)blockIdx.x * 2 * (L::kPart / 4);
  while (starts) {
    const int i = __ffs(starts) - 1;
    starts &= starts - 1;
    const uint32_t run = used & ~((1u << i) - 1) & (starts ? (1u << (__ffs(starts) - 1)) - 1 : 0xffffffffu);
    const Seq sq = sequence<PAIRS>(a, s_seq[i][0]);
    const int h = s_seq[i][1], ct = s_seq[i][2];
    for (int e = tid; e < PAIRS * HD / 4; e += NW * 32) {
      const int p = e / (HD / 4), c = e % (HD / 4) * 4;
      float M = -INFINITY, S = 0.f;
      for (uint32_t k = run; k; k &= k - 1) M = fmaxf(M, L::part(sm, __ffs(k) - 1)[PAIRS * HD + p]);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      const float base = M == -INFINITY ? 0.f : M;
      for (uint32_t k = run; k; k &= k - 1) {
        const float *pt = L::part(sm, __ffs(k) - 1);
        const float w = ex2(pt[PAIRS * HD + p] - base);
        S = fmaf(w, pt[PAIRS * (HD + 1) + p], S);
        const float4 x = *reinterpret_cast<const float4 *>(pt + p * HD + c);
        v.x = fmaf(w, x.x, v.x), v.y = fmaf(w, x.y, v.y), v.z = fmaf(w, x.z, v.z), v.w = fmaf(w, x.w, v.w);
      }
      if (s_whole[i]) {
        int head;
        const long long row = pair_row<PAIRS>(a, sq.q0, sq.ql, ct, p, &head);
        const float f = S == 0.f ? 0.f : 1.f / S;
        if (row >= 0) write4(a, row, (h * grp + head) * HD + c, make_float4(v.x * f, v.y * f, v.z * f, v.w * f));
      } else {
        float *dst = out_parts + s_join[i] * (L::kPart / 4);
        *reinterpret_cast<float4 *>(dst + p * HD + c) = v;
        if (c == 0) {
          dst[PAIRS * HD + p] = M;
          dst[PAIRS * (HD + 1) + p] = S;
        }
      }
    }
  }
}

// Joins the segments that lie across CTAs: block c takes the segment that
// holds CTA c's first tile if it began within CTA c - 1 (one block per
// segment), whose parts are c - 1's last and the first of c, c + 1, ...
constexpr int kJoinThreads = 256;

template <int PAIRS>
__global__ void __launch_bounds__(kJoinThreads) kv4_attn_join_kernel(const __grid_constant__ Kv4AttnArgs a) {
  __shared__ float s_w[2 * kNumSMs * PAIRS], s_l[2 * kNumSMs * PAIRS], s_inv[PAIRS];
  __shared__ float4 s_sum[kJoinThreads];
  pdl_wait();
  const RangeInfo *info = static_cast<const RangeInfo *>(a.ws);
  const int c = blockIdx.x + 1, HD = a.hd, grp = a.H / a.G, tid = threadIdx.x, lane = tid & 31;
  const RangeInfo r = info[c];
  if (!r.live) return;
  const Deal deal(r.total, r.live);
  const long long mine = deal.begin(c), prev = deal.begin(c - 1);
  if (r.begin >= mine || r.begin < prev) return;
  const int part = PAIRS * (HD + 2);
  const float *parts = reinterpret_cast<const float *>(static_cast<const uint8_t *>(a.ws) + (gridDim.x + 1) * sizeof(RangeInfo));
  // the parts: CTA c - 1's last (its first if the segment began there), then
  // the first of every CTA up to the one that holds the segment's last tile
  auto at = [&](int k) { return parts + (size_t)(2 * (c - 1 + k) + (k == 0 && r.begin > prev ? 1 : 0)) * part; };
  const int n = deal.owner(r.end - 1) - c + 2;
  for (int e = tid; e < n * PAIRS; e += kJoinThreads) {
    const float *pt = at(e / PAIRS) + PAIRS * HD + e % PAIRS;
    s_w[e] = pt[0];
    s_l[e] = pt[PAIRS];
  }
  __syncthreads();
  for (int p = tid >> 5; p < PAIRS; p += kJoinThreads / 32) {
    float M = -INFINITY, S = 0.f;
    for (int k = lane; k < n; k += 32) M = fmaxf(M, s_w[k * PAIRS + p]);
    M = warp_max(M);
    const float base = M == -INFINITY ? 0.f : M;
    for (int k = lane; k < n; k += 32) {
      const float w = ex2(s_w[k * PAIRS + p] - base);
      s_w[k * PAIRS + p] = w;
      S = fmaf(w, s_l[k * PAIRS + p], S);
    }
    S = warp_sum(S);
    if (lane == 0) s_inv[p] = S == 0.f ? 0.f : 1.f / S;
  }
  __syncthreads();
  const Seq sq = sequence<PAIRS>(a, r.seq);
  // `ways` threads share an output's parts
  const int cells = PAIRS * HD / 4, ways = max(1, kJoinThreads / cells);
  for (int e0 = 0; e0 < cells; e0 += kJoinThreads) {
    const int e = e0 + tid % cells, way = ways > 1 ? tid / cells : 0;
    const bool on = ways > 1 ? way < ways : e0 + tid < cells;
    const int cell = ways > 1 ? e : e0 + tid, p = on ? cell / (HD / 4) : 0, col = cell % (HD / 4) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (on) {
#pragma unroll 8
      for (int k = way; k < n; k += ways) {
        const float w = s_w[k * PAIRS + p];
        const float4 x = *reinterpret_cast<const float4 *>(at(k) + p * HD + col);
        v.x = fmaf(w, x.x, v.x), v.y = fmaf(w, x.y, v.y), v.z = fmaf(w, x.z, v.z), v.w = fmaf(w, x.w, v.w);
      }
    }
    if (ways > 1) {
      s_sum[tid] = v;
      __syncthreads();
      for (int k = 1; on && way == 0 && k < ways; ++k) {
        const float4 x = s_sum[tid + k * cells];
        v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
      }
    }
    int head;
    const long long row = pair_row<PAIRS>(a, sq.q0, sq.ql, r.ct, p, &head);
    if (on && way == 0 && row >= 0) {
      const float f = s_inv[p];
      write4(a, row, (r.h * grp + head) * HD + col, make_float4(v.x * f, v.y * f, v.z * f, v.w * f));
    }
  }
}

template <int NB, int NT, int NW, int MINB>
ifx_status run(const Kv4AttnArgs &args, bool alone, cudaStream_t st) {
  using L = Smem<NB, NT, NW>;
  auto kernel = kv4_attn_kernel<NB, NT, NW, MINB>;
  Kv4AttnArgs a = args;
  const size_t smem = L::kBytes + ((size_t)a.n_seqs + 1) * sizeof(long long);
  static std::atomic<uint64_t> done{0};
  IFX_TRY(raise_smem(kernel, L::kBytes + (kMaxAttnSeqs + 1) * 8, done));
  a.alone = alone;
  const int grid = alone ? a.n_seqs * a.G * ((a.H / a.G + 4 * NT - 1) / (4 * NT)) : kNumSMs * MINB;
  kernel<<<grid, NW * 32, smem, st>>>(a);
  IFX_CUDA(cudaGetLastError());
  if (!a.alone) IFX_CUDA(launch(kv4_attn_join_kernel<4 * NT>, dim3(grid - 1), dim3(kJoinThreads), 0, st, true, a));
  return IFX_OK;
}

template <int NB>
ifx_status run_nb(const Kv4AttnArgs &a, cudaStream_t st) {
  const int64_t columns = kv4_columns(a);
  // One row per sequence and short tables: a CTA per segment, whose warps
  // share its pages, and no second kernel. 16 sequences of 460 to 2300 keys,
  // 128 segments: 18 us against 23; 1100 keys: 13.4 us against 13.7, with
  // one launch less for the host. With more
  // than four pages a warp, or more segments than SMs, the dealt form is
  // even where this one waits for its longest segment.
  auto alone = [&](int pairs, int warps) {
    return !a.q_start && (int64_t)a.n_seqs * a.G * ((a.H / a.G + pairs - 1) / pairs) <= kNumSMs && a.max_pages <= 4 * warps;
  };
  if constexpr (NB <= 4) {
    if (columns > 4) return run<NB, 2, 12, 1>(a, alone(8, 12), st);
    if (alone(4, 12)) return run<NB, 1, 12, 1>(a, true, st);
    return run<NB, 1, 6, 2>(a, false, st);
  } else {
    return run<NB, 1, 8, 1>(a, alone(4, 8), st);
  }
}

}  // namespace

size_t kv4_attention_ws(int, int, int hd) { return kv4_chunks_ws(hd); }  // (the kernel above needs less)

ifx_status op_kv4_attention(const Kv4AttnArgs &a, cudaStream_t st) {
  if (!a.rows) return IFX_OK;
  if (kv4_chunks_take(a)) return kv4_attention_chunks(a, st);
  switch (a.hd / 32) {
    case 1: return run_nb<1>(a, st);
    case 2: return run_nb<2>(a, st);
    case 3: return run_nb<3>(a, st);
    case 4: return run_nb<4>(a, st);
    case 5: return run_nb<5>(a, st);
    case 6: return run_nb<6>(a, st);
    case 7: return run_nb<7>(a, st);
    default: return run_nb<8>(a, st);
  }
}

}  // namespace ifx
