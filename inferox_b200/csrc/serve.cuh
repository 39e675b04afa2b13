// The operators of a paged serving step: page tables and slot maps, the
// key/value cache in 4 bits with its attention, and row-wise sampling.
#pragma once
#include <atomic>

#include "common.cuh"

namespace ifx {

constexpr int kKv4PageRows = 64;  // rows of a page
constexpr int kKv4TileRows = 16;  // rows of a tile (four tiles per page and kv head)
constexpr int kMaxServeSeqs = 8192;  // pages_extend / pages_release
constexpr int kMaxAttnSeqs = 2048;   // kv4_attention: their running totals stay in shared memory

// The 4-bit cache (no reference counterpart; its KvCache holds f32 rows,
// src/model/cache.rs:7-14). A page holds 64 rows; for each kv head four
// tiles of 16 rows, each contiguous, so one bulk copy fetches any run of
// tiles of a page's head. With NB = hd / 32 blocks per row a tile is
//   key words    [row][t][b]      u32: values 32 b + 8 t + i in nibble i
//   key scales   [row][b]         f16
//   value words  [row / 2][g][b]  u32: values 32 b + 4 g + j of the even row in
//                                 nibble j of the low half, of the odd row
//                                 in the high half
//   value scales [row][b]         f16
// t = 0..3 and g = 0..7 are the lane coordinates of an m16n8k16 A fragment:
// a lane's words of one row are adjacent, and masking a word gives the
// fragment's f16 pairs without any byte permutation (keys pair dimensions,
// values pair rows, which is what the two products contract over).
// A block of 32 values is quantised as Q4_0 (the weights' Q4_0, dequant.rs:
// 54-75): value (q - 8) d.
struct Kv4Layout {
  __host__ __device__ static constexpr int tile_bytes(int nb) { return 576 * nb; }
  __host__ __device__ static constexpr int k_scales(int nb) { return 256 * nb; }
  __host__ __device__ static constexpr int v_words(int nb) { return 288 * nb; }
  __host__ __device__ static constexpr int v_scales(int nb) { return 544 * nb; }
  __host__ __device__ static constexpr int head_bytes(int nb) { return 4 * tile_bytes(nb); }
};

inline bool kv4_head_dim_ok(size_t hd) { return hd >= 32 && hd <= 256 && hd % 32 == 0; }
inline size_t kv4_page_bytes(size_t G, size_t hd) { return G * (size_t)Kv4Layout::head_bytes((int)(hd / 32)); }

// A wait of these kernels that gives up sets `err` where there is one; the rows
// that it held up come out as NaN (tokens as -1 with a NaN beside them).
constexpr int kErrKv4 = 601, kErrKv4Chunk = 602, kErrSample = 603;

// Raises a kernel's shared-memory limit, once per device: `done` holds a bit
// for each (the call costs a microsecond or two).
template <typename K>
ifx_status raise_smem(K kernel, int bytes, std::atomic<uint64_t> &done) {
  int dev = 0;
  IFX_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return IFX_OK;
  IFX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  done.fetch_or(bit, std::memory_order_relaxed);
  return IFX_OK;
}

struct PagesExtendArgs {
  const int *lens, *add;
  int n_seqs;
  int *table;
  int max_pages;
  const int *free_pages;
  int n_pages;
  const int *n_free;
  int64_t max_tokens;
  int *lens_out, *n_free_out, *q_start, *slots, *positions, *seqs, *status;
};
ifx_status op_pages_extend(const PagesExtendArgs &a, cudaStream_t st);

struct PagesReleaseArgs {
  const int *done, *lens;
  int n_seqs;
  const int *table;
  int max_pages;
  int *free_pages;
  int n_pages;
  const int *n_free;
  int *lens_out, *n_free_out;
};
ifx_status op_pages_release(const PagesReleaseArgs &a, cudaStream_t st);

struct Kv4RowsArgs {
  const void *k, *v;          // store: rows in; [n][G * hd] at k_stride / v_stride
  void *k_out, *v_out;        // load: rows out, contiguous
  int type;                   // IFX_TYPE_F32 or IFX_TYPE_F16
  int64_t n, k_stride, v_stride;
  const int *slots;
  uint8_t *pages;
  int64_t n_pages;
  int G, hd;
};
ifx_status op_kv4_store(const Kv4RowsArgs &a, cudaStream_t st);
ifx_status op_kv4_load(const Kv4RowsArgs &a, cudaStream_t st);

struct Kv4AttnArgs {
  const void *q;              // [rows][H * hd] at q_stride
  void *out;                  // [rows][H * hd] at out_stride
  int type;
  int64_t q_stride, out_stride, rows;
  const uint8_t *pages;
  int64_t n_pages;
  const int *table, *kv_len, *q_start;  // q_start null: one row per sequence
  int max_pages, n_seqs, H, G, hd, window;
  float scale;
  void *ws;
  bool zero_rest = false;     // rows of out that are no sequence's become 0
  bool alone = false;         // set by the launch: a CTA per segment
  int *err = nullptr;         // device word that a wait which gives up sets
};
ifx_status op_kv4_attention(const Kv4AttnArgs &a, cudaStream_t st);
// Bytes of scratch a call with these shapes needs.
size_t kv4_attention_ws(int H, int G, int hd);

struct SampleRowsArgs {
  const float *logits;        // [rows][n] at stride
  int64_t rows, n, stride;
  const float *u, *temperature;
  const int *top_k;
  const float *top_p, *min_p;
  int *token;
  float *logprob;
  int *err = nullptr;
};
ifx_status op_sample_rows(const SampleRowsArgs &a, cudaStream_t st);

}  // namespace ifx
