// Attention over the key/value cache in 4 bits.
#include <algorithm>

#include "serve.cuh"

namespace ifx {

namespace {

template <typename T>
__device__ __forceinline__ float to_f32(T x) { return (float)x; }

// Plain form: one warp per (query row, head), a running maximum and sum over
// the rows it sees; lane l holds dimensions l, l + 32, ...
template <typename T>
__global__ void __launch_bounds__(128) kv4_attn_plain_kernel(const __grid_constant__ Kv4AttnArgs a) {
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, nb = a.hd / 32;
  const int64_t row = unit / a.H;
  const int head = (int)(unit % a.H), h = head / (a.H / a.G);
  if (row >= a.rows) return;
  int seq = (int)row, i = 0, ql = 1;
  if (a.q_start) {
    int lo = 0, hi = a.n_seqs;  // the last sequence that starts at or before row
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.q_start[mid] <= row) lo = mid; else hi = mid - 1;
    }
    seq = lo;
    if (seq >= a.n_seqs) return;  // behind the last sequence: left as it was
    i = (int)row - a.q_start[seq];
    ql = a.q_start[seq + 1] - a.q_start[seq];
  }
  const int len = min(a.kv_len[seq], a.max_pages * kKv4PageRows);
  const int pos = len - ql + i;
  const int first = a.window ? max(0, pos - a.window + 1) : 0;
  const T *q = static_cast<const T *>(a.q) + row * a.q_stride + head * a.hd;
  float qv[8], o[8] = {}, m = -INFINITY, l = 0.f;
  for (int b = 0; b < nb; ++b) qv[b] = to_f32(q[b * 32 + lane]) * a.scale;
  for (int t = first; t <= pos; ++t) {
    const int page = a.table[(size_t)seq * a.max_pages + t / kKv4PageRows];
    if (page < 0 || page >= a.n_pages) continue;
    const int r = t % kKv4TileRows;
    const uint8_t *tile = a.pages + ((int64_t)page * a.G + h) * Kv4Layout::head_bytes(nb) +
                          t % kKv4PageRows / kKv4TileRows * Kv4Layout::tile_bytes(nb);
    float s = 0.f;
    for (int b = 0; b < nb; ++b) {
      const uint32_t w = reinterpret_cast<const uint32_t *>(tile)[(r * 4 + lane / 8) * nb + b];
      const float d = h2f(reinterpret_cast<const uint16_t *>(tile + Kv4Layout::k_scales(nb))[r * nb + b]);
      s += qv[b] * d * (float)((int)(w >> (4 * (lane % 8)) & 15u) - 8);
    }
    s = warp_sum(s);
    const float m2 = fmaxf(m, s), c = expf(m - m2), p = expf(s - m2);
    m = m2;
    l = l * c + p;
    for (int b = 0; b < nb; ++b) {
      const uint32_t w = reinterpret_cast<const uint32_t *>(tile + Kv4Layout::v_words(nb))[(r / 2 * 8 + lane / 4) * nb + b];
      const float d = h2f(reinterpret_cast<const uint16_t *>(tile + Kv4Layout::v_scales(nb))[r * nb + b]);
      o[b] = o[b] * c + p * d * (float)((int)(w >> (16 * (r & 1) + 4 * (lane % 4)) & 15u) - 8);
    }
  }
  T *out = static_cast<T *>(a.out) + row * a.out_stride + head * a.hd;
  for (int b = 0; b < nb; ++b) out[b * 32 + lane] = (T)(l > 0.f ? o[b] / l : 0.f);
}

}  // namespace

size_t kv4_attention_ws(int, int, int) { return 0; }

ifx_status op_kv4_attention(const Kv4AttnArgs &a, cudaStream_t st) {
  if (!a.rows) return IFX_OK;
  const unsigned grid = (unsigned)((a.rows * a.H + 3) / 4);
  if (a.type == IFX_TYPE_F16)
    kv4_attn_plain_kernel<__half><<<grid, 128, 0, st>>>(a);
  else
    kv4_attn_plain_kernel<float><<<grid, 128, 0, st>>>(a);
  IFX_CUDA(cudaGetLastError());
  return IFX_OK;
}

}  // namespace ifx
