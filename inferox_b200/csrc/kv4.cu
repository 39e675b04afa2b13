// Rows into and out of the key/value cache in 4 bits: per block of 32 values
// the Q4_0 rule of the weights, d = the first value of largest magnitude / -8
// as f16, q = trunc(x (1 / d) + 8.5) within 0 .. 15, value (q - 8) d.
//
// Bound by HBM: 4.5 bits a value beside the rows' 32 or 16. 4096 rows of 8
// heads of 128, f32, take 9.9 us each way (76 MB both ways together, 3.9
// TB/s); 16 rows 2.2 us, a launch.
#include <algorithm>

#include "serve.cuh"

namespace ifx {

namespace {

constexpr int kRowThreads = 256;

template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&x)[8]);
template <>
__device__ __forceinline__ void load8<float>(const float *p, float (&x)[8]) {
  const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
template <>
__device__ __forceinline__ void load8<__half>(const __half *p, float (&x)[8]) {
  const uint4 a = *reinterpret_cast<const uint4 *>(p);
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

__device__ __forceinline__ void store8(float *p, const float (&x)[8]) {
  reinterpret_cast<float4 *>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4 *>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__half *p, const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t *>(&h);
  }
  *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// Four adjacent lanes quantise one block of 32 values, eight each: the scale
// comes from the first value of the largest magnitude (kept with its sign,
// so that one end of -8..7 is exact), as the weights' Q4_0 has it. A NaN
// counts as 0 and the scale stops at f16's largest value, so every stored
// block reads back finite. Returns the eight nibbles, value i in nibble i.
__device__ __forceinline__ uint32_t quantise8(float (&x)[8], uint16_t &scale) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (x[i] != x[i]) x[i] = 0.f;
    if (fabsf(x[i]) > fabsf(m)) m = x[i];
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    const float y = __shfl_xor_sync(0xffffffffu, m, o);
    const bool low = threadIdx.x & o;  // the other lane holds earlier values
    if (fabsf(y) > fabsf(m) || (low && fabsf(y) == fabsf(m))) m = y;
  }
  const __half dh = __float2half_rn(fminf(fmaxf(m * -0.125f, -65504.f), 65504.f));
  const float d = __half2float(dh), id = d != 0.f ? 1.0f / d : 0.f;
  scale = __half_as_ushort(dh);
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // two roundings, as written (no fused multiply-add); x may be infinite
    // while id is not, and 0 * inf cannot occur: d = 0 only when all x are tiny
    const float y = __fadd_rn(__fmul_rn(x[i], id), 8.5f);
    w |= (uint32_t)fminf(fmaxf(y, 0.f), 15.f) << (4 * i);
  }
  return w;
}

// Where (slot, head) lives: its tile, and the row within it.
__device__ __forceinline__ int64_t tile_offset(int slot, int h, int G, int nb) {
  return ((int64_t)(slot / kKv4PageRows) * G + h) * Kv4Layout::head_bytes(nb) +
         (slot % kKv4PageRows / kKv4TileRows) * Kv4Layout::tile_bytes(nb);
}

// One thread: eight values of K and of V. Bound by memory (store: 8 or 4 B
// per value in, 9/16 B out); the value rows go out as 2-byte halves because
// the word they share belongs to the neighbouring row.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) kv4_store_kernel(const __grid_constant__ Kv4RowsArgs a) {
  const int nb = a.hd / 32, lanes = a.G * nb * 4;  // threads per row
  const uint32_t i = blockIdx.x * kRowThreads + threadIdx.x;  // below 2^31: the launch sees to it
  const int64_t row = i / (uint32_t)lanes;
  // whole groups of four lanes share a row and a block; lanes beyond the
  // rows keep running for the shuffles
  const uint32_t e = i - (uint32_t)row * lanes, h = e / (uint32_t)(nb * 4), b = e / 4 % (uint32_t)nb, t = e % 4;
  int slot = -1;
  if (row < a.n) slot = a.slots[row];
  if (slot < 0 || slot / kKv4PageRows >= a.n_pages) slot = -1;
  float x[8] = {}, y[8] = {};
  if (slot >= 0) {
    const int64_t at = h * a.hd + b * 32 + t * 8;
    load8(static_cast<const T *>(a.k) + row * a.k_stride + at, x);
    load8(static_cast<const T *>(a.v) + row * a.v_stride + at, y);
  }
  uint16_t kd, vd;
  const uint32_t kw = quantise8(x, kd), vw = quantise8(y, vd);
  if (slot < 0) return;
  uint8_t *tile = a.pages + tile_offset(slot, h, a.G, nb);
  const int r = slot % kKv4TileRows;
  reinterpret_cast<uint32_t *>(tile)[(r * 4 + t) * nb + b] = kw;
  uint16_t *vp = reinterpret_cast<uint16_t *>(tile + Kv4Layout::v_words(nb)) + (r & 1);
  vp[2 * ((r / 2 * 8 + 2 * t) * nb + b)] = (uint16_t)vw;
  vp[2 * ((r / 2 * 8 + 2 * t + 1) * nb + b)] = (uint16_t)(vw >> 16);
  if (t == 0) {
    reinterpret_cast<uint16_t *>(tile + Kv4Layout::k_scales(nb))[r * nb + b] = kd;
    reinterpret_cast<uint16_t *>(tile + Kv4Layout::v_scales(nb))[r * nb + b] = vd;
  }
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads) kv4_load_kernel(const __grid_constant__ Kv4RowsArgs a) {
  const int nb = a.hd / 32, lanes = a.G * nb * 4;
  const uint32_t i = blockIdx.x * kRowThreads + threadIdx.x;
  const int64_t row = i / (uint32_t)lanes;
  if (row >= a.n) return;
  const uint32_t e = i - (uint32_t)row * lanes, h = e / (uint32_t)(nb * 4), b = e / 4 % (uint32_t)nb, t = e % 4;
  const int slot = a.slots[row];
  float x[8] = {}, y[8] = {};
  if (slot >= 0 && slot / kKv4PageRows < a.n_pages) {
    const uint8_t *tile = a.pages + tile_offset(slot, h, a.G, nb);
    const int r = slot % kKv4TileRows;
    const uint32_t kw = reinterpret_cast<const uint32_t *>(tile)[(r * 4 + t) * nb + b];
    const uint16_t *vp = reinterpret_cast<const uint16_t *>(tile + Kv4Layout::v_words(nb)) + (r & 1);
    const uint32_t vw = vp[2 * ((r / 2 * 8 + 2 * t) * nb + b)] |
                        (uint32_t)vp[2 * ((r / 2 * 8 + 2 * t + 1) * nb + b)] << 16;
    const float kd = h2f(reinterpret_cast<const uint16_t *>(tile + Kv4Layout::k_scales(nb))[r * nb + b]);
    const float vd = h2f(reinterpret_cast<const uint16_t *>(tile + Kv4Layout::v_scales(nb))[r * nb + b]);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = (float)((int)(kw >> (4 * j) & 15u) - 8) * kd;
      y[j] = (float)((int)(vw >> (4 * j) & 15u) - 8) * vd;
    }
  }
  const int64_t at = row * a.G * a.hd + h * a.hd + b * 32 + t * 8;
  store8(static_cast<T *>(a.k_out) + at, x);
  store8(static_cast<T *>(a.v_out) + at, y);
}

// One launch per 2^31 - kRowThreads threads or less.
template <typename F>
ifx_status in_parts(const Kv4RowsArgs &all, F launch) {
  const int64_t lanes = (int64_t)all.G * (all.hd / 32) * 4, most = ((int64_t)INT32_MAX - kRowThreads) / lanes;
  const int64_t size = all.type == IFX_TYPE_F16 ? 2 : 4, out = (int64_t)all.G * all.hd * size;
  for (int64_t at = 0; at < all.n; at += most) {
    Kv4RowsArgs a = all;
    a.n = std::min(most, all.n - at);
    a.slots += at;
    if (a.k) a.k = static_cast<const char *>(a.k) + at * a.k_stride * size, a.v = static_cast<const char *>(a.v) + at * a.v_stride * size;
    if (a.k_out) a.k_out = static_cast<char *>(a.k_out) + at * out, a.v_out = static_cast<char *>(a.v_out) + at * out;
    launch((unsigned)((a.n * lanes + kRowThreads - 1) / kRowThreads), a);
    IFX_CUDA(cudaGetLastError());
  }
  return IFX_OK;
}

}  // namespace

ifx_status op_kv4_store(const Kv4RowsArgs &a, cudaStream_t st) {
  return in_parts(a, [&](unsigned grid, const Kv4RowsArgs &p) {
    if (p.type == IFX_TYPE_F16) kv4_store_kernel<__half><<<grid, kRowThreads, 0, st>>>(p);
    else kv4_store_kernel<float><<<grid, kRowThreads, 0, st>>>(p);
  });
}

ifx_status op_kv4_load(const Kv4RowsArgs &a, cudaStream_t st) {
  return in_parts(a, [&](unsigned grid, const Kv4RowsArgs &p) {
    if (p.type == IFX_TYPE_F16) kv4_load_kernel<__half><<<grid, kRowThreads, 0, st>>>(p);
    else kv4_load_kernel<float><<<grid, kRowThreads, 0, st>>>(p);
  });
}

}  // namespace ifx
