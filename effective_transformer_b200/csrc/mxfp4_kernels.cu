// Rows to MXFP4 and back, and weights to MXFP4 (layout and rounding: mxfp4.cuh).
//
// All three only move data: a row of K values is read once (2 or 4 bytes a value) and written as 17 / 32 byte a value,
// or back.  39778 x 4096 fp16 values, 413 MB: 72 us (5.7 TB/s) to MXFP4, 76 us (5.4 TB/s) back; a copy of the rows
// reaches 6.5 TB/s, stores alone 5.8 to 6.5.  Below some thousand rows both are latency: 3001 x 800 fp32 values from L2
// take 4 and 5.6 us.
#include "common.cuh"
#include "mxfp4.cuh"

namespace etb {

namespace {

constexpr int kThreads = 256;
constexpr int kBackTiles = 2;  // k-tiles of a row that a warp turns back at a time (four: 3001 x 800 12.6 us for both
                               // directions instead of 9.7, the same at 39778 x 4096)

// Two codes, j = 0..3 of a word of eight.
__device__ __forceinline__ __half2 mx_values2(uint32_t code, int j) {
  uint32_t h2;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t}"
      : "=r"(h2)
      : "r"(code >> (8 * j)));
  return *reinterpret_cast<const __half2*>(&h2);
}

// Sixteen consecutive values of a row: largest magnitude as fp32 bits, and the values.
template <typename T>
struct Sixteen;
template <>
struct Sixteen<__half> {
  Vec16 v[2];
  __device__ __forceinline__ void load(const __half* p) {
    v[0] = ld_activation_v4(p);
    v[1] = ld_activation_v4(p + 8);
  }
  __device__ __forceinline__ uint32_t top() const {
    const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
    __half2 h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = __habs2(*reinterpret_cast<const __half2*>(&w[i]));
#pragma unroll
    for (int n = 4; n >= 1; n >>= 1)
#pragma unroll
      for (int i = 0; i < n; ++i) h[i] = __hmax2_nan(h[i], h[i + n]);
    return abs_bits(__half2float(__hmax_nan(__low2half(h[0]), __high2half(h[0]))));
  }
  __device__ __forceinline__ void unpack(float* f) const {
    VecTraits<__half>::unpack(v[0], f);
    VecTraits<__half>::unpack(v[1], f + 8);
  }
};
template <>
struct Sixteen<float> {
  Vec16 v[4];
  __device__ __forceinline__ void load(const float* p) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = ld_activation_v4(p + 4 * i);
  }
  __device__ __forceinline__ uint32_t top() const {
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) m = max(m, w[j] & 0x7fffffffu);
    }
    return m;
  }
  __device__ __forceinline__ void unpack(float* f) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) VecTraits<float>::unpack(v[i], f + 4 * i);
  }
};

// A warp takes 512 values (two k-tiles) of kRows rows at a time: a lane holds sixteen values of each, two lanes a scale
// block.  (256 values, four lanes a block: twice the instructions for maxima, scales and addresses.)  32 bytes a lane
// in fp16, where eight CTAs per SM then keep enough of them in flight (two rows, six CTAs: 73 us as well, but 6.3 us
// instead of 5.7 at 11003 x 768); 128 bytes in fp32 (one row: 20.2 us instead of 16.0 at 20011 x 1024).
template <typename T>
constexpr int kRows = sizeof(T) == 2 ? 1 : 2;

template <typename T>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 8 : 4)
mx_quantize_kernel(const T* x, long long row_stride, const int* m_ptr, int max_m, int k, uint8_t* mx) {
  constexpr int R = kRows<T>;
  static_assert(kMxTileRows % R == 0, "the rows are of one tile");
  pdl_trigger();
  int rows = max_m;
  if (m_ptr != nullptr) rows = pdl_wait_row_count(m_ptr, max_m, 0);
  else pdl_wait();
  const int lane = threadIdx.x & 31;
  const uint32_t k_tiles = mx_k_tiles(k), pieces = (k_tiles + 1) / 2;
  const uint32_t tasks = (static_cast<uint32_t>(rows) + R - 1) / R * pieces;  // (2^32 would not fit any memory)
  const uint32_t warps = gridDim.x * (kThreads / 32);
  for (uint32_t task = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); task < tasks; task += warps) {
    const uint32_t row0 = task / pieces * R, col = (task % pieces) * 512 + lane * 16;
    const bool in = col < static_cast<uint32_t>(k);
    const bool tile_in = col < k_tiles * kMxTileK;  // (the row's last piece may be one k-tile)
    const T* src = x + static_cast<size_t>(row0) * row_stride + col;
    Sixteen<T> v[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (in && row0 + i < rows) {
        v[i].load(src + i * row_stride);
      } else {
#pragma unroll
        for (auto& w : v[i].v) w = Vec16{0u, 0u, 0u, 0u};
      }
    }
    uint8_t* tile = mx + mx_tile_offset(row0, col >> 8, k_tiles);  // (of all rows)
    const int b = (col & 255) >> 5;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      uint32_t top = v[i].top();
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      const MxScale s = mx_scale(top);
      if (!tile_in || row0 + i >= rows) continue;
      float f[16];
      v[i].unpack(f);
      const int r = (row0 & (kMxTileRows - 1)) + i;
      *reinterpret_cast<uint2*>(tile + mx_code_offset(r, b) + (lane & 1) * 8) =
          make_uint2(mx_codes8(f, s), mx_codes8(f + 8, s));
      if ((lane & 1) == 0) tile[mx_scale_offset(r, b)] = static_cast<uint8_t>(s.byte);
    }
  }
}

// Eight codes times a scale byte, as T.
__device__ __forceinline__ void mx_values8(uint32_t code, uint32_t scale, __half* dst) {
  // In fp16, with the scale as a product of two powers of two that fp16 has: the first product is exact (codes have two
  // bits behind the leading one), or infinite where the result is, so that the second one rounds as one would.  Exponents
  // outside of [-28, 30] are cut to them: from there on everything is zero, or infinite.
  const int e = static_cast<int>(scale) - 127, e1 = min(max(e, -14), 15), e2 = min(max(e - e1, -14), 15);
  const uint32_t w1 = scale == 255u ? 0x7fff7fffu : static_cast<uint32_t>(e1 + 15) * 0x04000400u;
  const uint32_t w2 = static_cast<uint32_t>(e2 + 15) * 0x04000400u;
  const __half2 s1 = *reinterpret_cast<const __half2*>(&w1), s2 = *reinterpret_cast<const __half2*>(&w2);
  uint32_t out[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const __half2 h = __hmul2(__hmul2(mx_values2(code, j), s1), s2);
    out[j] = *reinterpret_cast<const uint32_t*>(&h);
  }
  st_global_v4(dst, Vec16{out[0], out[1], out[2], out[3]});
}
__device__ __forceinline__ void mx_values8(uint32_t code, uint32_t scale, float* dst) {
  const float s = mx_scale_value(scale);
  float f[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 p = __half22float2(mx_values2(code, j));
    f[2 * j] = p.x * s;
    f[2 * j + 1] = p.y * s;
  }
  st_global_v4(dst, VecTraits<float>::pack(f));
  st_global_v4(dst + 4, VecTraits<float>::pack(f + 4));
}

// A warp takes kBackTiles k-tiles of a row at a time: a lane holds eight values of each, so that a warp reads lines of
// 128 bytes of codes and writes 512 or 1024 contiguous bytes.
template <typename T>
__global__ void __launch_bounds__(kThreads)
mx_dequantize_kernel(const uint8_t* mx, const int* m_ptr, int max_m, int k, T* out) {
  pdl_trigger();
  int rows = max_m;
  if (m_ptr != nullptr) rows = pdl_wait_row_count(m_ptr, max_m, 0);
  else pdl_wait();
  const int lane = threadIdx.x & 31;
  const uint32_t k_tiles = mx_k_tiles(k), pieces = (k_tiles + kBackTiles - 1) / kBackTiles;
  const uint32_t tasks = static_cast<uint32_t>(rows) * pieces;
  const uint32_t warps = gridDim.x * (kThreads / 32);
  for (uint32_t task = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); task < tasks; task += warps) {
    const uint32_t row = task / pieces, kt = (task - row * pieces) * kBackTiles, col = kt * kMxTileK + lane * 8;
    const int r = row & (kMxTileRows - 1), b = lane >> 2;
    const uint8_t* tile = mx + mx_tile_offset(row, kt, k_tiles);
    const uint8_t* codes = tile + mx_code_offset(r, b) + (lane & 3) * 4;
    const uint8_t* scales = tile + mx_scale_offset(r, b);
    uint32_t code[kBackTiles], scale[kBackTiles];
#pragma unroll
    for (int i = 0; i < kBackTiles; ++i)
      if (col + i * kMxTileK < static_cast<uint32_t>(k)) {
        code[i] = *reinterpret_cast<const uint32_t*>(codes + i * kMxTileBytes);
        scale[i] = scales[i * kMxTileBytes];
      }
    T* dst = out + static_cast<size_t>(row) * k + col;
#pragma unroll
    for (int i = 0; i < kBackTiles; ++i)
      if (col + i * kMxTileK < static_cast<uint32_t>(k)) mx_values8(code[i], scale[i], dst + i * kMxTileK);
  }
}

// W [K, N] -> MXFP4 rows of W^T [N, K].  A thread quantises one block: 32 values of a column, read beside its
// neighbours' columns.  Runs once per weight.
template <typename T>
__global__ void __launch_bounds__(kThreads)
mx_pack_weight_kernel(const T* w, uint8_t* mx, int k, int n) {
  const int col = blockIdx.x * kThreads + threadIdx.x;
  const int b = blockIdx.y;  // block along K, up to the width rounded up to 64
  if (col >= n) return;
  float f[kMxBlock];
  uint32_t top = 0u;
#pragma unroll
  for (int i = 0; i < kMxBlock; ++i) {
    const int kk = b * kMxBlock + i;
    f[i] = kk < k ? static_cast<float>(w[static_cast<size_t>(kk) * n + col]) : 0.f;
    top = max(top, abs_bits(f[i]));
  }
  const MxScale s = mx_scale(top);
  uint8_t* tile = mx + mx_tile_offset(col, b >> 3, mx_k_tiles(k));
  const int r = col & (kMxTileRows - 1);
  Vec16 v;
  v.x = mx_codes8(f, s);
  v.y = mx_codes8(f + 8, s);
  v.z = mx_codes8(f + 16, s);
  v.w = mx_codes8(f + 24, s);
  st_global_v4(tile + mx_code_offset(r, b & 7), v);
  tile[mx_scale_offset(r, b & 7)] = static_cast<uint8_t>(s.byte);
}

// CTAs for `tasks` warp tasks, at most 8 per SM.
inline dim3 mx_grid(long long tasks) {
  constexpr int kWarps = kThreads / 32;
  const long long ctas = (tasks + kWarps - 1) / kWarps, cap = static_cast<long long>(sm_count()) * 8;
  return dim3(static_cast<unsigned>(ctas > cap ? cap : ctas));
}

}  // namespace

template <typename T>
cudaError_t launch_mx_quantize(const T* x, long long row_stride, const int* m_ptr, int max_m, int k, void* mx,
                               cudaStream_t stream) {
  if (max_m <= 0) return cudaSuccess;
  if (k <= 0 || k % kMxBlock != 0 || row_stride < k) return cudaErrorInvalidValue;
  if ((reinterpret_cast<uintptr_t>(x) & 15u) || (row_stride * sizeof(T)) % 16 != 0 ||
      (reinterpret_cast<uintptr_t>(mx) & 127u))
    return cudaErrorMisalignedAddress;
  const long long tasks = (static_cast<long long>(max_m) + kRows<T> - 1) / kRows<T> * ((mx_k_tiles(k) + 1) / 2);
  return launch_pdl(mx_quantize_kernel<T>, mx_grid(tasks), dim3(kThreads), 0, stream, x, row_stride, m_ptr, max_m, k,
                    static_cast<uint8_t*>(mx));
}

template <typename T>
cudaError_t launch_mx_dequantize(const void* mx, const int* m_ptr, int max_m, int k, T* out, cudaStream_t stream) {
  if (max_m <= 0) return cudaSuccess;
  if (k <= 0 || k % kMxBlock != 0) return cudaErrorInvalidValue;
  if ((reinterpret_cast<uintptr_t>(out) & 15u) || (reinterpret_cast<uintptr_t>(mx) & 127u))
    return cudaErrorMisalignedAddress;
  const long long tasks = static_cast<long long>(max_m) * ((mx_k_tiles(k) + kBackTiles - 1) / kBackTiles);
  return launch_pdl(mx_dequantize_kernel<T>, mx_grid(tasks), dim3(kThreads), 0, stream,
                    static_cast<const uint8_t*>(mx), m_ptr, max_m, k, out);
}

template <typename T>
cudaError_t launch_mx_pack_weight(const T* w, void* mx, int k, int n, cudaStream_t stream) {
  if (k <= 0 || n <= 0 || k % kMxBlock != 0 || (k + 63) / 64 * 2 > 65535) return cudaErrorInvalidValue;
  if (reinterpret_cast<uintptr_t>(mx) & 127u) return cudaErrorMisalignedAddress;
  const dim3 grid((n + kThreads - 1) / kThreads, (k + 63) / 64 * 2);
  mx_pack_weight_kernel<T><<<grid, kThreads, 0, stream>>>(w, static_cast<uint8_t*>(mx), k, n);
  return cudaGetLastError();
}

#define ETB_INST(T)                                                                                             \
  template cudaError_t launch_mx_quantize<T>(const T*, long long, const int*, int, int, void*, cudaStream_t);   \
  template cudaError_t launch_mx_dequantize<T>(const void*, const int*, int, int, T*, cudaStream_t);            \
  template cudaError_t launch_mx_pack_weight<T>(const T*, void*, int, int, cudaStream_t);
ETB_INST(float)
ETB_INST(__half)
#undef ETB_INST

}  // namespace etb
