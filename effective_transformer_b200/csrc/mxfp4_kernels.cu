// Rows to MXFP4 and back, and weights to MXFP4 (layout and rounding: mxfp4.cuh).
//
// All three only move data: a row of K values is read once (2 or 4 bytes a value) and written as 17 / 32 byte a value.
#include "common.cuh"
#include "mxfp4.cuh"

namespace etb {

namespace {

constexpr int kThreads = 256;
constexpr int kTasks = 2;  // pieces of 512 values a warp has in flight

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
  // (the bits of non-negative fp16 numbers are in the order of the numbers, infinity and NaN on top)
  __device__ __forceinline__ uint32_t top() const {
    uint32_t m = v[0].x & 0x7fff7fffu;
    const uint32_t w[7] = {v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
    for (int i = 0; i < 7; ++i) asm("max.u16x2 %0, %0, %1;" : "+r"(m) : "r"(w[i] & 0x7fff7fffu));
    const uint32_t h = max(m & 0xffffu, m >> 16);
    return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(h))));
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

// A warp takes kTasks pieces of 512 values (two k-tiles of a row) at a time: a lane holds sixteen values, two lanes a
// scale block.  (Pieces of 256, four lanes a block, cost twice the instructions for maxima, scales and addresses.)
template <typename T>
__global__ void __launch_bounds__(kThreads)
mx_quantize_kernel(const T* x, long long row_stride, const int* m_ptr, int max_m, int k, uint8_t* mx) {
  pdl_trigger();
  int rows = max_m;
  if (m_ptr != nullptr) rows = pdl_wait_row_count(m_ptr, max_m, 0);
  else pdl_wait();
  const int lane = threadIdx.x & 31;
  const uint32_t k_tiles = mx_k_tiles(k), pieces = (k_tiles + 1) / 2;
  const uint32_t tasks = static_cast<uint32_t>(rows) * pieces;  // (2^32 of them would not fit any memory)
  const uint32_t warps = gridDim.x * (kThreads / 32);
  for (uint32_t t0 = (blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * kTasks; t0 < tasks; t0 += warps * kTasks) {
    Sixteen<T> v[kTasks];
    uint32_t row = t0 / pieces, piece = t0 - row * pieces;
    uint32_t rows_of[kTasks], cols[kTasks];
    bool in[kTasks], tile_in[kTasks];
#pragma unroll
    for (int i = 0; i < kTasks; ++i) {
      cols[i] = piece * 512 + lane * 16;
      rows_of[i] = row;
      tile_in[i] = t0 + i < tasks && cols[i] < k_tiles * kMxTileK;  // (the row's last piece may be one k-tile)
      in[i] = tile_in[i] && cols[i] < static_cast<uint32_t>(k);
      if (in[i]) {
        v[i].load(x + static_cast<size_t>(row) * row_stride + cols[i]);
      } else {
#pragma unroll
        for (auto& w : v[i].v) w = Vec16{0u, 0u, 0u, 0u};
      }
      if (++piece == pieces) piece = 0, ++row;
    }
#pragma unroll
    for (int i = 0; i < kTasks; ++i) {
      uint32_t top = v[i].top();
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      const MxScale s = mx_scale(top);
      uint32_t scales = s.byte | (__shfl_down_sync(0xffffffffu, s.byte, 2) << 8);
      scales |= __shfl_down_sync(0xffffffffu, scales, 4) << 16;  // four blocks' bytes in every eighth lane
      if (!tile_in[i]) continue;
      float f[16];
      v[i].unpack(f);
      uint8_t* tile = mx + mx_tile_offset(rows_of[i], cols[i] >> 8, k_tiles);
      const int r = rows_of[i] & (kMxTileRows - 1), b = (cols[i] & 255) >> 5;
      *reinterpret_cast<uint2*>(tile + mx_code_offset(r, b) + (lane & 1) * 8) =
          make_uint2(mx_codes8(f, s), mx_codes8(f + 8, s));
      if ((lane & 7) == 0) *reinterpret_cast<uint32_t*>(tile + mx_scale_offset(r, b)) = scales;
    }
  }
}

constexpr int kBackTasks = 4;  // (row, k-tile) pairs a warp has in flight

// One warp per (row, k-tile): a lane holds eight values, so that a warp reads one 128-byte line of codes and writes 512
// or 1024 contiguous bytes.
template <typename T>
__global__ void __launch_bounds__(kThreads)
mx_dequantize_kernel(const uint8_t* mx, const int* m_ptr, int max_m, int k, T* out) {
  pdl_trigger();
  int rows = max_m;
  if (m_ptr != nullptr) rows = pdl_wait_row_count(m_ptr, max_m, 0);
  else pdl_wait();
  const int lane = threadIdx.x & 31;
  const uint32_t k_tiles = mx_k_tiles(k);
  const uint32_t tasks = static_cast<uint32_t>(rows) * k_tiles;
  const uint32_t warps = gridDim.x * (kThreads / 32);
  for (uint32_t t0 = (blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * kBackTasks; t0 < tasks;
       t0 += warps * kBackTasks) {
    uint32_t code[kBackTasks], scale[kBackTasks];
    uint32_t row = t0 / k_tiles, kt = t0 - row * k_tiles;
    T* dst[kBackTasks];
#pragma unroll
    for (int i = 0; i < kBackTasks; ++i) {
      const int col = kt * kMxTileK + lane * 8;
      dst[i] = nullptr;
      code[i] = scale[i] = 0u;
      if (t0 + i < tasks && col < k) {
        const uint8_t* tile = mx + mx_tile_offset(row, kt, k_tiles);
        const int r = row & (kMxTileRows - 1);
        code[i] = *reinterpret_cast<const uint32_t*>(tile + mx_code_offset(r, lane >> 2) + (lane & 3) * 4);
        scale[i] = tile[mx_scale_offset(r, lane >> 2)];
        dst[i] = out + static_cast<size_t>(row) * k + col;
      }
      if (++kt == k_tiles) kt = 0, ++row;
    }
#pragma unroll
    for (int i = 0; i < kBackTasks; ++i) {
      if (dst[i] == nullptr) continue;
      const float s = mx_scale_value(scale[i]);
      float f[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t h2;
        asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %1;\n\t"
            "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t}"
            : "=r"(h2)
            : "r"(code[i] >> (8 * j)));
        const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&h2));
        f[2 * j] = p.x * s;
        f[2 * j + 1] = p.y * s;
      }
#pragma unroll
      for (int e = 0; e < 8; e += VecTraits<T>::kElems) st_global_v4(dst[i] + e, VecTraits<T>::pack(f + e));
    }
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

// CTAs for `tasks` warp tasks, `each` to a warp at a time, at most 8 per SM.
inline int mx_grid(long long tasks, int each) {
  const long long per_cta = static_cast<long long>(kThreads / 32) * each;
  long long ctas = (tasks + per_cta - 1) / per_cta;
  const long long cap = static_cast<long long>(sm_count()) * 8;
  if (ctas > cap) ctas = cap;
  return ctas < 1 ? 1 : static_cast<int>(ctas);
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
  return launch_pdl(mx_quantize_kernel<T>,
                    dim3(mx_grid(static_cast<long long>(max_m) * ((mx_k_tiles(k) + 1) / 2), kTasks)), dim3(kThreads), 0, stream, x, row_stride, m_ptr,
                    max_m, k, static_cast<uint8_t*>(mx));
}

template <typename T>
cudaError_t launch_mx_dequantize(const void* mx, const int* m_ptr, int max_m, int k, T* out, cudaStream_t stream) {
  if (max_m <= 0) return cudaSuccess;
  if (k <= 0 || k % kMxBlock != 0) return cudaErrorInvalidValue;
  if ((reinterpret_cast<uintptr_t>(out) & 15u) || (reinterpret_cast<uintptr_t>(mx) & 127u))
    return cudaErrorMisalignedAddress;
  return launch_pdl(mx_dequantize_kernel<T>, dim3(mx_grid(static_cast<long long>(max_m) * mx_k_tiles(k), kBackTasks)), dim3(kThreads), 0, stream,
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
