// Rows to MXFP4 and back, and weights to MXFP4 (layout and rounding: mxfp4.cuh).
//
// All three only move data: a row of K values is read once (2 or 4 bytes a value) and written as 17 / 32 byte a value.
#include "common.cuh"
#include "mxfp4.cuh"

namespace etb {

namespace {

constexpr int kThreads = 256;
constexpr int kTasks = 4;  // (row, k-tile) pairs a warp has in flight

// Eight consecutive values of a row, 16 or 32 bytes.
template <typename T>
struct Oct;
template <>
struct Oct<__half> {
  Vec16 v;
  __device__ void load(const __half* p) { v = ld_activation_v4(p); }
  __device__ void zero() { v = Vec16{0u, 0u, 0u, 0u}; }
  __device__ void unpack(float* f) const { VecTraits<__half>::unpack(v, f); }
};
template <>
struct Oct<float> {
  Vec16 a, b;
  __device__ void load(const float* p) {
    a = ld_activation_v4(p);
    b = ld_activation_v4(p + 4);
  }
  __device__ void zero() { a = b = Vec16{0u, 0u, 0u, 0u}; }
  __device__ void unpack(float* f) const {
    VecTraits<float>::unpack(a, f);
    VecTraits<float>::unpack(b, f + 4);
  }
};

// One warp per (row, k-tile): a lane holds eight values, four lanes a scale block, so that a warp reads 512 (fp16) or
// 1024 contiguous bytes and writes one 128-byte line of codes.
template <typename T>
__global__ void __launch_bounds__(kThreads)
mx_quantize_kernel(const T* x, long long row_stride, const int* m_ptr, int max_m, int k, uint8_t* mx) {
  pdl_trigger();
  int rows = max_m;
  if (m_ptr != nullptr) rows = pdl_wait_row_count(m_ptr, max_m, 0);
  else pdl_wait();
  const int lane = threadIdx.x & 31;
  const int k_tiles = mx_k_tiles(k);
  const long long tasks = static_cast<long long>(rows) * k_tiles;
  const long long warps = static_cast<long long>(gridDim.x) * (kThreads / 32);
  const long long first = static_cast<long long>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  for (long long t0 = first * kTasks; t0 < tasks; t0 += warps * kTasks) {
    Oct<T> v[kTasks];
    int row[kTasks], kt[kTasks];
#pragma unroll
    for (int i = 0; i < kTasks; ++i) {
      const long long t = t0 + i;
      row[i] = t < tasks ? static_cast<int>(t / k_tiles) : -1;
      kt[i] = static_cast<int>(t - t / k_tiles * k_tiles);
      const int col = kt[i] * kMxTileK + lane * 8;
      if (row[i] >= 0 && col < k) v[i].load(x + static_cast<size_t>(row[i]) * row_stride + col);
      else v[i].zero();
    }
#pragma unroll
    for (int i = 0; i < kTasks; ++i) {
      float f[8];
      v[i].unpack(f);
      uint32_t top = 0u;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, abs_bits(f[e]));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const MxScale s = mx_scale(top);
      uint32_t scales = s.byte | (__shfl_down_sync(0xffffffffu, s.byte, 4) << 8);
      scales |= __shfl_down_sync(0xffffffffu, scales, 8) << 16;  // four blocks' bytes in lanes 0 and 16
      if (row[i] < 0) continue;
      uint8_t* tile = mx + mx_tile_offset(row[i], kt[i], k_tiles);
      const int r = row[i] & (kMxTileRows - 1);
      *reinterpret_cast<uint32_t*>(tile + mx_code_offset(r, lane >> 2) + (lane & 3) * 4) = mx_codes8(f, s);
      if ((lane & 15) == 0) *reinterpret_cast<uint32_t*>(tile + mx_scale_offset(r, lane >> 2)) = scales;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
mx_dequantize_kernel(const uint8_t* mx, const int* m_ptr, int max_m, int k, T* out) {
  pdl_trigger();
  int rows = max_m;
  if (m_ptr != nullptr) rows = pdl_wait_row_count(m_ptr, max_m, 0);
  else pdl_wait();
  const int lane = threadIdx.x & 31;
  const int k_tiles = mx_k_tiles(k);
  const long long tasks = static_cast<long long>(rows) * k_tiles;
  const long long warps = static_cast<long long>(gridDim.x) * (kThreads / 32);
  const long long first = static_cast<long long>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  for (long long t0 = first * kTasks; t0 < tasks; t0 += warps * kTasks) {
    uint32_t code[kTasks], scale[kTasks];
    int row[kTasks], col[kTasks];
#pragma unroll
    for (int i = 0; i < kTasks; ++i) {
      const long long t = t0 + i;
      row[i] = t < tasks ? static_cast<int>(t / k_tiles) : -1;
      const int kt = static_cast<int>(t - t / k_tiles * k_tiles);
      col[i] = kt * kMxTileK + lane * 8;
      if (col[i] >= k) row[i] = -1;
      code[i] = scale[i] = 0u;
      if (row[i] >= 0) {
        const uint8_t* tile = mx + mx_tile_offset(row[i], kt, k_tiles);
        const int r = row[i] & (kMxTileRows - 1);
        code[i] = *reinterpret_cast<const uint32_t*>(tile + mx_code_offset(r, lane >> 2) + (lane & 3) * 4);
        scale[i] = tile[mx_scale_offset(r, lane >> 2)];
      }
    }
#pragma unroll
    for (int i = 0; i < kTasks; ++i) {
      if (row[i] < 0) continue;
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
      T* dst = out + static_cast<size_t>(row[i]) * k + col[i];
#pragma unroll
      for (int e = 0; e < 8; e += VecTraits<T>::kElems)
        st_global_v4(dst + e, VecTraits<T>::pack(f + e));
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

inline int mx_grid(long long rows, int k) {
  const long long tasks = rows * mx_k_tiles(k), per_cta = static_cast<long long>(kThreads / 32) * kTasks;
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
  return launch_pdl(mx_quantize_kernel<T>, dim3(mx_grid(max_m, k)), dim3(kThreads), 0, stream, x, row_stride, m_ptr,
                    max_m, k, static_cast<uint8_t*>(mx));
}

template <typename T>
cudaError_t launch_mx_dequantize(const void* mx, const int* m_ptr, int max_m, int k, T* out, cudaStream_t stream) {
  if (max_m <= 0) return cudaSuccess;
  if (k <= 0 || k % kMxBlock != 0) return cudaErrorInvalidValue;
  if ((reinterpret_cast<uintptr_t>(out) & 15u) || (reinterpret_cast<uintptr_t>(mx) & 127u))
    return cudaErrorMisalignedAddress;
  return launch_pdl(mx_dequantize_kernel<T>, dim3(mx_grid(max_m, k)), dim3(kThreads), 0, stream,
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
