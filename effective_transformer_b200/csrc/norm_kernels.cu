// The norm behind a block, its gate and residual scale, and the norm in front of the next block, in one pass:
//   p = post(x + bias)
//   h = residual_scale * residual + gate * p        (gate: per channel, or one row per sequence)
//   y = pre(h)
// post and pre are each a LayerNorm, (v - mean) * rsqrt(var + eps) * gamma + beta, an RMS norm,
// v * rsqrt(mean(v^2) + eps) * gamma, or nothing.  The plain post-norm encoder (add_bias_input_layernorm,
// cuda/cuda_kernels.cu:157-236) is post = nothing, gate = 1, residual_scale = 1, y only.
//
// Everything between the loads of x and residual and the stores of h and y stays in fp32 registers, so x and residual
// are read once and h and y written once: the kernel is bound by those bytes.  A row belongs to a group of WPR warps,
// a lane holds up to kMaxVec vectors of 16 bytes of it; means and variances are taken in two passes over the
// registers.  y can leave as MXFP4 too (mxfp4.cuh): four (fp16) or eight (fp32) neighbouring lanes hold a scale block.
#include "common.cuh"
#include "mxfp4.cuh"

namespace etb {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxVec = 4;

enum NormKind : int { kNormNone = 0, kNormLayer = 1, kNormRms = 2 };

// Sum over the WPR warps of a row group; every lane gets it.  `red`: WPR floats per group, double-buffered by `turn`.
template <int WPR>
__device__ __forceinline__ float group_sum(float v, float* red, int& turn, int group, int wig) {
  v = warp_sum(v);
  if (WPR == 1) return v;
  float* slot = red + turn * kWarps + group * WPR;
  turn ^= 1;
  if ((threadIdx.x & 31) == 0) slot[wig] = v;
  asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(WPR * 32) : "memory");
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < WPR; ++i) t += slot[i];
  return t;
}

// v := norm(v) over the row; elements past the row's end are zero before and are not read behind.
template <typename T, int V, int WPR>
__device__ __forceinline__ void normalise(float (&v)[V][VecTraits<T>::kElems], int kind, const T* gamma, const T* beta,
                                          int n, float eps, int vec0, int vecs, float* red, int& turn, int group,
                                          int wig) {
  constexpr int E = VecTraits<T>::kElems;
  const float inv_n = 1.0f / static_cast<float>(n);
  float mean = 0.f;
  if (kind == kNormLayer) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int e = 0; e < E; ++e) s += v[j][e];
    mean = group_sum<WPR>(s, red, turn, group, wig) * inv_n;
  }
  float sq = 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (vec0 + j * 32 * WPR < vecs) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        v[j][e] -= mean;
        sq = fmaf(v[j][e], v[j][e], sq);
      }
    }
  }
  const float rstd = rsqrtf(group_sum<WPR>(sq, red, turn, group, wig) * inv_n + eps);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = vec0 + j * 32 * WPR;
    if (c < vecs) {
      float g[E], b[E];
      VecTraits<T>::unpack(ld_global_v4(gamma + c * E), g);
      if (kind == kNormLayer) VecTraits<T>::unpack(ld_global_v4(beta + c * E), b);
#pragma unroll
      for (int e = 0; e < E; ++e)
        v[j][e] = kind == kNormLayer ? fmaf(v[j][e] * rstd, g[e], b[e]) : v[j][e] * rstd * g[e];
    }
  }
}

template <typename T, int V, int WPR>
__global__ void __launch_bounds__(kThreads)
gated_norm_kernel(const GatedNorm p) {
  constexpr int E = VecTraits<T>::kElems;
  constexpr int kGroups = kWarps / WPR;
  __shared__ float red[2 * kWarps];
  pdl_trigger();
  int rows = p.max_m;
  if (p.m_ptr != nullptr) rows = pdl_wait_row_count(p.m_ptr, p.max_m, 0);
  else pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = warp / WPR, wig = warp % WPR;
  const int n = p.n, vecs = n / E;
  const int vec0 = wig * 32 + lane;
  const T* x = static_cast<const T*>(p.x);
  const T* bias = static_cast<const T*>(p.bias);
  const T* residual = static_cast<const T*>(p.residual);
  const T* gate = static_cast<const T*>(p.gate);
  int turn = 0;
  for (long long row = static_cast<long long>(blockIdx.x) * kGroups + group; row < rows;
       row += static_cast<long long>(gridDim.x) * kGroups) {
    const size_t base = static_cast<size_t>(row) * n;
    float v[V][E];
    Vec16 vx[V], vr[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = vec0 + j * 32 * WPR;
      vx[j] = vr[j] = Vec16{0u, 0u, 0u, 0u};
      if (c < vecs) {
        vx[j] = ld_activation_v4(x + base + c * E);
        if (residual != nullptr) vr[j] = ld_activation_v4(residual + base + c * E);
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = vec0 + j * 32 * WPR;
      VecTraits<T>::unpack(vx[j], v[j]);
      if (bias != nullptr && c < vecs) {
        float b[E];
        VecTraits<T>::unpack(ld_global_v4(bias + c * E), b);
#pragma unroll
        for (int e = 0; e < E; ++e) v[j][e] += b[e];
      }
    }
    if (p.post_kind != kNormNone)
      normalise<T, V, WPR>(v, p.post_kind, static_cast<const T*>(p.post_gamma), static_cast<const T*>(p.post_beta), n,
                           p.eps, vec0, vecs, red, turn, group, wig);
    // a sequence number outside the gate's rows opens no gate: its row is zero
    const int gate_row = gate != nullptr && p.batch_idx != nullptr ? p.batch_idx[row] : 0;
    const bool gate_in = gate_row >= 0 && gate_row < p.gate_rows;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = vec0 + j * 32 * WPR;
      if (gate != nullptr) {
        float g[E];
        Vec16 vg = {0u, 0u, 0u, 0u};
        if (gate_in && c < vecs) vg = ld_activation_v4(gate + static_cast<size_t>(gate_row) * n + c * E);
        VecTraits<T>::unpack(vg, g);
#pragma unroll
        for (int e = 0; e < E; ++e) v[j][e] = gate_in ? v[j][e] * g[e] : 0.f;
      }
      if (residual != nullptr) {
        float r[E];
        VecTraits<T>::unpack(vr[j], r);
#pragma unroll
        for (int e = 0; e < E; ++e) v[j][e] = fmaf(r[e], p.residual_scale, v[j][e]);
      }
      if (p.h != nullptr && c < vecs) st_global_v4(static_cast<T*>(p.h) + base + c * E, VecTraits<T>::pack(v[j]));
    }
    if (p.pre_kind != kNormNone)
      normalise<T, V, WPR>(v, p.pre_kind, static_cast<const T*>(p.pre_gamma), static_cast<const T*>(p.pre_beta), n,
                           p.eps, vec0, vecs, red, turn, group, wig);
    if (p.y != nullptr) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = vec0 + j * 32 * WPR;
        if (c < vecs) st_global_v4(static_cast<T*>(p.y) + base + c * E, VecTraits<T>::pack(v[j]));
      }
    }
    if (p.y_mx != nullptr) {
      constexpr int kLanes = kMxBlock / E;     // lanes of a scale block
      constexpr int kBlocks = 32 / kLanes;     // blocks a warp holds per vector
      uint8_t* mx = static_cast<uint8_t*>(p.y_mx);
      const int k_tiles = mx_k_tiles(n), r = static_cast<int>(row) & (kMxTileRows - 1);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = vec0 + j * 32 * WPR, col = c * E;
        // (whole warps: the first column of a warp's vector decides)
        if ((c - lane) * E >= n) continue;
        float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        uint32_t top = 0u;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          f[e] = c < vecs ? v[j][e] : 0.f;
          top = max(top, abs_bits(f[e]));
        }
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const MxScale s = mx_scale(top);
        uint32_t scales = s.byte | (__shfl_down_sync(0xffffffffu, s.byte, kLanes) << 8);
        scales |= __shfl_down_sync(0xffffffffu, scales, 2 * kLanes) << 16;
        uint8_t* tile = mx + mx_tile_offset(static_cast<int>(row), col >> 8, k_tiles);
        const int b = (col & 255) >> 5;
        const uint32_t code = mx_codes8(f, s);
        uint8_t* dst = tile + mx_code_offset(r, b) + (lane & (kLanes - 1)) * (E / 2);
        if (E == 8) *reinterpret_cast<uint32_t*>(dst) = code;
        else *reinterpret_cast<uint16_t*>(dst) = static_cast<uint16_t>(code);
        if ((lane & (4 * kLanes - 1)) == 0) *reinterpret_cast<uint32_t*>(tile + mx_scale_offset(r, b)) = scales;
        (void)kBlocks;
      }
    }
  }
}

template <typename T, int V, int WPR>
cudaError_t launch_one(const GatedNorm& p, cudaStream_t stream) {
  auto kernel = gated_norm_kernel<T, V, WPR>;
  static std::atomic<int> resident[kMaxDevices] = {};
  const int dev = current_device();
  int per_sm = dev >= 0 ? resident[dev].load(std::memory_order_relaxed) : 0;
  if (per_sm == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kThreads, 0) != cudaSuccess || per_sm < 1)
      per_sm = 1;
    if (dev >= 0) resident[dev].store(per_sm, std::memory_order_relaxed);
  }
  constexpr int kGroups = kWarps / WPR;
  long long ctas = (static_cast<long long>(p.max_m) + kGroups - 1) / kGroups;
  const long long cap = static_cast<long long>(sm_count()) * per_sm;
  if (ctas > cap) ctas = cap;
  return launch_pdl(kernel, dim3(static_cast<int>(ctas)), dim3(kThreads), 0, stream, p);
}

template <typename T, int WPR>
cudaError_t launch_wpr(const GatedNorm& p, int v, cudaStream_t stream) {
  switch (v) {
    case 1: return launch_one<T, 1, WPR>(p, stream);
    case 2: return launch_one<T, 2, WPR>(p, stream);
    case 3: return launch_one<T, 3, WPR>(p, stream);
    case 4: return launch_one<T, 4, WPR>(p, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace

template <typename T>
cudaError_t launch_gated_norm(const GatedNorm& p, cudaStream_t stream) {
  constexpr int E = VecTraits<T>::kElems;
  if (p.max_m <= 0) return cudaSuccess;
  if (p.n <= 0 || p.n % E != 0 || (p.y_mx != nullptr && p.n % kMxBlock != 0)) return cudaErrorInvalidValue;
  if (p.post_kind < kNormNone || p.post_kind > kNormRms || p.pre_kind < kNormNone || p.pre_kind > kNormRms)
    return cudaErrorInvalidValue;
  if ((p.post_kind != kNormNone && p.post_gamma == nullptr) || (p.post_kind == kNormLayer && p.post_beta == nullptr) ||
      (p.pre_kind != kNormNone && p.pre_gamma == nullptr) || (p.pre_kind == kNormLayer && p.pre_beta == nullptr))
    return cudaErrorInvalidValue;
  if (p.x == nullptr || (p.h == nullptr && p.y == nullptr && p.y_mx == nullptr)) return cudaErrorInvalidValue;
  if (p.gate != nullptr && p.gate_rows < 1) return cudaErrorInvalidValue;
  for (const void* q : {p.x, p.bias, p.residual, p.gate, p.post_gamma, p.post_beta, p.pre_gamma, p.pre_beta,
                        static_cast<const void*>(p.h), static_cast<const void*>(p.y)})
    if (reinterpret_cast<uintptr_t>(q) & 15u) return cudaErrorMisalignedAddress;
  if (reinterpret_cast<uintptr_t>(p.y_mx) & 127u) return cudaErrorMisalignedAddress;
  const int vecs = p.n / E;
  for (int wpr = 1; wpr <= kWarps; wpr *= 2) {
    const int v = (vecs + 32 * wpr - 1) / (32 * wpr);
    if (v > kMaxVec) continue;
    switch (wpr) {
      case 1: return launch_wpr<T, 1>(p, v, stream);
      case 2: return launch_wpr<T, 2>(p, v, stream);
      case 4: return launch_wpr<T, 4>(p, v, stream);
      default: return launch_wpr<T, 8>(p, v, stream);
    }
  }
  return cudaErrorInvalidValue;  // wider than 8 warps of 4 vectors a lane
}

template cudaError_t launch_gated_norm<__half>(const GatedNorm&, cudaStream_t);
template cudaError_t launch_gated_norm<float>(const GatedNorm&, cudaStream_t);

}  // namespace etb
