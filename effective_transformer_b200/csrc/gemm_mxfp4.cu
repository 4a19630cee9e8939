// Projections in 4-bit microscaled floating point:
//   C[M,N] = act(A W + bias) (+ residual),  A [M,K] and W^T [N,K] as MXFP4 (mxfp4.cuh), fp32 accumulate,
//   C as fp16, fp32 or MXFP4 again (the operand of the next projection).
//
// A product of two e2m1 values and two power-of-two scales is exact, so the only roundings are those of the fp32
// sum and the one at the end.
//
// Structure (one persistent CTA per SM, 320 threads), tiles of 128 x 128:
//   warp 0    producer: one untiled bulk copy per operand and k-tile of 256 values (codes and scales, 17 KB) into a
//             ring of kStages stages
//   warp 1    MMA issuer: the stage's scales go to tensor memory (tcgen05.cp), then four tcgen05.mma kind::mxf4 of
//             K = 64, accumulating in one of two TMEM buffers
//   warps 2-9 epilogue: one TMEM lane quadrant and one half of the columns each
// Scales have a TMEM region per stage, so a stage's are replaced only after the MMAs that read them have retired.
#include "common.cuh"
#include "mxfp4.cuh"
#include "ptx_sm100.cuh"

namespace etb {

namespace {

using namespace ptx;

constexpr int BM = 128;
constexpr int kEpilogueWarps = 8;
constexpr int kNumThreads = 64 + kEpilogueWarps * 32;
constexpr int kStagingPerWarp = 32 * 128;
constexpr int kUmmaK = 64;

enum Site : int {
  kSiteProducerEmpty = 1,
  kSiteProducerDrain = 2,
  kSiteMmaTmemEmpty = 3,
  kSiteMmaFull = 4,
  kSiteMmaDrain = 5,
  kSiteEpilogueFull = 6,
  kSiteSmemAlign = 7,
};

struct MxArgs {
  const uint8_t* a;
  const uint8_t* w;
  void* c;               // T* or, for MXFP4 output, the tiles
  const void* residual;  // T* or null
  const int* m_ptr;      // null: max_m rows
  int max_m, n, k;
  int* status_word;
};

__device__ __forceinline__ void st_shared_v4(uint32_t addr, const Vec16& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
}
__device__ __forceinline__ Vec16 ld_shared_v4(uint32_t addr) {
  Vec16 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// Rows as MXFP4 instead of T.
struct MxOut {};
template <typename T>
struct BiasOf {
  typedef T type;
};

template <int ACT>
__device__ __forceinline__ float activate(float x) {
  if (ACT == kEpiBiasGelu) return gelu_tanh(x);
  if (ACT == kEpiBiasTanh) return tanhf(x);
  return x;
}

// 64 columns of 32 rows, a row per thread in r: bias and activation in fp32.
template <typename T, int ACT>
__device__ __forceinline__ void bias_act(float* f, const T* bias_s) {
  if (bias_s != nullptr) {
#pragma unroll
    for (int i = 0; i < 64; i += VecTraits<T>::kElems) {
      float b[VecTraits<T>::kElems];
      VecTraits<T>::unpack(*reinterpret_cast<const Vec16*>(bias_s + i), b);
#pragma unroll
      for (int e = 0; e < VecTraits<T>::kElems; ++e) f[i + e] += b[e];
    }
  }
#pragma unroll
  for (int i = 0; i < 64; ++i) f[i] = activate<ACT>(f[i]);
}

// Stores them to C, rows [0, rows_valid) and columns [0, cols_valid) of the piece; ctile / rtile: its first element.
// The warp's staging bytes turn one row per thread into whole row segments per instruction.  With a residual the
// sum is formed in fp32 and rounded once.
template <typename T>
__device__ __forceinline__ void store_rows(const float* f, T* ctile, const T* rtile, int n, int rows_valid,
                                           int cols_valid, uint32_t buf, int lane) {
  const int piece = lane & 7;
  if (sizeof(T) == 2 && rtile == nullptr) {
#pragma unroll
    for (int p = 0; p < 8; ++p)
      st_shared_v4(buf + lane * 128 + ((p ^ (lane & 7)) << 4), VecTraits<__half>::pack(f + 8 * p));
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int rr = 4 * i + (lane >> 3);
      const Vec16 v = ld_shared_v4(buf + rr * 128 + ((piece ^ (rr & 7)) << 4));
      if (rr < rows_valid && piece * 8 < cols_valid) st_global_v4(ctile + static_cast<size_t>(rr) * n + piece * 8, v);
    }
    __syncwarp();
    return;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int p = 0; p < 8; ++p)
      st_shared_v4(buf + lane * 128 + ((p ^ (lane & 7)) << 4), VecTraits<float>::pack(f + h * 32 + 4 * p));
    __syncwarp();
    const int col = h * 32 + piece * 4;
    float res[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int rr = 4 * i + (lane >> 3);
      const bool in = rtile != nullptr && rr < rows_valid && col < cols_valid;
      if (sizeof(T) == 2) {
        uint2 u = make_uint2(0u, 0u);
        if (in) u = *reinterpret_cast<const uint2*>(rtile + static_cast<size_t>(rr) * n + col);
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
        res[i][0] = a.x, res[i][1] = a.y, res[i][2] = b.x, res[i][3] = b.y;
      } else {
        Vec16 v = {0u, 0u, 0u, 0u};
        if (in) v = ld_activation_v4(rtile + static_cast<size_t>(rr) * n + col);
        VecTraits<float>::unpack(v, res[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int rr = 4 * i + (lane >> 3);
      float v[4];
      VecTraits<float>::unpack(ld_shared_v4(buf + rr * 128 + ((piece ^ (rr & 7)) << 4)), v);
      if (rtile != nullptr) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += res[i][e];
      }
      if (rr < rows_valid && col < cols_valid) {
        T* dst = ctile + static_cast<size_t>(rr) * n + col;
        if (sizeof(T) == 2) {
          const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
          *reinterpret_cast<uint2*>(dst) =
              make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
        } else {
          st_global_v4(dst, VecTraits<float>::pack(v));
        }
      }
    }
    __syncwarp();
  }
}

// The same 64 columns as two scale blocks of a row of MXFP4; a thread has whole blocks in its registers.
__device__ __forceinline__ void store_mx(const float* f, uint8_t* mx, int row, int col, int n, bool row_valid) {
  if (!row_valid || col >= n) return;  // (n is a multiple of 64)
  uint8_t* tile = mx + mx_tile_offset(row, col >> 8, mx_k_tiles(n));
  const int r = row & (kMxTileRows - 1), b0 = (col & 255) >> 5;
  uint32_t scales = 0u;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < 32; ++i) top = max(top, abs_bits(f[h * 32 + i]));
    const MxScale s = mx_scale(top);
    Vec16 v;
    v.x = mx_codes8(f + h * 32, s);
    v.y = mx_codes8(f + h * 32 + 8, s);
    v.z = mx_codes8(f + h * 32 + 16, s);
    v.w = mx_codes8(f + h * 32 + 24, s);
    st_global_v4(tile + mx_code_offset(r, b0 + h), v);
    scales |= s.byte << (8 * h);
  }
  *reinterpret_cast<uint16_t*>(tile + mx_scale_offset(r, b0)) = static_cast<uint16_t>(scales);
}

template <int BN>
struct Cfg {
  static constexpr int kStages = 5;
  static constexpr int kStageBytes = 2 * kMxTileBytes;
  static constexpr int kStagingBytes = kEpilogueWarps * kStagingPerWarp;
  static constexpr int kColsPerWarp = BN / 2;
  static constexpr int kBiasBytes = kEpilogueWarps * kColsPerWarp * 4;
  static constexpr int kNumBars = 2 * kStages + 5;
  static constexpr int kSmemBytes = kStages * kStageBytes + kStagingBytes + kBiasBytes + 256;
  static constexpr int kScaleCols = 16;  // per stage: 2 pieces of A, 2 of B, 4 columns each
  static constexpr int kTmemCols = 512;
  static_assert(2 * BN + kStages * kScaleCols <= kTmemCols, "tensor memory");
  static_assert(kSmemBytes <= 232448 && kNumBars * 8 + 8 <= 256, "shared memory");
};

// T: element type of bias, residual and C; OUT: T, or MxOut.
template <typename T, typename OUT, int ACT>
__global__ void __launch_bounds__(kNumThreads, 1)
gemm_mxfp4_kernel(const MxArgs g, const T* __restrict__ bias) {
  constexpr int BN = 128;
  using cfg = Cfg<BN>;
  constexpr int S = cfg::kStages;
  constexpr bool kMxOut = sizeof(OUT) != sizeof(T);
  pdl_trigger();

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t tiles_addr = smem_u32(smem_raw);
  if ((tiles_addr & 1023u) != 0u) {  // the swizzled tiles need 1024-byte alignment
    pdl_wait();
    if (threadIdx.x == 0) report_timeout(g.status_word, kKernelGemmMx, kSiteSmemAlign);
    return;
  }
  const uint32_t staging_addr = tiles_addr + S * cfg::kStageBytes;
  T* bias_all = reinterpret_cast<T*>(smem_raw + S * cfg::kStageBytes + cfg::kStagingBytes);
  uint64_t* bars =
      reinterpret_cast<uint64_t*>(smem_raw + S * cfg::kStageBytes + cfg::kStagingBytes + cfg::kBiasBytes);
  const uint32_t bar0 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto free_bar = [&](int s) { return bar0 + 8u * (S + s); };
  auto tmem_full_bar = [&](int a) { return bar0 + 8u * (2 * S + a); };
  auto tmem_empty_bar = [&](int a) { return bar0 + 8u * (2 * S + 2 + a); };
  const uint32_t drain_bar = bar0 + 8u * (2 * S + 4);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + cfg::kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(free_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tmem_full_bar(a), 1);
      mbar_init(tmem_empty_bar(a), kEpilogueWarps);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), cfg::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  int M = g.max_m;
  if (g.m_ptr != nullptr) M = pdl_wait_row_count(g.m_ptr, g.max_m, 0);
  else pdl_wait();
  const int N = g.n;
  const int n_tiles = (N + BN - 1) / BN;
  const int num_tiles = (M + BM - 1) / BM * n_tiles;
  const int k_tiles = mx_k_tiles(g.k);

  auto fail = [&](int site) {
    *abort_flag = 1;
    report_timeout(g.status_word, kKernelGemmMx, site);
  };

  if (warp == 0) {
    if (lane == 0) {
      uint32_t stage = 0, phase = 0;
      long long issued = 0;
      bool ok = true;
      for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x) {
        const int m_tile = tile / n_tiles, n_tile = tile - m_tile * n_tiles;
        const uint8_t* a_src = g.a + static_cast<size_t>(m_tile) * k_tiles * kMxTileBytes;
        const uint8_t* w_src = g.w + static_cast<size_t>(n_tile) * k_tiles * kMxTileBytes;
        for (int kt = 0; kt < k_tiles; ++kt) {
          if (!mbar_wait(free_bar(stage), phase ^ 1u, abort_flag)) {
            fail(kSiteProducerEmpty);
            ok = false;
            break;
          }
          const uint32_t dst = tiles_addr + stage * cfg::kStageBytes;
          mbar_arrive_expect_tx(full_bar(stage), cfg::kStageBytes);
          bulk_load(dst, a_src + static_cast<size_t>(kt) * kMxTileBytes, kMxTileBytes, full_bar(stage));
          bulk_load(dst + kMxTileBytes, w_src + static_cast<size_t>(kt) * kMxTileBytes, kMxTileBytes, full_bar(stage));
          ++issued;
          if (++stage == S) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // the issuer's commits on the ring are asynchronous arrivals: the last of them land before the barriers go away
      const long long pending = issued < S ? issued : S;
      for (long long i = 0; i < pending; ++i) {
        const long long f = issued - 1 - i;
        if (!mbar_wait(free_bar(static_cast<int>(f % S)), static_cast<uint32_t>((f / S) & 1), abort_flag) &&
            *abort_flag == 0)
          fail(kSiteProducerDrain);
      }
      // copies in flight land before the CTA's shared memory goes away, also behind a wait that ran out
      for (long long i = 0; i < pending; ++i) {
        const long long f = issued - 1 - i;
        if (!mbar_drain(full_bar(static_cast<int>(f % S)), static_cast<uint32_t>((f / S) & 1)) && *abort_flag == 0)
          fail(kSiteProducerDrain);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      uint32_t stage = 0, phase = 0;
      int it = 0;
      bool ok = true;
      for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x, ++it) {
        const int acc = it & 1;
        if (!mbar_wait(tmem_empty_bar(acc), ((it >> 1) & 1) ^ 1u, abort_flag)) {
          fail(kSiteMmaTmemEmpty);
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * BN;
        for (int kt = 0; kt < k_tiles; ++kt) {
          if (!mbar_wait(full_bar(stage), phase, abort_flag)) {
            fail(kSiteMmaFull);
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a_addr = tiles_addr + stage * cfg::kStageBytes, b_addr = a_addr + kMxTileBytes;
          const uint32_t sf = tmem_base + 2 * BN + stage * cfg::kScaleCols;
          const int left = g.k - kt * kMxTileK;
          const int steps = left >= kMxTileK ? 4 : (left + kUmmaK - 1) / kUmmaK;
          for (int p = 0; 2 * p < steps; ++p) {
            tmem_cp_scales(sf + 4 * p, make_scale_desc(a_addr + kMxCodeBytes + 512 * p));
            tmem_cp_scales(sf + 8 + 4 * p, make_scale_desc(b_addr + kMxCodeBytes + 512 * p));
          }
          const uint64_t adesc = make_kmajor_sw128_desc(a_addr), bdesc = make_kmajor_sw128_desc(b_addr);
          for (int j = 0; j < steps; ++j)
            umma_mxf4_ss(d_tmem, adesc + 2u * j, bdesc + 2u * j,
                         (j & 1) ? make_idesc_mxf4(BM, BN, 2) : make_idesc_mxf4(BM, BN, 0), sf + 4 * (j >> 1),
                         sf + 8 + 4 * (j >> 1), (kt | j) != 0 ? 1u : 0u);
          umma_commit(free_bar(stage));
          if (++stage == S) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (ok) umma_commit(tmem_full_bar(acc));
      }
      // all MMAs must have retired before TMEM is freed
      umma_commit(drain_bar);
      if (!mbar_drain(drain_bar, 0u) && *abort_flag == 0) fail(kSiteMmaDrain);
    }
  } else {
    const int quad = warp & 3, ew = warp - 2, half = ew >> 2;
    constexpr int kCols = cfg::kColsPerWarp;
    const uint32_t buf = staging_addr + ew * kStagingPerWarp;
    T* bias_s = bias_all + ew * kCols;
    int it = 0;
    for (int tile = blockIdx.x; tile < num_tiles; tile += gridDim.x, ++it) {
      const int m_tile = tile / n_tiles, n_tile = tile - m_tile * n_tiles;
      const int acc = it & 1;
      const int col0 = n_tile * BN + half * kCols;
      if (bias != nullptr) {
        for (int i = lane; i < kCols; i += 32) bias_s[i] = col0 + i < N ? bias[col0 + i] : T(0.f);
        __syncwarp();
      }
      const bool got = mbar_wait(tmem_full_bar(acc), (it >> 1) & 1, abort_flag);
      if (!__all_sync(0xffffffffu, got)) {
        if (lane == 0) fail(kSiteEpilogueFull);
        break;
      }
      tc_fence_after();
      const int row0 = m_tile * BM + quad * 32;
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + acc * BN + half * kCols;
      uint32_t r[64];
      tmem_ld_32x32b_x32(t_row, r);
      tmem_ld_32x32b_x32(t_row + 32, r + 32);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(tmem_empty_bar(acc));
      float f[64];
#pragma unroll
      for (int i = 0; i < 64; ++i) f[i] = __uint_as_float(r[i]);
      bias_act<T, ACT>(f, bias != nullptr ? bias_s : nullptr);
      if (kMxOut) {
        store_mx(f, static_cast<uint8_t*>(g.c), row0 + lane, col0, N, row0 + lane < M);
      } else {
        const size_t off = static_cast<size_t>(row0) * N + col0;
        const T* res = static_cast<const T*>(g.residual);
        store_rows<T>(f, static_cast<T*>(g.c) + off, res != nullptr ? res + off : nullptr, N, M - row0, N - col0, buf,
                      lane);
      }
      __syncwarp();  // bias_s is rewritten for the next tile
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, cfg::kTmemCols);
  }
}

template <typename T, typename OUT, int ACT>
cudaError_t launch_act(const MxArgs& g, const T* bias, cudaStream_t stream) {
  using cfg = Cfg<128>;
  static PerDeviceOnce once;
  const cudaError_t err = once.run([] {
    return cudaFuncSetAttribute(gemm_mxfp4_kernel<T, OUT, ACT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                cfg::kSmemBytes);
  });
  if (err != cudaSuccess) return err;
  const long long tiles = static_cast<long long>((g.max_m + BM - 1) / BM) * ((g.n + 127) / 128);
  if (tiles > 0x7fffffffll) return cudaErrorInvalidValue;
  const int grid = static_cast<int>(tiles < sm_count() ? tiles : sm_count());
  return launch_pdl(gemm_mxfp4_kernel<T, OUT, ACT>, dim3(grid), dim3(kNumThreads), cfg::kSmemBytes, stream, g, bias);
}

template <typename T, typename OUT>
cudaError_t launch_out(const MxArgs& g, const T* bias, int epilogue, cudaStream_t stream) {
  switch (epilogue) {
    case kEpiNone:
      return launch_act<T, OUT, kEpiBias>(g, nullptr, stream);
    case kEpiBias:
      return launch_act<T, OUT, kEpiBias>(g, bias, stream);
    case kEpiBiasGelu:
      return launch_act<T, OUT, kEpiBiasGelu>(g, bias, stream);
    case kEpiBiasTanh:
      return launch_act<T, OUT, kEpiBiasTanh>(g, bias, stream);
    default:
      return cudaErrorInvalidValue;
  }
}

}  // namespace

template <typename T>
cudaError_t launch_gemm_mxfp4(const MxGemm& p, const T* bias, const T* residual, T* c, int epilogue,
                              cudaStream_t stream) {
  if (p.max_m <= 0) return cudaSuccess;
  if (p.n <= 0 || p.k <= 0 || p.n % 32 != 0 || p.k % kMxBlock != 0) return cudaErrorInvalidValue;
  if ((c == nullptr) == (p.c_mx == nullptr)) return cudaErrorInvalidValue;
  if (p.c_mx != nullptr && (p.n % 64 != 0 || residual != nullptr)) return cudaErrorInvalidValue;
  if (epilogue != kEpiNone && bias == nullptr) return cudaErrorInvalidValue;
  for (const void* q : {p.a, p.w, static_cast<const void*>(c), static_cast<const void*>(p.c_mx),
                        static_cast<const void*>(bias), static_cast<const void*>(residual)})
    if (reinterpret_cast<uintptr_t>(q) & 15u) return cudaErrorMisalignedAddress;
  MxArgs g;
  g.a = static_cast<const uint8_t*>(p.a);
  g.w = static_cast<const uint8_t*>(p.w);
  g.c = c != nullptr ? static_cast<void*>(c) : p.c_mx;
  g.residual = residual;
  g.m_ptr = p.m_ptr;
  g.max_m = p.max_m, g.n = p.n, g.k = p.k;
  g.status_word = p.status_word;
  if (p.c_mx != nullptr) return launch_out<T, MxOut>(g, bias, epilogue, stream);
  return launch_out<T, T>(g, bias, epilogue, stream);
}

template cudaError_t launch_gemm_mxfp4<__half>(const MxGemm&, const __half*, const __half*, __half*, int,
                                               cudaStream_t);
template cudaError_t launch_gemm_mxfp4<float>(const MxGemm&, const float*, const float*, float*, int, cudaStream_t);

}  // namespace etb
