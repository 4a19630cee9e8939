// Projections in 4-bit microscaled floating point:
//   C[M,N] = act(A W + bias) (+ residual),  A [M,K] and W^T [N,K] as MXFP4 (mxfp4.cuh), fp32 accumulate,
//   C as fp16, fp32 or MXFP4 again (the operand of the next projection).
//
// A product of two e2m1 values and two power-of-two scales is exact, so the only roundings are those of the fp32
// sum and the one at the end.
//
// Three kernels.  Two are persistent, one CTA per SM:
//   warp 0    producer: operand tiles of 256 values of K, codes and scales, into a ring of kStages stages
//   warp 1    MMA issuer: the stage's scales go to tensor memory (tcgen05.cp), then tcgen05.mma kind::mxf4 of K = 64,
//             accumulating in one of two TMEM buffers
//   the rest  epilogue
// gemm_mxfp4_kernel works on tiles of 128 x 128, gemm_mxfp4_pair_kernel on tiles of 256 x 192 by CTA pairs.  The third,
// gemm_mxfp4_rows_kernel, takes few rows in fp16 or fp32 and quantises them itself.
// Scales have a TMEM region per stage, so a stage's are replaced only after the MMAs that read them have retired.
//
// Tensor memory is taken behind the wait for the kernels in front and before dependents are released.  A CTA of a dependent
// that held it while it waits could leave none for a CTA of the kernel that it waits for: a pair kernel's CTA (159 KB of
// shared memory, all 512 columns) fits an SM beside one of the attention, which releases its dependents before it allocates.
#include "common.cuh"
#include "mxfp4.cuh"
#include "packed_f32.cuh"
#include "ptx_sm100.cuh"

namespace etb {

namespace {

using namespace ptx;

constexpr int BM = 128;
// Epilogue warps of the 128 x 128 tiles: two sets of eight that take the tiles in turn, a set per accumulator buffer,
// so that one loads and computes while the other stores; in a set, a TMEM lane quadrant and one half of the columns each.
constexpr int kEpilogueSet = 8;
constexpr int kNumThreads = 64 + 2 * kEpilogueSet * 32;
constexpr int kUmmaK = 64;

enum Site : int {
  kSiteProducerEmpty = 1,
  kSiteProducerDrain = 2,
  kSiteMmaTmemEmpty = 3,
  kSiteMmaFull = 4,
  kSiteMmaDrain = 5,
  kSiteEpilogueFull = 6,
  kSiteSmemAlign = 7,
  kSiteMmaPeerTmem = 8,
};

struct MxArgs {
  const uint8_t* a;
  const uint8_t* w;
  void* c;               // T* or, for MXFP4 output, the tiles
  const void* residual;  // T* or null
  const int* m_ptr;      // null: max_m rows
  int max_m, n, k;
  int route_rows;  // rows by which the kernel is chosen
  bool sectors;    // c begins on a 32-byte boundary (its rows do then: n is a multiple of 32)
  int* status_word;
};

// Rows as MXFP4 instead of T.
struct MxOut {};

// tanh-form GELU of a pair, 0.5 x (1 + tanh u) as x / (1 + 2^z) with z = -2 u log2(e): nothing cancels for negative x, where
// 1 + tanh u does (with the hardware's tanh, right to 2^-11, the result at x = -3 would be off by a fifth of itself).  z is
// rounded four times, so the relative error is 4 |z| 2^-24 ln 2 at the most, 7e-6 at x = -6; 2^z overflows from x = -10 on
// and leaves -0, the limit.  Two special-function operations an element instead of tanh's one: 39778 x 1024 by 4096 103 ->
// 116 us in fp16, 98 -> 117 us in 4 bits (without activation 93 us).  One reciprocal for both elements, of the product of
// their denominators, takes clamps that keep a NaN from its neighbour and comes to 114 and 119 us; a polynomial and a Newton
// step in place of the reciprocal 122 and 133 us.
__device__ __forceinline__ Pair gelu_pair(const Pair& x) {
  const Pair c1 = pack2(-2.302208198144325f, -2.302208198144325f);
  const Pair c2 = pack2(-2.302208198144325f * 0.044715f, -2.302208198144325f * 0.044715f);
  Pair d = mul2(x, fma2(mul2(x, x), c2, c1));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(d.x));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(d.y));
  d = add2(d, pack2(1.f, 1.f));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(d.x));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(d.y));
  return mul2(x, d);
}

template <int ACT>
__device__ __forceinline__ Pair activate(const Pair& x) {
  if (ACT == kEpiBiasGelu) return gelu_pair(x);
  if (ACT == kEpiBiasTanh) return pack2(tanhf(x.x), tanhf(x.y));
  return x;
}

// Eight neighbouring values of a row of T.
template <typename T>
struct Oct {
  Vec16 v[sizeof(T) / 2];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) v[i] = Vec16{0u, 0u, 0u, 0u};
  }
  // (coherent loads for the bias too: a caller may have written it just before)
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) v[i] = ld_activation_v4(p + i * VecTraits<T>::kElems);
  }
  __device__ __forceinline__ void unpack(Pair* p) const {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
      float x[VecTraits<T>::kElems];
      VecTraits<T>::unpack(v[i], x);
#pragma unroll
      for (int e = 0; e < VecTraits<T>::kElems; e += 2)
        p[(i * VecTraits<T>::kElems + e) / 2] = pack2(x[e], x[e + 1]);
    }
  }
};
__device__ __forceinline__ void store_oct(__half* p, const Pair* f, bool) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __float22half2_rn(f[i]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  st_global_v4(p, Vec16{w[0], w[1], w[2], w[3]});
}
// (one whole sector where the result begins on one)
__device__ __forceinline__ void store_oct(float* p, const Pair* f, bool sectors) {
  if (sectors) {
    asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(f[0].x), "f"(f[0].y), "f"(f[1].x),
                 "f"(f[1].y), "f"(f[2].x), "f"(f[2].y), "f"(f[3].x), "f"(f[3].y)
                 : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float v[4] = {f[2 * i].x, f[2 * i].y, f[2 * i + 1].x, f[2 * i + 1].y};
      st_global_v4(p + 4 * i, VecTraits<float>::pack(v));
    }
  }
}

// Epilogues of the kernels: kEpiNone to kEpiBiasTanh, and this with a residual.  (Compile-time: as run-time branches
// they cost the plain epilogue an addition and two moves a value.)
constexpr int kWithResidual = 16;

// A column group of 32 columns of a warp's 32 rows: what is fetched for it ahead, how it comes from tensor memory, and
// what becomes of it.
//
// fp16 and fp32 results: a thread has, for each of 4 row groups of 8, eight neighbouring columns of one row (see
// mxfp4.cuh): bias and residual come in, and the result goes out, as 16 or 32 bytes a thread and 64 or 128 contiguous
// bytes a row.
template <typename T, typename OUT, int EPI>
struct Group {
  static constexpr int ACT = EPI & ~kWithResidual;
  static constexpr bool kBias = ACT != kEpiNone, kRes = (EPI & kWithResidual) != 0;
  Oct<T> bias, res[4];

  // Row of row group 0 (rows are lanes in the order of mx_row); the next groups' are 2, 4 and 6 further on.
  static __device__ __forceinline__ int first_row(int lane) { return mx_row(lane >> 2); }
  static_assert(mx_row(8 + 5) == mx_row(5) + 2 && mx_row(16 + 5) == mx_row(5) + 4 && mx_row(24 + 2) == mx_row(2) + 6, "");

  __device__ __forceinline__ void fetch(const MxArgs& g, const T* bias_ptr, int row0, int col0, int M, int lane) {
    const int col = col0 + (lane & 3) * 8, row = row0 + first_row(lane);
    if (kBias) {
      bias.zero();
      if (col < g.n) bias.load(bias_ptr + col);
    }
    if (kRes) {
      const T* src = static_cast<const T*>(g.residual) + static_cast<size_t>(row) * g.n + col;
      const size_t step = 2 * static_cast<size_t>(g.n);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        res[i].zero();
        if (row + 2 * i < M && col < g.n) res[i].load(src + i * step);
      }
    }
  }
  static __device__ __forceinline__ void load(uint32_t t_row, float* r) {
    tmem_ld_16x256b_x4(t_row, r);
    tmem_ld_16x256b_x4(t_row + (16u << 16), r + 16);
  }
  __device__ __forceinline__ void finish(const MxArgs& g, const T* bias_ptr, const float* r, int row0, int col0, int M,
                                         int lane) {
    if (col0 >= g.n) return;  // (n is a multiple of 32)
    const int row = row0 + first_row(lane);
    T* dst = static_cast<T*>(g.c) + static_cast<size_t>(row) * g.n + col0 + (lane & 3) * 8;
    const size_t step = 2 * static_cast<size_t>(g.n);
    Pair b[4];
    if (kBias) bias.unpack(b);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      Pair f[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = 16 * (i >> 1) + 4 * j + 2 * (i & 1);
        f[j] = pack2(r[at], r[at + 1]);
      }
      if (kBias) {
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = add2(f[j], b[j]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = activate<ACT>(f[j]);
      if (kRes) {
        Pair x[4];
        res[i].unpack(x);
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = add2(f[j], x[j]);
      }
      if (row + 2 * i < M) store_oct(dst, f, g.sectors);
      dst += step;
    }
  }
};

// MXFP4 results: a thread has the 32 columns of one row, a scale block, and needs no other's.
template <typename T, int ACT>
struct Group<T, MxOut, ACT> {
  static constexpr bool kBias = ACT != kEpiNone;
  Oct<T> bias[4];

  __device__ __forceinline__ void fetch(const MxArgs& g, const T* bias_ptr, int, int col0, int, int) {
    if (kBias) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        bias[i].zero();
        if (col0 < g.n) bias[i].load(bias_ptr + col0 + 8 * i);
      }
    }
  }
  static __device__ __forceinline__ void load(uint32_t t_row, float* r) { tmem_ld_32x32b_x32(t_row, r); }
  __device__ __forceinline__ void finish(const MxArgs& g, const T* bias_ptr, const float* r, int row0, int col0, int M,
                                         int lane) {
    const int row = row0 + mx_row(lane);
    if (row >= M || col0 >= g.n) return;
    Pair f[16];
    float top = 0.f;
    // neighbouring columns 2 m, 2 m + 1 are neighbours in tensor memory too, as a pair
#pragma unroll
    for (int m = 0; m < 16; ++m)
      f[m] = pack2(r[mx_row(2 * m)], r[mx_row(2 * m) + 1]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (kBias) {
        Pair b[4];
        bias[i].unpack(b);
#pragma unroll
        for (int j = 0; j < 4; ++j) f[4 * i + j] = add2(f[4 * i + j], b[j]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        Pair& v = f[4 * i + j];
        v = activate<ACT>(v);
        asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(top) : "f"(fabsf(v.x)), "f"(fabsf(v.y)));
      }
    }
    const MxScale s = mx_scale(abs_bits(top));
    uint8_t* tile = static_cast<uint8_t*>(g.c) + mx_tile_offset(row, col0 >> 8, mx_k_tiles(g.n));
    const int rt = row & (kMxTileRows - 1), b = (col0 & 255) >> 5;
    Vec16 v;
    v.x = mx_codes8(f, s);
    v.y = mx_codes8(f + 4, s);
    v.z = mx_codes8(f + 8, s);
    v.w = mx_codes8(f + 12, s);
    st_global_v4(tile + mx_code_offset(rt, b), v);
    tile[mx_scale_offset(rt, b)] = static_cast<uint8_t>(s.byte);
  }
};

// The epilogue of one warp: kGroups column groups of its 32 rows from (row0, col0) of a finished accumulator buffer
// (TMEM lanes at the lane field of t_row).  wait() returns whether the accumulator has come; release() hands the buffer
// back, when the last group is in registers.
// kAhead: what all groups need from global memory is fetched before the wait, and not a group's while its columns come
// from tensor memory.  kWhole: all groups are taken into registers first, so that the buffer goes back at once.
template <typename T, typename OUT, int EPI, int kGroups, bool kAhead, bool kWhole, typename Wait, typename Release>
__device__ __forceinline__ bool epilogue_warp(const MxArgs& g, const T* bias_ptr, uint32_t t_row, int row0,
                                              int col0, int M, int lane, Wait wait, Release release) {
  static_assert(kAhead || !kWhole, "");
  Group<T, OUT, EPI> group[kAhead ? kGroups : 1];
#pragma unroll
  for (int c = 0; c < (kAhead ? kGroups : 1); ++c) group[c].fetch(g, bias_ptr, row0, col0 + 32 * c, M, lane);
  if (!wait()) return false;
  tc_fence_after();
  float r[kWhole ? kGroups : 1][32];
#pragma unroll
  for (int c = 0; kWhole && c < kGroups; ++c) group[0].load(t_row + 32 * c, r[kWhole ? c : 0]);
#pragma unroll (kAhead ? kGroups : 1)
  for (int c = 0; c < kGroups; ++c) {
    if (!kWhole) group[0].load(t_row + 32 * c, r[0]);
    if (!kAhead && c > 0) group[0].fetch(g, bias_ptr, row0, col0 + 32 * c, M, lane);
    if (!kWhole || c == 0) tmem_ld_wait();
    if (c == (kWhole ? 0 : kGroups - 1)) {
      tc_fence_before();
      __syncwarp();
      release();
    }
    group[kAhead ? c : 0].finish(g, bias_ptr, r[kWhole ? c : 0], row0, col0 + 32 * c, M, lane);
  }
  return true;
}

// What one thread issues for a stage: the scales' copies and the MMAs of kSteps x 64 values of K.  The instruction
// stream of that thread is what the tensor core waits for when it is longer than an MMA (64 cycles at N = 128), so it is
// unrolled, with descriptors that differ by constants.
// kBlocks: W row blocks, each with its own 1 KB of scales, side by side; b_shift: columns to the scales of the tile's
// first W row; idesc0: the descriptor that reads the first two scales of a word.
template <bool kPair, int kBlocks>
__device__ __forceinline__ void issue_stage(int steps, uint32_t d_tmem, uint32_t a_addr, uint32_t b_addr,
                                            uint32_t bs_addr, uint32_t sfa, uint32_t sfb, uint32_t b_shift,
                                            uint32_t idesc0, bool first) {
  const uint64_t adesc = make_kmajor_sw128_desc(a_addr), bdesc = make_kmajor_sw128_desc(b_addr);
  const uint64_t as_desc = make_scale_desc(a_addr + kMxCodeBytes), bs_desc = make_scale_desc(bs_addr);
  auto cp = [&](uint32_t dst, uint64_t desc) {
    if (kPair) tmem_cp_scales_pair(dst, desc);
    else tmem_cp_scales(dst, desc);
  };
  auto copy = [&](int p) {
    cp(sfa + 4 * p, as_desc + 32u * p);
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) cp(sfb + 4 * (kBlocks * p + i), bs_desc + 32u * p + 64u * i);
  };
  auto mma = [&](int j) {
    const uint32_t idesc = idesc0 | ((j & 1) ? make_idesc_mxf4(0, 0, 2) : 0u), acc = first && j == 0 ? 0u : 1u;
    const uint32_t sa = sfa + 4 * (j >> 1), sb = sfb + 4 * kBlocks * (j >> 1) + b_shift;
    if (kPair) umma_mxf4_ss_pair(d_tmem, adesc + 2u * j, bdesc + 2u * j, idesc, sa, sb, acc);
    else umma_mxf4_ss(d_tmem, adesc + 2u * j, bdesc + 2u * j, idesc, sa, sb, acc);
  };
  if (steps == 4) {
    copy(0);
    copy(1);
#pragma unroll
    for (int j = 0; j < 4; ++j) mma(j);
  } else {  // the rest of a width that is no multiple of 256
    copy(0);
    if (steps > 2) copy(1);
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (j < steps) mma(j);
  }
}

// The kernels' tensor memory, behind their wait (see the top of the file).  Warp 1 allocates and then releases the
// dependents, since a CTA of theirs must not take what this one is about to; it waits for nobody, and the epilogue's warps
// (the other `threads`) ask for the address when they need it.
template <typename Alloc>
__device__ __forceinline__ uint32_t take_tmem(const uint32_t* slot, int threads, Alloc alloc) {
  alloc();
  __syncwarp();
  tc_fence_before();
  asm volatile("bar.arrive 1, %0;" ::"r"(threads + 32) : "memory");
  tc_fence_after();
  pdl_trigger();
  return __shfl_sync(0xffffffffu, *static_cast<const volatile uint32_t*>(slot), 0);
}
__device__ __forceinline__ uint32_t tmem_address(const uint32_t* slot, int threads) {
  asm volatile("bar.sync 1, %0;" ::"r"(threads + 32) : "memory");
  tc_fence_after();
  return __shfl_sync(0xffffffffu, *static_cast<const volatile uint32_t*>(slot), 0);
}

template <int BN>
struct Cfg {
  static constexpr int kStages = 6;
  static constexpr int kStageBytes = 2 * kMxTileBytes;
  static constexpr int kNumBars = 2 * kStages + 5;
  static constexpr int kSmemBytes = kStages * kStageBytes + 256;
  static constexpr int kScaleCols = 16;  // per stage: 2 pieces of A, 2 of B, 4 columns each
  static constexpr int kTmemCols = 512;
  static_assert(2 * BN + kStages * kScaleCols <= kTmemCols, "tensor memory");
  static_assert(kSmemBytes <= 232448 && kNumBars * 8 + 8 <= 256, "shared memory");
};

// T: element type of bias, residual and C; OUT: T, or MxOut.
template <typename T, typename OUT, int ACT>
__global__ void __launch_bounds__(kNumThreads, 1)
gemm_mxfp4_kernel(const MxArgs g, const T* bias) {
  constexpr int BN = 128;
  using cfg = Cfg<BN>;
  constexpr int S = cfg::kStages;

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t tiles_addr = smem_u32(smem_raw);
  if ((tiles_addr & 1023u) != 0u) {  // the swizzled tiles need 1024-byte alignment
    pdl_wait();
    if (threadIdx.x == 0) report_timeout(g.status_word, kKernelGemmMx, kSiteSmemAlign);
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem_raw + S * cfg::kStageBytes);
  const uint32_t bar0 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto free_bar = [&](int s) { return bar0 + 8u * (S + s); };
  auto tmem_full_bar = [&](int a) { return bar0 + 8u * (2 * S + a); };
  auto tmem_empty_bar = [&](int a) { return bar0 + 8u * (2 * S + 2 + a); };
  const uint32_t drain_bar = bar0 + 8u * (2 * S + 4);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + cfg::kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(free_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tmem_full_bar(a), 1);
      mbar_init(tmem_empty_bar(a), kEpilogueSet);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  __syncthreads();
  int M = g.max_m;
  if (g.m_ptr != nullptr) M = pdl_wait_row_count(g.m_ptr, g.max_m, 0);
  else pdl_wait();
  uint32_t tmem_base = 0;  // (the producer needs none)
  if (warp == 1)
    tmem_base = take_tmem(tmem_slot, kNumThreads - 64, [&] {
      tmem_alloc(smem_u32(tmem_slot), cfg::kTmemCols);
      tmem_relinquish();
    });

  const int N = g.n;
  const int n_tiles = (N + BN - 1) / BN;
  const int num_tiles = (M + BM - 1) / BM * n_tiles;
  const int k_tiles = mx_k_tiles(g.k);

  auto fail = [&](int site) {
    *abort_flag = 1;
    report_timeout(g.status_word, kKernelGemmMx, site);
  };

  if (warp == 0) {
    // all lanes walk through the loop, one issues (see elect_one)
    const bool issuer = elect_one();
    uint32_t stage = 0, phase = 0;
    long long issued = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x) {
      const int m_tile = tile / n_tiles, n_tile = tile - m_tile * n_tiles;
      const uint8_t* a_src = g.a + static_cast<size_t>(m_tile) * k_tiles * kMxTileBytes;
      const uint8_t* w_src = g.w + static_cast<size_t>(n_tile) * k_tiles * kMxTileBytes;
      for (int kt = 0; kt < k_tiles; ++kt) {
        if (!__all_sync(0xffffffffu, mbar_wait(free_bar(stage), phase ^ 1u, abort_flag))) {
          if (lane == 0) fail(kSiteProducerEmpty);
          ok = false;
          break;
        }
        const uint32_t dst = tiles_addr + stage * cfg::kStageBytes, bar = full_bar(stage);
        if (issuer) {
          mbar_arrive_expect_tx(bar, cfg::kStageBytes);
          bulk_load(dst, a_src, kMxTileBytes, bar);
          bulk_load(dst + kMxTileBytes, w_src, kMxTileBytes, bar);
        }
        __syncwarp();
        a_src += kMxTileBytes;
        w_src += kMxTileBytes;
        ++issued;
        if (++stage == S) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    if (issuer) {
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
    // all lanes walk through the loop, one issues (see elect_one)
    const bool issuer = elect_one();
    uint32_t stage = 0, phase = 0;
    int it = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x, ++it) {
      const int acc = it & 1;
      if (!__all_sync(0xffffffffu, mbar_wait(tmem_empty_bar(acc), ((it >> 1) & 1) ^ 1u, abort_flag))) {
        if (lane == 0) fail(kSiteMmaTmemEmpty);
        break;
      }
      tc_fence_after();
      const uint32_t d_tmem = tmem_base + acc * BN;
      for (int kt = 0; kt < k_tiles; ++kt) {
        if (!__all_sync(0xffffffffu, mbar_wait(full_bar(stage), phase, abort_flag))) {
          if (lane == 0) fail(kSiteMmaFull);
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t a_addr = tiles_addr + stage * cfg::kStageBytes, b_addr = a_addr + kMxTileBytes;
        const uint32_t sf = tmem_base + 2 * BN + stage * cfg::kScaleCols;
        const int left = g.k - kt * kMxTileK;
        const int steps = left >= kMxTileK ? 4 : (left + kUmmaK - 1) / kUmmaK;
        if (issuer) {
          issue_stage<false, 1>(steps, d_tmem, a_addr, b_addr, b_addr + kMxCodeBytes, sf, sf + 8, 0, make_idesc_mxf4(BM, BN, 0),
                                kt == 0);
          umma_commit(free_bar(stage));
          if (kt == k_tiles - 1) umma_commit(tmem_full_bar(acc));
        }
        __syncwarp();
        if (++stage == S) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    // all MMAs must have retired before TMEM is freed
    if (issuer) {
      umma_commit(drain_bar);
      if (!mbar_drain(drain_bar, 0u) && *abort_flag == 0) fail(kSiteMmaDrain);
    }
    __syncwarp();
  } else {
    tmem_base = tmem_address(tmem_slot, kNumThreads - 64);
    const int quad = warp & 3, half = ((warp - 2) >> 2) & 1, acc = (warp - 2) / kEpilogueSet;
    const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + acc * BN + half * (BN / 2);
    uint32_t phase = 0;
    for (int tile = blockIdx.x + acc * gridDim.x; tile < num_tiles; tile += 2 * gridDim.x, phase ^= 1u) {
      const int m_tile = tile / n_tiles, n_tile = tile - m_tile * n_tiles;
      const bool got = epilogue_warp<T, OUT, ACT, BN / 64, sizeof(OUT) == 2, false>(
          g, bias, t_row, m_tile * BM + quad * 32, n_tile * BN + half * (BN / 2), M, lane,
          [&] { return __all_sync(0xffffffffu, mbar_wait(tmem_full_bar(acc), phase, abort_flag)) != 0; },
          [&] {
            if (lane == 0) mbar_arrive(tmem_empty_bar(acc));
          });
      if (!got) {
        if (lane == 0) fail(kSiteEpilogueFull);
        break;
      }
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

// Tiles of 256 x 192 by a cluster of two CTAs.  Per 256 values of K a CTA loads its own 128 rows of A, half of the
// tile's W rows, and the scales of both: 31 KB for 128 x 192 of output, against 34 KB for 128 x 128 of the tile above.
// CTA 0 issues the MMAs (M = 256) of both.
//
// The width follows from three things.  The issuing thread needs 45 cycles for an MMA and, per stage, about 170 more
// for its waits, copies and commits: MMAs of N = 128 (64 cycles) do not cover that, of N = 192 (96 cycles) nearly do.
// A single accumulator buffer leaves the tensor core idle for 1000 to 1800 cycles a tile, the way from the last MMA
// to the epilogue and back.  And two buffers have to fit 512 columns beside the scales (24 columns a stage).
// 39778 x 1024 by 1024 x 4096, plain fp16 result / 39778 x 4096 by 4096 x 1024: 256 x 192 85 / 67 us, tiles of 128 x 128
// 104 / 83 us (and, with an earlier epilogue that took 104 / 76 us here: 256 x 256 in two column halves with three
// half-width buffers 120 / 82 us, 256 x 256 with one buffer 118 / 71 us).
//
// What bounds it now is the way of the operands from L2 to the SMs: 7.75 KB per 64 values of K and CTA, 124 cycles at 64
// bytes a cycle where the MMA needs 96; 62 bytes a cycle and SM are measured at 4096 -> 1024, 41 at 1024 -> 4096, where the
// results take 15 more.  With GELU it is the special functions (gelu_pair): their unit is 75 % busy, 70 % into 4 bits.
//
// Epilogue: all twelve warps on every tile, two column groups each that are in registers before the buffer goes back.
// Two sets of eight warps in turn, three groups each one after the other, took the same time for plain results (which
// the operands bound) but 190 us against 136 us with a residual, whose latency they met once per group.
//
// A tile's 192 W rows begin at the start or in the middle of a row block of 128: it takes the scales of two blocks, and
// in the second case the MMAs read them from two columns (64 rows) further on.
struct PairCfg {
  static constexpr int BN = 192;
  static constexpr int kStages = 5;
  static constexpr int kEpilogueWarps = 12;  // a TMEM lane quadrant and a third of the columns each
  static constexpr int kThreads = 64 + 32 * kEpilogueWarps;
  // both groups of a warp in registers at once, where they fit beside what is added to them (128 registers a thread)
  template <typename T, typename OUT, int EPI>
  static constexpr bool kWhole = sizeof(T) == 2 || (sizeof(OUT) == 4 && (EPI & kWithResidual) == 0);
  static constexpr int kBCodes = BN / 2 * 128;
  static constexpr int kStageBytes = kMxTileBytes + kBCodes + 2 * kMxScaleBytes;
  static constexpr int kScaleCols = 24;  // per stage: 2 pieces of A, 2 of each block of W, 4 columns each
  static constexpr int kTmemCols = 512;
  static constexpr int kNumBars = 2 * kStages + 6;
  static constexpr int kSmemBytes = kStages * kStageBytes + 256;
  static_assert(2 * BN + kStages * kScaleCols <= kTmemCols, "tensor memory");
  static_assert(kStageBytes % 1024 == 0 && kSmemBytes <= 232448 && kNumBars * 8 + 8 <= 256, "shared memory");
};

template <typename T, typename OUT, int ACT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PairCfg::kThreads, 1)
gemm_mxfp4_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w,
                       const __grid_constant__ CUtensorMap tmap_ws, const MxArgs g, const T* bias) {
  using cfg = PairCfg;
  constexpr int S = cfg::kStages;
  const uint32_t rank = cluster_ctarank();  // 0 issues the MMAs
  const int pair_id = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t tiles_addr = smem_u32(smem_raw);
  if ((tiles_addr & 1023u) != 0u) {  // same layout in both CTAs: uniform for the pair
    pdl_wait();
    if (threadIdx.x == 0) report_timeout(g.status_word, kKernelGemmMx, kSiteSmemAlign);
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem_raw + S * cfg::kStageBytes);
  const uint32_t bar0 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto free_bar = [&](int s) { return bar0 + 8u * (S + s); };
  auto tmem_full_bar = [&](int a) { return bar0 + 8u * (2 * S + a); };
  auto tmem_empty_bar = [&](int a) { return bar0 + 8u * (2 * S + 2 + a); };
  const uint32_t drain_bar = bar0 + 8u * (2 * S + 4), peer_tmem_bar = drain_bar + 8u;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + cfg::kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(free_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tmem_full_bar(a), 1);
      mbar_init(tmem_empty_bar(a), 2 * cfg::kEpilogueWarps);
    }
    mbar_init(drain_bar, 1);
    mbar_init(peer_tmem_bar, 1);
    *abort_flag = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  __syncthreads();
  cluster_sync_all();  // the peer's barriers are initialised before anything signals them
  int M = g.max_m;
  if (g.m_ptr != nullptr) M = pdl_wait_row_count(g.m_ptr, g.max_m, 0);
  else pdl_wait();
  uint32_t tmem_base = 0;  // (the producer needs none)
  if (warp == 1)
    tmem_base = take_tmem(tmem_slot, cfg::kThreads - 64, [&] {
      tmem_alloc_pair(smem_u32(tmem_slot), cfg::kTmemCols);
      tmem_relinquish_pair();
      __syncwarp();
      tc_fence_before();
      // (CTA 0 issues into both CTAs' tensor memory; a second cluster barrier instead: 0.7 us a launch)
      if (rank == 1 && lane == 0) mbar_arrive_cluster(mapa_shared(peer_tmem_bar, 0));
    });

  const int N = g.n;
  const int n_tiles = (N + cfg::BN - 1) / cfg::BN;
  const int num_tiles = (M + 255) / 256 * n_tiles;
  const int k_tiles = mx_k_tiles(g.k);
  // columns of a tile: the last one of a row of tiles has what is left of N, in steps of 64
  auto columns = [&](int n_tile) { return min(cfg::BN, (N - n_tile * cfg::BN + 63) / 64 * 64); };

  auto fail = [&](int site) {
    *abort_flag = 1;
    report_timeout(g.status_word, kKernelGemmMx, site);
  };

  if (warp == 0) {
    // ------------------------- producer (both CTAs) -------------------------
    // all lanes walk through the loop, one issues (see elect_one)
    const bool issuer = elect_one();
    if (issuer) {
      prefetch_tensormap(&tmap_a);
      prefetch_tensormap(&tmap_w);
      prefetch_tensormap(&tmap_ws);
    }
    {
      constexpr int kTileLines = kMxTileBytes / 1024;  // 16 of codes (8 rows each), 1 of scales
      uint32_t stage = 0, phase = 0;
      long long issued = 0;
      bool ok = true;
      for (int tile = pair_id; tile < num_tiles && ok; tile += num_pairs) {
        const int m_tile = tile / n_tiles, n_tile = tile - m_tile * n_tiles;
        const int cols = columns(n_tile), n0 = n_tile * cfg::BN;
        // (row blocks behind the last one are filled with zeros)
        int a_line = (m_tile * 2 + static_cast<int>(rank)) * k_tiles * kTileLines;
        const int w_row = n0 + static_cast<int>(rank) * (cols / 2);  // this CTA's first W row, of cols / 2
        int ws_line = n0 / kMxTileRows * k_tiles * kTileLines + kMxCodeBytes / 1024;
        int w_line[3];  // 32 W rows each, which never cross a row block
#pragma unroll
        for (int j = 0; j < 3; ++j)
          w_line[j] = (w_row + 32 * j) / kMxTileRows * k_tiles * kTileLines + (w_row + 32 * j) % kMxTileRows / 8;
        const uint32_t stage_tx = 2u * (kMxTileBytes + cols / 2 * 128 + 2 * kMxScaleBytes);
        for (int kt = 0; kt < k_tiles; ++kt) {
          if (!__all_sync(0xffffffffu, mbar_wait(free_bar(stage), phase ^ 1u, abort_flag))) {
            if (lane == 0) fail(kSiteProducerEmpty);
            ok = false;
            break;
          }
          const uint32_t dst = tiles_addr + stage * cfg::kStageBytes, w_dst = dst + kMxTileBytes;
          const uint32_t s_dst = w_dst + cfg::kBCodes, full0 = mapa_shared(full_bar(stage), 0);
          if (issuer) {
            if (rank == 0) mbar_arrive_expect_tx(full_bar(stage), stage_tx);
            tma_load_2d_pair(dst, &tmap_a, 0, a_line, full0);
            tma_load_2d_pair(w_dst, &tmap_w, 0, w_line[0], full0);
            if (cols > 64) tma_load_2d_pair(w_dst + 4096, &tmap_w, 0, w_line[1], full0);
            if (cols > 128) tma_load_2d_pair(w_dst + 8192, &tmap_w, 0, w_line[2], full0);
            tma_load_2d_pair(s_dst, &tmap_ws, 0, ws_line, full0);
            tma_load_2d_pair(s_dst + kMxScaleBytes, &tmap_ws, 0, ws_line + k_tiles * kTileLines, full0);
          }
          __syncwarp();
          a_line += kTileLines;
          ws_line += kTileLines;
#pragma unroll
          for (int j = 0; j < 3; ++j) w_line[j] += kTileLines;
          ++issued;
          if (++stage == S) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // the issuer's commits on the ring are asynchronous arrivals, in the peer from the other SM: the last of them
      // land before the barriers go away
      const long long pending = !issuer ? 0 : issued < S ? issued : S;
      for (long long i = 0; i < pending; ++i) {
        const long long f = issued - 1 - i;
        if (!mbar_wait(free_bar(static_cast<int>(f % S)), static_cast<uint32_t>((f / S) & 1), abort_flag) &&
            *abort_flag == 0)
          fail(kSiteProducerDrain);
      }
      if (rank == 0) {
        // full counts both CTAs' bytes: behind these phases no copy of the pair is in flight; the peer learns it at
        // the closing cluster barrier
        for (long long i = 0; i < pending; ++i) {
          const long long f = issued - 1 - i;
          if (!mbar_drain(full_bar(static_cast<int>(f % S)), static_cast<uint32_t>((f / S) & 1)) && *abort_flag == 0)
            fail(kSiteProducerDrain);
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------- MMA issuer (CTA 0 only) -------------------------
    // all lanes walk through the loop, one issues (see elect_one)
    if (rank == 0) {
      const bool issuer = elect_one();
      uint32_t stage = 0, phase = 0;
      int it = 0;
      bool ok = __all_sync(0xffffffffu, mbar_wait(peer_tmem_bar, 0u, abort_flag)) != 0;
      if (!ok && lane == 0) fail(kSiteMmaPeerTmem);
      tc_fence_after();
      for (int tile = pair_id; tile < num_tiles && ok; tile += num_pairs, ++it) {
        const int n_tile = tile % n_tiles, cols = columns(n_tile), acc = it & 1;
        if (!__all_sync(0xffffffffu, mbar_wait(tmem_empty_bar(acc), ((it >> 1) & 1) ^ 1u, abort_flag))) {
          if (lane == 0) fail(kSiteMmaTmemEmpty);
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * cfg::BN;
        const uint32_t shift = (n_tile & 1) * 2;  // the tile's W rows begin in the middle of a row block
        const uint32_t idesc0 = make_idesc_mxf4(2 * BM, cols, 0);
        for (int kt = 0; kt < k_tiles; ++kt) {
          if (!__all_sync(0xffffffffu, mbar_wait(full_bar(stage), phase, abort_flag))) {
            if (lane == 0) fail(kSiteMmaFull);
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a_addr = tiles_addr + stage * cfg::kStageBytes, b_addr = a_addr + kMxTileBytes;
          const uint32_t sf = tmem_base + 2 * cfg::BN + stage * cfg::kScaleCols;
          const int left = g.k - kt * kMxTileK;
          const int steps = left >= kMxTileK ? 4 : (left + kUmmaK - 1) / kUmmaK;
          if (issuer) {
            issue_stage<true, 2>(steps, d_tmem, a_addr, b_addr, b_addr + cfg::kBCodes, sf, sf + 8, shift, idesc0, kt == 0);
            umma_commit_both(free_bar(stage));
            if (kt == k_tiles - 1) umma_commit_both(tmem_full_bar(acc));
          }
          __syncwarp();
          if (++stage == S) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // all MMAs must have retired before TMEM is freed
      if (issuer) {
        umma_commit_pair(drain_bar);
        if (!mbar_drain(drain_bar, 0u) && *abort_flag == 0) fail(kSiteMmaDrain);
      }
      __syncwarp();
    }
  } else {
    // ------------------------- epilogue (both CTAs) -------------------------
    tmem_base = tmem_address(tmem_slot, cfg::kThreads - 64);
    const int quad = warp & 3, part = (warp - 2) >> 2;
    const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + part * 64;
    int it = 0;
    for (int tile = pair_id; tile < num_tiles; tile += num_pairs, ++it) {
      const int acc = it & 1;
      const int m_tile = tile / n_tiles, n_tile = tile - m_tile * n_tiles;
      const bool got = epilogue_warp<T, OUT, ACT, 2, true, cfg::kWhole<T, OUT, ACT>>(
          g, bias, t_row + acc * cfg::BN, m_tile * 256 + static_cast<int>(rank) * BM + quad * 32,
          n_tile * cfg::BN + part * 64, M, lane,
          [&] { return __all_sync(0xffffffffu, mbar_wait(tmem_full_bar(acc), (it >> 1) & 1, abort_flag)) != 0; },
          [&] {
            // (relaxed: the accumulator's values are in registers, and this tile's stores must not be waited for)
            if (lane == 0) mbar_arrive_cluster_relaxed(mapa_shared(tmem_empty_bar(acc), 0));
          });
      if (!got) {
        if (lane == 0) fail(kSiteEpilogueFull);
        break;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // neither CTA leaves while the other may still touch its barriers or TMEM
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, cfg::kTmemCols);
  }
}

// An MXFP4 tensor as lines of 1024 bytes, for boxes of `box` lines.  (Lines of 128 bytes move the same bytes at half
// the rate.)
bool encode_lines(CUtensorMap* map, const void* base, int rows, int k, uint32_t box) {
  EncodeTiledFn fn = get_encode_tiled();
  if (fn == nullptr) return false;
  const cuuint64_t dims[2] = {128, mx_bytes(rows, k) / 1024};
  const cuuint64_t strides[1] = {1024};
  const cuuint32_t boxes[2] = {128, box};
  const cuuint32_t elem_strides[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT64, 2, const_cast<void*>(base), dims, strides, boxes, elem_strides,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, typename OUT, int ACT>
cudaError_t launch_pair(const MxArgs& g, const T* bias, cudaStream_t stream) {
  using cfg = PairCfg;
  static PerDeviceOnce once;
  const cudaError_t err = once.run([] {
    return cudaFuncSetAttribute(gemm_mxfp4_pair_kernel<T, OUT, ACT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                cfg::kSmemBytes);
  });
  if (err != cudaSuccess) return err;
  CUtensorMap ta, tw, tws;
  if (!encode_lines(&ta, g.a, g.max_m, g.k, kMxTileBytes / 1024) || !encode_lines(&tw, g.w, g.n, g.k, 4) ||
      !encode_lines(&tws, g.w, g.n, g.k, 1))
    return cudaErrorInvalidValue;
  const long long tiles = static_cast<long long>((g.max_m + 255) / 256) * ((g.n + cfg::BN - 1) / cfg::BN);
  const int pairs = static_cast<int>(tiles < sm_count() / 2 ? tiles : sm_count() / 2);
  return launch_pdl(gemm_mxfp4_pair_kernel<T, OUT, ACT>, dim3(2 * pairs), dim3(cfg::kThreads), cfg::kSmemBytes, stream,
                    ta, tw, tws, g, bias);
}

// Few rows (a row tile or two) straight from fp16 or fp32: one CTA per tile of 128 x 64, all of K in shared memory at
// once.  Its 16 epilogue warps first quantise the tile's rows into the operand layout, while the producer fetches the W
// rows; there is no second kernel to launch and no 4-bit copy of the rows in memory.  Every CTA of a row tile
// quantises the same rows again, which is little work for few of them.  One row of 1024 through a 1024 x 4096
// projection with GELU: 3.7 us on the device against 5.4 us for quantisation and product, and one launch (3 us of host
// time) less.
struct RowsCfg {
  static constexpr int BN = 64;
  static constexpr int kMaxKTiles = 6;  // K up to 1536
  static constexpr int kStageBytes = kMxTileBytes + BN * 128 + kMxScaleBytes;
  static constexpr int kNumBars = kMaxKTiles + 3;
  static constexpr int kScaleCols = 16;
  static constexpr int kTmemCols = 256;
  static constexpr int smem_bytes(int k_tiles) { return k_tiles * kStageBytes + 256; }
  static_assert(BN + kMaxKTiles * kScaleCols <= kTmemCols, "tensor memory");
  static_assert(kStageBytes % 1024 == 0 && kMaxKTiles * kStageBytes + 256 <= 232448 && kNumBars * 8 + 8 <= 256,
                "shared memory");
};

template <typename T, typename OUT, int ACT>
__global__ void __launch_bounds__(kNumThreads, 1)
gemm_mxfp4_rows_kernel(const MxArgs g, const T* x, long long row_stride, const T* bias) {
  using cfg = RowsCfg;
  constexpr int BN = cfg::BN;
  const int k_tiles = mx_k_tiles(g.k);
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t tiles_addr = smem_u32(smem_raw);
  if ((tiles_addr & 1023u) != 0u) {  // the swizzled tiles need 1024-byte alignment
    pdl_wait();
    if (threadIdx.x == 0) report_timeout(g.status_word, kKernelGemmMx, kSiteSmemAlign);
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem_raw + k_tiles * cfg::kStageBytes);
  const uint32_t bar0 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  const uint32_t rows_bar = bar0 + 8u * cfg::kMaxKTiles, tmem_full_bar = rows_bar + 8u, drain_bar = rows_bar + 16u;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + cfg::kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < k_tiles; ++s) mbar_init(full_bar(s), 1);
    mbar_init(rows_bar, 2 * kEpilogueSet);
    mbar_init(tmem_full_bar, 1);
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  __syncthreads();
  int M = g.max_m;
  if (g.m_ptr != nullptr) M = pdl_wait_row_count(g.m_ptr, g.max_m, 0);
  else pdl_wait();

  const int N = g.n;
  const int n_tiles = (N + BN - 1) / BN;
  const int m_tile = blockIdx.x / n_tiles, n_tile = blockIdx.x - m_tile * n_tiles;
  const int row_tile = m_tile * BM;
  if (row_tile >= M) return;  // (the whole CTA, with nothing in flight)
  uint32_t tmem_base = 0;  // (the producer needs none)
  if (warp == 1)
    tmem_base = take_tmem(tmem_slot, kNumThreads - 64, [&] {
      tmem_alloc(smem_u32(tmem_slot), cfg::kTmemCols);
      tmem_relinquish();
    });

  auto fail = [&](int site) {
    *abort_flag = 1;
    report_timeout(g.status_word, kKernelGemmMx, site);
  };

  if (warp == 0) {
    const bool issuer = elect_one();
    if (issuer) {
      const uint8_t* w_src =
          g.w + static_cast<size_t>(n_tile * BN / kMxTileRows) * k_tiles * kMxTileBytes;  // the tile's W rows: half a block
      const int skip = n_tile * BN % kMxTileRows * 128;
      for (int kt = 0; kt < k_tiles; ++kt, w_src += kMxTileBytes) {
        const uint32_t w_dst = tiles_addr + kt * cfg::kStageBytes + kMxTileBytes;
        mbar_arrive_expect_tx(full_bar(kt), BN * 128 + kMxScaleBytes);
        bulk_load(w_dst, w_src + skip, BN * 128, full_bar(kt));
        bulk_load(w_dst + BN * 128, w_src + kMxCodeBytes, kMxScaleBytes, full_bar(kt));
      }
      // copies in flight land before the CTA's shared memory goes away, also behind a wait that ran out
      for (int kt = 0; kt < k_tiles; ++kt)
        if (!mbar_drain(full_bar(kt), 0u) && *abort_flag == 0) fail(kSiteProducerDrain);
    }
    __syncwarp();
  } else if (warp == 1) {
    // all lanes walk through the loop, one issues (see elect_one)
    const bool issuer = elect_one();
    bool ok = __all_sync(0xffffffffu, mbar_wait(rows_bar, 0u, abort_flag)) != 0;
    if (!ok && lane == 0) fail(kSiteMmaFull);
    const uint32_t shift = n_tile * BN % kMxTileRows / 32;
    for (int kt = 0; kt < k_tiles && ok; ++kt) {
      if (!__all_sync(0xffffffffu, mbar_wait(full_bar(kt), 0u, abort_flag))) {
        if (lane == 0) fail(kSiteMmaFull);
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t a_addr = tiles_addr + kt * cfg::kStageBytes, b_addr = a_addr + kMxTileBytes;
      const uint32_t sf = tmem_base + BN + kt * cfg::kScaleCols;
      const int left = g.k - kt * kMxTileK;
      const int steps = left >= kMxTileK ? 4 : (left + kUmmaK - 1) / kUmmaK;
      if (issuer) {
        issue_stage<false, 1>(steps, tmem_base, a_addr, b_addr, b_addr + BN * 128, sf, sf + 8, shift,
                              make_idesc_mxf4(BM, BN, 0), kt == 0);
        if (kt == k_tiles - 1) umma_commit(tmem_full_bar);
      }
      __syncwarp();
    }
    // all MMAs must have retired before TMEM is freed
    if (issuer) {
      umma_commit(drain_bar);
      if (!mbar_drain(drain_bar, 0u) && *abort_flag == 0) fail(kSiteMmaDrain);
    }
    __syncwarp();
  } else {
    // ---- the tile's rows, quantised as mx_quantize_kernel does: eight values a lane, four lanes a scale block ----
    // a piece is one k-tile of a row; they are dealt to the warps in turn, which have four each on their way at a time
    constexpr int kPieces = 4, kWarps = 2 * kEpilogueSet;
    const int rows = min(M - row_tile, BM), pieces = rows * k_tiles;
    for (int t0 = warp - 2; t0 < pieces; t0 += kWarps * kPieces) {
      Oct<T> v[kPieces];
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int t = t0 + i * kWarps, row = t / k_tiles, col = (t - row * k_tiles) * kMxTileK + lane * 8;
        v[i].zero();
        if (t < pieces && col < g.k) v[i].load(x + static_cast<size_t>(row_tile + row) * row_stride + col);
      }
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int t = t0 + i * kWarps, row = t / k_tiles, kt = t - row * k_tiles;
        if (t >= pieces) break;
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; e += VecTraits<T>::kElems) VecTraits<T>::unpack(v[i].v[e / VecTraits<T>::kElems], f + e);
        uint32_t top = 0u;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, abs_bits(f[e]));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const MxScale s = mx_scale(top);
        uint32_t scales = s.byte | (__shfl_down_sync(0xffffffffu, s.byte, 4) << 8);
        scales |= __shfl_down_sync(0xffffffffu, scales, 8) << 16;  // four blocks' bytes in lanes 0 and 16
        uint8_t* tile = smem_raw + kt * cfg::kStageBytes;
        *reinterpret_cast<uint32_t*>(tile + mx_code_offset(row, lane >> 2) + (lane & 3) * 4) = mx_codes8(f, s);
        if ((lane & 15) == 0) *reinterpret_cast<uint32_t*>(tile + mx_scale_offset(row, lane >> 2)) = scales;
      }
    }
    fence_proxy_async_smem();  // these stores are read by the tensor core
    __syncwarp();
    if (lane == 0) mbar_arrive(rows_bar);
    tmem_base = tmem_address(tmem_slot, kNumThreads - 64);
    // ---- epilogue: eight of the warps, a lane quadrant and 32 columns each ----
    if (warp < 2 + kEpilogueSet) {
      const int quad = warp & 3, half = (warp - 2) >> 2;
      const bool got = epilogue_warp<T, OUT, ACT, 1, true, true>(
          g, bias, tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + half * 32, row_tile + quad * 32,
          n_tile * BN + half * 32, M, lane,
          [&] { return __all_sync(0xffffffffu, mbar_wait(tmem_full_bar, 0u, abort_flag)) != 0; }, [] {});
      if (!got && lane == 0) fail(kSiteEpilogueFull);
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
cudaError_t launch_rows(const MxArgs& g, const T* x, long long row_stride, const T* bias, cudaStream_t stream) {
  using cfg = RowsCfg;
  static PerDeviceOnce once;
  const cudaError_t err = once.run([] {
    return cudaFuncSetAttribute(gemm_mxfp4_rows_kernel<T, OUT, ACT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                cfg::smem_bytes(cfg::kMaxKTiles));
  });
  if (err != cudaSuccess) return err;
  const int grid = (g.max_m + BM - 1) / BM * ((g.n + cfg::BN - 1) / cfg::BN);
  return launch_pdl(gemm_mxfp4_rows_kernel<T, OUT, ACT>, dim3(grid), dim3(kNumThreads),
                    cfg::smem_bytes(mx_k_tiles(g.k)), stream, g, x, row_stride, bias);
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
  if (mxfp4_route(sizeof(OUT) == 4, g.route_rows, g.n, g.k) == kMxPair) return launch_pair<T, OUT, ACT>(g, bias, stream);
  const int grid = static_cast<int>(tiles < sm_count() ? tiles : sm_count());
  return launch_pdl(gemm_mxfp4_kernel<T, OUT, ACT>, dim3(grid), dim3(kNumThreads), cfg::kSmemBytes, stream, g, bias);
}

// x given: few rows of T instead of MXFP4 ones.
template <typename T, typename OUT, int ACT>
cudaError_t launch_from(const MxArgs& g, const T* x, long long row_stride, const T* bias, cudaStream_t stream) {
  if (x != nullptr) return launch_rows<T, OUT, ACT>(g, x, row_stride, bias, stream);
  return launch_act<T, OUT, ACT>(g, bias, stream);
}

template <typename T, typename OUT>
cudaError_t launch_out(const MxArgs& g, const T* x, long long row_stride, const T* bias, int epilogue,
                       cudaStream_t stream) {
  constexpr int kRes = sizeof(OUT) == sizeof(T) ? kWithResidual : 0;  // (MXFP4 results take none)
#define ETB_MX_CASE(E)                                                                            \
  case E:                                                                                         \
    if (g.residual != nullptr) return launch_from<T, OUT, E + kRes>(g, x, row_stride, bias, stream); \
    return launch_from<T, OUT, E>(g, x, row_stride, bias, stream)
  switch (epilogue) {
    ETB_MX_CASE(kEpiNone);
    ETB_MX_CASE(kEpiBias);
    ETB_MX_CASE(kEpiBiasGelu);
    ETB_MX_CASE(kEpiBiasTanh);
    default:
      return cudaErrorInvalidValue;
  }
#undef ETB_MX_CASE
}

template <typename T>
cudaError_t launch_checked(const MxGemm& p, const T* x, long long row_stride, const T* bias, const T* residual, T* c,
                           int epilogue, cudaStream_t stream) {
  if (p.max_m <= 0) return cudaSuccess;
  if (p.n <= 0 || p.k <= 0 || p.n % 32 != 0 || p.k % kMxBlock != 0) return cudaErrorInvalidValue;
  if ((c == nullptr) == (p.c_mx == nullptr)) return cudaErrorInvalidValue;
  if (p.c_mx != nullptr && (p.n % 64 != 0 || residual != nullptr)) return cudaErrorInvalidValue;
  if (epilogue != kEpiNone && bias == nullptr) return cudaErrorInvalidValue;
  for (const void* q : {static_cast<const void*>(x), static_cast<const void*>(c), static_cast<const void*>(bias),
                        static_cast<const void*>(residual)})
    if (reinterpret_cast<uintptr_t>(q) & 15u) return cudaErrorMisalignedAddress;
  for (const void* q : {x != nullptr ? nullptr : p.a, p.w, static_cast<const void*>(p.c_mx)})
    if (reinterpret_cast<uintptr_t>(q) & 127u) return cudaErrorMisalignedAddress;
  MxArgs g;
  g.a = static_cast<const uint8_t*>(p.a);
  g.w = static_cast<const uint8_t*>(p.w);
  g.c = c != nullptr ? static_cast<void*>(c) : p.c_mx;
  g.residual = residual;
  g.m_ptr = p.m_ptr;
  g.max_m = p.max_m, g.n = p.n, g.k = p.k;
  g.route_rows = p.route_rows > 0 ? p.route_rows : p.max_m;
  g.status_word = p.status_word;
  g.sectors = (reinterpret_cast<uintptr_t>(c) & 31u) == 0;
  // (the kernels count tiles and 1 KB lines of an operand in 31 bits; a buffer beyond that would not fit any memory)
  if (mx_bytes(p.max_m, p.k) / 1024 > 0x7fffffffull || mx_bytes(p.n, p.k) / 1024 > 0x7fffffffull ||
      static_cast<long long>((p.max_m + BM - 1) / BM) * ((p.n + 63) / 64) > 0x7fffffffll)
    return cudaErrorInvalidValue;
  if (p.c_mx != nullptr) return launch_out<T, MxOut>(g, x, row_stride, bias, epilogue, stream);
  return launch_out<T, T>(g, x, row_stride, bias, epilogue, stream);
}

}  // namespace

// Tiles of 256 x 192 by CTA pairs need half the L2 traffic per product and 40 % fewer issue slots; tiles of 128 x 128
// start sooner, waste less at the edges and have the shorter epilogue.  Measured, 128 x 128 / pairs, us:
//   at least three rounds of 128 x 128 tiles, K = 4096: 8192 x 1024 23.2 / 17.0; K = 2048: 4096 x 2048 14.1 / 11.6;
//     K = 1024: 40000 x 4096 104 / 87, with GELU 115 / 115 to 123; K = 768: 16000 x 2304 22.8 / 19.1, with GELU 26.5 / 28,
//     with a residual 49 / 33 (fp32 31.8 / 30.2 and 93 / 56); but K = 256: 40000 x 1024 16.6 / 17.2, with GELU 26.7 / 31.4;
//   one to three rounds, K = 4096: 4096 x 1024 13.7 / 12.6; K = 2048: 2048 x 2048 9.1 / 8.7 (fp32 9.1 / 10.0);
//     K = 1024: 4096 x 1024 with GELU 6.7 / 7.9;
//   one round, K = 2048: 1024 x 2048 6.4 / 6.6.
MxRoute mxfp4_route(bool fp32_result, int rows, int n, int k) {
  const long long tiles = static_cast<long long>((rows + BM - 1) / BM) * ((n + 127) / 128);
  if (tiles > 3ll * sm_count()) return k >= 768 ? kMxPair : kMxSingle;
  return !fp32_result && k >= 2048 && tiles > sm_count() ? kMxPair : kMxSingle;
}
// The kernel that quantises the rows itself pays while its tiles are one round of CTAs, K fits its shared memory and the
// rows, which every CTA quantises again, are few: 128 pieces of 256 values.  1024 x 1024, 1 / 16 / 32 rows: 3.6 / 4.7 /
// 5.9 us on the device (64 would take 8.0), quantisation and product 5.2 / 5.5 / 5.4 us, and 3 us more on the host.
bool mxfp4_rows_supported(int rows, int n, int k) {
  return rows <= BM && mx_k_tiles(k) <= RowsCfg::kMaxKTiles && rows * mx_k_tiles(k) <= 128 &&
         (n + RowsCfg::BN - 1) / RowsCfg::BN <= sm_count();
}

template <typename T>
cudaError_t launch_gemm_mxfp4(const MxGemm& p, const T* bias, const T* residual, T* c, int epilogue,
                              cudaStream_t stream) {
  return launch_checked<T>(p, nullptr, 0, bias, residual, c, epilogue, stream);
}

template <typename T>
cudaError_t launch_linear_mxfp4(const MxGemm& p, const T* x, long long row_stride, void* x_mx, const T* bias,
                                const T* residual, T* c, int epilogue, cudaStream_t stream) {
  if (p.max_m <= 0) return cudaSuccess;
  if (x == nullptr || row_stride < p.k || row_stride * sizeof(T) % 16 != 0) return cudaErrorInvalidValue;
  // (the kernel of few rows reads x while other CTAs of it write: not in place)
  const size_t x_size = (static_cast<size_t>(p.max_m - 1) * row_stride + p.k) * sizeof(T);
  const bool in_place = overlap(x, x_size, c, static_cast<size_t>(p.max_m) * p.n * sizeof(T)) ||
                        (p.c_mx != nullptr && overlap(x, x_size, p.c_mx, mx_bytes(p.max_m, p.n)));
  if (!in_place && mxfp4_rows_supported(p.route_rows > 0 ? p.route_rows : p.max_m, p.n, p.k))
    return launch_checked<T>(p, x, row_stride, bias, residual, c, epilogue, stream);
  const cudaError_t err = launch_mx_quantize<T>(x, row_stride, p.m_ptr, p.max_m, p.k, x_mx, stream);
  if (err != cudaSuccess) return err;
  MxGemm q = p;
  q.a = x_mx;
  return launch_checked<T>(q, nullptr, 0, bias, residual, c, epilogue, stream);
}

#define ETB_INST(T)                                                                                                  \
  template cudaError_t launch_gemm_mxfp4<T>(const MxGemm&, const T*, const T*, T*, int, cudaStream_t);               \
  template cudaError_t launch_linear_mxfp4<T>(const MxGemm&, const T*, long long, void*, const T*, const T*, T*, int, \
                                              cudaStream_t);
ETB_INST(__half)
ETB_INST(float)
#undef ETB_INST

}  // namespace etb
