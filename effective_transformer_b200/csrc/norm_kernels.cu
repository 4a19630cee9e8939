// The norm behind a block, its gate and residual scale, and the norm in front of the next block, in one pass:
//   p = post(x + bias)
//   h = residual_scale * residual + gate * p        (gate: per channel, or one row per sequence)
//   y = pre(h)
// post and pre are each a LayerNorm, (v - mean) * rsqrt(var + eps) * gamma + beta, an RMS norm,
// v * rsqrt(mean(v^2) + eps) * gamma, or nothing.  The plain post-norm encoder (add_bias_input_layernorm,
// cuda/cuda_kernels.cu:157-236) is post = nothing, gate = 1, residual_scale = 1, y only.
//
// Everything between the loads of x and residual and the stores of h and y stays in fp32 registers, so x and residual
// are read once and h and y written once: the kernel is bound by those bytes once it spends few enough instructions.  A
// group of warps (at most 16) takes R rows at a time; a lane holds V vectors of 16 bytes of each, 1 or 2
// (launch_gated_norm has the rule).  So bias, gamma and beta stay in registers for all rows, and the R rows' sums go
// through their shuffles side by side.  Means and variances are taken in two passes over the registers.  y can leave as
// MXFP4 too (mxfp4.cuh): four (fp16) or eight (fp32) neighbouring lanes hold a scale block.
//
// 39778 rows of 1024 fp16 values with both norms and a gate: 68 us, 4.8 TB/s (328 MB; 50 us at the rate of a copy), 60 %
// of the issue slots at 16 warps an SM: the sums' shuffles and the conversions are what is left.  4099 rows of 2080 fp32
// values with RMS norms: 32 us, 4.2 TB/s.  One row of 768: 2.1 us.  The first of these by layout, while it took 81 us:
// one row to a warp with the parameters read from L1 for every row 118 us, from shared memory in fp32 88 us (128
// registers, and what is fetched ahead spills), four warps to one row 154 us, to four rows 82 us without and 96 us with
// fetching ahead.  Registers capped for more warps: spills, slower at every cap.  Rows counted in 32 bits: 78 us instead of
// 68 (and 34 of 32 in fp32), in the compiler's other order of the loads.
#include "common.cuh"
#include "mxfp4.cuh"
#include "packed_f32.cuh"

namespace etb {

namespace {

constexpr int kMaxWarps = 16;  // of a row
constexpr int kCtaWarps = 4;   // a CTA has as many whole groups as fit these, at least one

enum NormKind : int { kNormNone = 0, kNormLayer = 1, kNormRms = 2 };

// A vector of 16 bytes as pairs of fp32 values (packed_f32.cuh).
template <typename T>
struct Pairs {
  static constexpr int kCount = VecTraits<T>::kElems / 2;
  static __device__ __forceinline__ void unpack(const Vec16& v, Pair* p) {
    float f[2 * kCount];
    VecTraits<T>::unpack(v, f);
#pragma unroll
    for (int i = 0; i < kCount; ++i) p[i] = pack2(f[2 * i], f[2 * i + 1]);
  }
  static __device__ __forceinline__ Vec16 pack(const Pair* p) {
    float f[2 * kCount];
#pragma unroll
    for (int i = 0; i < kCount; ++i) unpack2(p[i], f[2 * i], f[2 * i + 1]);
    return VecTraits<T>::pack(f);
  }
};
__device__ __forceinline__ Pair both(float x) { return pack2(x, x); }

// One vector a lane of an MXFP4 row: c is the lane's vector, whose first column in the warp is that of lane 0.
template <typename T>
__device__ __forceinline__ void store_mx(const Pair* v, void* y_mx, int row, int c, int n, int lane) {
  constexpr int E = VecTraits<T>::kElems;
  constexpr int kLanes = kMxBlock / E;  // lanes of a scale block
  const int col = c * E;
  if ((c - lane) * E >= n) return;  // (uniform for the warp)
  float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  uint32_t top = 0u;
  if (col < n) {  // (zeros behind the row's end)
#pragma unroll
    for (int i = 0; i < E / 2; ++i) unpack2(v[i], f[2 * i], f[2 * i + 1]);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) top = max(top, abs_bits(f[e]));
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  const MxScale s = mx_scale(top);
  uint32_t scales = s.byte | (__shfl_down_sync(0xffffffffu, s.byte, kLanes) << 8);
  scales |= __shfl_down_sync(0xffffffffu, scales, 2 * kLanes) << 16;
  const int r = row & (kMxTileRows - 1), b = (col & 255) >> 5;
  uint8_t* tile = static_cast<uint8_t*>(y_mx) + mx_tile_offset(row, col >> 8, mx_k_tiles(n));
  const uint32_t code = mx_codes8(f, s);
  uint8_t* dst = tile + mx_code_offset(r, b) + (lane & (kLanes - 1)) * (E / 2);
  if (E == 8) *reinterpret_cast<uint32_t*>(dst) = code;
  else *reinterpret_cast<uint16_t*>(dst) = static_cast<uint16_t>(code);
  if ((lane & (4 * kLanes - 1)) == 0) *reinterpret_cast<uint32_t*>(tile + mx_scale_offset(r, b)) = scales;
}

// Where a lane stands: its group, the group's warps, the lane's first vector of a row.
struct Place {
  int group, wpr, wig, lane, vec0, vecs, turn;
  float* red;  // [2][R][kMaxWarps] of the group, used in turn
};

// Sums of R values over the lanes of a group, to every lane: in a warp the R rows' shuffles are merged (a lane passes on
// what its half of the warp is not to keep), between warps through shared memory.  kFew: at most four warps.
template <int R, bool kFew>
__device__ __forceinline__ void group_sum(float (&v)[R], Place& p) {
  int o = 16, row = 0;
#pragma unroll
  for (int h = R / 2; h >= 1; h >>= 1, o >>= 1) {
    const bool upper = (p.lane & o) != 0;
    row = 2 * row + (upper ? 1 : 0);
#pragma unroll
    for (int j = 0; j < h; ++j) {
      const float send = upper ? v[j] : v[j + h], keep = upper ? v[j + h] : v[j];
      v[j] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
  // row: the index of v that a lane ends with, most significant halving first
  const int lanes = o * 2;  // lanes that share it
#pragma unroll
  for (; o >= 1; o >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
  float* slot = p.red + p.turn * kMaxWarps * R;
  p.turn ^= 1;
  if ((p.lane & (lanes - 1)) == 0) slot[row * kMaxWarps + p.wig] = v[0];
  asm volatile("bar.sync %0, %1;" ::"r"(p.group + 1), "r"(p.wpr * 32) : "memory");
  // (slots of warps that the group does not have are zero)
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float4 f = *reinterpret_cast<const float4*>(slot + r * kMaxWarps);
    v[r] = (f.x + f.y) + (f.z + f.w);
  }
  for (int i = 4; !kFew && i < p.wpr; i += 4)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float4 f = *reinterpret_cast<const float4*>(slot + r * kMaxWarps + i);
      v[r] += (f.x + f.y) + (f.z + f.w);
    }
}

// v := norm(v) of R rows; elements past the row's end are zero before and behind.  kFull: no lane has such elements.
template <typename T, int V, int R, bool kFull, bool kFew>
__device__ __forceinline__ void normalise(Pair (&v)[R][V][Pairs<T>::kCount], int kind, const Vec16 (&gamma)[V],
                                          const Vec16 (&beta)[V], float inv_n, float eps, Place& p) {
  constexpr int P = Pairs<T>::kCount;
  float s[R];
  if (kind == kNormLayer) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      Pair a = v[r][0][0];
#pragma unroll
      for (int j = 0; j < V; ++j)
#pragma unroll
        for (int i = 0; i < P; ++i)
          if (i + j > 0) a = add2(a, v[r][j][i]);
      s[r] = a.x + a.y;
    }
    group_sum<R, kFew>(s, p);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float inside = kFull || p.vec0 + j * 32 * p.wpr < p.vecs ? -inv_n : 0.f;
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < P; ++i) v[r][j][i] = add2(v[r][j][i], both(s[r] * inside));
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    Pair a = mul2(v[r][0][0], v[r][0][0]);
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int i = 0; i < P; ++i)
        if (i + j > 0) a = fma2(v[r][j][i], v[r][j][i], a);
    s[r] = a.x + a.y;
  }
  group_sum<R, kFew>(s, p);
#pragma unroll
  for (int r = 0; r < R; ++r) s[r] = rsqrtf(fmaf(s[r], inv_n, eps));
#pragma unroll
  for (int j = 0; j < V; ++j) {
    Pair g[P], b[P];
    Pairs<T>::unpack(gamma[j], g);
    Pairs<T>::unpack(beta[j], b);  // (zeros for an RMS norm)
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < P; ++i) v[r][j][i] = fma2(mul2(v[r][j][i], both(s[r])), g[i], b[i]);
  }
}

// kRegs: 128, which a CTA of 512 threads may have, or 96.
template <typename T, int V, int R, bool kFull, bool kFew, int kRegs>
__global__ void __maxnreg__(kRegs)
gated_norm_kernel(const GatedNorm p, int wpr) {
  constexpr int E = VecTraits<T>::kElems, P = E / 2;
  __shared__ __align__(16) float red[kCtaWarps][2 * kMaxWarps * R];
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int groups = static_cast<int>(blockDim.x >> 5) / wpr;
  for (int i = threadIdx.x; i < kCtaWarps * 2 * kMaxWarps * R; i += blockDim.x) (&red[0][0])[i] = 0.f;
  __syncthreads();
  Place at;
  at.group = warp / wpr;
  at.wpr = wpr;
  at.wig = warp - at.group * wpr;
  at.lane = lane;
  at.vec0 = at.wig * 32 + lane;
  at.vecs = p.n / E;
  at.turn = 0;
  at.red = red[at.group];
  const int n = p.n;
  int rows = p.max_m;
  if (p.m_ptr != nullptr) rows = pdl_wait_row_count(p.m_ptr, p.max_m, 0);
  else pdl_wait();
  auto inside = [&](int j) { return kFull || at.vec0 + j * 32 * wpr < at.vecs; };
  // (a caller may have written the parameters just before: they come behind the wait too)
  Vec16 bias[V], pog[V], pob[V], prg[V], prb[V];
  auto param = [&](const void* src, bool used, Vec16(&dst)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      dst[j] = Vec16{0u, 0u, 0u, 0u};
      if (used && inside(j)) dst[j] = ld_global_v4(static_cast<const T*>(src) + (at.vec0 + j * 32 * wpr) * E);
    }
  };
  const int post_kind = p.post_kind, pre_kind = p.pre_kind, gate_rows = p.gate_rows;
  param(p.bias, p.bias != nullptr, bias);
  param(p.post_gamma, post_kind != kNormNone, pog);
  param(p.post_beta, post_kind == kNormLayer, pob);
  param(p.pre_gamma, pre_kind != kNormNone, prg);
  param(p.pre_beta, pre_kind == kNormLayer, prb);
  const float inv_n = 1.0f / static_cast<float>(n), eps = p.eps;
  const Pair scale = both(p.residual_scale);

  const long long stride = static_cast<long long>(gridDim.x) * groups * R;
  long long row0 = (static_cast<long long>(blockIdx.x) * groups + at.group) * R;
  // This lane's first vector of the first row in work, in bytes, and what lies between rows, vectors and rounds.
  const size_t pitch = static_cast<size_t>(n) * sizeof(T), lead = static_cast<size_t>(at.vec0) * 16;
  const size_t advance = static_cast<size_t>(stride) * pitch;
  const int vec_bytes = 512 * wpr;
  size_t off = static_cast<size_t>(row0) * pitch + lead;
  const char* const gate = p.gate != nullptr ? static_cast<const char*>(p.gate) + lead : nullptr;
  // The next round's vectors are fetched as soon as this round's have been unpacked, into the same registers; the gate
  // rows, through which the gate is found, a round before that.
  Vec16 vx[R][V], vr[R][V], vg[R][V];
  int gate_row[R], gate_next[R];
  auto fetch = [&](const void* base, size_t at_off, long long from, Vec16(&dst)[R][V]) {
    const char* src = static_cast<const char*>(base) + at_off;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (inside(j) && from + r < rows) dst[r][j] = ld_activation_v4(src + r * pitch + j * vec_bytes);
  };
  auto fetch_gate_rows = [&](long long from) {
#pragma unroll
    for (int r = 0; r < R; ++r) gate_next[r] = p.batch_idx != nullptr && from + r < rows ? p.batch_idx[from + r] : 0;
  };
  auto fetch_gate = [&](long long from) {  // and the gate rows of the round behind
#pragma unroll
    for (int r = 0; r < R; ++r) {
      gate_row[r] = gate_next[r];
      if (gate_row[r] >= 0 && gate_row[r] < gate_rows) {
        const char* src = gate + static_cast<size_t>(gate_row[r]) * pitch;
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (inside(j)) vg[r][j] = ld_activation_v4(src + j * vec_bytes);
      }
    }
    fetch_gate_rows(from + stride);
  };
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int j = 0; j < V; ++j) vx[r][j] = vr[r][j] = vg[r][j] = Vec16{0u, 0u, 0u, 0u};  // (zeros behind the row's end)
  fetch(p.x, off, row0, vx);
  if (p.residual != nullptr) fetch(p.residual, off, row0, vr);
  if (gate != nullptr) {
    fetch_gate_rows(row0);
    fetch_gate(row0);
  }
  for (; row0 < rows; row0 += stride, off += advance) {
    Pair v[R][V][P];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      Pair b[P];
      Pairs<T>::unpack(bias[j], b);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        Pairs<T>::unpack(vx[r][j], v[r][j]);
#pragma unroll
        for (int i = 0; i < P; ++i) v[r][j][i] = add2(v[r][j][i], b[i]);
      }
    }
    fetch(p.x, off + advance, row0 + stride, vx);
    if (post_kind != kNormNone) normalise<T, V, R, kFull, kFew>(v, post_kind, pog, pob, inv_n, eps, at);
    if (gate != nullptr) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (gate_row[r] >= 0 && gate_row[r] < gate_rows) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            Pair g[P];
            Pairs<T>::unpack(vg[r][j], g);
#pragma unroll
            for (int i = 0; i < P; ++i) v[r][j][i] = mul2(v[r][j][i], g[i]);
          }
        } else {  // a sequence number outside the gate's rows opens no gate
#pragma unroll
          for (int j = 0; j < V; ++j)
#pragma unroll
            for (int i = 0; i < P; ++i) v[r][j][i] = both(0.f);
        }
      }
      fetch_gate(row0 + stride);
    }
    if (p.residual != nullptr) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          Pair res[P];
          Pairs<T>::unpack(vr[r][j], res);
#pragma unroll
          for (int i = 0; i < P; ++i) v[r][j][i] = fma2(res[i], scale, v[r][j][i]);
        }
      fetch(p.residual, off + advance, row0 + stride, vr);
    }
    auto store = [&](void* base) {
      char* to = static_cast<char*>(base) + off;
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (inside(j) && row0 + r < rows) st_global_v4(to + r * pitch + j * vec_bytes, Pairs<T>::pack(v[r][j]));
    };
    if (p.h != nullptr) store(p.h);
    if (pre_kind != kNormNone) normalise<T, V, R, kFull, kFew>(v, pre_kind, prg, prb, inv_n, eps, at);
    if (p.y != nullptr) store(p.y);
    if (p.y_mx != nullptr) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (row0 + r < rows)
            store_mx<T>(v[r][j], p.y_mx, static_cast<int>(row0) + r, at.vec0 + j * 32 * wpr, n, lane);
    }
  }
}

template <typename T, int V, int R, bool kFull, bool kFew, int kRegs>
cudaError_t launch_full(const GatedNorm& p, int wpr, cudaStream_t stream) {
  auto kernel = gated_norm_kernel<T, V, R, kFull, kFew, kRegs>;
  const int groups = wpr >= kCtaWarps ? 1 : kCtaWarps / wpr, threads = groups * wpr * 32;
  static std::atomic<int> resident[kMaxDevices][kMaxWarps + 1] = {};
  const int dev = current_device();
  int per_sm = dev >= 0 ? resident[dev][wpr].load(std::memory_order_relaxed) : 0;
  if (per_sm == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, 0) != cudaSuccess || per_sm < 1)
      per_sm = 1;
    if (dev >= 0) resident[dev][wpr].store(per_sm, std::memory_order_relaxed);
  }
  const long long rows_per_cta = static_cast<long long>(groups) * R;
  long long ctas = (p.max_m + rows_per_cta - 1) / rows_per_cta;
  const long long cap = static_cast<long long>(sm_count()) * per_sm;
  if (ctas > cap) ctas = cap;
  return launch_pdl(kernel, dim3(static_cast<int>(ctas)), dim3(threads), 0, stream, p, wpr);
}

template <typename T, int V, int R, bool kFew, int kRegs = 128>
cudaError_t launch_rows(const GatedNorm& p, int wpr, cudaStream_t stream) {
  if (p.n == 32 * wpr * V * VecTraits<T>::kElems) return launch_full<T, V, R, true, kFew, kRegs>(p, wpr, stream);
  return launch_full<T, V, R, false, kFew, kRegs>(p, wpr, stream);
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
  int wpr = (vecs + 31) / 32;
  // Few rows: one at a time, so that they spread over the SMs.
  const int route = p.route_rows > 0 ? p.route_rows : p.max_m;
  const bool few_rows = route <= static_cast<long long>(sm_count()) * (wpr >= kCtaWarps ? 1 : kCtaWarps / wpr);
  // One vector a lane and two rows at a time, where 16 warps hold the row; but fp32 rows of eight warps and more leave
  // too few registers for two rows: 13000 rows of 1024 / 1536 / 2048, 47.9 / 61.1 / 107.6 us, and with two vectors a
  // lane 41.9 / 53.6 / 86.3.  (640, where they do not come out even, 27.4 and 32.1; fp16, 4096: 126 and 152.)
  if (wpr <= kMaxWarps && (sizeof(T) == 2 || wpr < 8 || few_rows)) {
    // (up to four warps to a row: without the loop over the further slots, 67.8 us instead of 70.3 at 39778 x 1024 fp16)
    if (wpr <= 4) return few_rows ? launch_rows<T, 1, 1, true>(p, wpr, stream) : launch_rows<T, 1, 2, true>(p, wpr, stream);
    return few_rows ? launch_rows<T, 1, 1, false>(p, wpr, stream) : launch_rows<T, 1, 2, false>(p, wpr, stream);
  }
  wpr = (vecs + 63) / 64;
  if (wpr > kMaxWarps) return cudaErrorInvalidValue;
  if constexpr (sizeof(T) == 4)
    if (wpr <= 4) return launch_rows<T, 2, 1, true>(p, wpr, stream);
  // Two vectors a lane spill with 96 registers (fp32 40 to 96 bytes a thread, fp16 330).  That pays where it brings two CTAs
  // to an SM instead of one, and in full rows, which spill least, of five and six warps (four instead of three, three instead
  // of two); not at seven.  128 / 96 registers, both norms and a gate per sequence, us:
  //   9 and 10 warps: 6699 rows fp32 2080 82 / 66, 2304 80 / 59, 2560 81 / 62; fp16 4608 141 / 91, 5120 147 / 96;
  //   full rows: 13000 rows fp32 1280 57.1 / 55.9, 1536 76 / 70; but 1792 (7 warps) 83 / 94;
  //   others: 1184 58 / 63, 1408 77 / 80, 1664 84 / 106.
  constexpr int kFile = 65536 / 32;
  const int more = kFile / (wpr * 96), few = kFile / (wpr * 128);
  const bool full = p.n == 64 * wpr * E;
  if (more >= 2 * few || (more > few && full && wpr <= 6)) return launch_rows<T, 2, 1, false, 96>(p, wpr, stream);
  return launch_rows<T, 2, 1, false>(p, wpr, stream);
}

template cudaError_t launch_gated_norm<__half>(const GatedNorm&, cudaStream_t);
template cudaError_t launch_gated_norm<float>(const GatedNorm&, cudaStream_t);

}  // namespace etb
