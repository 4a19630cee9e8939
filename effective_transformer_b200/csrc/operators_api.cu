// C ABI of the 4-bit projections and of the norms around a block (include/et_b200.h): argument checks and dispatch.
#include "../../include/et_b200.h"

#include "common.cuh"
#include "mxfp4.cuh"

using namespace etb;

namespace {

constexpr char kAlignment[] = "pointers must be 16-byte aligned, those of MXFP4 tensors 128-byte aligned";
constexpr char kElementAlignment[] =
    "m_ptr, batch_idx and status_word must be 4-byte aligned, w aligned to its elements";

int refuse(const char* msg) {
  set_global_error(msg);
  return ET_INVALID_ARGUMENT;
}

int status_of(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return ET_OK;
  set_global_error(std::string(what) + ": " + cudaGetErrorString(e));
  return e == cudaErrorInvalidValue || e == cudaErrorMisalignedAddress ? ET_INVALID_ARGUMENT : ET_CUDA_ERROR;
}

// No C++ exception crosses the boundary (the error texts allocate).
template <typename F>
int guarded(F f) {
  try {
    return f();
  } catch (...) {
    return ET_CUDA_ERROR;
  }
}

bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }
bool misaligned_mx(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 127u) != 0; }
// (an access through a pointer that its type does not allow is a fault on the GPU)
bool misaligned_to(const void* p, size_t size) { return reinterpret_cast<uintptr_t>(p) % size != 0; }
bool known_dtype(int dtype) { return dtype == ET_FP16 || dtype == ET_FP32; }
size_t size_of(int dtype) { return dtype == ET_FP16 ? 2 : 4; }
// Bytes from the first to behind the last value of `rows` rows (at least one).
size_t rows_size(int dtype, int rows, long long row_stride, int k) {
  return (static_cast<size_t>(rows - 1) * row_stride + k) * size_of(dtype);
}

int check_width(int k) {
  if (k <= 0 || k % kMxBlock != 0) return refuse("the width of an MXFP4 row must be a positive multiple of 32");
  return ET_OK;
}

// (an empty batch passes here: its tensors may have no address)
int check_gemm(int dtype, const void* a, const void* w_mx, const void* bias, const void* residual, const void* c,
               const void* c_mx, const int* m_ptr, const int* status_word, int max_m, int n, int k, int epilogue) {
  if (!known_dtype(dtype)) return refuse("dtype must be ET_FP16 or ET_FP32");
  if (int rc = check_width(k)) return rc;
  if (max_m < 0 || n <= 0 || n % 32 != 0) return refuse("max_m must not be negative, n a positive multiple of 32");
  if (epilogue < kEpiNone || epilogue > kEpiBiasTanh) return refuse("epilogue must be 0 to 3");
  if (max_m == 0) return ET_OK;
  if ((c == nullptr) == (c_mx == nullptr)) return refuse("exactly one of c and c_mx must be given");
  if (c_mx != nullptr && (n % 64 != 0 || residual != nullptr))
    return refuse("MXFP4 output needs n a multiple of 64 and takes no residual");
  if (a == nullptr || w_mx == nullptr || (epilogue != kEpiNone && bias == nullptr)) return refuse("null pointer");
  if (misaligned(a) || misaligned(bias) || misaligned(residual) || misaligned(c) || misaligned_mx(w_mx) || misaligned_mx(c_mx))
    return refuse(kAlignment);
  if (misaligned_to(m_ptr, sizeof(int)) || misaligned_to(status_word, sizeof(int))) return refuse(kElementAlignment);
  return ET_OK;
}

// The result may be the residual (every element is read where it is written), and nothing else.
int check_result(int dtype, const void* w_mx, const void* bias, const void* residual, const void* c, const void* c_mx,
                 const void* rows_mx, int max_m, int n, int k) {
  const size_t elem = size_of(dtype), c_size = static_cast<size_t>(max_m) * n * elem;
  const void* out = c != nullptr ? c : c_mx;
  const size_t size = c != nullptr ? c_size : mx_bytes(max_m, n);
  if (overlap(out, size, rows_mx, mx_bytes(max_m, k)) || overlap(out, size, w_mx, mx_bytes(n, k)) ||
      overlap(out, size, bias, n * elem) || (residual != c && overlap(out, size, residual, c_size)))
    return refuse("the result must not overlap an operand, except that c may be the residual");
  return ET_OK;
}

MxGemm gemm_of(const void* a_mx, const void* w_mx, void* c_mx, const int* m_ptr, int max_m, int n, int k,
               int* status_word) {
  MxGemm g;
  g.a = a_mx, g.w = w_mx, g.c_mx = c_mx;
  g.m_ptr = m_ptr, g.max_m = max_m, g.n = n, g.k = k;
  g.status_word = status_word;
  return g;
}

template <typename T>
int run_gemm(const MxGemm& g, const void* bias, const void* residual, void* c, int epilogue, cudaStream_t s) {
  return status_of(launch_gemm_mxfp4<T>(g, static_cast<const T*>(bias), static_cast<const T*>(residual),
                                        static_cast<T*>(c), epilogue, s),
                   "et_mxfp4_gemm");
}

template <typename T>
int run_linear(const MxGemm& g, const void* x, long long row_stride, void* x_mx, const void* bias, const void* residual,
               void* c, int epilogue, cudaStream_t s) {
  return status_of(launch_linear_mxfp4<T>(g, static_cast<const T*>(x), row_stride, x_mx, static_cast<const T*>(bias),
                                          static_cast<const T*>(residual), static_cast<T*>(c), epilogue, s),
                   "et_mxfp4_linear");
}

int run_quantize(int dtype, const void* x, long long row_stride, const int* m_ptr, int max_m, int k, void* mx,
                 cudaStream_t s) {
  if (dtype == ET_FP16)
    return status_of(launch_mx_quantize<__half>(static_cast<const __half*>(x), row_stride, m_ptr, max_m, k, mx, s),
                     "et_mxfp4_quantize");
  return status_of(launch_mx_quantize<float>(static_cast<const float*>(x), row_stride, m_ptr, max_m, k, mx, s),
                   "et_mxfp4_quantize");
}

}  // namespace

extern "C" {

size_t et_mxfp4_bytes(int rows, int k) {
  if (rows < 0 || k <= 0 || k % kMxBlock != 0) return 0;
  return mx_bytes(rows, k);
}

int et_mxfp4_quantize(int dtype, const void* x, long long row_stride, const int* m_ptr, int max_m, int k, void* mx,
                      void* stream) {
  return guarded([&] {
    if (!known_dtype(dtype)) return refuse("dtype must be ET_FP16 or ET_FP32");
    if (int rc = check_width(k)) return rc;
    if (max_m < 0 || row_stride < k || row_stride * size_of(dtype) % 16 != 0)
      return refuse("max_m must not be negative, row_stride at least k and a multiple of 16 bytes");
    if (max_m == 0) return static_cast<int>(ET_OK);
    if (x == nullptr || mx == nullptr) return refuse("null pointer");
    if (misaligned(x) || misaligned_mx(mx)) return refuse(kAlignment);
    if (misaligned_to(m_ptr, sizeof(int))) return refuse(kElementAlignment);
    if (overlap(x, rows_size(dtype, max_m, row_stride, k), mx, mx_bytes(max_m, k)))
      return refuse("x and mx must not overlap");
    return run_quantize(dtype, x, row_stride, m_ptr, max_m, k, mx, static_cast<cudaStream_t>(stream));
  });
}

int et_mxfp4_dequantize(int dtype, const void* mx, const int* m_ptr, int max_m, int k, void* out, void* stream) {
  return guarded([&] {
    if (!known_dtype(dtype)) return refuse("dtype must be ET_FP16 or ET_FP32");
    if (int rc = check_width(k)) return rc;
    if (max_m < 0) return refuse("max_m must not be negative");
    if (max_m == 0) return static_cast<int>(ET_OK);
    if (mx == nullptr || out == nullptr) return refuse("null pointer");
    if (misaligned_mx(mx) || misaligned(out)) return refuse(kAlignment);
    if (misaligned_to(m_ptr, sizeof(int))) return refuse(kElementAlignment);
    if (overlap(mx, mx_bytes(max_m, k), out, rows_size(dtype, max_m, k, k)))
      return refuse("mx and out must not overlap");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == ET_FP16)
      return status_of(launch_mx_dequantize<__half>(mx, m_ptr, max_m, k, static_cast<__half*>(out), s),
                       "et_mxfp4_dequantize");
    return status_of(launch_mx_dequantize<float>(mx, m_ptr, max_m, k, static_cast<float*>(out), s),
                     "et_mxfp4_dequantize");
  });
}

int et_mxfp4_pack_weight(int dtype, const void* w, void* w_mx, int k, int n, void* stream) {
  return guarded([&] {
    if (!known_dtype(dtype)) return refuse("dtype must be ET_FP16 or ET_FP32");
    if (int rc = check_width(k)) return rc;
    if (n <= 0 || n % 32 != 0) return refuse("n must be a positive multiple of 32");
    if (w == nullptr || w_mx == nullptr) return refuse("null pointer");
    if (misaligned_mx(w_mx)) return refuse(kAlignment);
    if (misaligned_to(w, size_of(dtype))) return refuse(kElementAlignment);
    if (overlap(w, rows_size(dtype, k, n, n), w_mx, mx_bytes(n, k))) return refuse("w and w_mx must not overlap");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == ET_FP16)
      return status_of(launch_mx_pack_weight<__half>(static_cast<const __half*>(w), w_mx, k, n, s),
                       "et_mxfp4_pack_weight");
    return status_of(launch_mx_pack_weight<float>(static_cast<const float*>(w), w_mx, k, n, s), "et_mxfp4_pack_weight");
  });
}

int et_mxfp4_gemm(int dtype, const void* a_mx, const void* w_mx, const void* bias, const void* residual, void* c,
                  void* c_mx, const int* m_ptr, int max_m, int n, int k, int epilogue, int* status_word, void* stream) {
  return guarded([&] {
    if (int rc = check_gemm(dtype, a_mx, w_mx, bias, residual, c, c_mx, m_ptr, status_word, max_m, n, k, epilogue)) return rc;
    if (max_m == 0) return static_cast<int>(ET_OK);
    if (misaligned_mx(a_mx)) return refuse(kAlignment);
    if (int rc = check_result(dtype, w_mx, bias, residual, c, c_mx, a_mx, max_m, n, k)) return rc;
    const MxGemm g = gemm_of(a_mx, w_mx, c_mx, m_ptr, max_m, n, k, status_word);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return dtype == ET_FP16 ? run_gemm<__half>(g, bias, residual, c, epilogue, s)
                            : run_gemm<float>(g, bias, residual, c, epilogue, s);
  });
}

int et_mxfp4_linear(int dtype, const void* x, long long row_stride, void* x_mx, const void* w_mx, const void* bias,
                    const void* residual, void* c, void* c_mx, const int* m_ptr, int max_m, int n, int k, int epilogue,
                    int* status_word, void* stream) {
  return guarded([&] {
    if (int rc = check_gemm(dtype, x, w_mx, bias, residual, c, c_mx, m_ptr, status_word, max_m, n, k, epilogue)) return rc;
    if (row_stride < k || row_stride * size_of(dtype) % 16 != 0)
      return refuse("row_stride must be at least k and a multiple of 16 bytes");
    if (max_m == 0) return static_cast<int>(ET_OK);
    if (x_mx == nullptr || misaligned_mx(x_mx)) return refuse("x_mx must be 128-byte aligned device memory");
    if (int rc = check_result(dtype, w_mx, bias, residual, c, c_mx, x_mx, max_m, n, k)) return rc;
    const size_t elem = size_of(dtype), mx_size = mx_bytes(max_m, k);
    if (overlap(x_mx, mx_size, x, rows_size(dtype, max_m, row_stride, k)) ||
        overlap(x_mx, mx_size, w_mx, mx_bytes(n, k)) || overlap(x_mx, mx_size, bias, n * elem) ||
        overlap(x_mx, mx_size, residual, static_cast<size_t>(max_m) * n * elem))
      return refuse("x_mx must not overlap an operand");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const MxGemm g = gemm_of(nullptr, w_mx, c_mx, m_ptr, max_m, n, k, status_word);
    return dtype == ET_FP16 ? run_linear<__half>(g, x, row_stride, x_mx, bias, residual, c, epilogue, s)
                            : run_linear<float>(g, x, row_stride, x_mx, bias, residual, c, epilogue, s);
  });
}

int et_mxfp4_route(int dtype, int rows, int n, int k, int* tile_m, int* tile_n, int* one_kernel) {
  return guarded([&] {
    if (!known_dtype(dtype)) return refuse("dtype must be ET_FP16 or ET_FP32");
    if (int rc = check_width(k)) return rc;
    if (rows <= 0 || n <= 0 || n % 32 != 0) return refuse("rows must be positive, n a positive multiple of 32");
    if (!tile_m || !tile_n || !one_kernel) return refuse("null pointer");
    const bool pair = mxfp4_route(dtype == ET_FP32, rows, n, k) == kMxPair;
    *tile_m = pair ? 256 : 128;
    *tile_n = pair ? 192 : 128;
    *one_kernel = mxfp4_rows_supported(rows, n, k) ? 1 : 0;
    return static_cast<int>(ET_OK);
  });
}

int et_gated_residual_norm(int dtype, const et_gated_norm_param_t* p, void* stream) {
  return guarded([&] {
    if (!known_dtype(dtype)) return refuse("dtype must be ET_FP16 or ET_FP32");
    if (p == nullptr) return refuse("null pointer");
    const int elems = dtype == ET_FP16 ? 8 : 4;
    if (p->max_m < 0 || p->n <= 0 || p->n % elems != 0)
      return refuse("max_m must not be negative, n a positive multiple of 16 bytes");
    if (p->n > 32 * 8 * 4 * elems) return refuse("n is limited to 8192 (ET_FP16) and 4096 (ET_FP32)");
    if (p->post_norm < ET_NORM_NONE || p->post_norm > ET_NORM_RMS || p->pre_norm < ET_NORM_NONE ||
        p->pre_norm > ET_NORM_RMS)
      return refuse("post_norm and pre_norm must be ET_NORM_NONE, ET_NORM_LAYER or ET_NORM_RMS");
    if ((p->post_norm != ET_NORM_NONE && !p->post_gamma) || (p->post_norm == ET_NORM_LAYER && !p->post_beta) ||
        (p->pre_norm != ET_NORM_NONE && !p->pre_gamma) || (p->pre_norm == ET_NORM_LAYER && !p->pre_beta))
      return refuse("a norm needs its gamma, a LayerNorm its beta too");
    if (p->max_m == 0) return static_cast<int>(ET_OK);  // (an empty batch's tensors may have no address)
    if (!p->h_out && !p->y_out && !p->y_mx) return refuse("at least one of h_out, y_out and y_mx must be given");
    if (p->y_mx != nullptr && p->n % kMxBlock != 0) return refuse("y_mx needs n a multiple of 32");
    if (p->gate != nullptr && (p->gate_rows < 1 || (p->gate_rows > 1 && !p->batch_idx)))
      return refuse("gate needs gate_rows >= 1, and batch_idx with more than one row");
    if (p->x == nullptr) return refuse("null pointer");
    for (const void* q : {p->x, p->bias, p->residual, p->gate, p->post_gamma, p->post_beta, p->pre_gamma, p->pre_beta,
                          static_cast<const void*>(p->h_out), static_cast<const void*>(p->y_out)})
      if (misaligned(q)) return refuse(kAlignment);
    if (misaligned_mx(p->y_mx)) return refuse(kAlignment);
    if (misaligned_to(p->m_ptr, sizeof(int)) ||
        (p->gate != nullptr && p->gate_rows > 1 && misaligned_to(p->batch_idx, sizeof(int))))
      return refuse(kElementAlignment);
    {
      // every element of x and residual is read where h and y are written, nothing else is
      const size_t row = p->n * size_of(dtype), all = p->max_m * row;
      const struct { const void* at; size_t size; } outs[] = {
          {p->h_out, all}, {p->y_out, all}, {p->y_mx, p->y_mx != nullptr ? mx_bytes(p->max_m, p->n) : 0}};
      for (int i = 0; i < 3; ++i) {
        const auto& o = outs[i];
        bool bad = false;
        for (const void* q : {p->x, p->residual}) bad = bad || ((q != o.at || i == 2) && overlap(o.at, o.size, q, all));
        for (const void* q : {p->bias, p->post_gamma, p->post_beta, p->pre_gamma, p->pre_beta})
          bad = bad || overlap(o.at, o.size, q, row);
        bad = bad || overlap(o.at, o.size, p->gate, static_cast<size_t>(p->gate_rows) * row) ||
              (p->gate_rows > 1 && overlap(o.at, o.size, p->batch_idx, p->max_m * sizeof(int)));
        for (int j = 0; j < i; ++j) bad = bad || overlap(o.at, o.size, outs[j].at, outs[j].size);
        if (bad) return refuse("outputs must not overlap each other or an input, except that h_out or y_out may be x or residual");
      }
    }
    GatedNorm g;
    g.x = p->x, g.bias = p->bias, g.residual = p->residual, g.gate = p->gate;
    g.batch_idx = p->gate_rows > 1 ? p->batch_idx : nullptr;
    g.gate_rows = p->gate_rows;
    g.residual_scale = p->residual_scale;
    g.eps = p->eps > 0.f ? p->eps : 1e-6f;
    g.post_kind = p->post_norm, g.pre_kind = p->pre_norm;
    g.post_gamma = p->post_gamma, g.post_beta = p->post_beta, g.pre_gamma = p->pre_gamma, g.pre_beta = p->pre_beta;
    g.h = p->h_out, g.y = p->y_out, g.y_mx = p->y_mx;
    g.m_ptr = p->m_ptr, g.max_m = p->max_m, g.n = p->n;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return dtype == ET_FP16 ? status_of(launch_gated_norm<__half>(g, s), "et_gated_residual_norm")
                            : status_of(launch_gated_norm<float>(g, s), "et_gated_residual_norm");
  });
}

}  // extern "C"
