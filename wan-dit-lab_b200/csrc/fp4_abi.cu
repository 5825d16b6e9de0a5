// The extern "C" entry points of the FP4 operators (include/wdl_b200.h): argument validation before any launch.
#include <climits>

#include "../../include/wdl_b200.h"
#include "fp4.cuh"
#include "fp4.h"

namespace wdl {
// Defined in abi.cu (C++ linkage): the per-thread message of wdl_last_error and the current device's error word.
int set_last_error(int code, const char* message);
uint32_t* device_error_word();
}  // namespace wdl

namespace {

using wdl::fp4::block_columns;

int refuse(const char* message) { return wdl::set_last_error(WDL_ERR_ARGUMENT, message); }
int ok() { return wdl::set_last_error(WDL_OK, nullptr); }
int cuda_status(cudaError_t e) {
  return e == cudaSuccess ? ok() : wdl::set_last_error(WDL_ERR_CUDA, cudaGetErrorString(e));
}
bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
bool known_dtype(int d) { return d == WDL_BF16 || d == WDL_F16 || d == WDL_F32; }
int size_of(int d) { return d == WDL_F32 ? 4 : 2; }
bool rows_aligned(const void* p, int64_t ld, int size) { return aligned(p, 16) && (ld * size) % 16 == 0; }

// Rows and columns that leave room for a tile in 32-bit row numbers and for a grid's second dimension.
constexpr int kMostRows = INT_MAX - 65535, kMostColumns = 1 << 26;

// What every FP4 entry point asks of a matrix in this format.
const char* bad_matrix(int M, int K, int fmt) {
  if (M > kMostRows || K > kMostColumns) return "more than 2^31 - 2^16 rows or 2^26 columns";
  if (fmt != WDL_NVFP4 && fmt != WDL_MXFP4) return "unknown FP4 format";
  if (M < 0 || K <= 0 || K % 32 != 0) return "the number of columns must be a positive multiple of 32";
  return nullptr;
}

// Rows of values to be quantized.
const char* bad_source(const void* x, int dtype, int64_t ld, int M, int K) {
  if (!known_dtype(dtype)) return "x must be bf16, f16 or f32";
  if (ld < K) return "ldx must be at least K";
  if (M > 0 && !x) return "x must not be null";
  return M > 0 && !rows_aligned(x, ld, size_of(dtype)) ? "x rows must be 16-byte aligned" : nullptr;
}

}  // namespace

extern "C" {

size_t wdl_fp4_scale_bytes(int M, int K, int format) {
  if (bad_matrix(M, K, format)) return 0;
  return (static_cast<size_t>(M) + 127) / 128 * wdl::fp4::tiles_along(format, K) * wdl::fp4::kTileBytes;
}

int wdl_fp4_quantize_rows(const void* x, int x_dtype, int64_t ldx, int M, int K, int format, const float* tensor_scale,
                          uint8_t* codes, uint8_t* scales, void* stream) {
  if (const char* why = bad_matrix(M, K, format)) return refuse(why);
  if (const char* why = bad_source(x, x_dtype, ldx, M, K)) return refuse(why);
  if (format == WDL_MXFP4 && tensor_scale) return refuse("mxfp4 takes no tensor scale");
  if (M == 0) return ok();
  if (!codes || !scales) return refuse("codes and scales must not be null");
  if (!aligned(codes, 16) || !aligned(scales, 16) || !aligned(tensor_scale, 4))
    return refuse("codes and scales must be 16-byte aligned");
  return cuda_status(wdl::fp4::quantize_rows_launch(x, x_dtype, ldx, M, K, format, tensor_scale, codes, scales,
                                                    static_cast<cudaStream_t>(stream)));
}

int wdl_fp4_dequantize_rows(const uint8_t* codes, const uint8_t* scales, int M, int K, int format,
                            const float* tensor_scale, void* out, int out_dtype, int64_t ldo, void* stream) {
  if (const char* why = bad_matrix(M, K, format)) return refuse(why);
  if (!known_dtype(out_dtype)) return refuse("out must be bf16, f16 or f32");
  if (ldo < K) return refuse("ldo must be at least K");
  if (format == WDL_MXFP4 && tensor_scale) return refuse("mxfp4 takes no tensor scale");
  if (M == 0) return ok();
  if (!codes || !scales || !out) return refuse("codes, scales and out must not be null");
  if (!rows_aligned(out, ldo, size_of(out_dtype))) return refuse("out rows must be 16-byte aligned");
  if (!aligned(codes, 16) || !aligned(scales, 16) || !aligned(tensor_scale, 4))
    return refuse("codes and scales must be 16-byte aligned");
  return cuda_status(wdl::fp4::dequantize_rows_launch(codes, scales, M, K, format, tensor_scale, out, out_dtype, ldo,
                                                      static_cast<cudaStream_t>(stream)));
}

int wdl_fp4_gemm_rows_per_cta(int M, int N, int K, int sms) {
  return M <= 0 || N <= 0 || K <= 0 || sms <= 0 ? -1 : wdl::fp4::gemm_rows_per_cta(M, N, K, sms);
}

static int run_gemm(wdl::fp4::GemmArgs& g, const wdl_fp4_rows* a, const wdl_fp4_rows* w, const float* bias, int M, int N,
                    int K, bool early_w, void* stream) {
  if (!a || !w) return refuse("null operand");
  if (a->format != w->format) return refuse("both operands must be in the same FP4 format");
  if ((static_cast<int64_t>(M) + 127) / 128 * ((static_cast<int64_t>(N) + 15) / 16) > INT_MAX) return refuse("too many tiles");
  if (const char* why = bad_matrix(M, K, a->format)) return refuse(why);
  if (N <= 0 || N > kMostRows) return refuse("N must be positive and at most 2^31 - 2^16");
  if (a->format == WDL_MXFP4 && (a->tensor_scale || w->tensor_scale || g.ep.tout))
    return refuse("mxfp4 takes no tensor scale");
  if (M == 0) return ok();
  if ((!g.raw.p && (!a->codes || !a->scales)) || !w->codes || !w->scales || !g.ep.out) return refuse("null operand pointer");
  if (!aligned(a->codes, 16) || !aligned(a->scales, 16) || !aligned(w->codes, 16) || !aligned(w->scales, 16))
    return refuse("codes and scales must be 16-byte aligned");
  if (!aligned(bias, 4) || !aligned(a->tensor_scale, 4) || !aligned(w->tensor_scale, 4) || !aligned(g.ep.tout, 4))
    return refuse("float32 arguments must be 4-byte aligned");
  g.a = a->codes, g.a_scales = a->scales, g.b = w->codes, g.b_scales = w->scales;
  g.M = M, g.N = N, g.K = K, g.fmt = a->format, g.early_w = early_w;
  g.ep.bias = bias, g.ep.ta = a->tensor_scale, g.ep.tb = w->tensor_scale;
  g.err = wdl::device_error_word();
  if (!g.err) return wdl::set_last_error(WDL_ERR_CUDA, "cannot resolve the device error word");
  const char* why = "";
  if (wdl::fp4::gemm_launch(g, static_cast<cudaStream_t>(stream), &why) != 0)
    return wdl::set_last_error(WDL_ERR_CUDA, why);
  return ok();
}

// The plain output of a product.
static const char* set_output(wdl::fp4::GemmArgs& g, int N, void* out, int out_dtype, int64_t ldo) {
  if (!known_dtype(out_dtype)) return "out must be bf16, f16 or f32";
  if (ldo < N || ldo > INT_MAX) return "ldo must be at least N and below 2^31";
  if (!aligned(out, size_of(out_dtype))) return "out is not aligned to its type";
  g.mode = out_dtype == WDL_BF16 ? wdl::fp4::kEpiBf16 : out_dtype == WDL_F16 ? wdl::fp4::kEpiF16 : wdl::fp4::kEpiF32;
  g.ep.out = out, g.ep.ld_out = static_cast<int>(ldo), g.ep.rows_per_group = 1;
  g.ep.vector = rows_aligned(out, ldo, size_of(out_dtype));
  return nullptr;
}

// The gated residual update as a product's output.
static const char* set_residual(wdl::fp4::GemmArgs& g, int M, int N, const float* gate, int groups, int64_t ld_gate,
                                const float* residual, int64_t ldr, float* out, int64_t ldo) {
  if (ldo < N || ldo > INT_MAX || ldr < N || ldr > INT_MAX) return "ldo and ldr must be at least N and below 2^31";
  if (gate && (groups <= 0 || M % groups != 0)) return "M must be a multiple of the gate's groups";
  if (gate && groups > 1 && (ld_gate < N || ld_gate > INT_MAX)) return "ld_gate must be at least N and below 2^31";
  if (M > 0 && !residual) return "residual must not be null";
  if (!aligned(out, 4) || !aligned(residual, 4) || !aligned(gate, 4)) return "float32 arguments must be 4-byte aligned";
  g.mode = wdl::fp4::kEpiResidual;
  g.ep.out = out, g.ep.ld_out = static_cast<int>(ldo), g.ep.residual = residual, g.ep.ld_res = static_cast<int>(ldr);
  g.ep.gate = gate, g.ep.ld_gate = gate && groups > 1 ? static_cast<int>(ld_gate) : 0;
  g.ep.rows_per_group = gate && M > 0 ? M / groups : 1;
  g.ep.vector = rows_aligned(out, ldo, 4) && rows_aligned(residual, ldr, 4) && rows_aligned(gate, g.ep.ld_gate, 4);
  return nullptr;
}

int wdl_fp4_gemm(const wdl_fp4_rows* a, const wdl_fp4_rows* w, const float* bias, int M, int N, int K, void* out,
                 int out_dtype, int64_t ldo, void* stream) {
  wdl::fp4::GemmArgs g{};
  if (const char* why = set_output(g, N, out, out_dtype, ldo)) return refuse(why);
  return run_gemm(g, a, w, bias, M, N, K, false, stream);
}

int wdl_fp4_gemm_residual(const wdl_fp4_rows* a, const wdl_fp4_rows* w, const float* bias, const float* gate, int groups,
                          int64_t ld_gate, const float* residual, int64_t ldr, int M, int N, int K, float* out,
                          int64_t ldo, void* stream) {
  wdl::fp4::GemmArgs g{};
  if (const char* why = set_residual(g, M, N, gate, groups, ld_gate, residual, ldr, out, ldo)) return refuse(why);
  return run_gemm(g, a, w, bias, M, N, K, false, stream);
}

static const char* set_gelu(wdl::fp4::GemmArgs& g, int M, int N, const float* t, uint8_t* codes, uint8_t* scales) {
  if (N <= 0 || N % 32 != 0) return "the hidden layer's width must be a positive multiple of 32";
  if (M > 0 && (!scales || !aligned(scales, 16) || !aligned(codes, 16)))
    return "codes and scales must be 16-byte aligned and not null";
  g.mode = wdl::fp4::kEpiGelu;
  g.ep.out = codes, g.ep.out_scales = scales, g.ep.tout = t, g.ep.rows_per_group = 1, g.ep.vector = 1;
  return nullptr;
}

int wdl_fp4_gemm_gelu(const wdl_fp4_rows* a, const wdl_fp4_rows* w, const float* bias, int M, int N, int K,
                      const float* out_tensor_scale, uint8_t* codes, uint8_t* scales, void* stream) {
  wdl::fp4::GemmArgs g{};
  if (const char* why = set_gelu(g, M, N, out_tensor_scale, codes, scales)) return refuse(why);
  return run_gemm(g, a, w, bias, M, N, K, false, stream);
}

// A matrix's codes and scales inside a workspace: each rounded up to 256 bytes.
static size_t up256(size_t n) { return (n + 255) / 256 * 256; }
static size_t rows_bytes(int M, int K, int format) {
  return up256(static_cast<size_t>(M) * (K / 2)) + up256(wdl_fp4_scale_bytes(M, K, format));
}
static wdl_fp4_rows place(uint8_t* work, int M, int K, int format, const float* t) {
  return wdl_fp4_rows{work, work + up256(static_cast<size_t>(M) * (K / 2)), t, format};
}

size_t wdl_fp4_linear_workspace(int M, int K, int format) {
  return bad_matrix(M, K, format) || M == 1 ? 0 : rows_bytes(M, K, format);
}

size_t wdl_fp4_gelu_mlp_workspace(int M, int K, int H, int format) {
  return bad_matrix(M, K, format) || bad_matrix(M, H, format) ? 0 : wdl_fp4_linear_workspace(M, K, format) + rows_bytes(M, H, format);
}

// A product with x quantized to w's format: a single row by the product itself, more into `work` first.
static int run_linear(wdl::fp4::GemmArgs& g, const void* x, int x_dtype, int64_t ldx, const float* x_scale,
                      const wdl_fp4_rows* w, const float* bias, int M, int N, int K, uint8_t* work, void* stream) {
  if (M != 1) {
    const wdl_fp4_rows a = place(work, M, K, w->format, x_scale);
    const int st = wdl_fp4_quantize_rows(x, x_dtype, ldx, M, K, w->format, x_scale, const_cast<uint8_t*>(a.codes),
                                         const_cast<uint8_t*>(a.scales), stream);
    return st != WDL_OK ? st : run_gemm(g, &a, w, bias, M, N, K, true, stream);
  }
  if (const char* why = bad_source(x, x_dtype, ldx, M, K)) return refuse(why);
  const wdl_fp4_rows a{nullptr, nullptr, x_scale, w->format};
  g.raw = {x, x_dtype};
  return run_gemm(g, &a, w, bias, M, N, K, false, stream);
}

static const char* bad_workspace(const void* work, size_t bytes, size_t need, int M) {
  if (M <= 0 || need == 0) return nullptr;
  if (!work || !aligned(work, 256)) return "the workspace must be 256-byte aligned and not null";
  return bytes < need ? "the workspace is too small" : nullptr;
}

int wdl_fp4_linear(const void* x, int x_dtype, int64_t ldx, const float* x_scale, const wdl_fp4_rows* w, const float* bias,
                   const float* gate, int groups, int64_t ld_gate, const float* residual, int64_t ldr, int M, int N, int K,
                   void* out, int out_dtype, int64_t ldo, void* workspace, size_t workspace_bytes, void* stream) {
  if (!w) return refuse("null operand");
  if (const char* why = bad_matrix(M, K, w->format)) return refuse(why);
  wdl::fp4::GemmArgs g{};
  const char* why = residual ? set_residual(g, M, N, gate, groups, ld_gate, residual, ldr, static_cast<float*>(out), ldo)
                             : set_output(g, N, out, out_dtype, ldo);
  if (!why && residual && out_dtype != WDL_F32) why = "the residual update writes f32";
  if (!why && !residual && gate) why = "a gate needs a residual";
  if (!why) why = bad_workspace(workspace, workspace_bytes, wdl_fp4_linear_workspace(M, K, w->format), M);
  if (!why && (!out || !w->codes || !w->scales) && M > 0) why = "null operand pointer";
  if (why) return refuse(why);
  return run_linear(g, x, x_dtype, ldx, x_scale, w, bias, M, N, K, static_cast<uint8_t*>(workspace), stream);
}

int wdl_fp4_gelu_mlp(const void* x, int x_dtype, int64_t ldx, const float* x_scale, const wdl_fp4_rows* x_rows,
                     const wdl_fp4_rows* w1, const float* bias1, const float* hidden_scale, const wdl_fp4_rows* w2,
                     const float* bias2, const float* gate, int groups, int64_t ld_gate, const float* residual,
                     int64_t ldr, int M, int H, int N, int K, void* out, int out_dtype, int64_t ldo, void* workspace,
                     size_t workspace_bytes, void* stream) {
  if (!w1 || !w2) return refuse("null operand");
  const int format = w1->format;
  if (const char* why = bad_matrix(M, K, format)) return refuse(why);
  if (const char* why = bad_matrix(M, H, format)) return refuse(why);
  if (w2->format != format || (x_rows && x_rows->format != format)) return refuse("all operands must be in the same FP4 format");
  if ((x != nullptr) == (x_rows != nullptr) && M > 0) return refuse("either x or x_rows must be given");
  wdl::fp4::GemmArgs g1{}, g2{};
  const char* why = residual ? set_residual(g2, M, N, gate, groups, ld_gate, residual, ldr, static_cast<float*>(out), ldo)
                             : set_output(g2, N, out, out_dtype, ldo);
  if (!why && residual && out_dtype != WDL_F32) why = "the residual update writes f32";
  if (!why && !residual && gate) why = "a gate needs a residual";
  const size_t first = x_rows ? 0 : wdl_fp4_linear_workspace(M, K, format);
  if (!why) why = bad_workspace(workspace, workspace_bytes, first + rows_bytes(M, H, format), M);
  if (!why && M > 0 && (!out || !w1->codes || !w1->scales || !w2->codes || !w2->scales)) why = "null operand pointer";
  uint8_t* work = static_cast<uint8_t*>(workspace);
  const wdl_fp4_rows h = place(work + first, M, H, format, hidden_scale);
  if (!why) why = set_gelu(g1, M, H, hidden_scale, const_cast<uint8_t*>(h.codes), const_cast<uint8_t*>(h.scales));
  if (why) return refuse(why);
  const int st = x_rows ? run_gemm(g1, x_rows, w1, bias1, M, H, K, false, stream)
                        : run_linear(g1, x, x_dtype, ldx, x_scale, w1, bias1, M, H, K, work, stream);
  return st != WDL_OK ? st : run_gemm(g2, &h, w2, bias2, M, N, H, true, stream);
}

int wdl_gated_norm(const wdl_gated_norm_args* p, void* stream) {
  if (!p) return refuse("null arguments");
  const wdl_gated_norm_args& a = *p;
  const bool fp4 = a.out == WDL_OUT_NVFP4 || a.out == WDL_OUT_MXFP4;
  if (!fp4 && !known_dtype(a.out)) return refuse("unknown output type");
  if (a.M < 0 || a.K <= 0 || a.K > 16384 || a.K % (fp4 ? 32 : 8) != 0)
    return refuse(fp4 ? "K must be a positive multiple of 32, at most 16384"
                      : "K must be a positive multiple of 8, at most 16384");
  if ((a.x_dtype != WDL_BF16 && a.x_dtype != WDL_F32) || (a.y && a.y_dtype != WDL_BF16 && a.y_dtype != WDL_F32))
    return refuse("x and y must be bf16 or f32");
  if (a.M > kMostRows) return refuse("more than 2^31 - 2^16 rows");
  if (a.groups <= 0 || a.M % a.groups != 0) return refuse("M must be a multiple of the modulation's groups");
  if (!a.y && (a.gate || a.x_out)) return refuse("a gate or an updated stream needs a branch y");
  if (a.tensor_scale && a.out != WDL_OUT_NVFP4) return refuse("only nvfp4 takes a tensor scale");
  if (!(a.eps >= 0.f)) return refuse("eps must not be negative");
  if (a.M == 0) return ok();
  if (!a.x || !a.h || (a.y && !a.x_out) || (fp4 && !a.h_scales)) return refuse("null pointer");
  if (a.ldx < a.K || (a.y && (a.ldy < a.K || a.ldxo < a.K)) || (!fp4 && a.ldh < a.K)) return refuse("a row stride is below K");
  if (!rows_aligned(a.x, a.ldx, size_of(a.x_dtype)) ||
      (a.y && (!rows_aligned(a.y, a.ldy, size_of(a.y_dtype)) || !rows_aligned(a.x_out, a.ldxo, size_of(a.x_dtype)))) ||
      (fp4 ? !aligned(a.h, 16) || !aligned(a.h_scales, 16) : !rows_aligned(a.h, a.ldh, size_of(a.out))))
    return refuse("rows must be 16-byte aligned");
  if (!aligned(a.weight, 16) || !aligned(a.bias, 16) || !rows_aligned(a.gate, a.gate ? a.ld_gate : 0, 4) ||
      !rows_aligned(a.shift, a.shift ? a.ld_shift : 0, 4) || !rows_aligned(a.scale, a.scale ? a.ld_scale : 0, 4) ||
      !aligned(a.tensor_scale, 4))
    return refuse("weight, bias, gate, shift and scale rows must be 16-byte aligned");
  if (a.groups > 1 && ((a.gate && a.ld_gate < a.K) || (a.shift && a.ld_shift < a.K) || (a.scale && a.ld_scale < a.K)))
    return refuse("a modulation row stride is below K");
  wdl::fp4::GatedNormArgs g{};
  g.x = a.x, g.x_dtype = a.x_dtype, g.ldx = a.ldx;
  g.y = a.y, g.y_dtype = a.y ? a.y_dtype : WDL_F32, g.ldy = a.ldy;
  g.gate = a.gate, g.ld_gate = a.ld_gate, g.weight = a.weight, g.bias = a.bias;
  g.shift = a.shift, g.ld_shift = a.ld_shift, g.scale = a.scale, g.ld_scale = a.ld_scale;
  g.M = a.M, g.K = a.K, g.rows_per_group = a.M / a.groups, g.rms = a.rms != 0, g.eps = a.eps;
  g.inverse_k = 1.f / static_cast<float>(a.K);
  g.x_out = a.x_out, g.ldxo = a.ldxo;
  g.out = a.out == WDL_OUT_NVFP4 ? 3 : a.out == WDL_OUT_MXFP4 ? 4 : a.out;
  g.h = a.h, g.ldh = a.ldh, g.h_scales = a.h_scales, g.t = a.tensor_scale;
  return cuda_status(wdl::fp4::gated_norm_launch(g, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
