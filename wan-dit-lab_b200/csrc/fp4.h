// Internal interface of the FP4 kernels (not part of the public C ABI).
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace wdl {
namespace fp4 {

// Launches a kernel that may begin while the one before it on the stream still runs (fp4.cuh).
template <typename Kernel, typename... Args>
inline cudaError_t launch_dependent(Kernel kernel, dim3 grid, int threads, cudaStream_t s, Args... args) {
  cudaLaunchConfig_t c = {};
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  c.gridDim = grid, c.blockDim = dim3(threads), c.stream = s, c.attrs = &at, c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kernel, args...);
}

// x [M, K] (dtype 0 bf16, 1 f16, 2 f32; row stride ldx elements) to codes [M, K / 2] and tiled scales.
cudaError_t quantize_rows_launch(const void* x, int x_dtype, int64_t ldx, int M, int K, int fmt, const float* t,
                                 uint8_t* codes, uint8_t* scales, cudaStream_t s);
cudaError_t dequantize_rows_launch(const uint8_t* codes, const uint8_t* scales, int M, int K, int fmt, const float* t,
                                   void* out, int out_dtype, int64_t ldo, cudaStream_t s);

enum EpilogueMode : int {
  kEpiBf16 = 0,  // out = alpha acc + bias
  kEpiF16 = 1,
  kEpiF32 = 2,
  kEpiResidual = 3,  // out f32 = residual + gate (alpha acc + bias)
  kEpiGelu = 4,      // out codes [M, N / 2] and out_scales: GELU(alpha acc + bias) in the operands' own format
};

// Taken by value as a launch parameter, within 128 bytes (larger blocks ran the W4A4 epilogues far slower).
struct Epilogue {
  void* out;
  uint8_t* out_scales;    // kEpiGelu: tiles of the hidden layer's scales
  const float* bias;      // [N] or null
  const float* gate;      // [groups, ld_gate] or null: row m uses group m / rows_per_group
  const float* residual;  // [M, ld_res]
  const float* ta;        // tensor scales of the operands and of the GELU output (null: 1)
  const float* tb;
  const float* tout;
  int ld_out, ld_res, ld_gate, rows_per_group;
  int vector;  // every row of out, residual and gate can be read and written 16 bytes at a time (kEpiGelu: 1)
};
static_assert(sizeof(Epilogue) <= 128, "the epilogue parameter block must stay within 128 bytes");

// A row that a product takes as it is and quantizes itself (p null: none).
struct RawRow {
  const void* p;
  int dtype;  // 0 bf16, 1 f16, 2 f32
};

struct GemmArgs {
  RawRow raw;               // M 1: instead of a and a_scales
  const uint8_t* a;         // [M, K / 2] codes
  const uint8_t* a_scales;  // tiles
  const uint8_t* b;         // [N, K / 2]
  const uint8_t* b_scales;
  int M, N, K, fmt, mode;
  bool early_w;  // the kernel before this one on the stream is this library's and writes a: w may be read before it ends
  Epilogue ep;
  uint32_t* err;
};
// Rows of a that one CTA of the few-row kernel takes, 0 for the many-row kernel (which does not split K).
int gemm_rows_per_cta(int M, int N, int K, int sms);
// Validated by the caller. 0, or nonzero with *why set.
int gemm_launch(const GemmArgs& a, cudaStream_t s, const char** why);

struct GatedNormArgs {
  const void* x;  // [M, ldx] the stream, bf16 or f32
  int x_dtype;
  int64_t ldx;
  const void* y;  // [M, ldy] the branch (nullable: no update), bf16 or f32
  int y_dtype;
  int64_t ldy;
  const float* gate;  // [groups, ld_gate] (nullable: 1)
  int64_t ld_gate;
  const float* weight;  // [K] (nullable)
  const float* bias;    // [K] (nullable)
  const float* shift;   // [groups, ld_shift] (nullable)
  int64_t ld_shift;
  const float* scale;  // [groups, ld_scale] (nullable)
  int64_t ld_scale;
  int M, K, rows_per_group, rms;
  float eps, inverse_k;  // inverse_k: 1 / K, rounded to nearest
  void* x_out;  // [M, ldxo] the updated stream (null without a branch)
  int64_t ldxo;
  int out;   // 0 bf16, 1 f16, 2 f32, 3 nvfp4, 4 mxfp4
  void* h;   // [M, ldh] (codes [M, K / 2])
  int64_t ldh;
  uint8_t* h_scales;  // FP4: tiles
  const float* t;     // nvfp4: the tensor scale (null: 1)
};
cudaError_t gated_norm_launch(const GatedNormArgs& a, cudaStream_t s);

}  // namespace fp4
}  // namespace wdl
