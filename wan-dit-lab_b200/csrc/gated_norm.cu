// The gated residual update of a block and the normalization that follows it, in one pass over the row:
//
//   x' = x + gate y                                            stored in the stream's type, and read as stored by
//   u  = (x' - mean x') / sqrt(var x' + eps)                   LayerNorm, or x' / sqrt(mean x'^2 + eps)
//   h  = (u weight + bias) (1 + scale) + shift                 as bf16, f16, f32, or codes and scales in FP4 (fp4.cuh)
//
// gate, shift and scale are rows [groups, K]: row m of x takes group m / rows_per_group (a modulation per frame).
// A CTA takes neighbouring rows; a row lies in its registers (8 columns a thread and chunk) between the statistics and
// the output, and the next row's x and y are on their way meanwhile. Up to 4096 columns (one chunk) the modulation stays
// in registers as well, until the group changes: read again for every row it was three quarters of the L1 traffic, which
// bound the kernel. Bytes: x and y read once, x' and h written once.
//
// Every step is one float32 operation, rounded to nearest (gate y, then the sum; the division by the root, not a product
// with its inverse). Of the two statistics only the sums of 64 columns are float32 (of 8 in rows of several chunks), the sums
// of these are float64: a statistic's error before its own rounding is at most 6 (3) half steps of float32 relative to the
// mean magnitude of what it adds, and mostly a fraction of one, since the parts' errors differ. A value of h next to a border
// of the FP4 codes falls to one side or the other by its last bit, and an error of the row's statistics moves all of the
// row's values.
//
// What bounds it: instructions and the chain of two reductions a row, not HBM, at the block widths. Measured on a B200 with
// gate, LayerNorm and modulation, rows of 3072: 1392 rows (x float32, y bf16) into NVFP4 14.3 us; 7040 rows (bf16, 8 groups)
// into bf16 42.3 us, 4.1 TB/s, 62 % of the issue slots. Without the reductions these are 11.3 and 36.9, without the FP4
// store the first is 12.0. Slower: sums in float64 from the threads on (14.7 us for the first), three or four CTAs an SM
// with fewer registers (19.8, 24), 192 or 128 threads a row with two or three chunks each (16.4, 18.4; the second 45.7 at
// best), the modulation in shared memory (15.0), rows through a ring of bulk copies in shared memory (15.0 and 46.8). Rows of
// several chunks read the modulation again for each row: 1392 rows of 5120 into NVFP4 37.5 us, 4224 of them (bf16) into bf16
// 62.8 us, 2.8 TB/s; 700 rows of 16384 (bf16) into bf16 32.3 us, 2.8 TB/s.
#include <atomic>
#include <type_traits>

#include "fp4.cuh"
#include "fp4.h"

namespace wdl {
namespace fp4 {
namespace {

// 8 values as they lie in memory, and as four pairs of float32.
template <typename T>
struct Raw {
  uint4 w[sizeof(T) / 2];
};
struct Eight {
  uint64_t p[4];
};
template <typename T>
__device__ __forceinline__ Raw<T> load_raw(const T* p) {
  Raw<T> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.w[i] = reinterpret_cast<const uint4*>(p)[i];
  return r;
}
__device__ __forceinline__ uint64_t join(uint32_t lo, uint32_t hi) { return pack2(__uint_as_float(lo), __uint_as_float(hi)); }
template <typename T>
__device__ __forceinline__ Eight values(const Raw<T>& r) {
  if constexpr (sizeof(T) == 4) {
    return {join(r.w[0].x, r.w[0].y), join(r.w[0].z, r.w[0].w), join(r.w[1].x, r.w[1].y), join(r.w[1].z, r.w[1].w)};
  } else {
    const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
    Eight v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v.p[i] = join(w[i] << 16, w[i] & 0xFFFF0000u);
    return v;
  }
}
__device__ __forceinline__ Eight load8(const float* p) {
  const ulonglong2 a = __ldg(reinterpret_cast<const ulonglong2*>(p)), b = __ldg(reinterpret_cast<const ulonglong2*>(p + 4));
  return {a.x, a.y, b.x, b.y};
}
__device__ __forceinline__ uint32_t bf16_pair(uint64_t v) {
  float a, b;
  unpack2(v, a, b);
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t f16_pair(uint64_t v) {
  float a, b;
  unpack2(v, a, b);
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void store8(float* p, const Eight& v) {
  reinterpret_cast<ulonglong2*>(p)[0] = make_ulonglong2(v.p[0], v.p[1]);
  reinterpret_cast<ulonglong2*>(p)[1] = make_ulonglong2(v.p[2], v.p[3]);
}

// The CTA's sum over the row, in a fixed order, rounded to float32 and divided by K. part: a thread's 8 columns in float32,
// which 8 threads add up to 64 of them, or the float64 sum of its chunks. red: one number a warp, not the array of the call
// before.
template <int kWarps, typename Sum>
__device__ __forceinline__ float block_mean(Sum part, double* red, float K, float inverse_k) {
  constexpr int kFirst = sizeof(Sum) == 4 ? 8 : 1;
#pragma unroll
  for (int o = 1; o < kFirst; o *= 2) part += __shfl_xor_sync(0xFFFFFFFFu, part, o);
  double v = part;
#pragma unroll
  for (int o = kFirst; o < 32; o *= 2) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double s[kWarps];
#pragma unroll
  for (int i = 0; i < kWarps; ++i) s[i] = red[i];
#pragma unroll
  for (int w = 1; w < kWarps; w *= 2)  // pairwise
#pragma unroll
    for (int i = 0; i + w < kWarps; i += 2 * w) s[i] += s[i + w];
  const float sum = static_cast<float>(s[0]);
  // the short division makes a NaN of an infinity (and of sums below 2^-100 a quotient one bit off)
  return fabsf(sum) < INFINITY ? div_rn_by(sum, K, inverse_k) : sum;
}

__device__ __forceinline__ float sum8(const Eight& v) {
  float a, b;
  unpack2(add2(add2(v.p[0], v.p[1]), add2(v.p[2], v.p[3])), a, b);
  return a + b;
}
__device__ __forceinline__ float squares8(const Eight& v) {
  float a, b;
  unpack2(add2(fma2(v.p[1], v.p[1], mul2(v.p[0], v.p[0])), fma2(v.p[3], v.p[3], mul2(v.p[2], v.p[2]))), a, b);
  return a + b;
}

// Codes of this thread's 8 columns k .. k + 7 (a block is 2 or 4 neighbouring threads); every lane calls it.
template <int kFmt>
__device__ __forceinline__ void store_fp4(const GatedNormArgs& a, int m, int k, bool valid, const Eight& e) {
  float v[8], amax = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) unpack2(e.p[i], v[2 * i], v[2 * i + 1]);
  if (valid) {
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = max_nan(amax, fabsf(v[i]));
  }
#pragma unroll
  for (int o = 1; o < block_columns(kFmt) / 8; o *= 2) amax = max_nan(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
  const int bt = tiles_along(kFmt, a.K), b = k / block_columns(kFmt);
  const BlockScale sc = block_scale<kFmt>(amax, a.t ? __ldg(a.t) : 1.f);
  if (valid) {
    *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.h) + static_cast<int64_t>(m) * (a.K / 2) + k / 2) =
        encode8<kFmt>(v, sc);
    if (k % block_columns(kFmt) == 0) a.h_scales[scale_offset(m, b, bt)] = static_cast<uint8_t>(sc.byte);
  } else if (k % block_columns(kFmt) == 0 && b < bt * 4) {
    a.h_scales[scale_offset(m, b, bt)] = 0;  // the last tile's padding blocks
  }
}

template <typename TX, typename TY, int kThreads, int kChunks>
__global__ void __launch_bounds__(kThreads) gated_norm_kernel(const GatedNormArgs a) {
  constexpr int kWarps = kThreads / 32;
  using Sum = std::conditional_t<kChunks == 1, float, double>;
  __shared__ double red[3][kWarps];  // in turn: two sums a row, so that none is written again before all have read it
  grid_dependency_wait();
  grid_dependents_launch();
  const int t = threadIdx.x, K = a.K;
  const float k_float = static_cast<float>(K);
  Raw<TX> rx[kChunks];
  Raw<TY> ry[kChunks];
  auto fetch = [&](int m) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int k = (c * kThreads + t) * 8;
      if (k >= K) continue;
      rx[c] = load_raw(static_cast<const TX*>(a.x) + static_cast<int64_t>(m) * a.ldx + k);
      if (a.y) ry[c] = load_raw(static_cast<const TY*>(a.y) + static_cast<int64_t>(m) * a.ldy + k);
    }
  };
  // gate, 1 + scale and shift of a chunk; `kept`: of the one chunk, for as long as the group lasts
  struct Modulation {
    Eight gate, scale, shift;
  };
  auto modulation = [&](int64_t group, int k) {
    Modulation w = {};
    if (k >= K) return w;
    if (a.gate) w.gate = load8(a.gate + group * a.ld_gate + k);
    if (a.scale) {
      w.scale = load8(a.scale + group * a.ld_scale + k);
#pragma unroll
      for (int i = 0; i < 4; ++i) w.scale.p[i] = add2(pack2(1.f, 1.f), w.scale.p[i]);
    }
    if (a.shift) w.shift = load8(a.shift + group * a.ld_shift + k);
    return w;
  };
  const int per = (a.M + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
  const int first = blockIdx.x * per, last = min(a.M, first + per);
  if (first >= last) return;
  fetch(first);
  int group = a.rows_per_group < a.M ? first / a.rows_per_group : 0;
  int64_t group_end = static_cast<int64_t>(group + 1) * a.rows_per_group;
  Modulation kept = modulation(group, t * 8);
  int turn = 0;
  for (int m = first; m < last; ++m) {
    if (m >= group_end) {
      ++group, group_end += a.rows_per_group;
      if (kChunks == 1) kept = modulation(group, t * 8);
    }
    Eight v[kChunks];
    Sum s = 0;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int k = (c * kThreads + t) * 8;
      if (k >= K) continue;
      v[c] = values(rx[c]);
      if (a.y) {
        Eight y = values(ry[c]);
        if (a.gate) {
          const Eight g = kChunks == 1 ? kept.gate : load8(a.gate + static_cast<int64_t>(group) * a.ld_gate + k);
#pragma unroll
          for (int i = 0; i < 4; ++i) y.p[i] = mul2(g.p[i], y.p[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) v[c].p[i] = add2(v[c].p[i], y.p[i]);
        TX* out = static_cast<TX*>(a.x_out) + static_cast<int64_t>(m) * a.ldxo + k;
        if constexpr (sizeof(TX) == 2) {
          Raw<TX> r;
          r.w[0] = make_uint4(bf16_pair(v[c].p[0]), bf16_pair(v[c].p[1]), bf16_pair(v[c].p[2]), bf16_pair(v[c].p[3]));
          *reinterpret_cast<uint4*>(out) = r.w[0];
          v[c] = values(r);
        } else {
          store8(out, v[c]);
        }
      }
      s += a.rms ? squares8(v[c]) : sum8(v[c]);
    }
    if (m + 1 < last) fetch(m + 1);
    float var = block_mean<kWarps>(s, red[turn], k_float, a.inverse_k);
    turn = turn == 2 ? 0 : turn + 1;
    if (!a.rms) {
      const uint64_t minus = pack2(-var, -var);
      s = 0;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        if ((c * kThreads + t) * 8 >= K) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[c].p[i] = add2(v[c].p[i], minus);
        s += squares8(v[c]);
      }
      var = block_mean<kWarps>(s, red[turn], k_float, a.inverse_k);
      turn = turn == 2 ? 0 : turn + 1;
    }
    const float root = __fsqrt_rn(__fadd_rn(var, a.eps)), inverse = __frcp_rn(root);
    // the short division (div_rn_by, two at a time) is exact here: beyond these bounds a quotient or its remainder could
    // leave float32's normal range
    const bool plain = root >= 0x1p-60f && root <= 0x1p60f;
    const uint64_t r2 = pack2(inverse, inverse), minus_root = pack2(-root, -root);
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int k = (c * kThreads + t) * 8;
      const bool valid = k < K;
      if (valid) {
        if (plain) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint64_t q = mul2(v[c].p[i], r2);
            v[c].p[i] = fma2(fma2(q, minus_root, v[c].p[i]), r2, q);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float lo, hi;
            unpack2(v[c].p[i], lo, hi);
            v[c].p[i] = pack2(__fdiv_rn(lo, root), __fdiv_rn(hi, root));
          }
        }
        if (a.weight) {
          const Eight p = load8(a.weight + k);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[c].p[i] = mul2(v[c].p[i], p.p[i]);
        }
        if (a.bias) {
          const Eight p = load8(a.bias + k);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[c].p[i] = add2(v[c].p[i], p.p[i]);
        }
        const Modulation w = kChunks == 1 ? kept : modulation(group, k);
        if (a.scale) {
#pragma unroll
          for (int i = 0; i < 4; ++i) v[c].p[i] = mul2(v[c].p[i], w.scale.p[i]);
        }
        if (a.shift) {
#pragma unroll
          for (int i = 0; i < 4; ++i) v[c].p[i] = add2(v[c].p[i], w.shift.p[i]);
        }
        const int64_t at = static_cast<int64_t>(m) * a.ldh + k;
        if (a.out == 0)
          *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.h) + at) =
              make_uint4(bf16_pair(v[c].p[0]), bf16_pair(v[c].p[1]), bf16_pair(v[c].p[2]), bf16_pair(v[c].p[3]));
        else if (a.out == 1)
          *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.h) + at) =
              make_uint4(f16_pair(v[c].p[0]), f16_pair(v[c].p[1]), f16_pair(v[c].p[2]), f16_pair(v[c].p[3]));
        else if (a.out == 2)
          store8(static_cast<float*>(a.h) + at, v[c]);
      }
      if (a.out == 3) store_fp4<kNv>(a, m, k, valid, v[c]);
      if (a.out == 4) store_fp4<kMx>(a, m, k, valid, v[c]);
    }
  }
}

}  // namespace

// As many CTAs as fit the device (asked once per device), each with an equal share of neighbouring rows.
template <typename TX, typename TY, int kThreads, int kChunks>
static cudaError_t launch_rows(const GatedNormArgs& a, cudaStream_t s) {
  static std::atomic<int> room[64] = {};
  auto kernel = gated_norm_kernel<TX, TY, kThreads, kChunks>;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  int fit = room[dev].load(std::memory_order_relaxed);
  if (fit == 0) {
    int blocks = 1, sms = 148;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, kernel, kThreads, 0) != cudaSuccess) cudaGetLastError();
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    fit = (blocks < 1 ? 1 : blocks) * sms;
    room[dev].store(fit, std::memory_order_relaxed);
  }
  return launch_dependent(kernel, dim3(a.M < fit ? a.M : fit), kThreads, s, a);
}

cudaError_t gated_norm_launch(const GatedNormArgs& a, cudaStream_t s) {
  // the padding blocks of an FP4 row's last tile (at most three) belong to threads past the row: columns to cover
  const int cover = a.out >= 3 ? (a.K + 127) / 128 * 128 : a.K;
  auto shape = [&](auto xt, auto yt) {
    using TX = decltype(xt);
    using TY = decltype(yt);
    if (cover <= 1024) return launch_rows<TX, TY, 128, 1>(a, s);
    if (cover <= 2048) return launch_rows<TX, TY, 256, 1>(a, s);
    if (cover <= 3072) return launch_rows<TX, TY, 384, 1>(a, s);
    if (cover <= 4096) return launch_rows<TX, TY, 512, 1>(a, s);
    if (cover <= 8192) return launch_rows<TX, TY, 512, 2>(a, s);
    return launch_rows<TX, TY, 512, 4>(a, s);
  };
  const __nv_bfloat16 b{};
  if (a.x_dtype == 2) return a.y_dtype == 2 ? shape(float{}, float{}) : shape(float{}, b);
  return a.y_dtype == 2 ? shape(b, float{}) : shape(b, b);
}

}  // namespace fp4
}  // namespace wdl
