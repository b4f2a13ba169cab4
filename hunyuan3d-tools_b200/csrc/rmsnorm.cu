// Root-mean-square norm over the last dimension, with the residual's addition in front of it and 16-bit values or the
// per-token quantiser's int8 codes behind it, in one pass over memory.
//
//     t     = round16(x + add)                       (t = x without add; stored in `sum` when there is one)
//     rstd  = 1 / sqrt(sum(t^2) / K + eps)           (fp32 sum in a fixed order, IEEE square root and reciprocal)
//     y     = round16((t * rstd) * gamma)
//     scale = max(max|y|, 1e-8) / 127,  q = rint(y / scale)
//
// so q and scale equal hy3d_quantize_rows of the 16-bit output bit for bit (quantize.cu has the proof of its rounding).
// A row with a NaN or an infinity gets a scale that is not finite, hence values that are NaN, as the 16-bit output has.
#include "common.cuh"

namespace hy3d {
int device_ok();
namespace rms {
namespace {

using quant::RowQuant;
using quant::row_quant;
using quant::quant8;
using quant::unpack8;

constexpr int kThreads = 256;

// Running packed maximum of |x| that keeps a NaN.
template <bool kBf16>
__device__ __forceinline__ void absmax8_nan(const uint4& v, uint32_t& acc) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (kBf16) asm("max.NaN.xorsign.abs.bf16x2 %0, %0, %1;" : "+r"(acc) : "r"(w[i]));
    else asm("max.NaN.xorsign.abs.f16x2 %0, %0, %1;" : "+r"(acc) : "r"(w[i]));
  }
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
template <bool kBf16>
__device__ __forceinline__ float absmax_nan_to_float(uint32_t acc) {
  acc &= 0x7FFF7FFFu;
  if (kBf16) return max_nan(__uint_as_float(acc << 16), __uint_as_float(acc & 0xFFFF0000u));
  const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&acc));
  return max_nan(t.x, t.y);
}

struct Args {
  const uint16_t *x, *add;
  int64_t ldx, ld_add;
  uint16_t *sum, *y;
  const void* gamma;
  int8_t* q;
  float* scale;
  int64_t M;
  float eps, inv_k;
  int K, lg, g_dtype;
};

// Eight of gamma's values as pairs.  kOwn: of the activations' type, `raw` loaded earlier.
template <bool kBf16, bool kOwn>
__device__ __forceinline__ void gamma_pairs(const Args& a, int vec, const uint4& raw, float2 (&g)[4]) {
  float f[8];
  if (kOwn) {
    unpack8<kBf16>(raw, f);
  } else if (!a.gamma) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = 1.0f;
  } else if (a.g_dtype == HY3D_F32) {
    const float4* p = reinterpret_cast<const float4*>(a.gamma) + 2 * vec;
    const float4 u = __ldg(p), v = __ldg(p + 1);
    f[0] = u.x; f[1] = u.y; f[2] = u.z; f[3] = u.w;
    f[4] = v.x; f[5] = v.y; f[6] = v.z; f[7] = v.w;
  } else {
    unpack8<!kBf16>(__ldg(reinterpret_cast<const uint4*>(a.gamma) + vec), f);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) g[j] = make_float2(f[2 * j], f[2 * j + 1]);
}

// 2^lg threads share a row, each with up to kV 16-byte vectors that stay in registers between the statistics and the
// output.  A block holds blockDim >> lg rows; threads past the last row compute it too and store nothing.
// Bound by HBM with a residual (12288 x 640 to 16 bits 8.6 us, 7.4 TB/s, part of it still in L2; to codes 9.9, 5.6; 8192 x 8192
// to 16 bits 80.3, 6.7).  Without one, to codes, by instructions and the chain of load, two reductions and store (3855 x 1536
// 7.2 us, 2.5 TB/s; 49152 x 320 13.0, 3.6).  Blocks per SM follow from the registers kV needs, none of which may spill: with
// three blocks for every kV those two took 8 and 6 % more.  (A grid-stride loop that requests the next row ahead of the current
// one's work spilled: 12288 x 640 to codes 10.8 -> 13.2.)
// kOwn: gamma is of the activations' type, and its values are requested with the row's, not after its statistics, where there
// are registers for both.  With its type looked up for every vector one row of 4096 took 2.5 us instead of 2.1, 3855 x 1536
// 7.9, 12288 x 640 to codes 10.7 and 4096 x 4096 23.0 instead of 19.4.
template <bool kBf16, int kV, bool kAdd, bool kCodes, bool kWide, bool kOwn>
__global__ void __launch_bounds__(kWide ? 512 : kThreads, kWide ? 2 : kV == 1 ? 6 : kV == 2 ? 5 : kV == 3 ? 4 : 3)
rmsnorm_kernel(const __grid_constant__ Args a) {
  __shared__ float s_part[2][16];
  pdl_launch_dependents();
  const int tid = threadIdx.x, G = 1 << a.lg, sub = tid & (G - 1);
  int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> a.lg) + (tid >> a.lg);
  const bool live = row < a.M;
  if (!live) row = a.M - 1;
  const int nvec = a.K >> 3;
  const int warp = tid >> 5, warps_per_row = G >> 5, first = warp & ~(warps_per_row - 1);
  pdl_wait();
  uint4 v[kV];
  {
    const uint4* src = reinterpret_cast<const uint4*>(a.x + row * a.ldx) + sub;
#pragma unroll
    for (int i = 0; i < kV; ++i) v[i] = sub + i * G < nvec ? __ldcs(src + i * G) : make_uint4(0, 0, 0, 0);
  }
  if (kAdd) {
    const uint4* src = reinterpret_cast<const uint4*>(a.add + row * a.ld_add) + sub;
    uint4 w[kV];
#pragma unroll
    for (int i = 0; i < kV; ++i) w[i] = sub + i * G < nvec ? __ldcs(src + i * G) : make_uint4(0, 0, 0, 0);
    uint4* dst = reinterpret_cast<uint4*>(a.sum + row * static_cast<int64_t>(a.K)) + sub;
#pragma unroll
    for (int i = 0; i < kV; ++i) {
      v[i] = add8_16<kBf16>(v[i], w[i]);
      if (live && sub + i * G < nvec) dst[i * G] = v[i];
    }
  }
  constexpr bool kEarly = kOwn && (!kCodes || kV <= (kWide ? 3 : 4));
  uint4 graw[kV];
  if (kEarly)
#pragma unroll
    for (int i = 0; i < kV; ++i)
      graw[i] = sub + i * G < nvec ? __ldg(reinterpret_cast<const uint4*>(a.gamma) + sub + i * G) : make_uint4(0, 0, 0, 0);
  float2 ss2 = make_float2(0.0f, 0.0f);
#pragma unroll
  for (int i = 0; i < kV; ++i) {
    float f[8];
    unpack8<kBf16>(v[i], f);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 p = make_float2(f[2 * j], f[2 * j + 1]);
      ss2 = __ffma2_rn(p, p, ss2);
    }
  }
  float ss = ss2.x + ss2.y;
  for (int off = (G < 32 ? G : 32) >> 1; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
  if (G > 32) {
    if ((tid & 31) == 0) s_part[0][warp] = ss;
    __syncthreads();
    ss = s_part[0][first];
    for (int i = 1; i < warps_per_row; ++i) ss += s_part[0][first + i];
  }
  const float rstd = __frcp_rn(__fsqrt_rn(fmaf(ss, a.inv_k, a.eps)));
  const float2 rstd2 = make_float2(rstd, rstd);
  uint32_t amax2 = 0;
  uint4* ydst = reinterpret_cast<uint4*>(a.y + row * static_cast<int64_t>(a.K)) + sub;
#pragma unroll
  for (int i = 0; i < kV; ++i) {
    if (sub + i * G < nvec) {
      float2 g[4];
      if (kOwn && !kEarly) graw[i] = __ldg(reinterpret_cast<const uint4*>(a.gamma) + sub + i * G);
      gamma_pairs<kBf16, kOwn>(a, sub + i * G, graw[i], g);
      float f[8];
      unpack8<kBf16>(v[i], f);
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 y = __fmul2_rn(__fmul2_rn(make_float2(f[2 * j], f[2 * j + 1]), rstd2), g[j]);
        w[j] = pack2(y.x, y.y, kBf16 ? HY3D_BF16 : HY3D_F16);
      }
      v[i] = make_uint4(w[0], w[1], w[2], w[3]);
      if (kCodes) absmax8_nan<kBf16>(v[i], amax2);
      if (live && (!kCodes || a.y)) ydst[i * G] = v[i];
    }
  }
  if (kCodes) {
    float amax = absmax_nan_to_float<kBf16>(amax2);
    for (int off = (G < 32 ? G : 32) >> 1; off > 0; off >>= 1)
      amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, off));
    if (G > 32) {
      if ((tid & 31) == 0) s_part[1][warp] = amax;
      __syncthreads();
      amax = s_part[1][first];
      for (int i = 1; i < warps_per_row; ++i) amax = max_nan(amax, s_part[1][first + i]);
    }
    const RowQuant rq = row_quant(amax);
    if (live && sub == 0) a.scale[row] = amax == amax ? rq.scale : amax;
    uint2* dst = reinterpret_cast<uint2*>(a.q + row * static_cast<int64_t>(a.K)) + sub;
    auto write = [&](auto exact) {
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        if (live && sub + i * G < nvec) {
          float f[8];
          unpack8<kBf16>(v[i], f);
          dst[i * G] = quant8<decltype(exact)::value>(f, rq);
        }
      }
    };
    if (rq.exact) write(quant::True{}); else write(quant::False{});
  }
}

template <bool kBf16>
int launch(const Args& in, cudaStream_t stream) {
  Args a = in;
  const int nvec = a.K >> 3;
  // Threads per row: the fewest (a power of two, eight where the row has as many vectors, so that a load touches whole 128-byte
  // lines: 30000 x 64 a third less) that hold it with 4 vectors each; eight threads take 5.  More vectors a thread and fewer
  // threads save reductions and barriers (at most 3 vectors: 5000 x 2048 to codes and 49152 x 320 18 % more),
  // fewer vectors leave registers for more blocks on an SM (5: 12288 x 640 to 16 bits 8 % more).  By K alone: the number
  // of threads fixes the order of the row's sum, so a row's result does not depend on how many others there are.
  a.lg = 0;
  while ((a.lg < 3 && (1 << a.lg) < nvec) || ((nvec + (1 << a.lg) - 1) >> a.lg) > (a.lg == 3 ? 5 : 4)) ++a.lg;
  const int v = (nvec + (1 << a.lg) - 1) >> a.lg;
  const int threads = a.lg > 8 ? 1 << a.lg : kThreads;
  const int rows = threads >> a.lg;
  const int64_t blocks = (a.M + rows - 1) / rows;
  if (blocks > 0x7FFFFFFF) return HY3D_ERR_SHAPE;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2] = {pdl_attribute(), carveout_attribute(4, 128)};
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  using KernelFn = void (*)(const Args);
#define HY3D_RMS2(V, A, C, W) {rmsnorm_kernel<kBf16, V, A, C, W, false>, rmsnorm_kernel<kBf16, V, A, C, W, true>}
#define HY3D_RMS(V, W)                                                    \
  {{HY3D_RMS2(V, false, false, W), HY3D_RMS2(V, false, true, W)},         \
   {HY3D_RMS2(V, true, false, W), HY3D_RMS2(V, true, true, W)}}
  static const KernelFn kernels[5][2][2][2] = {HY3D_RMS(1, false), HY3D_RMS(2, false), HY3D_RMS(3, false), HY3D_RMS(4, false),
                                               HY3D_RMS(5, false)};
  static const KernelFn wide[2][2][2][2] = {HY3D_RMS(3, true), HY3D_RMS(4, true)};      // 512 threads: K from 8200 on
#undef HY3D_RMS
#undef HY3D_RMS2
  const int own = a.gamma && a.g_dtype == (kBf16 ? HY3D_BF16 : HY3D_F16) ? 1 : 0;
  const KernelFn kernel = (a.lg > 8 ? wide[v - 3] : kernels[v - 1])[a.add ? 1 : 0][a.q ? 1 : 0][own];
  if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess) {
    cudaGetLastError();
    return HY3D_ERR_CUDA;
  }
  return HY3D_OK;
}

// Codes back to the values they stand for: round16(q * scale).  A block takes kUnroll * kThreads adjacent vectors of eight;
// a vector's row comes from one division per thread and additions from there on.
__global__ void __launch_bounds__(kThreads)
dequantize_rows_kernel(const uint2* __restrict__ q, const float* __restrict__ scale, uint4* __restrict__ y, int64_t total,
                       int vec_cols, int out_dtype) {
  pdl_launch_dependents();
  constexpr int kUnroll = 4;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (kUnroll * kThreads) + threadIdx.x;
  int64_t row = total <= 0xFFFFFFFFll ? static_cast<int64_t>(static_cast<uint32_t>(first) / static_cast<uint32_t>(vec_cols)) : first / vec_cols;
  int col = static_cast<int>(first - row * vec_cols);
  const int step_row = kThreads / vec_cols, step_col = kThreads - step_row * vec_cols;
  pdl_wait();
  uint2 v[kUnroll];
  float s[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t at = first + u * kThreads;
    if (at < total) {
      v[u] = __ldcs(q + at);
      s[u] = __ldg(scale + row);
    }
    row += step_row;
    col += step_col;
    if (col >= vec_cols) { col -= vec_cols; ++row; }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t at = first + u * kThreads;
    if (at < total) {
      const uint32_t w[2] = {v[u].x, v[u].y};
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t h = w[j >> 1] >> (16 * (j & 1));
        o[j] = pack2(static_cast<float>(static_cast<signed char>(h)) * s[u],
                     static_cast<float>(static_cast<signed char>(h >> 8)) * s[u], out_dtype);
      }
      y[at] = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

}  // namespace

int rmsnorm(const void* x, int64_t ldx, const void* add, int64_t ld_add, void* sum, int x_dtype, int64_t M, int64_t K,
            const void* gamma, int g_dtype, float eps, void* y, int8_t* q, float* scale, cudaStream_t stream) {
  if (x_dtype != HY3D_F16 && x_dtype != HY3D_BF16) return HY3D_ERR_ARG;
  if (gamma && (g_dtype < HY3D_F16 || g_dtype > HY3D_F32)) return HY3D_ERR_ARG;
  if (!(eps >= 0.0f)) return HY3D_ERR_ARG;
  if (M < 0 || K <= 0 || (K & 7) || K > 16384 || ldx < K || (ldx & 7)) return HY3D_ERR_SHAPE;
  if (add && (ld_add < K || (ld_add & 7))) return HY3D_ERR_SHAPE;
  if (M == 0) return HY3D_OK;
  if (!x || (!y && !q) || (q && !scale) || (add && !sum)) return HY3D_ERR_ARG;
  const uintptr_t at16 = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(add) | reinterpret_cast<uintptr_t>(add ? sum : nullptr) |
                         reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(gamma);
  if ((at16 & 15) || (reinterpret_cast<uintptr_t>(q) & 7)) return HY3D_ERR_SHAPE;
  const int rc = device_ok();
  if (rc != HY3D_OK) return rc;
  Args a;
  a.x = static_cast<const uint16_t*>(x);
  a.add = static_cast<const uint16_t*>(add);
  a.ldx = ldx;
  a.ld_add = ld_add;
  a.sum = static_cast<uint16_t*>(sum);
  a.y = static_cast<uint16_t*>(y);
  a.gamma = gamma;
  a.q = q;
  a.scale = scale;
  a.M = M;
  a.eps = eps;
  a.inv_k = 1.0f / static_cast<float>(K);
  a.K = static_cast<int>(K);
  a.g_dtype = g_dtype;
  return x_dtype == HY3D_BF16 ? launch<true>(a, stream) : launch<false>(a, stream);
}

int dequantize_rows(const int8_t* q, const float* scale, int64_t M, int64_t K, int out_dtype, void* y, cudaStream_t stream) {
  if (out_dtype != HY3D_F16 && out_dtype != HY3D_BF16) return HY3D_ERR_ARG;
  if (M < 0 || K <= 0 || (K & 7) || K > 0x7FFFFFFF) return HY3D_ERR_SHAPE;
  if (M == 0) return HY3D_OK;
  if (!q || !scale || !y) return HY3D_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(q) & 7) || (reinterpret_cast<uintptr_t>(y) & 15)) return HY3D_ERR_SHAPE;
  const int64_t total = M * (K >> 3), blocks = (total + 4 * kThreads - 1) / (4 * kThreads);
  if (blocks > 0x7FFFFFFF) return HY3D_ERR_SHAPE;
  const int rc = device_ok();
  if (rc != HY3D_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1] = {pdl_attribute()};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, dequantize_rows_kernel, reinterpret_cast<const uint2*>(q), scale, static_cast<uint4*>(y), total,
                         static_cast<int>(K >> 3), out_dtype) != cudaSuccess) {
    cudaGetLastError();
    return HY3D_ERR_CUDA;
  }
  return HY3D_OK;
}

}  // namespace rms
}  // namespace hy3d
