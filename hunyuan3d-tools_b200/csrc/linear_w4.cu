// Linear layers with 4-bit weights and group scales, 16-bit activations:
//     W[n,k] = s[n, k/G] * (c[n,k] - z[n, k/G]),   c in 0..15, z = 8 or a whole number of 0..15 per group
//     y[m,n] = epilogue( sum over groups of s[n,g] * (sum over k of the group of x[m,k] * (c[n,k] - z[n,g])) + bias[n] )
// The products x * (c - z) are exact in fp32 and summed there, the scale multiplies a group's sum in fp32, and the result
// is rounded once: the codes meet the activations as the whole numbers they are, which both 16-bit types hold exactly.
//
// Layout of the codes: tiles of 16 rows x 64 columns, 512 bytes, [N/16][K/64][lane][word].  Lane (g = lane / 4,
// t = lane % 4) of a warp owns rows g and g + 8: word 0 has columns 8t .. 8t+7 of row g, word 1 those of row g + 8, words 2
// and 3 the same of columns 32 + 8t ...  In a word, nibble j < 4 is column 2j and nibble 4 + j column 2j + 1, so that
// (word >> 4j) & 0x000F000F is a pair of neighbouring columns.  One 16-byte load per lane is then the whole A operand of
// four m16n8k16 products, in an order of k that the activations' 16-byte vectors have by themselves.
// Scales and zero points: [N/16][K/G][16] with rows g and g + 8 next to each other (places 2g and 2g + 1).
#include "common.cuh"

namespace hy3d {
int device_sm_count();
int device_ok();
int ensure_max_smem(const void* kernel, int bytes);
namespace w4 {
namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps;

struct Args {
  const uint16_t* x;
  int64_t ldx;
  const uint4* w;
  const uint32_t* scale;      // pairs (row g, row g + 8)
  const uint16_t* zero;       // the same, a byte each; or null
  const void* bias;
  uint16_t* out;
  uint64_t tiles_inv;         // ceil(2^32 / tiles of a group)
  int M, N, K, groups, epilogue, bias_dtype, scale_bf16, ks;
};

__device__ __forceinline__ void mma_16816(bool bf16, float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  if (bf16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A nibble c under the exponent of 2^7 (bf16) or 2^10 (fp16) is the number 128 + c or 1024 + c; the same with the zero
// point is subtracted, exactly.
template <bool kBf16> constexpr uint32_t kMagic = kBf16 ? 0x43004300u : 0x64006400u;
template <bool kBf16>
__device__ __forceinline__ void unpack_codes(uint32_t w, uint32_t bias, uint32_t (&out)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t v = ((w >> (4 * j)) & 0x000F000Fu) | kMagic<kBf16>;
    if (kBf16) asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(out[j]) : "r"(v), "r"(bias));
    else asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(out[j]) : "r"(v), "r"(bias));
  }
}

// A CTA computes kR blocks of 16 rows for kNT * 8 tokens; its warps (and the CTAs of its cluster) take the tiles of K in
// turn and their sums are added in a fixed order.
template <bool kBf16, int kNT, int kR, int kSub, int kUnroll>
__global__ void __launch_bounds__(kThreads)
linear_w4_kernel(const __grid_constant__ Args a) {
  extern __shared__ float s_part[];             // [warp][row][token]
  constexpr int kRows = 16 * kR, kTok = 8 * kNT, kPitch = kTok + 1;
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = a.ks > 1 ? static_cast<int>(cluster_cta_rank()) : 0;
  const int rb0 = (blockIdx.x / a.ks) * kR, tok0 = blockIdx.y * kTok;
  const int blocks = a.N >> 4, tiles = a.K >> 6, groups = a.groups;
  const int step = a.ks * kWarps;
  float acc[kR][kNT][4] = {};
  pdl_wait();

  const uint4* wp[kR];
  const uint32_t* sp[kR];
  const uint16_t* zp[kR];
#pragma unroll
  for (int r = 0; r < kR; ++r) {
    const int rb = min(rb0 + r, blocks - 1);
    wp[r] = a.w + static_cast<int64_t>(rb) * tiles * 32 + lane;
    sp[r] = a.scale + static_cast<int64_t>(rb) * groups * 8 + g;
    zp[r] = a.zero ? a.zero + static_cast<int64_t>(rb) * groups * 8 + g : nullptr;
  }
  const uint16_t* xp[kNT];
  bool live[kNT];
#pragma unroll
  for (int i = 0; i < kNT; ++i) {
    live[i] = tok0 + 8 * i + g < a.M;
    xp[i] = a.x + static_cast<int64_t>(min(tok0 + 8 * i + g, a.M - 1)) * a.ldx + 8 * t;
  }

  for (int base = rank * kWarps + warp; base < tiles; base += step * kUnroll) {
    uint4 w[kUnroll][kR], xv[kUnroll][kNT][2];
    uint32_t s[kUnroll][kR][kSub], z[kUnroll][kR][kSub];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int tile = base + u * step;
      const bool on = tile < tiles;
      const int grp = kSub == 2 ? 2 * tile : static_cast<int>(static_cast<uint32_t>(tile) * a.tiles_inv >> 32);
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        w[u][r] = on ? __ldcs(wp[r] + static_cast<int64_t>(tile) * 32) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int h = 0; h < kSub; ++h) {
          s[u][r][h] = on ? __ldg(sp[r] + (grp + h) * 8) : 0;
          z[u][r][h] = on && a.zero ? __ldg(zp[r] + (grp + h) * 8) : 0x0808u;
        }
      }
#pragma unroll
      for (int i = 0; i < kNT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          xv[u][i][h] = on && live[i] ? __ldg(reinterpret_cast<const uint4*>(xp[i] + tile * 64 + 32 * h)) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        float part[kNT][4] = {};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int sg = kSub == 2 ? h : 0;
          const uint32_t zz = z[u][r][sg];
          const uint32_t zlo = kMagic<kBf16> | (zz & 0xFFu) * 0x00010001u, zhi = kMagic<kBf16> | (zz >> 8) * 0x00010001u;
          uint32_t lo[4], hi[4];
          unpack_codes<kBf16>(h ? w[u][r].z : w[u][r].x, zlo, lo);
          unpack_codes<kBf16>(h ? w[u][r].w : w[u][r].y, zhi, hi);
#pragma unroll
          for (int i = 0; i < kNT; ++i) {
            mma_16816(kBf16, part[i], lo[0], hi[0], lo[1], hi[1], xv[u][i][h].x, xv[u][i][h].y);
            mma_16816(kBf16, part[i], lo[2], hi[2], lo[3], hi[3], xv[u][i][h].z, xv[u][i][h].w);
          }
          if (kSub == 2 || h == 1) {
            const uint32_t sw = s[u][r][sg];
            float slo, shi;
            if (a.scale_bf16) {
              slo = __uint_as_float(sw << 16);
              shi = __uint_as_float(sw & 0xFFFF0000u);
            } else {
              const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&sw));
              slo = f.x;
              shi = f.y;
            }
#pragma unroll
            for (int i = 0; i < kNT; ++i) {
              acc[r][i][0] = fmaf(slo, part[i][0], acc[r][i][0]);
              acc[r][i][1] = fmaf(slo, part[i][1], acc[r][i][1]);
              acc[r][i][2] = fmaf(shi, part[i][2], acc[r][i][2]);
              acc[r][i][3] = fmaf(shi, part[i][3], acc[r][i][3]);
              part[i][0] = part[i][1] = part[i][2] = part[i][3] = 0.0f;
            }
          }
        }
      }
    }
  }

  // Lane (g, t) has rows g and g + 8 of tokens 2t and 2t + 1.
  float* mine = s_part + warp * kRows * kPitch;
#pragma unroll
  for (int r = 0; r < kR; ++r)
#pragma unroll
    for (int i = 0; i < kNT; ++i) {
      float* p = mine + (16 * r + g) * kPitch + 8 * i + 2 * t;
      p[0] = acc[r][i][0];
      p[1] = acc[r][i][1];
      p[8 * kPitch] = acc[r][i][2];
      p[8 * kPitch + 1] = acc[r][i][3];
    }
  __syncthreads();
  for (int e = threadIdx.x; e < kRows * kTok; e += kThreads) {
    const int at = (e / kTok) * kPitch + e % kTok;
    float y = s_part[at];
#pragma unroll
    for (int v = 1; v < kWarps; ++v) y += s_part[v * kRows * kPitch + at];
    s_part[at] = y;              // only this thread reads or writes the place
  }
  __syncwarp();
  if (a.ks > 1) cluster_sync_all(); else __syncthreads();

  // Every CTA of the cluster finishes a share of the outputs.
  const bool geglu = a.epilogue == HY3D_EPI_GEGLU;
  const int out_rows = geglu ? kRows / 2 : kRows, n_out = geglu ? a.N >> 1 : a.N;
  for (int e = rank * kThreads + threadIdx.x; e < out_rows * kTok; e += step * 32) {
    const int tok = e / out_rows, row = e - tok * out_rows, m = tok0 + tok;
    const int in_row = geglu ? (row >> 4) * 32 + (row & 15) : row;
    const int n = rb0 * 16 + in_row;
    if (m >= a.M || n >= a.N) continue;
    auto total = [&](int rr) {
      const uint32_t local = smem_u32(s_part + rr * kPitch + tok);
      if (a.ks == 1) return s_part[rr * kPitch + tok];
      float y = 0.0f;
      for (int c = 0; c < a.ks; ++c) {
        float v;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(map_to_cta(local, c)));
        y += v;
      }
      return y;
    };
    float y = total(in_row);
    if (a.bias) y += load_scalar(a.bias, a.bias_dtype, n);
    if (a.epilogue == HY3D_EPI_GELU) {
      y = gelu_phi(y);
    } else if (geglu) {
      float gate = total(in_row + 16);
      if (a.bias) gate += load_scalar(a.bias, a.bias_dtype, n + 16);
      y *= gelu_phi(gate);
    }
    const int col = geglu ? (rb0 >> 1) * 16 + row : n;
    a.out[static_cast<int64_t>(m) * n_out + col] = static_cast<uint16_t>(pack2(y, 0.0f, kBf16 ? HY3D_BF16 : HY3D_F16));
  }
  __syncwarp();
  if (a.ks > 1) cluster_sync_all();      // a CTA's sums stay until the others have read them
}

using KernelFn = void (*)(const Args);
template <bool kBf16, int kSub>
KernelFn kernel_of(int nt, int r) {
  if (nt == 1) return r == 1 ? linear_w4_kernel<kBf16, 1, 1, kSub, 4> : linear_w4_kernel<kBf16, 1, 2, kSub, 2>;
  if (nt == 2) return linear_w4_kernel<kBf16, 2, 2, kSub, 2>;
  return linear_w4_kernel<kBf16, 4, 4, kSub, 1>;
}

}  // namespace

int linear(const void* x, int x_dtype, int64_t ldx, const void* w, const void* scale, int scale_dtype, const void* zero, int64_t group, const void* bias,
           int bias_dtype, void* out, int64_t M, int64_t N, int64_t K, int epilogue, cudaStream_t stream) {
  if (x_dtype != HY3D_F16 && x_dtype != HY3D_BF16) return HY3D_ERR_ARG;
  if (scale_dtype != HY3D_F16 && scale_dtype != HY3D_BF16) return HY3D_ERR_ARG;
  if (epilogue < HY3D_EPI_LINEAR || epilogue > HY3D_EPI_GEGLU) return HY3D_ERR_ARG;
  if (bias && (bias_dtype < HY3D_F16 || bias_dtype > HY3D_F32)) return HY3D_ERR_ARG;
  if (M < 0 || M > 0x7FFFFFFF || N <= 0 || N > 0x7FFFFFFF || K <= 0 || K > 1 << 20 || (K & 63) || (N & 15)) return HY3D_ERR_SHAPE;
  if (epilogue == HY3D_EPI_GEGLU && (N & 31)) return HY3D_ERR_SHAPE;
  if (group < 32 || (group & 31) || (group != 32 && (group & 63)) || K % group) return HY3D_ERR_SHAPE;
  if (ldx < K || (ldx & 7)) return HY3D_ERR_SHAPE;
  if (M == 0) return HY3D_OK;
  if (!x || !w || !scale || !out) return HY3D_ERR_ARG;
  if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & 15) || (reinterpret_cast<uintptr_t>(scale) & 3) ||
      ((reinterpret_cast<uintptr_t>(zero) | reinterpret_cast<uintptr_t>(out)) & 1))
    return HY3D_ERR_SHAPE;
  int rc = device_ok();
  if (rc != HY3D_OK) return rc;
  Args a;
  a.x = static_cast<const uint16_t*>(x);
  a.ldx = ldx;
  a.w = static_cast<const uint4*>(w);
  a.scale = static_cast<const uint32_t*>(scale);
  a.zero = static_cast<const uint16_t*>(zero);
  a.bias = bias;
  a.bias_dtype = bias_dtype;
  a.out = static_cast<uint16_t*>(out);
  a.M = static_cast<int>(M);
  a.N = static_cast<int>(N);
  a.K = static_cast<int>(K);
  a.groups = static_cast<int>(K / group);
  const uint64_t group_tiles = group == 32 ? 1 : static_cast<uint64_t>(group / 64);
  a.tiles_inv = ((1ull << 32) + group_tiles - 1) / group_tiles;
  a.scale_bf16 = scale_dtype == HY3D_BF16;
  a.epilogue = epilogue;
  const int nt = M <= 8 ? 1 : M <= 16 ? 2 : 4;
  const int r = nt == 4 ? 4 : nt == 2 || epilogue == HY3D_EPI_GEGLU ? 2 : 1;
  const int64_t by = (M + 8 * nt - 1) / (8 * nt);
  if (by > 65535) return HY3D_ERR_SHAPE;
  const int64_t bx = (N / 16 + r - 1) / r;
  const int sms = device_sm_count() > 0 ? device_sm_count() : 148;
  int ks = 1;
  while (ks < 8 && bx * by * ks * 2 <= sms && K / 64 >= kWarps * ks * 2) ks *= 2;
  a.ks = ks;
  const bool bf16 = x_dtype == HY3D_BF16, sub = group == 32;
  const KernelFn kernel = bf16 ? (sub ? kernel_of<true, 2>(nt, r) : kernel_of<true, 1>(nt, r))
                               : (sub ? kernel_of<false, 2>(nt, r) : kernel_of<false, 1>(nt, r));
  const int smem = kWarps * 16 * r * (8 * nt + 1) * 4;
  if (smem > 48 * 1024) {
    rc = ensure_max_smem(reinterpret_cast<const void*>(kernel), smem);
    if (rc != HY3D_OK) return rc;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(bx * ks), static_cast<unsigned>(by));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2] = {pdl_attribute(), {}};
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(ks);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ks > 1 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess) {
    cudaGetLastError();
    return HY3D_ERR_CUDA;
  }
  return HY3D_OK;
}

}  // namespace w4
}  // namespace hy3d
