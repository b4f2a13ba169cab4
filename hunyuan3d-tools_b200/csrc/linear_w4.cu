// Linear layers with 4-bit weights and group scales, 16-bit activations:
//     W[n,k] = s[n, k/G] * (c[n,k] - z[n, k/G]),   c in 0..15, z = 8 or a whole number of 0..15 per group
//     y[m,n] = epilogue( sum over groups of s[n,g] * (sum over k of the group of x[m,k] * (c[n,k] - z[n,g])) + bias[n] )
// The products x * (c - z) are exact in fp32 and summed there, the scale multiplies a group's sum in fp32, and the result
// is rounded once: the codes meet the activations as the whole numbers they are, which both 16-bit types hold exactly.
//
// Layout of the codes: tiles of 16 rows x 64 columns, 512 bytes, [N/16][K/64][lane][word].  Lane (g = lane / 4,
// t = lane % 4) of a warp owns rows g and g + 8: words 0 and 1 are these rows' columns 4t .. 4t+3 and 16 + 4t .. 16 + 4t+3,
// words 2 and 3 the same of columns 32 on.  In a word, nibble j < 4 is the 2j-th of its columns and nibble 4 + j the one
// behind it, so that (word >> 4j) & 0x000F000F is a pair of neighbouring columns.  One 16-byte load per lane is then the
// whole A operand of four m16n8k16 products whose columns are those of the activations' 8-byte vectors, and also what the
// lane stores of a 16 x 64 operand in tensor memory (gemm_w4.cu).
// Scales and zero points: [N/16][K/G][16] with rows g and g + 8 next to each other (places 2g and 2g + 1).
#include "common.cuh"

namespace hy3d {
int device_sm_count();
int device_ok();
int ensure_max_smem(const void* kernel, int bytes);
namespace w4 {
namespace {

constexpr int kWarps = 16, kThreads = 32 * kWarps;
constexpr int kMaxTrips = 8;
constexpr int kSmem = 226 * 1024;
constexpr int64_t kMaxGridY = 65535;
constexpr int kTiles = 4, kStages = 2;      // tiles of a stage, stages of a warp's ring
// Bytes of a stage for one block of rows: codes, scales, zero points.
__host__ __device__ constexpr int stage_row(int sub, bool plain) { return kTiles * (512 + 32 * sub + (plain ? 0 : 16 * sub)); }

struct Args {
  const uint16_t* x;
  int64_t ldx;
  const uint4* w;
  const uint32_t* scale;      // pairs (row g, row g + 8)
  const uint8_t* zero;        // the same, a byte each; or null
  const void* bias;
  uint16_t* out;
  uint32_t tiles_inv;         // ceil(2^31 / tiles of a group)
  int M, N, K, groups, epilogue, bias_dtype, scale_bf16;
  int tokens;                 // of a CTA, at most 8
  int lg_wk, trips, units;    // 2^lg_wk warps share a unit (kR blocks of rows); units a warp takes, and their number
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

// Integers as the low bits of a number whose exponent is fixed, the usual conversion of packed weights (Y. J. Kim et al., "Who
// Says Elephants Can't Run", 2022, describe it for these types; the constants follow from the formats):
// a nibble c under the exponent of 2^7 (bf16) or 2^10 (fp16) is the number 128 + c or 1024 + c; `minus` is the negative of
// that with the zero point, and the sum is exact.  (As a multiply-add by one: bf16 has no addition of its own.)  fp16 has
// room for the next nibble where it lies, 1024 + 16 c, and the multiply-add scales it: two shifts in three less.
template <bool kBf16> constexpr uint32_t kMagic = kBf16 ? 0x43004300u : 0x64006400u;
__device__ __forceinline__ uint32_t masked(uint32_t w, uint32_t mask, uint32_t magic) {
  uint32_t v;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(w), "r"(mask), "r"(magic));     // (w & mask) | magic
  return v;
}
struct Minus { uint32_t one, sixteenth; };
template <bool kBf16>
__device__ __forceinline__ Minus minus_of(uint32_t z) {         // z in both halves
  return {kMagic<kBf16> | 0x80008000u | z, 0xD400D400u | z << 4};       // -(2^10 + z), and -(2^6 + z) for fp16
}
template <bool kBf16>
__device__ __forceinline__ void unpack_codes(uint32_t w, const Minus& m, uint32_t (&out)[4]) {
  if (kBf16) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(out[j]) : "r"(masked(w >> (4 * j), 0x000F000Fu, kMagic<true>)), "r"(0x3F803F80u), "r"(m.one));
  } else {
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      const uint32_t v = w >> (4 * j);
      asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(out[j]) : "r"(masked(v, 0x000F000Fu, kMagic<false>)), "r"(0x3C003C00u), "r"(m.one));
      asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(out[j + 1]) : "r"(masked(v, 0x00F000F0u, kMagic<false>)), "r"(0x2C002C00u), "r"(m.sixteenth));
    }
  }
}

// The scales of rows g and g + 8.
__device__ __forceinline__ float2 scale_pair(uint32_t w, bool bf16) {
  if (bf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

__device__ __forceinline__ void bulk_prefetch_l2(const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src), "r"(bytes) : "memory");
}
template <int kBytes>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  if (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory"); }

// Few tokens (8 at most).  1 x 8192 -> 8192 with groups of 128 takes 10.0 us, 3.5 TB/s (with the loop over a stage's tiles rolled
// up 16), 12 x 1280 -> 640 2.8: neither the stream of codes (5.3 us) nor the instructions that unpack them (72 a tile, 4.7 us on the
// 128 SMs that a power of two of warps a unit leaves at work; issue slots 56 % used) fill it, but the tiles that a warp has in
// series, its ring of two stages and the start.  One CTA per SM.  The activations of its tokens lie in shared memory whole; 2^lg_wk warps share a unit of kR blocks of 16
// rows, each with a range of K, and take `trips` units one after the other without a pause, through rings of their own in
// shared memory: nothing waits for another warp until the sums are added at the end, in a fixed order.
// kPlain: no zero points, and scales of the activations' type.
template <bool kBf16, int kR, int kSub, bool kPlain>
__global__ void __launch_bounds__(kThreads, 1)
linear_w4_kernel(const __grid_constant__ Args a) {
  constexpr int kRows = 16 * kR, kScales = kTiles * 512, kZeros = kScales + kTiles * 32 * kSub;
  constexpr int kRow = stage_row(kSub, kPlain), kStage = kR * kRow;
  extern __shared__ __align__(128) uint8_t s_mem[];      // [warp][stage]; activations [token][K]; sums [trip][warp][row][token]
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int wk = 1 << a.lg_wk, per_cta = kWarps >> a.lg_wk;
  const int group = static_cast<int>(blockIdx.x) * per_cta + (warp >> a.lg_wk), all_groups = static_cast<int>(gridDim.x) * per_cta;
  const int tok0 = blockIdx.y * a.tokens, mt = min(a.tokens, a.M - tok0);
  const int blocks = a.N >> 4, tiles = a.K >> 6, part = warp & (wk - 1);
  const int first = tiles * part >> a.lg_wk, count = (tiles * (part + 1) >> a.lg_wk) - first;
  const int mine = group < a.units ? min(a.trips, (a.units - group + all_groups - 1) / all_groups) : 0;
  uint8_t* ring = s_mem + warp * (kStages * kStage);
  const int x_pitch = a.K * 2 + 32;                      // 32 bytes off a multiple of 128: no bank conflicts
  uint8_t* s_x = s_mem + kWarps * kStages * kStage;
  float* s_part = reinterpret_cast<float*>(s_x + a.tokens * x_pitch);

  // What comes next into the ring: tiles [in_tile, in_tile + kTiles) of the range, of unit in_unit.
  int in_tile = 0, in_trip = 0;
  const uint8_t* wp[kR];
  const uint8_t* sp[kR];
  const uint8_t* zp[kR];
  auto point = [&] {
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      const int64_t block = min((group + in_trip * all_groups) * kR + r, blocks - 1);
      wp[r] = reinterpret_cast<const uint8_t*>(a.w) + (block * tiles + first) * 512 + lane * 16;
      sp[r] = reinterpret_cast<const uint8_t*>(a.scale) + block * a.groups * 32 + (lane & 7) * 4;
      zp[r] = !kPlain && a.zero ? a.zero + block * a.groups * 16 + (lane & 3) * 4 : nullptr;
    }
  };
  auto group_of = [&](int tile) { return kSub == 2 ? 2 * tile : static_cast<int>(__umulhi(2 * tile, a.tiles_inv)); };
  auto issue = [&](const uint8_t* into) {
    const uint32_t slot = smem_u32(into);
    if (in_trip < mine) {
      const int n = min(kTiles, count - in_tile);
      // scales: lane 8u + i has words i of tile u's group, zero points: lane 4u + i
      const int u8 = lane >> 3, u4 = lane >> 2;
      const int s_at = group_of(first + in_tile + min(u8, n - 1)) * 32, z_at = group_of(first + in_tile + min(u4 & 3, n - 1)) * 16;
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        const uint32_t to = slot + r * kRow;
#pragma unroll
        for (int u = 0; u < kTiles; ++u)
          if (u < n) copy_async<16>(to + u * 512 + lane * 16, wp[r] + u * 512);
        wp[r] += kTiles * 512;
#pragma unroll
        for (int h = 0; h < kSub; ++h) {
          copy_async<4>(to + kScales + u8 * (32 * kSub) + h * 32 + (lane & 7) * 4, sp[r] + s_at + h * 32);
          if (!kPlain && a.zero && lane < 16) copy_async<4>(to + kZeros + u4 * (16 * kSub) + h * 16 + (lane & 3) * 4, zp[r] + z_at + h * 16);
        }
      }
      in_tile += kTiles;
      if (in_tile >= count) {
        in_tile = 0;
        ++in_trip;
        point();
      }
    }
    copies_commit();
  };
  const int trips = count > 0 ? mine : 0;
  if (trips == 0) {
    in_trip = mine;
  } else {
    point();
    // into L2 while the previous kernel ends: its tail hides what memory takes to answer
    if (lane == 0)
#pragma unroll
      for (int r = 0; r < kR; ++r) bulk_prefetch_l2(wp[r], min(count, kTiles * kStages) * 512);
  }
  pdl_wait();
  // the activations, all threads together
  for (int m = 0; m < mt; ++m) {
    const uint16_t* src = a.x + static_cast<int64_t>(tok0 + m) * a.ldx;
    for (int v = threadIdx.x; v < a.K >> 3; v += kThreads) copy_async<16>(smem_u32(s_x + m * x_pitch + v * 16), src + v * 8);
  }
  copies_commit();
#pragma unroll
  for (int i = 0; i < kStages; ++i) issue(ring + i * kStage);
  copies_wait<kStages>();
  __syncthreads();

  float acc[kR][4] = {};
  const uint8_t* x_lane = s_x + min(g, mt - 1) * x_pitch + first * 128 + t * 8;      // tokens past the last: its columns again, not read
  auto multiply = [&](const uint8_t* slot, const uint8_t* at_x, int u) {
    uint2 x[4];                        // columns 16i + 4t .. 16i + 4t + 3
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const uint2*>(at_x + 32 * i);
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      const uint8_t* from = slot + r * kRow;
      const uint4 w = *reinterpret_cast<const uint4*>(from + u * 512 + lane * 16);
      float part_sum[4] = {};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int sg = u * kSub + (kSub == 2 ? h : 0);
        uint32_t zlo = 0x00080008u, zhi = 0x00080008u;
        if (!kPlain && a.zero) {
          const uint32_t z = *reinterpret_cast<const uint16_t*>(from + kZeros + sg * 16 + g * 2);
          zlo = (z & 0xFFu) * 0x00010001u;
          zhi = (z >> 8 & 0xFFu) * 0x00010001u;
        }
        uint32_t lo[4], hi[4];
        unpack_codes<kBf16>(h ? w.z : w.x, minus_of<kBf16>(zlo), lo);
        unpack_codes<kBf16>(h ? w.w : w.y, minus_of<kBf16>(zhi), hi);
        mma_16816(kBf16, part_sum, lo[0], hi[0], lo[1], hi[1], x[2 * h].x, x[2 * h].y);
        mma_16816(kBf16, part_sum, lo[2], hi[2], lo[3], hi[3], x[2 * h + 1].x, x[2 * h + 1].y);
        if (kSub == 2 || h == 1) {
          const float2 sc = scale_pair(*reinterpret_cast<const uint32_t*>(from + kScales + sg * 32 + g * 4), kPlain ? kBf16 : a.scale_bf16 != 0);
          acc[r][0] = fmaf(sc.x, part_sum[0], acc[r][0]);
          acc[r][1] = fmaf(sc.x, part_sum[1], acc[r][1]);
          acc[r][2] = fmaf(sc.y, part_sum[2], acc[r][2]);
          acc[r][3] = fmaf(sc.y, part_sum[3], acc[r][3]);
          part_sum[0] = part_sum[1] = part_sum[2] = part_sum[3] = 0.0f;
        }
      }
    }
  };
  float* sums = s_part + warp * kRows * a.tokens;
  const uint8_t* slot = ring;
  static_assert(kStages == 2, "two slots in turn");
  for (int trip = 0; trip < trips; ++trip) {
    for (int k = 0; k < count; k += kTiles) {
      copies_wait<kStages - 1>();
      __syncwarp();                    // scales and zero points are other lanes' copies
      const uint8_t* at_x = x_lane + k * 128;
      if (count - k >= kTiles) {
#pragma unroll
        for (int u = 0; u < kTiles; ++u) multiply(slot, at_x + u * 128, u);
      } else {
#pragma unroll
        for (int u = 0; u < kTiles - 1; ++u)
          if (u < count - k) multiply(slot, at_x + u * 128, u);
      }
      __syncwarp();
      issue(slot);
      slot = slot == ring ? ring + kStage : ring;
    }
    // lane (g, t) has rows g and g + 8 of tokens 2t and 2t + 1
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      float* p = sums + (16 * r + g) * a.tokens + 2 * t;
      if (2 * t < mt) {
        p[0] = acc[r][0];
        p[8 * a.tokens] = acc[r][2];
      }
      if (2 * t + 1 < mt) {
        p[1] = acc[r][1];
        p[8 * a.tokens + 1] = acc[r][3];
      }
      acc[r][0] = acc[r][1] = acc[r][2] = acc[r][3] = 0.0f;
    }
    sums += kWarps * kRows * a.tokens;
  }
  copies_wait<0>();
  __syncthreads();

  // Rows of a trip: per_cta units side by side.  A range without tiles (more warps than tiles) wrote no sums.
  const bool geglu = a.epilogue == HY3D_EPI_GEGLU;
  const int n_out = geglu ? a.N >> 1 : a.N, out_rows = geglu ? kRows / 2 : kRows, parts = min(wk, tiles);
  for (int e = threadIdx.x; e < a.trips * per_cta * out_rows * mt; e += kThreads) {
    const int row = e % out_rows, rest = e / out_rows, tok = rest % mt, at = rest / mt, trip = at >> (4 - a.lg_wk), sub = at & (per_cta - 1);
    const int unit = static_cast<int>(blockIdx.x) * per_cta + sub + trip * all_groups;
    const int n = unit * kRows + row;
    if (unit >= a.units || n >= a.N) continue;
    auto sum_of = [&](int r) {
      const float* p = s_part + ((trip * kWarps + sub * wk) * kRows + r) * a.tokens + tok;
      float y = 0.0f;
      for (int v = 0; v < wk; ++v)
        if (parts == wk || (tiles * (v + 1) >> a.lg_wk) > (tiles * v >> a.lg_wk)) y += p[v * kRows * a.tokens];
      return y;
    };
    float y = sum_of(row);
    if (a.bias) y += load_scalar(a.bias, a.bias_dtype, n);
    int col = n;
    if (a.epilogue == HY3D_EPI_GELU) {
      y = gelu_phi(y);
    } else if (geglu) {
      float gate = sum_of(row + 16);
      if (a.bias) gate += load_scalar(a.bias, a.bias_dtype, n + 16);
      y *= gelu_phi(gate);
      col = unit * 16 + row;
    }
    a.out[static_cast<int64_t>(tok0 + tok) * n_out + col] = static_cast<uint16_t>(pack2(y, 0.0f, kBf16 ? HY3D_BF16 : HY3D_F16));
  }
}

using KernelFn = void (*)(const Args);
template <bool kBf16>
KernelFn kernel_of(int r, bool sub, bool plain) {
  if (r == 1) {
    if (plain) return sub ? linear_w4_kernel<kBf16, 1, 2, true> : linear_w4_kernel<kBf16, 1, 1, true>;
    return sub ? linear_w4_kernel<kBf16, 1, 2, false> : linear_w4_kernel<kBf16, 1, 1, false>;
  }
  if (plain) return sub ? linear_w4_kernel<kBf16, 2, 2, true> : linear_w4_kernel<kBf16, 2, 1, true>;
  return sub ? linear_w4_kernel<kBf16, 2, 2, false> : linear_w4_kernel<kBf16, 2, 1, false>;
}

// How the few-token kernel would run a layer.
struct Plan {
  int tokens, lg_wk, trips, smem;
  int64_t bx, by, cycles;      // CTAs, and about what the busiest SM takes
};
// A tile takes a warp 380 cycles beside three others of its scheduler; about 2500 cycles go to the start, the first codes
// and the sums, and the activations arrive at 100 bytes a cycle.
Plan plan_of(int64_t M, int64_t N, int64_t K, int64_t by, int r, int sub, bool plain, int sms) {
  Plan p = {};
  const int tiles = static_cast<int>(K / 64);
  const int64_t units = N / 16 / r, row = K * 2 + 32;
  const int ring = kWarps * kStages * r * stage_row(sub, plain);
  p.tokens = static_cast<int>((M + by - 1) / by);
  while (ring + p.tokens * (row + kWarps * 16 * r * 4) > kSmem) --p.tokens;      // one at least: K is bounded
  p.by = (M + p.tokens - 1) / p.tokens;
  const int64_t sms_each = sms / p.by > 1 ? sms / p.by : 1;
  const int trip_bytes = kWarps * 16 * r * p.tokens * 4;
  const int64_t fixed = ring + p.tokens * row, most_trips = (kSmem - fixed) / trip_bytes < kMaxTrips ? (kSmem - fixed) / trip_bytes : kMaxTrips;
  p.cycles = INT64_MAX;
  for (int lg = 0; lg <= 4; ++lg) {      // warps of a unit
    const int per_cta = kWarps >> lg;
    int64_t trips = (units + sms_each * per_cta - 1) / (sms_each * per_cta);
    if (trips > most_trips) trips = most_trips;
    const int64_t bx = (units + per_cta * trips - 1) / (per_cta * trips), waves = (bx * p.by + sms - 1) / sms;
    const int64_t cycles = waves * (trips * ((tiles + (1 << lg) - 1) >> lg) * 380 * r + 2500 + p.tokens * row / 100);
    if (cycles < p.cycles) {
      p.cycles = cycles;
      p.lg_wk = lg;
      p.trips = static_cast<int>(trips);
      p.bx = bx;
      p.smem = static_cast<int>(fixed + trips * trip_bytes);
    }
  }
  return p;
}

}  // namespace

// The kernel of gemm_w4.cu, and how it would run a layer.
struct TcPlan {
  int tokens, ks;
  int64_t cycles;
};
TcPlan tc_plan(int64_t M, int64_t N, int64_t K);
int gemm(const void* x, int x_dtype, int64_t ldx, const void* w, const void* scale, const void* zero, int64_t group, const void* bias,
         int bias_dtype, void* out, int64_t M, int64_t N, int64_t K, int epilogue, const TcPlan& plan, cudaStream_t stream);

int linear(const void* x, int x_dtype, int64_t ldx, const void* w, const void* scale, int scale_dtype, const void* zero, int64_t group, const void* bias,
           int bias_dtype, void* out, int64_t M, int64_t N, int64_t K, int epilogue, cudaStream_t stream) {
  if (x_dtype != HY3D_F16 && x_dtype != HY3D_BF16) return HY3D_ERR_ARG;
  if (scale_dtype != HY3D_F16 && scale_dtype != HY3D_BF16) return HY3D_ERR_ARG;
  if (epilogue < HY3D_EPI_LINEAR || epilogue > HY3D_EPI_GEGLU) return HY3D_ERR_ARG;
  if (bias && (bias_dtype < HY3D_F16 || bias_dtype > HY3D_F32)) return HY3D_ERR_ARG;
  if (M < 0 || M > 0x7FFFFFFF || N <= 0 || N > 0x7FFFFFFF || K <= 0 || K > 32768 || (K & 63) || (N & 15)) return HY3D_ERR_SHAPE;
  if (epilogue == HY3D_EPI_GEGLU && (N & 31)) return HY3D_ERR_SHAPE;
  if (group < 32 || (group & 31) || (group != 32 && (group & 63)) || K % group) return HY3D_ERR_SHAPE;
  if (ldx < K || (ldx & 7)) return HY3D_ERR_SHAPE;
  if (M == 0) return HY3D_OK;
  if (!x || !w || !scale || !out) return HY3D_ERR_ARG;
  if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(scale) |
        reinterpret_cast<uintptr_t>(zero)) & 15) || (reinterpret_cast<uintptr_t>(out) & 7))
    return HY3D_ERR_SHAPE;
  int rc = device_ok();
  if (rc != HY3D_OK) return rc;
  const int sms = device_sm_count() > 0 ? device_sm_count() : 148;
  const int r = epilogue == HY3D_EPI_GEGLU ? 2 : 1, sub = group == 32 ? 2 : 1;
  const bool plain = !zero && scale_dtype == x_dtype;
  // Up to 8 tokens the kernel above reads the weights once; up to 64 it may still be the faster one with CTAs for every 8
  // (24 x 1280 -> 1280 3.3 us, the other 5.7; 64 x 4096 -> 4096 18.6 and 12.0).
  const int64_t passes = (M + 7) / 8;
  const Plan p = plan_of(M, N, K, passes, r, sub, plain, sms);
  if (M > 8 && scale_dtype == x_dtype) {
    TcPlan tc = tc_plan(M, N, K);
    if (M > 64 || tc.cycles < p.cycles)
      return gemm(x, x_dtype, ldx, w, scale, zero, group, bias, bias_dtype, out, M, N, K, epilogue, tc, stream);
  }
  Args a;
  a.ldx = ldx;
  a.w = static_cast<const uint4*>(w);
  a.scale = static_cast<const uint32_t*>(scale);
  a.zero = static_cast<const uint8_t*>(zero);
  a.bias = bias;
  a.bias_dtype = bias_dtype;
  a.N = static_cast<int>(N);
  a.K = static_cast<int>(K);
  a.groups = static_cast<int>(K / group);
  const uint64_t group_tiles = group == 32 ? 1 : static_cast<uint64_t>(group / 64);
  a.tiles_inv = static_cast<uint32_t>(((1ull << 31) + group_tiles - 1) / group_tiles);
  a.scale_bf16 = scale_dtype == HY3D_BF16;
  a.epilogue = epilogue;
  a.units = static_cast<int>(N / 16 / r);
  a.tokens = p.tokens;
  a.lg_wk = p.lg_wk;
  a.trips = p.trips;
  const KernelFn kernel = x_dtype == HY3D_BF16 ? kernel_of<true>(r, sub == 2, plain) : kernel_of<false>(r, sub == 2, plain);
  rc = ensure_max_smem(reinterpret_cast<const void*>(kernel), 227 * 1024);
  if (rc != HY3D_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(p.smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1] = {pdl_attribute()};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // A launch takes as many rows as a grid has places in y; the next goes on behind them.
  const int64_t n_out = epilogue == HY3D_EPI_GEGLU ? N / 2 : N, most = kMaxGridY * p.tokens;
  for (int64_t first = 0; first < M; first += most) {
    const int64_t rows = M - first < most ? M - first : most;
    a.x = static_cast<const uint16_t*>(x) + first * ldx;
    a.out = static_cast<uint16_t*>(out) + first * n_out;
    a.M = static_cast<int>(rows);
    cfg.gridDim = dim3(static_cast<unsigned>(p.bx), static_cast<unsigned>((rows + p.tokens - 1) / p.tokens));
    if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess) {
      cudaGetLastError();
      return HY3D_ERR_CUDA;
    }
  }
  return HY3D_OK;
}

}  // namespace w4
}  // namespace hy3d
