// The 4-bit linear layer of linear_w4.cu for more than a few tokens: tcgen05.mma with the weight rows as M, the tokens as
// N, and the weights unpacked into tensor memory as a 16-bit A operand.
//
// A weight s * (c - z) has up to 4 bits more than its scale, so one 16-bit number would round it, and the output would be
// off by as much again as its own rounding.  Two hold it exactly:
//     hi = round16(s * (c - z)),   -lo = hi - s * (c - z)    (one multiplication, one multiply-add: at most 5 bits are left
//                                                             over, multiples of the scale's own last place)
// and the products of both, the second with the instruction's negation of A, go to the same fp32 accumulator.  That
// doubles the tensor work, which bounds the layer from about 136 tokens a CTA on: 4096 x 4096 -> 4096 takes 174 us, with one
// rounded number it would take 125.  (The other exact way, a sum per group in tensor memory that warps scale and add up in
// registers, took 225 us there with groups of 64: a hand-over every 64 columns is too often.)
//
// A CTA has 128 rows and up to 256 tokens, over a range of K (the CTAs of its cluster have the others, and the sums are
// added through distributed shared memory).  Sixteen warps unpack, 16 rows and every second tile of 64 columns each: the
// codes come through rings in shared memory that a lane has to itself, and go to tensor memory in the fragment order of
// tcgen05.st.16x256b, which the packed layout is made for -- through shared memory A would be written and read at more
// than its bandwidth.  One thread issues the products, one the tokens' TMA loads.
#include "common.cuh"

namespace hy3d {
int resident_clusters(int ranks, int per_sm);
int encode_tmap_2d_u8(CUtensorMap* map, const void* base, uint64_t inner_bytes, uint64_t rows, uint64_t pitch_bytes,
                      uint32_t box_inner, uint32_t box_rows, int swizzle_bytes);
namespace w4 {
namespace {

constexpr int kUnpackWarps = 16, kTcThreads = 32 * (kUnpackWarps + 2);
constexpr int kTcMaxStages = 3, kSumPitch = 132;      // floats of a token's sums
constexpr int kACols = 64;                  // of tensor memory: hi and lo of 128 rows x 64 columns; a stage has two tiles
// A lane's codes, scales and zero points of a tile, all lanes together, and how many tiles a warp's ring holds.
__host__ __device__ constexpr int slot_bytes(int sub, bool plain) { return 512 + 128 * sub * (plain ? 1 : 2); }
__host__ __device__ constexpr int ring_depth(int sub, bool plain) { return slot_bytes(sub, plain) <= 640 ? 8 : 5; }

struct TcArgs {
  const uint16_t* x;
  int64_t ldx;
  const uint4* w;
  const uint32_t* scale;      // pairs (row g, row g + 8)
  const uint8_t* zero;        // the same, a byte each; or null
  const void* bias;
  uint16_t* out;
  uint32_t tiles_inv;
  int M, N, K, groups, epilogue, bias_dtype;
  int tokens, stages, ks, d_cols, tmem_cols;     // tokens of a CTA (a multiple of 16), columns of the accumulator, of all
};

struct TcControl {
  uint64_t full[kTcMaxStages], empty[kTcMaxStages], done;
  uint32_t tmem;
  int abort_flag;
};

// One MMA with A in tensor memory: D[tmem] (+)= A[tmem] * B[smem]^T.
__device__ __forceinline__ void mma_f16_ta(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t desc_hi, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "r"(b_lo), "r"(desc_hi), "r"(idesc), "r"(accumulate) : "memory");
}
// 16 lanes x 32 columns, in the fragment order of tmem_ld_16x256b_x4.
__device__ __forceinline__ void tmem_st_16x256b_x4(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Instruction descriptor for kind::f16: fp32 sums (bits 4-5 = 1), both operands f16 (0) or bf16 (1) in bits 7-9 and 10-12.
__host__ __device__ constexpr uint32_t make_idesc_f16(bool bf16, uint32_t m, uint32_t n) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

constexpr uint32_t kNegateA = 1u << 13;

// The sum of one output as the definition has it, in order, up to the first NaN.  Rolled up: unrolled it needs 94 registers,
// 22 more than the kernel, and those leave the next kernel's blocks less room (924 x 1024 -> 2560 10.8 us instead of 10.6).
template <bool kBf16>
__device__ __noinline__ float sum_by_definition(const TcArgs& a, int token, int row) {
  const int tiles = a.K >> 6, group = a.K / a.groups, half = row >> 3 & 1, g = row & 7;
  const int64_t block = row >> 4;
  const uint16_t* x = a.x + token * a.ldx;
  const uint32_t* w = reinterpret_cast<const uint32_t*>(a.w) + block * tiles * 128 + 16 * g + half;
  float y = 0.0f;
#pragma unroll 1
  for (int k = 0; k < a.K && y == y; k += 32) {
    const int64_t at = (block * a.groups + k / group) * 16 + 2 * g + half;
    const uint16_t bits = reinterpret_cast<const uint16_t*>(a.scale)[at];
    const float scale = kBf16 ? __uint_as_float(static_cast<uint32_t>(bits) << 16) : __half2float(__ushort_as_half(bits));
    const int zero = a.zero ? a.zero[at] : 8;
    float sum = 0.0f;
#pragma unroll 1
    for (int t = 0; t < 4; ++t) {      // columns 4t .. 4t + 3 and 16 + 4t .. 16 + 4t + 3
      const uint32_t codes = w[(k >> 6) * 128 + 4 * t + (k >> 4 & 2)];
#pragma unroll 1
      for (int i = 0; i < 8; ++i) {
        const int code = static_cast<int>(codes >> (4 * (i >> 1) + 16 * (i & 1)) & 15u);
        const uint16_t v = x[k + 4 * t + 16 * (i >> 2) + (i & 3)];
        sum = fmaf(kBf16 ? __uint_as_float(static_cast<uint32_t>(v) << 16) : __half2float(__ushort_as_half(v)),
                   static_cast<float>(code - zero), sum);
      }
    }
    y = fmaf(scale, sum, y);
  }
  return y;
}

// A lane's outputs of a token, packed: from the sums of rows `row` and `row + 1` and of those `gates` behind.
template <bool kBf16>
__device__ __forceinline__ uint2 outputs_of(int epilogue, const float (&y)[4]) {
  constexpr int kType = kBf16 ? HY3D_BF16 : HY3D_F16;
  if (epilogue == HY3D_EPI_GEGLU) {
    const float2 gate = gelu_phi2(make_float2(y[2], y[3]));
    return make_uint2(pack2(y[0] * gate.x, y[1] * gate.y, kType), 0u);
  }
  float2 u = make_float2(y[0], y[1]), v = make_float2(y[2], y[3]);
  if (epilogue == HY3D_EPI_GELU) {
    u = gelu_phi2(u);
    v = gelu_phi2(v);
  }
  return make_uint2(pack2(u.x, u.y, kType), pack2(v.x, v.y, kType));
}

// A running maximum of packed pairs, in which a NaN stays.
template <bool kBf16>
__device__ __forceinline__ uint32_t max_or_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  if (kBf16) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <bool kBf16>
__device__ __forceinline__ bool has_nan(uint32_t w) {
  constexpr uint32_t kInf = kBf16 ? 0x7F80u : 0x7C00u;
  return (w & 0x7FFFu) > kInf || (w >> 16 & 0x7FFFu) > kInf;
}

// kPlain: no zero points.
template <bool kBf16, int kSub, bool kPlain>
__global__ void __launch_bounds__(kTcThreads, 1)
gemm_w4_kernel(const __grid_constant__ TcArgs a, const __grid_constant__ CUtensorMap tm_x) {
  constexpr int kSlot = slot_bytes(kSub, kPlain), kDepth = ring_depth(kSub, kPlain), kZeroAt = 512 + 128 * kSub;
  extern __shared__ uint8_t s_raw[];
  __shared__ TcControl ctrl;
  uint8_t* s_tiles = s_raw + ((1024u - (smem_u32(s_raw) & 1023u)) & 1023u);      // [stage][2] tokens, [warp][slot] codes; at the end sums
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = a.ks > 1 ? static_cast<int>(cluster_cta_rank()) : 0;
  const int row0 = static_cast<int>(blockIdx.x / static_cast<unsigned>(a.ks)) * 128, tok0 = blockIdx.y * a.tokens;
  const int tiles = a.K >> 6;
  const int first = static_cast<int>(static_cast<uint32_t>(tiles) * static_cast<uint32_t>(rank) / static_cast<uint32_t>(a.ks));
  const int end = static_cast<int>(static_cast<uint32_t>(tiles) * static_cast<uint32_t>(rank + 1) / static_cast<uint32_t>(a.ks));
  const int b_bytes = a.tokens * 128, stage_bytes = 2 * b_bytes, n = end - first, pairs = (n + 1) >> 1;
  volatile int* abort_flag = &ctrl.abort_flag;

  if (warp == kUnpackWarps) {
    if (lane == 0) {
      for (int i = 0; i < a.stages; ++i) {
        mbar_init(smem_u32(&ctrl.full[i]), kUnpackWarps + 1);
        mbar_init(smem_u32(&ctrl.empty[i]), 1);
      }
      mbar_init(smem_u32(&ctrl.done), 1);
      ctrl.abort_flag = 0;
      fence_barrier_init();
    }
    __syncwarp();
    tmem_alloc_1cta(smem_u32(&ctrl.tmem), static_cast<uint32_t>(a.tmem_cols));
    tmem_relinquish_1cta();
  } else if (warp == kUnpackWarps + 1 && lane == 0) {
    tma_prefetch_desc(&tm_x);
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = ctrl.tmem, tmem_a = tmem + static_cast<uint32_t>(a.d_cols);
  // Not before every CTA of the grid has its tensor memory: the next kernel takes its own and then waits for this one to
  // end, so a CTA still without would wait for columns that are held until it is done.
  pdl_launch_dependents();

  bool ok = true;
  if (warp < kUnpackWarps) {
    // ---------------- unpack ----------------
    // a warp reaches the 32 lanes of tensor memory that its number modulo 4 names: two blocks of 16 rows, for warps of two
    // kinds; of those, one takes the even tiles and one the odd ones
    const int b = 2 * (warp & 3) + (warp >> 2 & 1), odd = warp >> 3, g = lane >> 2;
    const int64_t block = min((row0 >> 4) + b, (a.N >> 4) - 1);
    const uint4* wp = a.w + (block * tiles + first + odd) * 32 + lane;
    const uint32_t* sp = a.scale + block * a.groups * 8 + g;
    const bool zeros = !kPlain && a.zero;
    const uint8_t* zp = zeros ? a.zero + block * a.groups * 16 + 4 * (g >> 1) : nullptr;
    const int mine = (n - odd + 1) >> 1;
    uint8_t* ring = s_tiles + a.stages * stage_bytes + warp * (kDepth * kSlot);
    if (lane == 0 && mine > 0) bulk_prefetch_l2(wp, (n < 2 * kDepth ? n - odd : 2 * kDepth - 1) * 512);      // while the previous kernel ends
    pdl_wait();
    auto issue = [&](int i, int slot) {
      if (i < mine) {
        const uint32_t to = smem_u32(ring + slot * kSlot);
        copy_async<16>(to + lane * 16, wp + i * 64);
        const int tile = first + odd + 2 * i;
        const int grp = kSub == 2 ? 2 * tile : static_cast<int>(__umulhi(2 * tile, a.tiles_inv));
#pragma unroll
        for (int h = 0; h < kSub; ++h) {
          copy_async<4>(to + 512 + 128 * h + lane * 4, sp + (grp + h) * 8);
          if (zeros) copy_async<4>(to + kZeroAt + 128 * h + lane * 4, zp + (grp + h) * 16);
        }
      }
      copies_commit();
    };
#pragma unroll
    for (int i = 0; i < kDepth - 1; ++i) issue(i, i);
    const uint32_t a_lanes = tmem_a + (static_cast<uint32_t>(16 * b) << 16) + static_cast<uint32_t>(odd * kACols);
    int stage = 0, slot = 0, next = kDepth - 1;
    uint32_t parity = 1;
    uint32_t hi[16], lo[16];           // [16 columns][row g, row g + 8][two pairs]
    auto unpack = [&](int i) {         // my i-th tile
      copies_wait<kDepth - 2>();
      if (i < mine) {
        const uint8_t* from = ring + slot * kSlot;
        const uint4 w = *reinterpret_cast<const uint4*>(from + lane * 16);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t zlo = 0x00080008u, zhi = 0x00080008u;
          if (zeros) {
            const uint32_t z = *reinterpret_cast<const uint32_t*>(from + kZeroAt + 128 * (h % kSub) + lane * 4) >> (16 * (g & 1));
            zlo = (z & 0xFFu) * 0x00010001u;
            zhi = (z >> 8 & 0xFFu) * 0x00010001u;
          }
          const uint32_t sw = *reinterpret_cast<const uint32_t*>(from + 512 + 128 * (h % kSub) + lane * 4);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t s2 = __byte_perm(sw, sw, e ? 0x3232 : 0x1010), minus_s2 = s2 ^ 0x80008000u;
            uint32_t c[4];
            unpack_codes<kBf16>(e ? (h ? w.w : w.y) : (h ? w.z : w.x), minus_of<kBf16>(e ? zhi : zlo), c);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int at = 8 * h + 4 * (j >> 1) + 2 * e + (j & 1);
              if (kBf16) {
                asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(hi[at]) : "r"(c[j]), "r"(s2));
                asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(lo[at]) : "r"(c[j]), "r"(minus_s2), "r"(hi[at]));
              } else {
                asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(hi[at]) : "r"(c[j]), "r"(s2));
                asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(lo[at]) : "r"(c[j]), "r"(minus_s2), "r"(hi[at]));
              }
            }
          }
        }
      }
      issue(i + kDepth - 1, next);
      next = slot;
      if (++slot == kDepth) slot = 0;
    };
    unpack(0);
    for (int i = 0; i < pairs; ++i) {
      ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&ctrl.empty[stage]), parity, abort_flag, kDevTimeoutEmpty)) != 0;
      if (!ok) break;
      if (i < mine) {
        tc_fence_after_sync();
        const uint32_t to = a_lanes + static_cast<uint32_t>(stage * 2 * kACols);
        tmem_st_16x256b_x4(to, hi);
        tmem_st_16x256b_x4(to + kACols / 2, lo);
      }
      if (i + 1 < pairs) unpack(i + 1);          // while the stores are under way
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&ctrl.full[stage]));
      if (++stage == a.stages) {
        stage = 0;
        parity ^= 1;
      }
    }
    copies_wait<0>();
  } else if (warp == kUnpackWarps) {
    // ---------------- products ----------------
    pdl_wait();
    const uint32_t idesc = make_idesc_f16(kBf16, 128, static_cast<uint32_t>(a.tokens));
    const uint64_t desc_const = make_smem_desc(0, 1024, 128);
    const uint32_t desc_hi = static_cast<uint32_t>(desc_const >> 32);
    const uint32_t b_at0 = static_cast<uint32_t>(desc_const) | (smem_u32(s_tiles) >> 4), b_atom = static_cast<uint32_t>(b_bytes) >> 4;
    if (elect_one()) {                 // one thread: nothing here waits for the rest of the warp
      int stage = 0;
      uint32_t parity = 0, a_at = tmem_a, b_at = b_at0, more = 0;
      for (int left = n; left > 0; left -= 2) {
        ok = mbar_wait<true>(smem_u32(&ctrl.full[stage]), parity, abort_flag, kDevTimeoutFull);
        if (!ok) break;
        tc_fence_after_sync();
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if (u == 0 || left > 1) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              mma_f16_ta(tmem, a_at + u * kACols + 8 * k, b_at + u * b_atom + 2 * k, desc_hi, idesc, u + k ? 1u : more);
              mma_f16_ta(tmem, a_at + u * kACols + kACols / 2 + 8 * k, b_at + u * b_atom + 2 * k, desc_hi, idesc | kNegateA, 1u);
            }
          }
        }
        tc_commit_1cta(smem_u32(&ctrl.empty[stage]));
        more = 1;
        a_at += 2 * kACols;
        b_at += 2 * b_atom;
        if (++stage == a.stages) {
          stage = 0;
          parity ^= 1;
          a_at = tmem_a;
          b_at = b_at0;
        }
      }
      if (ok) tc_commit_1cta(smem_u32(&ctrl.done));
    }
  } else {
    // ---------------- tokens ----------------
    pdl_wait();
    if (elect_one()) {
      int stage = 0;
      uint32_t parity = 1;
      for (int at = first; at < end && ok; at += 2) {
        ok = mbar_wait(smem_u32(&ctrl.empty[stage]), parity, abort_flag, kDevTimeoutEmpty);
        if (!ok) break;
        const uint32_t bar = smem_u32(&ctrl.full[stage]), to = smem_u32(s_tiles) + stage * stage_bytes;
        const int count = min(2, end - at);
        mbar_arrive_expect_tx(bar, static_cast<uint32_t>(count * b_bytes));
        for (int u = 0; u < count; ++u) tma_load_2d(to + u * b_bytes, &tm_x, bar, (at + u) * 128, tok0);
        if (++stage == a.stages) {
          stage = 0;
          parity ^= 1;
        }
      }
    }
  }
  __syncwarp();
  // ---------------- outputs ----------------
  // Once the last products are done the stages and rings are free: the sums go there, [token][row], and a loop over the
  // tokens -- short code, run by all warps -- finishes them.  (Straight from the registers it was a few thousand
  // instructions that run once, and fetching those took 10 us.)  With several ranges of K every CTA of the cluster finishes
  // a share of the tokens.
  __syncthreads();
  if (!*abort_flag) mbar_wait(smem_u32(&ctrl.done), 0, abort_flag, kDevTimeoutTmemFull);
  tc_fence_after_sync();
  float* s_sum = reinterpret_cast<float*>(s_tiles);
  __syncthreads();
  if (*abort_flag) {      // copies that may still be in flight land before the shared memory is used again or released
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) { }
    __syncthreads();
  }
  if (warp < kUnpackWarps) {
    const uint32_t from = tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16);
    float* to = s_sum + 32 * (warp & 3) + lane;
#pragma unroll 1
    for (int c = 16 * (warp >> 2); c < a.tokens; c += 64) {
      uint32_t v[16];
      tmem_ld_x16(from + static_cast<uint32_t>(c), v);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 16; ++i) to[(c + i) * kSumPitch] = __uint_as_float(v[i]);
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  // Before the cluster's barrier: a CTA that has tensor memory never waits for one that may be waiting for some.
  if (warp == kUnpackWarps) {
    tc_fence_after_sync();
    tmem_dealloc_1cta(tmem, static_cast<uint32_t>(a.tmem_cols));
  }
  __syncwarp();
  if (a.ks > 1) cluster_sync_all();
  const bool geglu = a.epilogue == HY3D_EPI_GEGLU;
  const int n_out = geglu ? a.N >> 1 : a.N;
  // A lane has four neighbouring rows, or with a gate the values of two outputs: two rows and the two 16 behind them.
  const int local = geglu ? (lane >> 3) * 32 + (lane & 7) * 2 : 4 * lane, gates = geglu ? 16 : 2;
  const int row = row0 + local, col = geglu ? (row >> 5) * 16 + (row & 15) : row;
  float bias[4] = {};
  if (a.bias && row < a.N) {
#pragma unroll
    for (int i = 0; i < 4; ++i) bias[i] = load_scalar(a.bias, a.bias_dtype, row + (i & 1) + (i >> 1) * gates);
  }
  uint32_t seen = 0;
  const uint32_t at0 = smem_u32(s_sum + local);
#pragma unroll 1
  for (int tok = rank + a.ks * warp; tok < a.tokens; tok += a.ks * static_cast<int>(blockDim.x >> 5)) {
    if (tok0 + tok >= a.M || row >= a.N) break;
    const uint32_t at = at0 + tok * (kSumPitch * 4);
    float y[4];
    if (a.ks == 1) {
      const float2 u = *reinterpret_cast<const float2*>(s_sum + tok * kSumPitch + local);
      const float2 v = *reinterpret_cast<const float2*>(s_sum + tok * kSumPitch + local + gates);
      y[0] = u.x; y[1] = u.y; y[2] = v.x; y[3] = v.y;
    } else {
      float2 p[8][2];
#pragma unroll
      for (int c = 0; c < 8; ++c) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          p[c][i] = make_float2(0.0f, 0.0f);
          if (c < a.ks)
            asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(p[c][i].x), "=f"(p[c][i].y)
                         : "r"(map_to_cta(at + i * gates * 4, static_cast<uint32_t>(c))));
        }
      }
      y[0] = y[1] = y[2] = y[3] = 0.0f;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        y[0] += p[c][0].x; y[1] += p[c][0].y;
        y[2] += p[c][1].x; y[3] += p[c][1].y;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] += bias[i];
    const uint2 w = outputs_of<kBf16>(a.epilogue, y);
    uint16_t* out = a.out + static_cast<int64_t>(tok0 + tok) * n_out + col;
    seen = max_or_nan<kBf16>(seen, w.x);
    if (geglu) {
      *reinterpret_cast<uint32_t*>(out) = w.x;
    } else {
      *reinterpret_cast<uint2*>(out) = w;
      seen = max_or_nan<kBf16>(seen, w.y);
    }
  }
  // Two numbers a weight cannot give the sum where an activation is infinite: lo is 0 for most weights, and infinity times that
  // is NaN, where infinity times the weight keeps its sign.  A lane's outputs that are NaN are made once more, from the
  // definition.  (The look for them costs 0.5 %.)
  if (has_nan<kBf16>(seen)) {
    for (int tok = rank + a.ks * warp; tok < a.tokens && tok0 + tok < a.M; tok += a.ks * static_cast<int>(blockDim.x >> 5)) {
      uint16_t* out = a.out + static_cast<int64_t>(tok0 + tok) * n_out + col;
      uint32_t* out2 = reinterpret_cast<uint32_t*>(out);
      if (!has_nan<kBf16>(out2[0]) && (geglu || !has_nan<kBf16>(out2[1]))) continue;
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = sum_by_definition<kBf16>(a, tok0 + tok, row + (i & 1) + (i >> 1) * gates) + bias[i];
      const uint2 w = outputs_of<kBf16>(a.epilogue, y);
      out2[0] = w.x;
      if (!geglu) out2[1] = w.y;
    }
  }
  __syncwarp();
  if (a.ks > 1) cluster_sync_all();      // a CTA's sums stay until the others have read them
}

using TcFn = void (*)(const TcArgs, const CUtensorMap);
template <bool kBf16>
TcFn tc_kernel_of(bool sub, bool plain) {
  if (sub) return plain ? gemm_w4_kernel<kBf16, 2, true> : gemm_w4_kernel<kBf16, 2, false>;
  return plain ? gemm_w4_kernel<kBf16, 1, true> : gemm_w4_kernel<kBf16, 1, false>;
}

}  // namespace

// CTAs along the tokens and along K: the fewest cycles for the busiest SM, at what was measured for a tile (the products of
// T tokens 4 T cycles, the unpacking 540), for a CTA's start and end, and for a cluster's.  Rounds are counted in clusters that
// run at the same time, not in SMs: 15 of eight, and with 16 (148 SMs have room for their
// CTAs) 200 x 8192 -> 2048 took 41.9 us instead of 18.1, 66 x 4096 -> 1024 14.1 instead of 9.4.
TcPlan tc_plan(int64_t M, int64_t N, int64_t K) {
  TcPlan p = {16, 1, INT64_MAX};
  const int64_t bx = (N + 127) / 128, tiles = K / 64, fewest = (M + 255) / 256;
  int64_t at_once[9];
  for (int ks = 1; ks <= 8; ++ks) at_once[ks] = resident_clusters(ks, 1) > 0 ? resident_clusters(ks, 1) : 128 / ks;
  for (int64_t ctas = fewest; ctas <= (M + 15) / 16 && ctas <= fewest + 15; ++ctas) {
    const int64_t t = ((M + ctas - 1) / ctas + 15) / 16 * 16, by = (M + t - 1) / t;
    for (int ks = 1; ks <= 8 && (ks == 1 || tiles >= 4 * ks); ++ks) {
      const int64_t tile = 4 * t > 540 ? 4 * t : 540, waves = (bx * by + at_once[ks] - 1) / at_once[ks];
      const int64_t cycles = waves * ((tiles + ks - 1) / ks * tile + 6000 + 12 * t + (ks > 1 ? 1500 : 0));
      if (cycles < p.cycles) p = {static_cast<int>(t), ks, cycles};
    }
  }
  return p;
}

// Checked arguments; scale of x's type.
int gemm(const void* x, int x_dtype, int64_t ldx, const void* w, const void* scale, const void* zero, int64_t group, const void* bias,
         int bias_dtype, void* out, int64_t M, int64_t N, int64_t K, int epilogue, const TcPlan& plan, cudaStream_t stream) {
  TcArgs a;
  a.ldx = ldx;
  a.w = static_cast<const uint4*>(w);
  a.scale = static_cast<const uint32_t*>(scale);
  a.zero = static_cast<const uint8_t*>(zero);
  a.bias = bias;
  const uint64_t group_tiles = group == 32 ? 1 : static_cast<uint64_t>(group / 64);
  a.tiles_inv = static_cast<uint32_t>(((1ull << 31) + group_tiles - 1) / group_tiles);
  a.N = static_cast<int>(N);
  a.K = static_cast<int>(K);
  a.groups = static_cast<int>(K / group);
  a.epilogue = epilogue;
  a.bias_dtype = bias_dtype;
  const int64_t bx = (N + 127) / 128;
  a.tokens = plan.tokens;
  a.ks = plan.ks;
  const bool plain = !zero, sub = group == 32;
  const int stage_bytes = 2 * a.tokens * 128, rings = kUnpackWarps * ring_depth(sub ? 2 : 1, plain) * slot_bytes(sub ? 2 : 1, plain);
  a.d_cols = (a.tokens + 31) / 32 * 32;
  a.stages = (225 * 1024 - rings) / stage_bytes;
  if (a.stages > (512 - a.d_cols) / (2 * kACols)) a.stages = (512 - a.d_cols) / (2 * kACols);
  if (a.stages > kTcMaxStages) a.stages = kTcMaxStages;
  a.tmem_cols = 32;
  while (a.tmem_cols < a.d_cols + 2 * kACols * a.stages) a.tmem_cols *= 2;
  int smem = a.stages * stage_bytes + rings;
  if (smem < a.tokens * kSumPitch * 4) smem = a.tokens * kSumPitch * 4;
  smem += 1024;
  // One CTA per SM: each takes all 512 columns of tensor memory, so a second could only wait for them.
  if (smem < 120 * 1024) smem = 120 * 1024;
  const TcFn kernel = x_dtype == HY3D_BF16 ? tc_kernel_of<true>(sub, plain) : tc_kernel_of<false>(sub, plain);
  int rc = ensure_max_smem(reinterpret_cast<const void*>(kernel), 226 * 1024);
  if (rc != HY3D_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kTcThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2] = {pdl_attribute(), {}};
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(a.ks);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.ks > 1 ? 2 : 1;
  const int64_t n_out = epilogue == HY3D_EPI_GEGLU ? N / 2 : N, most = kMaxGridY * a.tokens;
  for (int64_t first = 0; first < M; first += most) {      // as many rows as a grid has places in y
    const int64_t rows = M - first < most ? M - first : most;
    a.x = static_cast<const uint16_t*>(x) + first * ldx;
    a.out = static_cast<uint16_t*>(out) + first * n_out;
    a.M = static_cast<int>(rows);
    CUtensorMap tm_x;
    rc = encode_tmap_2d_u8(&tm_x, a.x, static_cast<uint64_t>(2 * K), static_cast<uint64_t>(rows), static_cast<uint64_t>(2 * ldx), 128,
                           static_cast<uint32_t>(a.tokens), 128);
    if (rc != HY3D_OK) return rc;
    cfg.gridDim = dim3(static_cast<unsigned>(bx * a.ks), static_cast<unsigned>((rows + a.tokens - 1) / a.tokens));
    if (cudaLaunchKernelEx(&cfg, kernel, a, tm_x) != cudaSuccess) {
      cudaGetLastError();
      return HY3D_ERR_CUDA;
    }
  }
  return HY3D_OK;
}

}  // namespace w4
}  // namespace hy3d
