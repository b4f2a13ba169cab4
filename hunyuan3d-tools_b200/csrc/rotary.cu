// Rotary positions: pairs (u, v) of a head's dimensions turn by an angle proportional to the token's position,
//     (u, v) -> (u cos a - v sin a, v cos a + u sin a) * amplitude,    a = position[axis(i)] * w_i
// for the queries and the keys of one call, out of place or in place, in either direction (the inverse turns by -a).
//
// The angle loses next to nothing at far positions: w_i comes as a 64-bit fraction of a turn, 2^64 w_i / (2 pi) to the
// nearest, so the product with the integer position is the angle modulo one turn by itself -- the integer product wraps
// where the circle does.  Its error is position * 2^-65 turns (4e-10 radians at 2^31, 2e-7 at 2^40), and 2^-32 turns, 1.5e-9
// radians, for the low half that is left out; the fp32 product position * w_i would be off by 0.06 at a million.  There is
// no table of cosines to build, to keep or to outgrow.  The angle's top two bits are its quadrant, and the rest is small
// enough for the Taylor polynomials of sine and cosine.
//
// Bound by HBM: 4 bytes of traffic per value (32768 tokens of 40 heads of 128: 105 us, 6.4 TB/s; 8 x 1 tokens: 2.0 us).
// A thread has the sines and cosines of 8 pairs and turns those of up to 8 heads with them, loads of four heads in flight at
// a time: one head after the other with sincospif took 146 and 3.4.  Where few heads share the sines the instructions count
// as much (2 x 6144 tokens over three axes, 20 heads of 64: 13.2 us, 4.8 TB/s, a thousand instructions per warp of 5 heads;
// with each head's addresses from its strides instead of additions 15.9).
#include "common.cuh"

namespace hy3d {
int device_sm_count();
int device_ok();
namespace rotary {
namespace {

constexpr int kThreads = 128;
constexpr int kMaxPairs = 256;

struct Side {                     // queries or keys
  const uint16_t* src;
  uint16_t* dst;
  int64_t sb, sn, sh, db, dn, dh; // strides of batch, token and head, elements
  int heads, lanes;               // threads of a token that share a unit's heads, lanes apart
};
struct Args {
  Side side[2];
  const void* positions;          // null: the token's index + offset
  int64_t pb, pn, pa, offset;
  int64_t tokens;                 // batch * n
  uint32_t n;                     // tokens of a sequence
  int units, tail_units;          // of a head: turned, and only copied
  uint32_t turn_blocks;           // blocks that turn; the others copy
  int lanes;                      // of both sides
  int half, dim;                  // rotated pairs; dimensions of a head
  float amplitude;
  uint8_t pos64, inverse, small;
  uint8_t axis[kMaxPairs];
  uint64_t turns[kMaxPairs];
};

// kP pairs per unit: kP elements at 2 places, half apart, in both layouts -- interleaved, each of the two vectors holds
// kP / 2 whole pairs.  With one pair nothing is known of the alignment, and its elements are moved one by one.
template <int kBytes>
__device__ __forceinline__ void copy_in(uint32_t* w, const uint16_t* p) {
  if (kBytes == 2) w[0] = *p;
  else if (kBytes == 4) w[0] = *reinterpret_cast<const uint32_t*>(p);
  else if (kBytes == 8) { const uint2 v = *reinterpret_cast<const uint2*>(p); w[0] = v.x; w[1] = v.y; }
  else {
#pragma unroll
    for (int i = 0; i < kBytes / 16; ++i) {
      const uint4 v = reinterpret_cast<const uint4*>(p)[i];
      w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
  }
}
template <int kBytes>
__device__ __forceinline__ void copy_out(uint16_t* p, const uint32_t* w) {
  if (kBytes == 2) *p = static_cast<uint16_t>(w[0]);
  else if (kBytes == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
  else if (kBytes == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  else {
#pragma unroll
    for (int i = 0; i < kBytes / 16; ++i)
      reinterpret_cast<uint4*>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  }
}
template <bool kBf16>
__device__ __forceinline__ float2 widen(uint32_t w) {
  if (kBf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// Sine and cosine of a 64-bit fraction of a turn, whose top 32 bits are given: x = angle past the nearest quarter turn,
// |x| <= pi / 4, where the next terms are below 2.3e-9 (sine, relative) and 3e-8 (cosine).
__device__ __forceinline__ void sincos_turn(uint32_t phase, float& s, float& c) {
  const uint32_t shifted = phase + 0x20000000u, quadrant = shifted >> 30;
  const float x = static_cast<float>(static_cast<int32_t>(shifted & 0x3FFFFFFFu) - 0x20000000) * 1.4629180792671596e-9f;     // 2 pi / 2^32
  const float y = x * x;
  float sine = fmaf(y, 2.7557319e-6f, -1.9841270e-4f), cosine = fmaf(y, 2.4801587e-5f, -1.3888889e-3f);
  sine = fmaf(sine, y, 8.3333333e-3f);
  cosine = fmaf(cosine, y, 4.1666667e-2f);
  sine = fmaf(sine, y, -1.6666667e-1f);
  cosine = fmaf(cosine, y, -0.5f);
  sine = fmaf(sine * y, x, x);
  cosine = fmaf(cosine, y, 1.0f);
  const bool swap = quadrant & 1;
  s = swap ? cosine : sine;
  c = swap ? sine : cosine;
  s = __uint_as_float(__float_as_uint(s) ^ (quadrant & 2) << 30);
  c = __uint_as_float(__float_as_uint(c) ^ ((quadrant + 1) & 2) << 30);
}

constexpr int kBatch = 4;         // heads whose loads are in flight together

// The first blocks turn: a thread has one unit of one token and walks over that token's heads of one side, by additions to
// two addresses.  Neighbouring threads have neighbouring units, then neighbouring heads, the keys' behind the queries'.  The blocks behind them copy the dimensions that
// are not turned, in the same order.
// kAxes: pairs of several axes, each with a position of its own.  Five blocks an SM leave the registers for four heads without
// spills (six: 107 us and 22.8 for 105 and 22.2); with several axes six are better all the same (13.2 us, five 14.9).
template <bool kBf16, bool kInterleaved, int kP, bool kAxes>
__global__ void __launch_bounds__(kThreads, kAxes ? 6 : 5)
rotary_kernel(const __grid_constant__ Args a) {
  __shared__ uint64_t s_turns[kMaxPairs];
  __shared__ uint8_t s_axis[kAxes ? kMaxPairs : 1];
  pdl_launch_dependents();
  constexpr int kType = kBf16 ? HY3D_BF16 : HY3D_F16;
  const bool copies = blockIdx.x >= a.turn_blocks;
  if (!copies) {                  // indexed by lane, the parameter itself would be read one address after the other
    for (int i = threadIdx.x; i < a.half; i += kThreads) {
      s_turns[i] = a.turns[i];
      if (kAxes) s_axis[i] = a.axis[i];
    }
    __syncthreads();
  }
  const int units = copies ? a.tail_units : a.units;
  const int64_t id = static_cast<int64_t>(copies ? blockIdx.x - a.turn_blocks : blockIdx.x) * kThreads + threadIdx.x;
  const uint32_t per_token = static_cast<uint32_t>(a.lanes * units);
  int64_t token, b;
  if (a.small) {                  // a 64-bit division costs as much as the sines
    token = static_cast<uint32_t>(id) / per_token;
    b = static_cast<uint32_t>(token) / a.n;
  } else {
    token = id / per_token;
    b = token / a.n;
  }
  if (token >= a.tokens) return;
  const uint32_t rest = static_cast<uint32_t>(id - token * per_token);
  const int lane = static_cast<int>(rest / static_cast<uint32_t>(units)), unit = static_cast<int>(rest) - lane * units;
  const uint32_t n = static_cast<uint32_t>(token - b * a.n);
  const bool second = lane >= a.side[0].lanes;
  const Side& side = a.side[second];
  const int first_head = second ? lane - a.side[0].lanes : lane, lanes = side.lanes;
  int left = (side.heads - first_head + lanes - 1) / lanes;      // heads to go
  const int64_t step_src = lanes * side.sh, step_dst = lanes * side.dh;
  const uint16_t* src = side.src + b * side.sb + n * side.sn + first_head * side.sh;
  uint16_t* dst = side.dst + b * side.db + n * side.dn + first_head * side.dh;
  pdl_wait();

  if (copies) {
    const int at = 2 * a.half + unit * 2 * kP;
    src += at;
    dst += at;
    for (; left > 0; left -= kBatch) {
      if (kP == 1) {
        for (int j = 0; j < kBatch && j < left; ++j, src += step_src, dst += step_dst) {
          dst[0] = src[0];
          if (at + 1 < a.dim) dst[1] = src[1];
        }
      } else {
        uint32_t w[kBatch][kP];
#pragma unroll
        for (int j = 0; j < kBatch; ++j, src += step_src)
          if (j < left) copy_in<4 * kP>(w[j], src);
#pragma unroll
        for (int j = 0; j < kBatch; ++j, dst += step_dst)
          if (j < left) copy_out<4 * kP>(dst, w[j]);
      }
    }
    return;
  }

  float cs[kP], sn[kP];
  const int at = kInterleaved && kP == 1 ? 2 * unit : unit * kP, apart = kInterleaved && kP == 1 ? 1 : a.half;
  constexpr int kW = kP > 1 ? kP / 2 : 1;
  src += at;
  dst += at;
  for (bool first = true; left > 0; left -= kBatch, first = false) {
    uint32_t u[kBatch][kW], v[kBatch][kW];         // the vectors at the two places
#pragma unroll
    for (int j = 0; j < kBatch; ++j, src += step_src) {
      if (j >= left) continue;
      copy_in<2 * kP>(u[j], src);
      copy_in<2 * kP>(v[j], src + apart);
    }
    if (first) {                        // while the first loads are under way
      const int64_t row = b * a.pb + n * a.pn;
      auto position = [&](int64_t place) {
        return a.pos64 ? static_cast<const int64_t*>(a.positions)[place] : static_cast<int64_t>(static_cast<const int32_t*>(a.positions)[place]);
      };
      const float sine_amplitude = a.inverse ? -a.amplitude : a.amplitude;
      int64_t p = !kAxes && a.positions ? position(row) : a.offset + n;
      int axis = -1;
#pragma unroll
      for (int i = 0; i < kP; ++i) {
        const int pair = kInterleaved && kP > 1 ? unit * kW + i + (i < kW ? 0 : (a.half >> 1) - kW) : unit * kP + i;
        if (kAxes && s_axis[pair] != axis) {       // neighbouring pairs are of one axis mostly
          axis = s_axis[pair];
          p = position(row + axis * a.pa);
        }
        sincos_turn(static_cast<uint32_t>(static_cast<uint64_t>(p) * s_turns[pair] >> 32), sn[i], cs[i]);      // modulo one turn
        cs[i] *= a.amplitude;
        sn[i] *= sine_amplitude;
      }
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j, dst += step_dst) {
      if (j >= left) continue;
      if (kP == 1) {
        const float2 f = widen<kBf16>(u[j][0] | v[j][0] << 16);
        const uint32_t w = pack2(fmaf(f.x, cs[0], -f.y * sn[0]), fmaf(f.y, cs[0], f.x * sn[0]), kType);
        u[j][0] = w & 0xFFFFu;
        v[j][0] = w >> 16;
      } else if (kInterleaved) {
#pragma unroll
        for (int i = 0; i < kP; ++i) {
          uint32_t& w = i < kW ? u[j][i % kW] : v[j][i % kW];
          const float2 f = widen<kBf16>(w);
          w = pack2(fmaf(f.x, cs[i], -f.y * sn[i]), fmaf(f.y, cs[i], f.x * sn[i]), kType);
        }
      } else {
#pragma unroll
        for (int i = 0; i < kW; ++i) {
          const float2 fu = widen<kBf16>(u[j][i]), fv = widen<kBf16>(v[j][i]);
          const float2 c = make_float2(cs[2 * i], cs[(2 * i + 1) % kP]), s = make_float2(sn[2 * i], sn[(2 * i + 1) % kP]);
          const float2 x = __ffma2_rn(fu, c, __fmul2_rn(fv, make_float2(-s.x, -s.y))), y = __ffma2_rn(fv, c, __fmul2_rn(fu, s));
          u[j][i] = pack2(x.x, x.y, kType);
          v[j][i] = pack2(y.x, y.y, kType);
        }
      }
      copy_out<2 * kP>(dst, u[j]);
      copy_out<2 * kP>(dst + apart, v[j]);
    }
  }
}

using KernelFn = void (*)(const Args);
template <bool kBf16, bool kInterleaved, bool kAxes>
KernelFn kernel_of(int pairs) {
  switch (pairs) {
    case 8: return rotary_kernel<kBf16, kInterleaved, 8, kAxes>;
    case 4: return rotary_kernel<kBf16, kInterleaved, 4, kAxes>;
    case 2: return rotary_kernel<kBf16, kInterleaved, 2, kAxes>;
    default: return rotary_kernel<kBf16, kInterleaved, 1, kAxes>;
  }
}

}  // namespace

int apply(const hy3d_rotary_side* sides, int n_sides, int dtype, int64_t batch, int64_t n, int dim, int rot, int interleaved,
          const void* positions, int pos64, int64_t pb, int64_t pn, int64_t pa, int64_t offset, const uint64_t* turns,
          const uint8_t* axis, float amplitude, int inverse, cudaStream_t stream) {
  if (dtype != HY3D_F16 && dtype != HY3D_BF16) return HY3D_ERR_ARG;
  if (!sides || n_sides < 1 || n_sides > 2 || !turns || !axis) return HY3D_ERR_ARG;
  if (batch < 0 || n < 0 || n > 0x7FFFFFFF || dim <= 0 || rot <= 0 || (rot & 1) || rot > dim || rot > 2 * kMaxPairs) return HY3D_ERR_SHAPE;
  if (batch == 0 || n == 0) return HY3D_OK;
  if (batch > INT64_MAX / n) return HY3D_ERR_SHAPE;
  Args a = {};
  a.half = rot / 2;
  a.dim = dim;
  a.n = static_cast<uint32_t>(n);
  a.tokens = batch * n;
  bool in_place = true;
  for (int i = 0; i < n_sides; ++i) {
    const hy3d_rotary_side& s = sides[i];
    if (s.heads < 0 || s.heads > 1 << 20) return HY3D_ERR_SHAPE;
    if (s.heads > 0 && (!s.src || !s.dst)) return HY3D_ERR_ARG;
    if ((reinterpret_cast<uintptr_t>(s.src) | reinterpret_cast<uintptr_t>(s.dst)) & 1) return HY3D_ERR_SHAPE;
    a.side[i] = {static_cast<const uint16_t*>(s.src), static_cast<uint16_t*>(s.dst), s.src_b, s.src_n, s.src_h, s.dst_b, s.dst_n, s.dst_h, s.heads, 0};
    in_place = in_place && (s.heads == 0 || s.src == s.dst);
  }
  if (a.side[0].heads + a.side[1].heads == 0) return HY3D_OK;
  // Pairs of a unit: the most whose vectors are whole and aligned everywhere.
  const int tail = in_place ? 0 : dim - rot;
  int pairs = 8;
  for (; pairs > 1; pairs >>= 1) {
    if (a.half % pairs || tail % (2 * pairs)) continue;
    // 2 * pairs bytes at multiples of that; the copied rest: 4 * pairs bytes, as 16-byte vectors at most
    const int el = tail ? 2 * pairs : pairs, align = el < 8 ? el : 8;
    uint64_t all = 0;
    for (int i = 0; i < n_sides; ++i) {
      const hy3d_rotary_side& s = sides[i];
      if (s.heads == 0) continue;
      all |= reinterpret_cast<uintptr_t>(s.src) / 2 | reinterpret_cast<uintptr_t>(s.dst) / 2;
      if (batch > 1) all |= static_cast<uint64_t>(s.src_b) | static_cast<uint64_t>(s.dst_b);
      if (n > 1) all |= static_cast<uint64_t>(s.src_n) | static_cast<uint64_t>(s.dst_n);
      if (s.heads > 1) all |= static_cast<uint64_t>(s.src_h) | static_cast<uint64_t>(s.dst_h);
    }
    if ((all & (align - 1)) == 0 && (!tail || rot % align == 0)) break;
  }
  a.units = a.half / pairs;
  a.tail_units = (tail + 2 * pairs - 1) / (2 * pairs);
  const int rc = device_ok();
  if (rc != HY3D_OK) return rc;
  // Heads of a thread: up to 8 share its sines and cosines; fewer where that leaves an SM less than 1024 threads.
  const int sms = device_sm_count() > 0 ? device_sm_count() : 148;
  for (int per = 8; per > 0; per >>= 1) {
    a.lanes = 0;
    for (Side& side : a.side) a.lanes += side.lanes = (side.heads + per - 1) / per;
    if (a.tokens * a.units * a.lanes >= static_cast<int64_t>(sms) * 1024) break;
  }
  a.positions = positions;
  a.pos64 = pos64 != 0;
  a.pb = pb;
  a.pn = pn;
  a.pa = pa;
  a.offset = offset;
  a.amplitude = amplitude;
  a.inverse = inverse != 0;
  bool many_axes = false;         // without positions every axis has the token's index
  for (int i = 0; i < a.half; ++i) {
    a.turns[i] = turns[i];
    a.axis[i] = axis[i];
    if (axis[i] && positions) many_axes = true;
  }
  const int64_t per_token = static_cast<int64_t>(a.lanes) * a.units, per_tail = static_cast<int64_t>(a.lanes) * a.tail_units;
  const int64_t most = per_token > per_tail ? per_token : per_tail;
  if (most > 0x3FFFFFFF || a.tokens > (int64_t{0x3FFFFFFF} * kThreads) / most) return HY3D_ERR_SHAPE;
  a.small = a.tokens * most <= 0xFFFFFFFFll - kThreads;
  a.turn_blocks = static_cast<uint32_t>((a.tokens * per_token + kThreads - 1) / kThreads);
  const uint32_t copy_blocks = static_cast<uint32_t>((a.tokens * per_tail + kThreads - 1) / kThreads);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.turn_blocks + copy_blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1] = {pdl_attribute()};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const KernelFn kernel =
      many_axes ? (dtype == HY3D_BF16 ? (interleaved ? kernel_of<true, true, true>(pairs) : kernel_of<true, false, true>(pairs))
                                      : (interleaved ? kernel_of<false, true, true>(pairs) : kernel_of<false, false, true>(pairs)))
                : (dtype == HY3D_BF16 ? (interleaved ? kernel_of<true, true, false>(pairs) : kernel_of<true, false, false>(pairs))
                                      : (interleaved ? kernel_of<false, true, false>(pairs) : kernel_of<false, false, false>(pairs)));
  if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess) {
    cudaGetLastError();
    return HY3D_ERR_CUDA;
  }
  return HY3D_OK;
}

}  // namespace rotary
}  // namespace hy3d
