// Rotary positions: pairs (u, v) of a head's dimensions turn by an angle proportional to the token's position,
//     (u, v) -> (u cos a - v sin a, v cos a + u sin a) * amplitude,    a = position[axis(i)] * w_i
// for the queries and the keys of one call, out of place or in place, in either direction (the inverse turns by -a).
//
// The angle is exact at any position: w_i comes as a 64-bit fraction of a turn, 2^64 w_i / (2 pi), so the product with
// the integer position is the angle modulo one turn by itself -- the integer product wraps where the circle does.  Its
// error is position * 2^-65 turns; the fp32 product position * w_i would be off by 0.06 radians at a million.  There is
// no table of cosines to build, to keep or to outgrow.
#include "common.cuh"

namespace hy3d {
int device_sm_count();
int device_ok();
namespace rotary {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 256;

struct Side {                     // queries or keys
  const uint16_t* src;
  uint16_t* dst;
  int64_t sb, sn, sh, db, dn, dh; // strides of batch, token and head, elements
};
struct Args {
  Side side[2];
  const void* positions;          // null: the token's index + offset
  int64_t pb, pn, pa, offset;
  int64_t tokens;                 // batch * n
  uint32_t n;                     // tokens of a sequence
  int heads0, heads;              // of the first side, of both
  int units, units_all;           // rotated units of a head, and with those that are only copied
  int lanes_h;                    // threads of a token that share a unit's heads
  int half, dim;                  // rotated pairs; dimensions of a head
  float amplitude;
  uint8_t pos64, inverse, small;
  uint8_t axis[kMaxPairs];
  uint64_t turns[kMaxPairs];
};

// kP pairs per unit.  Half layout: kP elements at 2 places, half apart; interleaved: 2 kP adjacent elements.  With one
// pair nothing is known of the alignment, and elements are moved one by one.
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

// A thread has one unit of one token and walks over that token's heads, lanes_h apart: the sines and cosines are
// computed once for all of them.  Neighbouring threads have neighbouring units, then neighbouring heads.
template <bool kBf16, bool kInterleaved, int kP>
__global__ void __launch_bounds__(kThreads)
rotary_kernel(const __grid_constant__ Args a) {
  pdl_launch_dependents();
  constexpr int kType = kBf16 ? HY3D_BF16 : HY3D_F16;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const uint32_t per_token = static_cast<uint32_t>(a.lanes_h * a.units_all);
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
  const int first_head = rest / a.units_all, unit = rest - first_head * a.units_all;
  const uint32_t n = static_cast<uint32_t>(token - b * a.n);
  pdl_wait();

  if (unit >= a.units) {          // dimensions behind the rotated ones
    const int at = 2 * a.half + (unit - a.units) * 2 * kP;
    for (int h = first_head; h < a.heads; h += a.lanes_h) {
      const Side& s = a.side[h >= a.heads0];
      const int hh = h >= a.heads0 ? h - a.heads0 : h;
      const uint16_t* src = s.src + b * s.sb + n * s.sn + hh * s.sh + at;
      uint16_t* dst = s.dst + b * s.db + n * s.dn + hh * s.dh + at;
      if (kP == 1) {
        dst[0] = src[0];
        if (at + 1 < a.dim) dst[1] = src[1];
      } else {
        uint32_t w[kP];
        copy_in<4 * kP>(w, src);
        copy_out<4 * kP>(dst, w);
      }
    }
    return;
  }

  float cs[kP], sn[kP];
#pragma unroll
  for (int i = 0; i < kP; ++i) {
    const int pair = unit * kP + i;
    int64_t p = a.offset + n;
    if (a.positions) {
      const int64_t at = b * a.pb + n * a.pn + a.axis[pair] * a.pa;
      p = a.pos64 ? static_cast<const int64_t*>(a.positions)[at] : static_cast<const int32_t*>(a.positions)[at];
    }
    const uint64_t phase = static_cast<uint64_t>(p) * a.turns[pair];                       // modulo one turn
    const float t = static_cast<float>(static_cast<int32_t>(phase >> 32)) * 4.656612873077393e-10f;   // half turns, [-1, 1)
    sincospif(t, &sn[i], &cs[i]);
    cs[i] *= a.amplitude;
    sn[i] *= a.inverse ? -a.amplitude : a.amplitude;
  }
  for (int h = first_head; h < a.heads; h += a.lanes_h) {
    const Side& s = a.side[h >= a.heads0];
    const int hh = h >= a.heads0 ? h - a.heads0 : h;
    const uint16_t* src = s.src + b * s.sb + n * s.sn + hh * s.sh;
    uint16_t* dst = s.dst + b * s.db + n * s.dn + hh * s.dh;
    if (kInterleaved) {
      uint32_t w[kP];
      if (kP == 1) w[0] = src[unit * 2] | static_cast<uint32_t>(src[unit * 2 + 1]) << 16;
      else copy_in<4 * kP>(w, src + unit * 2 * kP);
#pragma unroll
      for (int i = 0; i < kP; ++i) {
        const float2 f = widen<kBf16>(w[i]);
        w[i] = pack2(fmaf(f.x, cs[i], -f.y * sn[i]), fmaf(f.y, cs[i], f.x * sn[i]), kType);
      }
      if (kP == 1) {
        dst[unit * 2] = static_cast<uint16_t>(w[0]);
        dst[unit * 2 + 1] = static_cast<uint16_t>(w[0] >> 16);
      } else {
        copy_out<4 * kP>(dst + unit * 2 * kP, w);
      }
    } else {
      constexpr int kW = kP > 1 ? kP / 2 : 1;
      uint32_t u[kW], v[kW];
      copy_in<2 * kP>(u, src + unit * kP);
      copy_in<2 * kP>(v, src + a.half + unit * kP);
#pragma unroll
      for (int i = 0; i < kW; ++i) {
        const float2 fu = widen<kBf16>(u[i]), fv = widen<kBf16>(v[i]);
        const float c1 = kP > 1 ? cs[(2 * i + 1) % kP] : 0.0f, s1 = kP > 1 ? sn[(2 * i + 1) % kP] : 0.0f;
        u[i] = pack2(fmaf(fu.x, cs[2 * i], -fv.x * sn[2 * i]), fmaf(fu.y, c1, -fv.y * s1), kType);
        v[i] = pack2(fmaf(fv.x, cs[2 * i], fu.x * sn[2 * i]), fmaf(fv.y, c1, fu.y * s1), kType);
      }
      copy_out<2 * kP>(dst + unit * kP, u);
      copy_out<2 * kP>(dst + a.half + unit * kP, v);
    }
  }
}

using KernelFn = void (*)(const Args);
template <bool kBf16, bool kInterleaved>
KernelFn kernel_of(int pairs) {
  switch (pairs) {
    case 8: return rotary_kernel<kBf16, kInterleaved, 8>;
    case 4: return rotary_kernel<kBf16, kInterleaved, 4>;
    case 2: return rotary_kernel<kBf16, kInterleaved, 2>;
    default: return rotary_kernel<kBf16, kInterleaved, 1>;
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
    a.side[i] = {static_cast<const uint16_t*>(s.src), static_cast<uint16_t*>(s.dst), s.src_b, s.src_n, s.src_h, s.dst_b, s.dst_n, s.dst_h};
    a.heads += s.heads;
    if (i == 0) a.heads0 = s.heads;
    in_place = in_place && (s.heads == 0 || s.src == s.dst);
  }
  if (a.heads == 0) return HY3D_OK;
  // Pairs of a unit: the most whose vectors are whole and aligned everywhere.
  const int tail = in_place ? 0 : dim - rot;
  int pairs = 8;
  for (; pairs > 1; pairs >>= 1) {
    if (a.half % pairs || tail % (2 * pairs)) continue;
    // half: 2 * pairs bytes at multiples of that; interleaved, and the copied rest: 4 * pairs bytes, as 16-byte vectors at most
    const int el = (interleaved || tail) ? 2 * pairs : pairs, align = el < 8 ? el : 8;
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
  a.units_all = a.units + (tail + 2 * pairs - 1) / (2 * pairs);
  const int rc = device_ok();
  if (rc != HY3D_OK) return rc;
  // Heads of a thread: up to 8 share its sines and cosines; fewer where there are too few tokens to fill the SMs.
  const int sms = device_sm_count() > 0 ? device_sm_count() : 148;
  int per = 8;
  while (per > 1 && a.tokens * a.units_all * ((a.heads + per - 1) / per) < static_cast<int64_t>(sms) * 2048) per >>= 1;
  a.lanes_h = (a.heads + per - 1) / per;
  a.positions = positions;
  a.pos64 = pos64 != 0;
  a.pb = pb;
  a.pn = pn;
  a.pa = pa;
  a.offset = offset;
  a.amplitude = amplitude;
  a.inverse = inverse != 0;
  for (int i = 0; i < a.half; ++i) {
    a.turns[i] = turns[i];
    a.axis[i] = axis[i];
  }
  const int64_t per_token = static_cast<int64_t>(a.lanes_h) * a.units_all;
  if (per_token > 0x7FFFFFFF || a.tokens > (int64_t{0x7FFFFFFF} * kThreads) / per_token) return HY3D_ERR_SHAPE;
  a.small = a.tokens * per_token <= 0xFFFFFFFFll - kThreads;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((a.tokens * per_token + kThreads - 1) / kThreads));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1] = {pdl_attribute()};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const KernelFn kernel = dtype == HY3D_BF16 ? (interleaved ? kernel_of<true, true>(pairs) : kernel_of<true, false>(pairs))
                                             : (interleaved ? kernel_of<false, true>(pairs) : kernel_of<false, false>(pairs));
  if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess) {
    cudaGetLastError();
    return HY3D_ERR_CUDA;
  }
  return HY3D_OK;
}

}  // namespace rotary
}  // namespace hy3d
