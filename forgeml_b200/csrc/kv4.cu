// 4-bit key/value cache: rows quantised as they are written (neb_kv4_append)
// and read back (neb_kv4_read).  Format: kv4.cuh.
#include <algorithm>
#include <cmath>
#include <string>
#include <type_traits>

#include "kv4.cuh"

namespace fml {
namespace kv4 {

// Eight consecutive channels of a row as they lie; those past D repeat the
// last real one (a thread without any repeats channel 0 of its group's first
// thread, which changes neither minimum nor maximum).
template <typename T, bool VEC>
struct Row8 {
  uint4 raw[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p, int c0, int D) {
    if (VEC) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw[i] = __ldcs(reinterpret_cast<const uint4*>(p + min(c0, D - 8)) + i);
    } else {
      T e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = p[min(c0 + i, D - 1)];
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw[i] = reinterpret_cast<const uint4*>(e)[i];
    }
  }
  __device__ __forceinline__ void floats(float (&x)[8]) const {
    const T* e = reinterpret_cast<const T*>(raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32<T>(e[i]);
  }
};

// Minimum and maximum of a group over its four neighbouring lanes; NaN where the
// group holds one.  The 16-bit types compare two numbers at once, and maximum
// and negated minimum travel together.
__device__ __forceinline__ __nv_bfloat162 max2(__nv_bfloat162 a, __nv_bfloat162 b) { return __hmax2_nan(a, b); }
__device__ __forceinline__ __nv_bfloat162 min2(__nv_bfloat162 a, __nv_bfloat162 b) { return __hmin2_nan(a, b); }
__device__ __forceinline__ __half2 max2(__half2 a, __half2 b) { return __hmax2_nan(a, b); }
__device__ __forceinline__ __half2 min2(__half2 a, __half2 b) { return __hmin2_nan(a, b); }
template <typename T2, bool VEC, typename T>
__device__ __forceinline__ void range16(const Row8<T, VEC>& r, float& lo, float& hi) {
  const T2* e = reinterpret_cast<const T2*>(r.raw);
  const T2 mx = max2(max2(e[0], e[1]), max2(e[2], e[3])), mn = min2(min2(e[0], e[1]), min2(e[2], e[3]));
  // (maximum, -minimum) of the two halves
  T2 both;
  both.x = __hmax_nan(mx.x, mx.y);
  both.y = __hneg(__hmin_nan(mn.x, mn.y));
#pragma unroll
  for (int off = 1; off <= 2; off <<= 1) {
    const uint32_t o = __shfl_xor_sync(0xffffffffu, *reinterpret_cast<uint32_t*>(&both), off);
    both = max2(both, *reinterpret_cast<const T2*>(&o));
  }
  hi = to_f32<T>(both.x);
  lo = -to_f32<T>(both.y);
}
template <typename T, bool VEC>
__device__ __forceinline__ void range(const Row8<T, VEC>& r, const float (&x)[8], float& lo, float& hi) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    range16<__nv_bfloat162>(r, lo, hi);
  } else if constexpr (std::is_same<T, __half>::value) {
    range16<__half2>(r, lo, hi);
  } else {
    lo = hi = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
      lo = fminf(lo, x[i]);
      hi = fmaxf(hi, x[i]);
    }
    float sum = 0.f;  // NaN and infinities stay in it
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(x[i], 0.f, sum);
    if (sum != sum) hi = INFINITY;
#pragma unroll
    for (int off = 1; off <= 2; off <<= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, off));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, off));
    }
  }
}

// Codes of eight channels of a group, as eight nibbles, and the group's s and z.
//
// Quotients.  d = (x - z) / 2 and u = s / 2 (halved so that the widest range
// stays finite; scaled by a power of two when s is tiny so that 1 / u does).
// With y near 1 / u, q0 = d y, r = d - q0 u (exact) and q = q0 + r y rounded
// once, q is the quotient rounded to fp32 but for 2^-44 of it (Markstein's
// correction step).  For the 16-bit types, where d is exact, a quotient that is not
// itself a border k + 1/2 is at least 2^-20 of it away from one, so q falls on a border
// only where the quotient does, and adding 1.5 * 2^23 (to nearest, ties to even) gives
// its code.  d is exact where no number is below 2^-16 (bf16) or 2^-13 (fp16) of the
// group's span (`exact`).  Elsewhere the remainder, with what d lost, decides where q is a
// border (the borders times u are exact, so rounding d and q does not pass one); for
// fp32, whose borders are not, it always does.
constexpr float kRound = 12582912.f;  // 1.5 * 2^23
template <typename T> __device__ __forceinline__ float smallest_normal();
template <> __device__ __forceinline__ float smallest_normal<float>() { return 1.17549435e-38f; }
template <> __device__ __forceinline__ float smallest_normal<__half>() { return 6.103515625e-05f; }
template <> __device__ __forceinline__ float smallest_normal<__nv_bfloat16>() { return 1.17549435e-38f; }

// Rounds eight quotients and lays the codes side by side, on the fp32 pipe (the
// integer one is what bounds the kernel).  Adding 16^i q to 1.5 * 2^(23 + 4 i), whose
// last place is 16^i, rounds q to an integer (ties to even: what lies above is a
// multiple of 2 * 16^i) above the codes still to come; taking it down to 1.5 *
// 2^(19 + 4 i) is exact.  Four codes a sum.
__device__ __forceinline__ uint32_t pack4(const float* q) {
  constexpr float k3 = kRound * 4096.f, k2 = kRound * 256.f, k1 = kRound * 16.f;
  float x = __fadd_rn(fmaf(q[3], 4096.f, k3), -(k3 - k2));
  x = __fadd_rn(fmaf(q[2], 256.f, x), -(k2 - k1));
  x = __fadd_rn(fmaf(q[1], 16.f, x), -(k1 - kRound));
  return __float_as_uint(__fadd_rn(x, q[0]));
}
__device__ __forceinline__ uint32_t pack8(const float (&q)[8]) { return __byte_perm(pack4(q), pack4(q + 4), 0x5410); }
__device__ __forceinline__ float near_reciprocal(float u) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(u));
  return y;
}
constexpr float kPerStep = 1.0f / 7.5f;  // s / half_range
// A 16-bit step that needs none of the checks below: whether half_range is large
// enough for a normal step and no underflow, and finite.
template <typename T>
__device__ __forceinline__ bool plain(float half_range) {
  return sizeof(T) == 2 && half_range >= (std::is_same<T, __half>::value ? 5e-4f : 1e-15f) &&
         half_range <= 3.402823466e38f;
}
// Whether x - z is exact in fp32 for a thread's eight numbers and the group's minimum (a
// sufficient condition: numbers of p bits that are at least 2^(p - 24) of the span are
// multiples of the difference's last place).
__device__ __forceinline__ float least2(__nv_bfloat162 a) { return __bfloat162float(__hmin(a.x, a.y)); }
__device__ __forceinline__ float least2(__half2 a) { return __half2float(__hmin(a.x, a.y)); }
template <typename T, bool VEC>
__device__ __forceinline__ bool exact(const Row8<T, VEC>& r, float half_range, float z) {
  if constexpr (sizeof(T) == 4) {
    return true;  // not looked at
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const T2* e = reinterpret_cast<const T2*>(r.raw);
    const float smallest = least2(__hmin2(__hmin2(__habs2(e[0]), __habs2(e[1])), __hmin2(__habs2(e[2]), __habs2(e[3]))));
    return fminf(smallest, fabsf(z)) >= half_range * (std::is_same<T, __half>::value ? 2.44140625e-4f : 3.0517578125e-5f);  // 2^-12, 2^-15
  }
}
// Where a quotient q of d + lost = x - z by u is a border, moves it off to the side that
// the exact remainder says.
__device__ __forceinline__ float off_border(float q, float x, float scale, float zs, float u) {
  if (fabsf(q - rintf(q)) != 0.5f) return q;
  const float xs = x * scale, d = xs + zs, b = d - xs;
  const float lost = (xs - (d - b)) + (zs - b);  // x - z = d + lost exactly
  const float r = fmaf(-q, u, d) + lost;  // (the first is exact; it is 0 or far above what d lost)
  return r > 0.f ? q + 0.25f : r < 0.f ? q - 0.25f : q;
}
template <typename T>
__device__ __forceinline__ uint32_t quantise8_plain(const float (&x)[8], float half_range, float z, bool exact, float& s) {
  const float s0 = half_range * kPerStep;
  s = to_f32<T>(from_f32<T>(fmaf(fmaf(-s0, 7.5f, half_range), kPerStep, s0)));
  const float u = 0.5f * s, zs = -0.5f * z, y = near_reciprocal(u);
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float d = fmaf(x[i], 0.5f, zs), q0 = d * y;
    q[i] = fmaf(fmaf(-q0, u, d), y, q0);
  }
  if (!exact) {
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = off_border(q[i], x[i], 0.5f, zs, u);
  }
  return pack8(q);
}

template <typename T>
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], float half_range, float hi, float& s, float& z) {
  if (!(half_range <= 3.402823466e38f)) {  // an infinity or a NaN in the group
    s = z = NAN;
    return 0u;
  }
  // s = (max - min) / 15 rounded to T.  The 16-bit types' differences have few
  // enough bits for one fp32 quotient (by the same correction step, with the
  // constant 1 / 7.5); fp32 takes the 64-bit one.
  if constexpr (sizeof(T) == 4) {
    s = (float)(((double)hi - (double)z) / 15.0);
  } else {
    const float s0 = half_range * kPerStep;
    s = fmaf(fmaf(-s0, 7.5f, half_range), kPerStep, s0);
    if (half_range < 1e-30f) s = __fdiv_rn(half_range, 7.5f);  // the remainder would underflow
    s = to_f32<T>(from_f32<T>(s));
  }
  if (s == 0.f) return 0u;
  float scale = 0.5f;
  if (s < 8.6736174e-19f) scale = 0.5f * 1.1529215e18f;  // 2^-60, 2^60
  const float u = s * scale, zs = -z * scale, y = near_reciprocal(u);
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float d = fmaf(x[i], scale, zs), q0 = d * y;
    q[i] = fmaf(fmaf(-q0, u, d), y, q0);
    float c = rintf(q[i]);
    const float xs = x[i] * scale, b = d - xs;
    const float lost = (xs - (d - b)) + (zs - b);  // x - z = d + lost exactly
    // the remainder's distance above the upper border and below the lower one; both
    // differences are exact near 0
    const float r = fmaf(-c, u, d), h = 0.5f * u, above = (r - h) + lost, below = (r + h) + lost;
    const bool odd = ((int)c & 1) != 0;
    if (above > 0.f || (above == 0.f && odd)) c += 1.f;
    else if (below < 0.f || (below == 0.f && odd)) c -= 1.f;
    q[i] = c;
  }
  if (s < smallest_normal<T>()) {  // a step without all its bits: quotients may pass 15.5
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = fminf(q[i], 15.f);
  }
  return pack8(q);
}

// Duplicate requests: true when an earlier request of the batch holds the same
// slot and its rows [start, start + tq) overlap this one's.  Whole warp, same b.
__device__ __forceinline__ bool written_before(const int32_t* slot_of, const int32_t* start_pos, int b, int slot,
                                               int start, int tq) {
  bool dup = false;
  for (int i = threadIdx.x & 31; i < b; i += 32)
    if (slot_of[i] == slot) {
      const long long gap = (long long)start_pos[i] - start;
      dup |= gap < tq && gap > -(long long)tq;
    }
  return __any_sync(0xffffffffu, dup);
}

// The values' codes of a group's quarter q (channels 8 q .. 8 q + 7) are the half
// words 2 q and 2 q + 1 of the row's order.  With an even number of groups two
// neighbouring groups (lanes 4 apart) exchange one each, so that both move a
// whole word: the even group's half words 2 q, the odd group's 2 q + 1.
__device__ __forceinline__ uint32_t swap_halves(uint32_t w, bool odd) {
  const uint32_t other = __shfl_xor_sync(0xffffffffu, odd ? w : w >> 16, 4);  // low half counts
  return odd ? __byte_perm(other, w, 0x7610) : __byte_perm(w, other, 0x5410);
}

// Work: 2 bytes read and 0.6 written a number, and some 20 instructions (minimum
// and maximum, the quotient with its correction, rounding, packing), whose issue
// bounds it (0.8 of the slots): 32 x 512 tokens x 16 heads of 128 in bf16 take 47.4
// us, 3.7 TB/s, where the bytes alone take 27.
//
// One thread: eight channels of one head, keys and values, of a run of a
// request's tokens.  threadIdx.x (and blockIdx.y) = (head, group, quarter);
// blockIdx.x = (request, run).
template <typename T, bool VEC>
__global__ void __launch_bounds__(256, 3)  // three blocks an SM (with 87 registers two fit: 54.6 us for 47.4)
    append_kernel(const T* __restrict__ k, long long ks0, long long ks1, long long ks2, const T* __restrict__ v,
                  long long vs0, long long vs1, long long vs2, const Pool p, const int32_t* __restrict__ slot_of,
                  const int32_t* __restrict__ start_pos, int tq, int run, int runs) {
  pdl_wait();
  pdl_trigger();
  const int b = blockIdx.x / runs, t0 = (blockIdx.x - b * runs) * run;
  const int slot = slot_of[b], start = start_pos[b];
  // the run's tokens that have a place
  int t1 = min(tq, t0 + run);
  if (slot < 0 || slot >= p.slots || start < 0 || written_before(slot_of, start_pos, b, slot, start, tq)) t1 = t0;
  else t1 = min(t1, max(t0, p.max_seq - min(start, p.max_seq)));
  if (t1 < min(tq, t0 + run) && threadIdx.x == 0) raise_device_error(DEV_ERR_ATTN_RANGE);
  const int per_head = 4 * p.G;
  const int j = blockIdx.y * blockDim.x + threadIdx.x;
  const bool live = j < p.H * per_head;
  const int h = live ? j / per_head : 0, part = live ? j - h * per_head : 0, g = part >> 2, quarter = part & 3;
  const int c0 = g * kGroup + quarter * 8, n = min(8, max(0, p.D - c0));
  const uint32_t real = n == 8 ? 0xffffffffu : (1u << (4 * n)) - 1;  // codes of real channels
  const int src_c = n > 0 ? c0 : g * kGroup;  // a quarter without channels looks at its group's first
  const T* kr = k + b * ks0 + t0 * ks1 + h * ks2;
  const T* vr = v + b * vs0 + t0 * vs1 + h * vs2;
  uint8_t* const tiles = head_tiles(p, max(slot, 0), h);
  const bool pairs = (p.G & 1) == 0, odd = (g & 1) != 0;
  const int k_at = k_byte(p.G, c0), v_at = v_byte(p.G, pairs ? (g & ~1) * kGroup + quarter * 8 + (odd ? 4 : 0) : c0, 0);
  int r = (start + t0) % kTile;
  uint8_t* tile = tiles + (long long)((start + t0) / kTile) * (2 * p.half);
  // the next token's rows are on their way while this one's are quantised
  Row8<T, VEC> kn, vn;
  if (t0 < t1) {
    kn.load(kr, src_c, p.D);
    vn.load(vr, src_c, p.D);
  }
#pragma unroll 1
  for (int t = t0; t < t1; ++t, kr += ks1, vr += vs1) {
    const Row8<T, VEC> kx = kn, vx = vn;
    if (t + 1 < t1) {
      kn.load(kr + ks1, src_c, p.D);
      vn.load(vr + vs1, src_c, p.D);
    }
    float kf[8], vf[8], ks, kz, k_hi, vs, vz, v_hi;
    kx.floats(kf);
    vx.floats(vf);
    range(kx, kf, kz, k_hi);
    range(vx, vf, vz, v_hi);
    const float k_half = fmaf(0.5f, k_hi, -0.5f * kz), v_half = fmaf(0.5f, v_hi, -0.5f * vz);
    uint32_t kw, vw;
    if (plain<T>(k_half) && plain<T>(v_half)) {
      kw = quantise8_plain<T>(kf, k_half, kz, exact(kx, k_half, kz), ks) & real;
      vw = quantise8_plain<T>(vf, v_half, vz, exact(vx, v_half, vz), vs) & real;
    } else {
      kw = quantise8<T>(kf, k_half, k_hi, ks, kz) & real;
      vw = quantise8<T>(vf, v_half, v_hi, vs, vz) & real;
    }
    uint8_t* const vrow = tile + p.half + r * 16 * p.G;
    const uint32_t vx2 = pairs ? swap_halves(vw, odd) : 0u;
    if (live) {
      *reinterpret_cast<uint32_t*>(tile + r * 16 * p.G + k_at) = kw;
      if (pairs) {
        *reinterpret_cast<uint32_t*>(vrow + (v_at ^ v_swizzle(p.G, r))) = vx2;
      } else {
        *reinterpret_cast<uint16_t*>(vrow + v_at) = (uint16_t)vw;
        *reinterpret_cast<uint16_t*>(vrow + v_at + 2 * p.G) = (uint16_t)(vw >> 16);
      }
      if (quarter < 2) {  // the first lane writes the keys' parameters, the second the values'
        T sz[2] = {from_f32<T>(quarter ? vs : ks), from_f32<T>(quarter ? vz : kz)};
        uint8_t* at = tile + quarter * p.half + kTile * 16 * p.G + (r * p.G + g) * 2 * (int)sizeof(T);
        if (sizeof(T) == 4) *reinterpret_cast<uint2*>(at) = *reinterpret_cast<uint2*>(sz);
        else *reinterpret_cast<uint32_t*>(at) = *reinterpret_cast<uint32_t*>(sz);
      }
    }
    if (++r == kTile) {
      r = 0;
      tile += 2 * p.half;
    }
  }
}

// z + c * s rounded to T, within T's finite range (a rounded-up step can carry
// code 15 of the widest groups past it); NaN stays.  Eight channels of a group.
// The 16-bit types work on pairs: a code under the exponent of 128 (or 1024) is
// 128 + c, exact in both, and one fused product rounds once.
// Only a step of at least half a last place of the largest number / (15 times its own
// rounding) gets there: above the limits below, which are well under that.
template <typename T>
__device__ __forceinline__ bool may_overflow(T s) {
  return to_f32<T>(s) > (std::is_same<T, __half>::value ? 2000.f : 1e36f);
}
template <typename T>
__device__ __forceinline__ void values8(uint32_t w, T s, T z, uint4 (&out)[sizeof(T) / 2]) {
  if constexpr (sizeof(T) == 4) {
    float e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      e[i] = fmaf((float)((w >> (4 * i)) & 0xf), s, z);
    }
    if (may_overflow<T>(s))
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = e[i] > 3.402823466e38f ? 3.402823466e38f : e[i];
#pragma unroll
    for (int i = 0; i < 2; ++i) out[i] = reinterpret_cast<const uint4*>(e)[i];
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    constexpr bool kHalf = std::is_same<T, __half>::value;
    const uint32_t exponent = kHalf ? 0x64006400u : 0x43004300u, top = kHalf ? 0x7bff7bffu : 0x7f7f7f7fu;
    const T2 base = *reinterpret_cast<const T2*>(&exponent), most = *reinterpret_cast<const T2*>(&top);
    T2 s2, z2;
    s2.x = s2.y = s;
    z2.x = z2.y = z;
    uint32_t e[4];  // channels i and i + 4
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t c = ((w >> (4 * i)) & 0x000f000fu) | exponent;
      const T2 x = __hfma2(__hsub2(*reinterpret_cast<const T2*>(&c), base), s2, z2);
      e[i] = *reinterpret_cast<const uint32_t*>(&x);
    }
    if (may_overflow<T>(s))
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const T2 x = min2(*reinterpret_cast<const T2*>(&e[i]), most);
        e[i] = *reinterpret_cast<const uint32_t*>(&x);
      }
    out[0] = make_uint4(__byte_perm(e[0], e[1], 0x5410), __byte_perm(e[2], e[3], 0x5410),
                        __byte_perm(e[0], e[1], 0x7632), __byte_perm(e[2], e[3], 0x7632));
  }
}

// 32 x 2048 positions x 16 heads of 128, bf16: 136 us, 5.2 TB/s (705 MB, three
// quarters of it written).
//
// out[b, h, i, :] = the numbers that row start + i of request b stands for.  A
// thread: eight channels of one row, keys and values; blockIdx.y = (request,
// head), the block's rows side by side, blockIdx.x and steps along the rows.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
    read_kernel(const Pool p, const int32_t* __restrict__ slot_of, const int32_t* __restrict__ start_pos, int count,
                T* __restrict__ ko, T* __restrict__ vo, int heads_first) {
  pdl_wait();
  pdl_trigger();
  const int per_row = 4 * p.G, rows = blockDim.x / per_row;
  const int bh = blockIdx.y + heads_first, b = bh / p.H, h = bh - b * p.H;
  const int sub = threadIdx.x / per_row, part = threadIdx.x - sub * per_row, g = part >> 2, quarter = part & 3;
  const int slot = slot_of[b], start = start_pos ? start_pos[b] : 0;
  const bool in_pool = slot >= 0 && slot < p.slots && start >= 0;
  const uint8_t* const tiles = head_tiles(p, in_pool ? slot : 0, h);
  const int c0 = g * kGroup + quarter * 8;
  const bool pairs = (p.G & 1) == 0, odd = (g & 1) != 0;
  const int k_at = k_byte(p.G, c0), v_at = v_byte(p.G, pairs ? (g & ~1) * kGroup + quarter * 8 + (odd ? 4 : 0) : c0, 0);
#pragma unroll 1  // (unrolled twice: 146 us where this takes 136)
  for (int i0 = blockIdx.x * rows; i0 < count; i0 += gridDim.x * rows) {
    const int i = i0 + sub;
    const bool live = sub < rows && i < count;
    const bool ok = in_pool && live && start <= p.max_seq - 1 - i;
    if (live && !ok) raise_device_error(DEV_ERR_ATTN_RANGE);
    const unsigned pos = ok ? start + i : 0, r = pos % kTile;
    const uint8_t* const tile = tiles + (unsigned long long)(pos / kTile) * (unsigned)(2 * p.half);
    const int at = kTile * 16 * p.G + (r * p.G + g) * 2 * (int)sizeof(T);
    uint32_t kw = 0, vw = 0;
    T kp[2], vp[2];
    kp[0] = kp[1] = vp[0] = vp[1] = from_f32<T>(0.f);
    if (ok) {
      const uint8_t* const vrow = tile + p.half + r * 16 * p.G;
      kw = __ldcs(reinterpret_cast<const uint32_t*>(tile + r * 16 * p.G + k_at));
      if (pairs)
        vw = __ldcs(reinterpret_cast<const uint32_t*>(vrow + (v_at ^ v_swizzle(p.G, pos))));
      else
        vw = *reinterpret_cast<const uint16_t*>(vrow + v_at) |
             (uint32_t) * reinterpret_cast<const uint16_t*>(vrow + v_at + 2 * p.G) << 16;
      if (sizeof(T) == 4) {
        *reinterpret_cast<uint2*>(kp) = *reinterpret_cast<const uint2*>(tile + at);
        *reinterpret_cast<uint2*>(vp) = *reinterpret_cast<const uint2*>(tile + p.half + at);
      } else {
        *reinterpret_cast<uint32_t*>(kp) = *reinterpret_cast<const uint32_t*>(tile + at);
        *reinterpret_cast<uint32_t*>(vp) = *reinterpret_cast<const uint32_t*>(tile + p.half + at);
      }
    }
    if (pairs) vw = swap_halves(vw, odd);  // its own inverse
    uint4 kx[sizeof(T) / 2], vx[sizeof(T) / 2];
    values8<T>(kw, kp[0], kp[1], kx);
    values8<T>(vw, vp[0], vp[1], vx);
    if (!live) continue;
    const long long o = ((long long)bh * count + i) * p.D + c0;
    if (VEC) {
      if (c0 < p.D) {
#pragma unroll
        for (int e = 0; e < (int)sizeof(T) / 2; ++e) {
          __stcs(reinterpret_cast<uint4*>(ko + o) + e, kx[e]);
          __stcs(reinterpret_cast<uint4*>(vo + o) + e, vx[e]);
        }
      }
    } else {
      for (int e = 0; e < 8 && c0 + e < p.D; ++e) {
        ko[o + e] = reinterpret_cast<const T*>(kx)[e];
        vo[o + e] = reinterpret_cast<const T*>(vx)[e];
      }
    }
  }
}

int pool_from(const neb_kv4_pool* pool, const char* who, Pool* p) {
  const std::string name(who);
  if (!pool) return fail(FML_EINVAL, name + ": null pool");
  if (!valid_dtype(pool->dtype)) return fail(FML_EINVAL, name + ": bad dtype");
  if (!pool->data)
    return fail(FML_EINVAL, name + ": null pointer");
  if (pool->slots <= 0 || pool->heads <= 0 || pool->max_seq <= 0 || pool->head_dim <= 0)
    return fail(FML_EINVAL, name + ": sizes must be positive");
  if (pool->head_dim > kMaxD) return fail(FML_EUNSUPPORTED, name + ": head_dim > 256");
  if (pool->slots > (1 << 30) || pool->heads > (1 << 18) || pool->max_seq > (1 << 30))
    return fail(FML_EUNSUPPORTED, name + ": pool too large");
  if (reinterpret_cast<uintptr_t>(pool->data) & 127) return fail(FML_EINVAL, name + ": the pool must be 128-byte aligned");
  p->data = static_cast<uint8_t*>(pool->data);
  p->tiles = (pool->max_seq + kTile - 1) / kTile;
  p->slots = (int)pool->slots;
  p->H = (int)pool->heads;
  p->max_seq = (int)pool->max_seq;
  p->D = (int)pool->head_dim;
  p->G = groups_of(p->D);
  p->half = kTile * p->G * (16 + 2 * (int)dtype_size(pool->dtype));
  return FML_OK;
}

template <typename T>
static int append(const void* k, const int64_t* ks, const void* v, const int64_t* vs, const Pool& p,
                  const int32_t* slot_of, const int32_t* start_pos, int64_t batch, int64_t t, cudaStream_t st) {
  const int lanes = p.H * 4 * p.G;
  const int block = lanes >= 256 ? 256 : (lanes + 31) / 32 * 32;
  const long long gy = (lanes + block - 1) / block;
  // Tokens per block: one while blocks are few, up to 16 where they are many
  // (the request's look-ups and addresses are made once a block: about two waves of
  // blocks, 81 us, against six, 82.4, for 32 x 512 tokens and their reading back).
  const long long spread = 148LL * 6;
  const int run = (int)std::min<long long>(16, std::max<long long>(1, batch * t * gy / spread));
  const long long runs = (t + run - 1) / run;
  auto addressable = [&](const void* x, const int64_t* s) {
    return p.D % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && s[0] * sizeof(T) % 16 == 0 &&
           s[1] * sizeof(T) % 16 == 0 && s[2] * sizeof(T) % 16 == 0;
  };
  auto go = [&](auto kernel) {
    return launch_pdl(kernel, dim3((unsigned)(batch * runs), (unsigned)gy), dim3(block), 0, st, 1,
                      static_cast<const T*>(k), (long long)ks[0], (long long)ks[1], (long long)ks[2],
                      static_cast<const T*>(v), (long long)vs[0], (long long)vs[1], (long long)vs[2], p, slot_of,
                      start_pos, (int)t, run, (int)runs);
  };
  const bool vec = addressable(k, ks) && addressable(v, vs);
  const cudaError_t e = vec ? go(append_kernel<T, true>) : go(append_kernel<T, false>);
  count_launch();
  return check_cuda(e, "neb_kv4_append launch");
}

template <typename T>
static int read(const Pool& p, const int32_t* slot_of, const int32_t* start_pos, int64_t count, void* ko, void* vo,
                int64_t batch, cudaStream_t st) {
  const int per_row = 4 * p.G;
  const int rows = 256 / per_row;
  const int block = (rows * per_row + 31) / 32 * 32;
  const bool vec = p.D % 8 == 0 && reinterpret_cast<uintptr_t>(ko) % 16 == 0 && reinterpret_cast<uintptr_t>(vo) % 16 == 0;
  const long long heads = batch * p.H;
  for (long long first = 0; first < heads; first += 65535) {  // grid.y
    const long long gy = std::min<long long>(65535, heads - first);
    // up to eight steps along the rows a block, where that leaves blocks enough (one:
    // 179 us for 32 x 2048 positions, four 136.4, eight 135.7, sixteen 137.7)
    const long long steps = (count + rows - 1) / rows;
    const long long gx = std::max<long long>(1, std::min(steps, std::max((steps + 7) / 8, 148LL * 16 / gy)));
    auto go = [&](auto kernel) {
      return launch_pdl(kernel, dim3((unsigned)gx, (unsigned)gy), dim3(block), 0, st, 1, p, slot_of, start_pos,
                        (int)count, static_cast<T*>(ko), static_cast<T*>(vo), (int)first);
    };
    const cudaError_t e = vec ? go(read_kernel<T, true>) : go(read_kernel<T, false>);
    count_launch();
    if (e != cudaSuccess) return check_cuda(e, "neb_kv4_read launch");
  }
  return FML_OK;
}

}  // namespace kv4
}  // namespace fml

using namespace fml;

extern "C" size_t neb_kv4_pool_bytes(int64_t slots, int64_t heads, int64_t max_seq, int64_t head_dim, int dtype) {
  if (slots <= 0 || heads <= 0 || max_seq <= 0 || head_dim <= 0 || head_dim > kv4::kMaxD || !valid_dtype(dtype)) return 0;
  if (slots > (1 << 30) || heads > (1 << 18) || max_seq > (1 << 30)) return 0;
  const size_t tiles = (size_t)((max_seq + kv4::kTile - 1) / kv4::kTile);
  const size_t row = 2 * kv4::kTile * (size_t)kv4::groups_of((int)head_dim) * (16 + 2 * dtype_size(dtype));
  const size_t heads_bytes = (size_t)heads * tiles * row;  // below 2^58
  if (heads_bytes > (1ull << 62) / (size_t)slots) return 0;
  return (size_t)slots * heads_bytes;
}

extern "C" int neb_kv4_append(const void* k, const int64_t k_strides[4], const void* v, const int64_t v_strides[4],
                              const neb_kv4_pool* pool, const int32_t* slot_of, const int32_t* start_pos,
                              int64_t batch, int64_t t, void* stream) {
  kv4::Pool p;
  if (const int rc = kv4::pool_from(pool, "neb_kv4_append", &p)) return rc;
  if (!k || !v || !k_strides || !v_strides || !slot_of || !start_pos)
    return fail(FML_EINVAL, "neb_kv4_append: null pointer");
  if (batch <= 0 || t <= 0) return fail(FML_EINVAL, "neb_kv4_append: sizes must be positive");
  if (k_strides[3] != 1 || v_strides[3] != 1)
    return fail(FML_EUNSUPPORTED, "neb_kv4_append: innermost stride must be 1");
  if (t > p.max_seq || batch > (1 << 24) || batch * t > (1ll << 30))
    return fail(FML_EUNSUPPORTED, "neb_kv4_append: too many rows");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (pool->dtype == FML_F32) return kv4::append<float>(k, k_strides, v, v_strides, p, slot_of, start_pos, batch, t, st);
  if (pool->dtype == FML_BF16)
    return kv4::append<__nv_bfloat16>(k, k_strides, v, v_strides, p, slot_of, start_pos, batch, t, st);
  return kv4::append<__half>(k, k_strides, v, v_strides, p, slot_of, start_pos, batch, t, st);
}

extern "C" int neb_kv4_read(const neb_kv4_pool* pool, const int32_t* slot_of, const int32_t* start_pos, int64_t count,
                            void* k_out, void* v_out, int64_t batch, void* stream) {
  kv4::Pool p;
  if (const int rc = kv4::pool_from(pool, "neb_kv4_read", &p)) return rc;
  if (!slot_of || !k_out || !v_out) return fail(FML_EINVAL, "neb_kv4_read: null pointer");
  if (batch <= 0 || count <= 0) return fail(FML_EINVAL, "neb_kv4_read: sizes must be positive");
  if (count > p.max_seq) return fail(FML_EINVAL, "neb_kv4_read: count exceeds max_seq");
  if (batch > (1 << 24)) return fail(FML_EUNSUPPORTED, "neb_kv4_read: too many requests");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (pool->dtype == FML_F32) return kv4::read<float>(p, slot_of, start_pos, count, k_out, v_out, batch, st);
  if (pool->dtype == FML_BF16) return kv4::read<__nv_bfloat16>(p, slot_of, start_pos, count, k_out, v_out, batch, st);
  return kv4::read<__half>(p, slot_of, start_pos, count, k_out, v_out, batch, st);
}
