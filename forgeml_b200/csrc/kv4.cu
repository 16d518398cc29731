// 4-bit key/value cache: rows quantised as they are written (neb_kv4_append)
// and read back (neb_kv4_read).  Format: kv4.cuh.
#include <cmath>
#include <string>

#include "kv4.cuh"

namespace fml {
namespace kv4 {

// Eight consecutive channels of one row as floats; channels past D give 0 and
// ok[i] false.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int c0, int D, float (&x)[8]) {
  if (VEC) {
    constexpr int N = (int)sizeof(T) / 2;  // 16-byte loads: 1 for 16-bit, 2 for fp32
    uint4 raw[N];
#pragma unroll
    for (int i = 0; i < N; ++i) raw[i] = reinterpret_cast<const uint4*>(p + c0)[i];
    const T* e = reinterpret_cast<const T*>(raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32<T>(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = c0 + i < D ? to_f32<T>(p[c0 + i]) : 0.f;
  }
}

// Codes of eight channels (n of them real) of a group whose four threads are
// neighbouring lanes: the group's s and z, and the codes as eight nibbles.
//
// Quotients.  d = (x - z) / 2 and u = s / 2 (halved so that the widest range
// stays finite; scaled by a power of two when s is tiny so that 1 / u does):
// with y = RN(1 / u), q0 = RN(d y), r = d - q0 u (exact), RN(q0 + r y) is the
// correctly rounded d / u (Markstein 1990).  Numerators of at most 20 bits
// and steps of at most 11 cannot round onto a border k + 1/2 that they do not
// hit, so adding 1.5 * 2^23 (round to nearest even) gives the code of the
// exact quotient for the 16-bit types.  For fp32 the exact remainder,
// including what x - z lost, decides the borders.
template <typename T>
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], int n, float& s_out, float& z_out) {
  float lo = INFINITY, hi = -INFINITY;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (i < n) {
      lo = fminf(lo, x[i]);
      hi = fmaxf(hi, x[i]);
      bad |= !(fabsf(x[i]) <= 3.402823466e38f);
    }
  }
  if (bad) hi = INFINITY;
#pragma unroll
  for (int off = 1; off <= 2; off <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, off));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, off));
  }
  const float half_range = fmaf(0.5f, hi, -0.5f * lo);
  if (!(half_range <= 3.402823466e38f)) {  // an infinity or a NaN in the group
    s_out = z_out = NAN;
    return 0u;
  }
  // (max - min) / 15 rounded to T: for the 16-bit types the difference has few
  // enough bits for one fp32 division; fp32 takes the 64-bit quotient.
  float s;
  if (sizeof(T) == 4) s = (float)(((double)hi - (double)lo) / 15.0);
  else s = to_f32<T>(from_f32<T>(__fdiv_rn(half_range, 7.5f)));
  s_out = s;
  z_out = lo;
  if (s == 0.f) return 0u;
  const float scale = s < 8.6736174e-19f ? 0.5f * 1.1529215e18f : 0.5f;  // 2^-60, 2^60
  const float u = s * scale, y = __frcp_rn(u), z = -lo * scale;
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float d = fmaf(x[i], scale, z);
    const float q0 = d * y;
    float q = fmaf(fmaf(-q0, u, d), y, q0);
    if (sizeof(T) == 4) {
      float c = rintf(q);
      const float xs = x[i] * scale, b = d - xs;
      const float lost = (xs - (d - b)) + (z - b);  // x - z = d + lost exactly
      const float r = fmaf(-c, u, d) + lost, h = 0.5f * u;
      const bool odd = ((int)c & 1) != 0;
      if (r > h || (r == h && odd)) c += 1.f;
      else if (r < -h || (r == -h && odd)) c -= 1.f;
      q = c;
    }
    q = fminf(q, 15.f);
    const uint32_t code = __float_as_uint(q + 12582912.f) & 0xfu;
    if (i < n) w |= code << (4 * i);
  }
  return w;
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

// One thread: eight channels of one head of one token, keys and values.
// blockIdx.y * blockDim.x + threadIdx.x = (head, group, quarter); tokens are
// dealt to blockIdx.x.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
    append_kernel(const T* __restrict__ k, long long ks0, long long ks1, long long ks2, const T* __restrict__ v,
                  long long vs0, long long vs1, long long vs2, const Pool p, const int32_t* __restrict__ slot_of,
                  const int32_t* __restrict__ start_pos, int tq, int tokens) {
  pdl_wait();
  pdl_trigger();
  const int per_head = 4 * p.G;
  const int j = blockIdx.y * blockDim.x + threadIdx.x;
  const int h = j / per_head;
  const bool live = h < p.H;
  const int part = j - h * per_head, g = part >> 2, quarter = part & 3;
  const int c0 = g * kGroup + quarter * 8;
  const int n = live ? max(0, min(8, p.D - c0)) : 0;
  for (int row = blockIdx.x; row < tokens; row += gridDim.x) {
    const int b = row / tq, t = row - b * tq;
    const int slot = slot_of[b], start = start_pos[b];
    if (slot < 0 || slot >= p.slots || start < 0 || start > p.max_seq - 1 - t ||
        written_before(slot_of, start_pos, b, slot, start, tq)) {
      if (threadIdx.x == 0) raise_device_error(DEV_ERR_ATTN_RANGE);
      continue;
    }
    const int pos = start + t;
    uint8_t* const tile = live ? head_tiles(p, slot, h) + (long long)(pos / kTile) * (2 * p.half) : nullptr;
    const int r = pos % kTile;
    float x[2][8];
    if (n > 0) {
      load8<T, VEC>(k + b * ks0 + t * ks1 + h * ks2, c0, p.D, x[0]);
      load8<T, VEC>(v + b * vs0 + t * vs1 + h * vs2, c0, p.D, x[1]);
    }
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      float s, z;
      const uint32_t w = quantise8<T>(x[kv], n, s, z);
      if (live && quarter == 0) {
        T* pr = reinterpret_cast<T*>(tile + kv * p.half + kTile * 16 * p.G) + (r * p.G + g) * 2;
        pr[0] = from_f32<T>(s);
        pr[1] = from_f32<T>(z);
      }
      if (kv == 0) {
        if (live) *reinterpret_cast<uint32_t*>(tile + r * 16 * p.G + k_byte(p.G, c0)) = w;
      } else if (live) {
        uint8_t* vr = tile + p.half + r * 16 * p.G;
        *reinterpret_cast<uint16_t*>(vr + v_byte(p.G, c0, pos)) = (uint16_t)w;
        *reinterpret_cast<uint16_t*>(vr + v_byte(p.G, c0 + 4, pos)) = (uint16_t)(w >> 16);
      }
    }
  }
}

// z + c * s rounded to T, within T's finite range (a rounded-up step can carry
// code 15 of the widest groups past it); NaN stays.
template <typename T>
__device__ __forceinline__ float largest();
template <> __device__ __forceinline__ float largest<float>() { return 3.402823466e38f; }
template <> __device__ __forceinline__ float largest<__half>() { return 65504.f; }
template <> __device__ __forceinline__ float largest<__nv_bfloat16>() { return 3.3895313892515355e38f; }
template <typename T>
__device__ __forceinline__ float value_of(uint32_t code, float s, float z) {
  const float x = fmaf((float)code, s, z);
  return x > largest<T>() ? largest<T>() : x;
}

// out[b, h, i, :] = the numbers that row start + i of request b stands for.
template <typename T>
__global__ void __launch_bounds__(256)
    read_kernel(const Pool p, const int32_t* __restrict__ slot_of, const int32_t* __restrict__ start_pos, int count,
                T* __restrict__ ko, T* __restrict__ vo, long long total) {
  pdl_wait();
  pdl_trigger();
  const int per_row = 4 * p.G;
  for (long long idx = (long long)blockIdx.x * blockDim.x + threadIdx.x; idx < total;
       idx += (long long)gridDim.x * blockDim.x) {
    const int part = (int)(idx % per_row), g = part >> 2;
    const long long o = idx / per_row;  // output row: (b, h, i)
    const int i = (int)(o % count);
    const int h = (int)((o / count) % p.H), b = (int)(o / count / p.H);
    const int c0 = g * kGroup + (part & 3) * 8;
    const int slot = slot_of[b], start = start_pos ? start_pos[b] : 0;
    const bool ok = slot >= 0 && slot < p.slots && start >= 0 && start <= p.max_seq - 1 - i;
    if (!ok) raise_device_error(DEV_ERR_ATTN_RANGE);
    const int pos = ok ? start + i : 0;
    const uint8_t* const tile = ok ? head_tiles(p, slot, h) + (long long)(pos / kTile) * (2 * p.half) : nullptr;
    const int r = pos % kTile;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      T* out = (kv ? vo : ko) + o * p.D;
      float s = 0.f, z = 0.f;
      uint32_t w = 0;
      if (ok) {
        const T* pr = reinterpret_cast<const T*>(tile + kv * p.half + kTile * 16 * p.G) + (r * p.G + g) * 2;
        s = to_f32<T>(pr[0]);
        z = to_f32<T>(pr[1]);
        if (kv == 0) {
          w = *reinterpret_cast<const uint32_t*>(tile + r * 16 * p.G + k_byte(p.G, c0));
        } else {
          const uint8_t* vr = tile + p.half + r * 16 * p.G;
          w = *reinterpret_cast<const uint16_t*>(vr + v_byte(p.G, c0, pos)) |
              (uint32_t) * reinterpret_cast<const uint16_t*>(vr + v_byte(p.G, c0 + 4, pos)) << 16;
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c0 + e < p.D) out[c0 + e] = from_f32<T>(value_of<T>((w >> (4 * e)) & 0xf, s, z));
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
  if (pool->slots > (1 << 30) || pool->heads > (1 << 20) || pool->max_seq > (1 << 30))
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
  const int per_head = 4 * p.G;
  const int lanes = p.H * per_head;
  const int block = lanes >= 256 ? 256 : (lanes + 31) / 32 * 32;
  const long long tokens = batch * t;
  const unsigned gy = (unsigned)((lanes + block - 1) / block);
  const long long gx = std::min<long long>(tokens, std::max<long long>(1, 148LL * 64 / gy));
  constexpr int W = 8;
  auto addressable = [&](const void* x, const int64_t* s) {
    return p.D % W == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && s[0] * sizeof(T) % 16 == 0 &&
           s[1] * sizeof(T) % 16 == 0 && s[2] * sizeof(T) % 16 == 0;
  };
  auto go = [&](auto kernel) {
    return launch_pdl(kernel, dim3((unsigned)gx, gy), dim3(block), 0, st, 1, static_cast<const T*>(k),
                      (long long)ks[0], (long long)ks[1], (long long)ks[2], static_cast<const T*>(v), (long long)vs[0],
                      (long long)vs[1], (long long)vs[2], p, slot_of, start_pos, (int)t, (int)tokens);
  };
  const bool vec = addressable(k, ks) && addressable(v, vs);
  const cudaError_t e = vec ? go(append_kernel<T, true>) : go(append_kernel<T, false>);
  count_launch();
  return check_cuda(e, "neb_kv4_append launch");
}

template <typename T>
static int read(const Pool& p, const int32_t* slot_of, const int32_t* start_pos, int64_t count, void* ko, void* vo,
                int64_t batch, cudaStream_t st) {
  const long long total = batch * p.H * count * 4 * p.G;
  const long long blocks = std::min<long long>((total + 255) / 256, 148LL * 64);
  const cudaError_t e = launch_pdl(read_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, st, 1, p, slot_of, start_pos,
                                   (int)count, static_cast<T*>(ko), static_cast<T*>(vo), total);
  count_launch();
  return check_cuda(e, "neb_kv4_read launch");
}

}  // namespace kv4
}  // namespace fml

using namespace fml;

extern "C" size_t neb_kv4_pool_bytes(int64_t slots, int64_t heads, int64_t max_seq, int64_t head_dim, int dtype) {
  if (slots <= 0 || heads <= 0 || max_seq <= 0 || head_dim <= 0 || head_dim > kv4::kMaxD || !valid_dtype(dtype)) return 0;
  const size_t tiles = (size_t)((max_seq + kv4::kTile - 1) / kv4::kTile);
  return (size_t)slots * (size_t)heads * tiles * 2 * kv4::kTile * (size_t)kv4::groups_of((int)head_dim) *
         (16 + 2 * dtype_size(dtype));
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
