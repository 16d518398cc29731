// Attention over the 4-bit key/value cache (neb_kv4_attention).
//
//   out[b,t,h,:] = sum_j p_j v_j,  p = softmax_j(scale * q[b,t,h,:] . k_j),
//   j = 0 .. start_pos[b] + t,     k_j, v_j = z + c s per group (kv4.cuh)
//
// Per group of 32 channels the row's step and minimum leave the sums:
//   q . k_j = sum_g s_g[j] (q_g . c_g[j]) + z_g[j] sum(q_g)
//   out_g   = sum_j (p_j s_g[j]) c_g[j] + sum_j p_j z_g[j]
// so the matrix instructions multiply the codes themselves, as 8-bit integers
// (mma.sync m16n8k32, exact 32-bit sums).  A byte of the cache holds two codes,
// lo + 16 hi.  It is used twice: as it lies, and with its upper half masked off:
//   16 (q0 lo + q1 hi) = q1 (lo + 16 hi) + (16 q0 - q1) lo
//   sum P hi = (sum P (lo + 16 hi) - sum P lo) / 16
// so eight codes cost one logic instruction for the keys.  (Spreading them into
// bfloat16 operands costs seven, and the integer ALU was what bounded that
// form: 44 us against 15 us for 64 requests of 128 .. 2303 positions.)
//
// What is rounded: q to 27 bits below its largest channel (four 8-bit digits;
// the 16-bit types and all but the smallest channels of fp32 are exact), the
// weights p s to 16 bits below their running bound (two digits; three, 23
// bits, for fp16 and fp32, whose outputs keep more bits than bf16's).  Scores,
// maxima, sums and outputs are fp32.
#include <algorithm>
#include <string>
#include <type_traits>

#include "kv4.cuh"

namespace fml {
namespace kv4 {

// Each warp is a worker with its own contiguous share of all (request, query
// row) segments of the batch, counted in units of 32 positions, so the work is
// even whatever the lengths are.  A worker streams its units through its own
// ring of shared memory with cp.async and keeps a running maximum, sum and
// output; a segment that it holds whole is written out, the others leave
// (maximum, sum, output) in the workspace for the join kernel.
constexpr int kUnit = 32;
constexpr int kWarps = 4;
constexpr int kStages = 2;

template <typename T> struct Parts { static constexpr int p = 3; };
template <> struct Parts<__nv_bfloat16> { static constexpr int p = 2; };

template <typename T, int G>
struct Unit {
  static constexpr int SETS = (G + 3) / 4;           // groups are handled four at a time
  static constexpr int CR = 16 * G;                  // bytes of a row's codes
  static constexpr int PR = 2 * G * (int)sizeof(T);  // bytes of a row's parameters
  static constexpr int kc = 0, vc = kUnit * CR, kp = 2 * kUnit * CR, vp = kp + kUnit * PR;
  static constexpr int bytes = vp + kUnit * PR;
  // A warp's shared memory: the ring, the scores' parts [set][8][36] fp32 (36:
  // distinct banks), the weights' digits [set][8 or 16][32].
  static constexpr int dots = kStages * bytes;
  static constexpr int digits = dots + SETS * 8 * 36 * 4;
  static constexpr int warp_bytes = digits + SETS * (Parts<T>::p == 3 ? 16 : 8) * 32;
  // CTAs per SM, by registers: the sums of every group (of three digits twice).
  static constexpr int resident = G > 4 ? 2 : G == 4 && Parts<T>::p == 3 ? 3 : 4;
  static_assert(resident * (kWarps * warp_bytes + 1024) <= 227 * 1024, "shared memory");
};

struct Problem {
  const int32_t *slot_of, *start_pos;
  int B, tq, QH, group;  // group: query heads of a key/value head
  long long qs0, qs1, qs2;
  float scale_log2;  // softmax scale * log2(e)
  const void* q;
  void* out;
  float* ws;  // [worker][first / last segment][4 + 32 G]: maximum, sum, -, -, output
};

// Positions that request b's last query attends; 0 for a bad slot or position.
__device__ __forceinline__ int keys_of(const Pool& p, const Problem& a, int b) {
  const int slot = a.slot_of[b], start = a.start_pos[b];
  if (slot < 0 || slot >= p.slots || start < 0 || start >= p.max_seq) return 0;
  return min(start + a.tq, p.max_seq);
}
__device__ __forceinline__ int units_of(int keys) { return (keys + kUnit - 1) / kUnit; }

// Where a worker is.  A request's segments are its query rows, (head, token)
// in this order, each of all the request's units (an earlier token's last
// units may be masked whole).
struct Cursor {
  int b, seg, unit, keys, units;
  int segs;  // segments of a request
  __device__ __forceinline__ void request(const Pool& p, const Problem& a, int nb) {
    b = nb;
    keys = units = 0;
    while (b < a.B) {
      keys = keys_of(p, a, b);
      units = units_of(keys);
      if (units > 0) break;
      ++b;
    }
  }
  __device__ __forceinline__ void next(const Pool& p, const Problem& a) {
    if (++unit < units) return;
    unit = 0;
    if (++seg < segs) return;
    seg = 0;
    request(p, a, b + 1);
  }
};

// Units of the whole batch; the whole warp calls.
__device__ __forceinline__ long long all_units(const Pool& p, const Problem& a, int segs) {
  long long n = 0;
  for (int i = threadIdx.x & 31; i < a.B; i += 32) n += units_of(keys_of(p, a, i));
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) n += __shfl_xor_sync(0xffffffffu, n, off);
  return n * segs;
}

// The unit at place `at` of the batch's order (request, segment, unit); the
// whole warp calls, 0 <= at < all_units.
__device__ __forceinline__ Cursor seek(const Pool& p, const Problem& a, int segs, long long at) {
  Cursor c;
  c.segs = segs;
  const int lane = threadIdx.x & 31;
  long long before = 0;
  for (int base = 0; base < a.B; base += 32) {
    const int i = base + lane;
    const long long mine = i < a.B ? (long long)units_of(keys_of(p, a, i)) * segs : 0;
    long long incl = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long o = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += o;
    }
    const unsigned past = __ballot_sync(0xffffffffu, before + incl > at);
    if (past) {
      const int l = __ffs(past) - 1;
      const long long rest = at - before - __shfl_sync(0xffffffffu, incl - mine, l);
      c.request(p, a, base + l);
      c.seg = (int)(rest / c.units);
      c.unit = (int)(rest - (long long)c.seg * c.units);
      return c;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  c.b = a.B;
  c.seg = c.unit = c.keys = c.units = 0;
  return c;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Copies a unit's first nk rows into a stage (the rest of the stage keeps what
// it held and is masked).  Copies are whole 16 bytes: up to 15 rows' worth of
// parameters past nk, inside the head's padded rows.
template <typename T, int G>
__device__ __forceinline__ void load_unit(const Pool& p, long long row, int nk, uint32_t dst) {
  using U = Unit<T, G>;
  const int lane = threadIdx.x & 31;
  const uint8_t* kc = p.kc + row * U::CR + lane * 16;
  const uint8_t* vc = p.vc + row * U::CR + lane * 16;
  const uint8_t* kp = static_cast<const uint8_t*>(p.kp) + row * U::PR + lane * 16;
  const uint8_t* vp = static_cast<const uint8_t*>(p.vp) + row * U::PR + lane * 16;
  dst += lane * 16;
#pragma unroll
  for (int i = 0; i < G; ++i)
    if (i * 512 + lane * 16 < nk * U::CR) {
      cp_async16(dst + U::kc + i * 512, kc + i * 512);
      cp_async16(dst + U::vc + i * 512, vc + i * 512);
    }
#pragma unroll
  for (int i = 0; i < (kUnit * U::PR + 511) / 512; ++i)
    if (i * 512 + lane * 16 < nk * U::PR) {
      cp_async16(dst + U::kp + i * 512, kp + i * 512);
      cp_async16(dst + U::vp + i * 512, vp + i * 512);
    }
}

// d = a b + c: a 16 x 32 signed or unsigned bytes, b 32 x 8 unsigned bytes.
__device__ __forceinline__ void mma_s8u8(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_u8u8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.u8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  return x;
}
// Largest of a warp's floats by their bits' order as signed integers, negative
// numbers' bits turned round (a NaN with a clear sign is the largest).
__device__ __forceinline__ float warp_max(float x) {
  int i = __float_as_int(x);
  i ^= (i >> 31) & 0x7fffffff;
  i = __reduce_max_sync(0xffffffffu, i);
  return __int_as_float(i ^ ((i >> 31) & 0x7fffffff));
}

// N consecutive words of shared memory, in the widest loads that their
// alignment (their own size's largest power of two) allows.
template <int N>
__device__ __forceinline__ void lds_words(const uint8_t* s, uint32_t* w) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) *reinterpret_cast<uint4*>(w + i) = *reinterpret_cast<const uint4*>(s + 4 * i);
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) *reinterpret_cast<uint2*>(w + i) = *reinterpret_cast<const uint2*>(s + 4 * i);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = *reinterpret_cast<const uint32_t*>(s + 4 * i);
  }
}
// Pairs of half words (two groups a word); an odd last one sits alone.
template <int G>
__device__ __forceinline__ void lds_halves(const uint8_t* s, uint32_t* w) {
  if constexpr (G % 2 == 0) {
    lds_words<G / 2>(s, w);
  } else {
#pragma unroll
    for (int i = 0; i < (G + 1) / 2; ++i) {
      w[i] = *reinterpret_cast<const uint16_t*>(s + 4 * i);
      if (2 * i + 1 < G) w[i] |= (uint32_t) * reinterpret_cast<const uint16_t*>(s + 4 * i + 2) << 16;
    }
  }
}
// A row's parameters, (s, z) per group; zeros unless ok.
template <typename T, int G>
__device__ __forceinline__ void lds_params(const uint8_t* s, bool ok, float (&step)[G], float (&low)[G]) {
  constexpr int N = 2 * G * (int)sizeof(T) / 4;
  uint32_t w[N];
  lds_words<N>(s, w);
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = ok ? w[i] : 0u;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    if constexpr (std::is_same<T, float>::value) {
      step[g] = __uint_as_float(w[2 * g]);
      low[g] = __uint_as_float(w[2 * g + 1]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      step[g] = __uint_as_float(w[g] << 16);
      low[g] = __uint_as_float(w[g] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[g]));
      step[g] = f.x;
      low[g] = f.y;
    }
  }
}

// Balanced base-256 digit d (0: lowest) of x, |x| <= 127 (2^24 + 2^16 + 2^8 + 1).
__device__ __forceinline__ uint32_t digit(int x, int d) {
  // Adding 128 to every lower digit carries into the ones above as needed.
  const uint32_t biased = (uint32_t)x + 0x00808080u;
  const uint32_t byte = (biased >> (8 * d)) & 0xffu;
  return d == 3 ? byte : byte ^ 0x80u;  // take the 128 off again, modulo 256
}

// ---------------------------------------------------------------------------
// One query row per segment.
//
// Scores, 8 positions a product (A = query digits, B = codes): rows j and 8 + j
// of A hold q's digits 3 and 2 restricted to group j, rows 4 + j and 12 + j its
// digits 1 and 0 (groups 4 .. 7 in a second set of products).  Lane (g, t) =
// (lane / 4, lane % 4) gets two digits' sums for two positions, joins them in
// integers and leaves them in shared memory, where one lane a position picks
// up its eight parts, applies the row's steps and minima and takes the
// exponential.  It then writes the weights' digits, byte by byte, in the order
// of the B operand of the second product:
// Output (A = codes: 16 bytes of the rows, B = weights): column j of B holds
// the upper digit of p s for group j, column 4 + j the lower one (for three
// digits, column j of a second product the lowest).  Bytes of group j take
// their column j (+ 4 + j).  The integer sums are taken over into fp32 when a
// maximum or a bound moves, at the latest after kFlush units: a sum grows by at
// most 32 * 255 * 255 a unit.
//
// Position i of lane t: 16 (i / 4) + (t, 4 + (t ^ 1), 8 + t, 12 + (t ^ 1))[i % 4].
// The scores' columns and the weights' rows are then the same positions, and
// the rows that a quarter or half of the warp reads at once lie in distinct
// banks (kv4.cuh).
// ---------------------------------------------------------------------------
constexpr int kFlush = 1000;
constexpr float kQMax = 1.2e8f;  // |16 q0 - q1| stays within four digits

template <typename T, int G>
__global__ void __launch_bounds__(kWarps * 32, Unit<T, G>::resident) attn_row_kernel(const Pool p, const Problem a) {
  using U = Unit<T, G>;
  constexpr int PP = Parts<T>::p, SETS = U::SETS;
  constexpr float kPMax = PP == 3 ? 8388600.f : 65530.f;
  extern __shared__ __align__(128) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * U::warp_bytes;
  const uint32_t ring_u32 = smem_u32(ring);
  float* dots = reinterpret_cast<float*>(ring + U::dots);
  uint8_t* digits = ring + U::digits;
  T* const out = static_cast<T*>(a.out);
  pdl_wait();
  pdl_trigger();

  const int segs = a.QH * a.tq;
  const long long w = (long long)blockIdx.x * kWarps + warp, nw = (long long)gridDim.x * kWarps;
  // zeros for queries without a place in the pool
  for (long long b = w; b < a.B; b += nw) {
    const int keys = keys_of(p, a, (int)b), good = keys == 0 ? 0 : min(a.tq, keys - a.start_pos[b]);
    if (good == a.tq) continue;
    if (lane == 0) raise_device_error(DEV_ERR_ATTN_RANGE);
    const long long n = (long long)(a.tq - good) * a.QH * p.D;
    for (long long i = lane; i < n; i += 32) out[(b * a.tq + good) * a.QH * p.D + i] = from_f32<T>(0.f);
  }
  const long long total = all_units(p, a, segs);
  const long long W = min(nw, total);
  if (w >= W) return;  // every worker holds a unit
  const long long begin = total * w / W, end = total * (w + 1) / W;
  Cursor cur = seek(p, a, segs, begin), pre = cur;
  long long left = end - begin, ahead = left;
  auto prefetch = [&](int stage) {
    if (ahead > 0) {
      const int h = pre.seg / a.tq / a.group;
      const long long row = head_row(p, a.slot_of[pre.b], h) + pre.unit * kUnit;
      load_unit<T, G>(p, row, min(kUnit, pre.keys - pre.unit * kUnit), ring_u32 + stage * U::bytes);
      pre.next(p, a);
      --ahead;
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) prefetch(i);

  // Offsets of this lane's reads within a stage.
  const int krow = (g & 1) ? 4 + ((g >> 1) ^ 1) : (g >> 1);  // position (of 8) that column g of a product stands for
  const int k_off = U::kc + krow * U::CR + t * 4 * G;
  const int v_off0 = U::vc + t * U::CR + ((g * 2 * G) ^ v_swizzle(G, t));
  const int v_off1 = U::vc + (4 + (t ^ 1)) * U::CR + ((g * 2 * G) ^ v_swizzle(G, t ^ 1));
  // the position that this lane turns into a weight: number `lane` of the order (t, i)
  const int lt = lane >> 3, li = lane & 7;
  const int my_pos = 16 * (li >> 2) + 4 * (li & 3) + ((li & 1) ? lt ^ 1 : lt);

  uint32_t qa[G][4];  // A: this lane's bytes, zero outside its row's group
  float qsum[G], unit_q = 0.f;
  int accm[G][4], accr[G][4];                                // sums of P lo and of P (lo + 16 hi)
  int accm3[PP == 3 ? G : 1][4], accr3[PP == 3 ? G : 1][4];  // third digits
  float o[G][4], zacc[G], bound[G], to_int[G], m = -INFINITY, l = 0.f;
  int stage = 0, since = 0, row_keys = 0;
  bool fresh = true;

  // Takes the integer sums over into o (channels 32 gi + 4 g .. + 3, valid in
  // the lanes whose columns are group gi's).
  auto flush = [&]() {
#pragma unroll
    for (int gi = 0; gi < G; ++gi) {
      const float u = bound[gi] * (1.0f / kPMax);
      const float d1 = t < 2 ? (PP == 3 ? 65536.f : 256.f) * u : (PP == 3 ? 256.f : 1.f) * u;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int e = 2 * h + (gi & 1);
        o[gi][2 * h] = fmaf((float)accm[gi][e], d1, o[gi][2 * h]);
        o[gi][2 * h + 1] = fmaf((float)(accr[gi][e] - accm[gi][e]), d1 * 0.0625f, o[gi][2 * h + 1]);
        if constexpr (PP == 3) {
          if (t < 2) {
            o[gi][2 * h] = fmaf((float)accm3[gi][e], u, o[gi][2 * h]);
            o[gi][2 * h + 1] = fmaf((float)(accr3[gi][e] - accm3[gi][e]), u * 0.0625f, o[gi][2 * h + 1]);
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        accm[gi][e] = accr[gi][e] = 0;
        if constexpr (PP == 3) accm3[gi][e] = accr3[gi][e] = 0;
      }
    }
    since = 0;
  };

  while (left > 0) {
    if (fresh) {  // a segment begins: its query, empty sums
      const int qh = cur.seg / a.tq, tok = cur.seg - qh * a.tq;
      const T* qp = static_cast<const T*>(a.q) + cur.b * a.qs0 + tok * a.qs1 + qh * a.qs2;
      row_keys = a.start_pos[cur.b] + tok + 1;
      float x[G][8], big = 0.f;
#pragma unroll
      for (int gi = 0; gi < G; ++gi)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int c = gi * 32 + 8 * t + i;
          x[gi][i] = c < p.D ? to_f32<T>(qp[c]) : 0.f;
          big = fmaxf(big, fabsf(x[gi][i]));
          if (!(fabsf(x[gi][i]) <= 3.402823466e38f)) big = INFINITY;
        }
      big = warp_max(big);
      const bool sound = big <= 3.402823466e38f;
      const float to_q = big > 0.f && sound ? fminf(kQMax / big, 1e37f) : 0.f;
      // scores = (integer sums / 16) * unit_q + minima's share, in log2 units
      unit_q = sound ? (to_q > 0.f ? 0.0625f / to_q * a.scale_log2 : 0.f) : NAN;
#pragma unroll
      for (int gi = 0; gi < G; ++gi) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += x[gi][i];
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        qsum[gi] = sum * a.scale_log2;
        uint32_t r[4] = {0u, 0u, 0u, 0u};
        if ((gi & 3) == (g & 3)) {
          const int hi = g < 4 ? 3 : 1;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int q0 = __float2int_rn(x[gi][2 * i] * to_q), q1 = __float2int_rn(x[gi][2 * i + 1] * to_q);
            const int q01 = 16 * q0 - q1;
            r[0] |= digit(q01, hi) << (8 * i);
            r[1] |= digit(q01, hi - 1) << (8 * i);
            r[2] |= digit(q1, hi) << (8 * i);
            r[3] |= digit(q1, hi - 1) << (8 * i);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          qa[gi][i] = r[i];
          accm[gi][i] = accr[gi][i] = 0;
          if constexpr (PP == 3) accm3[gi][i] = accr3[gi][i] = 0;
          o[gi][i] = 0.f;
        }
        zacc[gi] = bound[gi] = to_int[gi] = 0.f;
      }
      m = -INFINITY;
      l = 0.f;
      since = 0;
      fresh = false;
    }
    cp_async_wait<kStages - 2>();
    __syncwarp();
    prefetch(stage == 0 ? kStages - 1 : stage - 1);
    const uint8_t* st = ring + stage * U::bytes;
    const int nk = row_keys - cur.unit * kUnit;  // positions of the unit that the row attends
    if (nk > 0) {
      // ---- scores
      int c[SETS][4][4];
#pragma unroll
      for (int nt = 0; nt < 4; ++nt) {
        uint32_t kw[G];
        lds_words<G>(st + k_off + nt * 8 * U::CR, kw);
#pragma unroll
        for (int s = 0; s < SETS; ++s)
#pragma unroll
          for (int e = 0; e < 4; ++e) c[s][nt][e] = 0;
#pragma unroll
        for (int gi = 0; gi < G; ++gi) mma_s8u8(c[gi / 4][nt], qa[gi], kw[gi] & 0x0f0f0f0fu, kw[gi]);
      }
#pragma unroll
      for (int s = 0; s < SETS; ++s)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float4 f;
          f.x = (float)(c[s][2 * i][0] * 256 + c[s][2 * i][2]);
          f.y = (float)(c[s][2 * i][1] * 256 + c[s][2 * i][3]);
          f.z = (float)(c[s][2 * i + 1][0] * 256 + c[s][2 * i + 1][2]);
          f.w = (float)(c[s][2 * i + 1][1] * 256 + c[s][2 * i + 1][3]);
          *reinterpret_cast<float4*>(dots + s * 8 * 36 + g * 36 + t * 8 + 4 * i) = f;
        }
      __syncwarp();
      const bool valid = my_pos < nk;
      float step[G], low[G];
      lds_params<T, G>(st + U::kp + my_pos * U::PR, valid, step, low);
      float x = 0.f, y = 0.f;
#pragma unroll
      for (int gi = 0; gi < G; ++gi) {
        const float* d = dots + (gi / 4) * 8 * 36 + (gi & 3) * 36 + lane;
        x = fmaf(step[gi], fmaf(d[0], 65536.f, d[4 * 36]), x);
        y = fmaf(low[gi], qsum[gi], y);
      }
      const float sc = valid ? fmaf(x, unit_q, y) : -INFINITY;
      const float mx = warp_max(sc);
      lds_params<T, G>(st + U::vp + my_pos * U::PR, valid, step, low);
      bool grow = mx > m, over = false;
#pragma unroll
      for (int gi = 0; gi < G; ++gi) over |= step[gi] > bound[gi];
      over = __any_sync(0xffffffffu, over);
      if (grow || over || since == kFlush) {  // the same in every lane
        flush();
        if (over) {
#pragma unroll
          for (int gi = 0; gi < G; ++gi) {
            // a quarter of headroom, so that it moves seldom
            const float s = warp_max(step[gi]);
            if (s > bound[gi]) bound[gi] = fmaxf(1.25f * s, 1e-32f);
            to_int[gi] = bound[gi] > 0.f ? kPMax / bound[gi] : 0.f;
          }
        }
        if (grow) {
          const float alpha = ex2(m - mx);
          m = mx;
          l *= alpha;
#pragma unroll
          for (int gi = 0; gi < G; ++gi) {
            zacc[gi] *= alpha;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[gi][e] *= alpha;
          }
        }
      }
      ++since;

      // ---- weights
      const float pr = valid ? ex2(sc - m) : 0.f;
      l += pr;
#pragma unroll
      for (int gi = 0; gi < G; ++gi) {
        zacc[gi] = fmaf(pr, low[gi], zacc[gi]);
        const uint32_t n = __float_as_uint(fmaf(pr * step[gi], to_int[gi], 8388608.f));
        uint8_t* d = digits + (gi / 4) * (PP == 3 ? 16 : 8) * 32 + (gi & 3) * 32 + lane;
        if constexpr (PP == 3) {
          d[0] = (uint8_t)((n >> 16) & 0x7f);
          d[4 * 32] = (uint8_t)(n >> 8);
          d[8 * 32] = (uint8_t)n;
        } else {
          d[0] = (uint8_t)(n >> 8);
          d[4 * 32] = (uint8_t)n;
        }
      }
      __syncwarp();
      uint2 pb[SETS], pb3[SETS];
#pragma unroll
      for (int s = 0; s < SETS; ++s) {
        const uint8_t* d = digits + s * (PP == 3 ? 16 : 8) * 32 + t * 8;
        pb[s] = *reinterpret_cast<const uint2*>(d + g * 32);
        if constexpr (PP == 3) pb3[s] = *reinterpret_cast<const uint2*>(d + (8 + (g & 3)) * 32);
      }

      // ---- output: per word (two groups) the bytes of four rows change places
      uint32_t vw[8][(G + 1) / 2];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        lds_halves<G>(st + ((i & 1) ? v_off1 : v_off0) + (16 * (i >> 2) + 8 * ((i >> 1) & 1)) * U::CR, vw[i]);
#pragma unroll
      for (int wi = 0; wi < (G + 1) / 2; ++wi) {
        uint32_t by[2][4];  // [rows 0-3 / 4-7][byte of the word]
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const uint32_t lo01 = __byte_perm(vw[4 * hf][wi], vw[4 * hf + 1][wi], 0x5140);
          const uint32_t lo23 = __byte_perm(vw[4 * hf + 2][wi], vw[4 * hf + 3][wi], 0x5140);
          by[hf][0] = __byte_perm(lo01, lo23, 0x5410);
          by[hf][1] = __byte_perm(lo01, lo23, 0x7632);
          if (2 * wi + 1 < G) {
            const uint32_t hi01 = __byte_perm(vw[4 * hf][wi], vw[4 * hf + 1][wi], 0x7362);
            const uint32_t hi23 = __byte_perm(vw[4 * hf + 2][wi], vw[4 * hf + 3][wi], 0x7362);
            by[hf][2] = __byte_perm(hi01, hi23, 0x5410);
            by[hf][3] = __byte_perm(hi01, hi23, 0x7632);
          }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int gi = 2 * wi + k;
          if (gi < G) {
            const uint32_t a0 = by[0][2 * k], a1 = by[0][2 * k + 1], a2 = by[1][2 * k], a3 = by[1][2 * k + 1];
            const uint32_t m0 = a0 & 0x0f0f0f0fu, m1 = a1 & 0x0f0f0f0fu, m2 = a2 & 0x0f0f0f0fu, m3 = a3 & 0x0f0f0f0fu;
            mma_u8u8(accr[gi], a0, a1, a2, a3, pb[gi / 4].x, pb[gi / 4].y);
            mma_u8u8(accm[gi], m0, m1, m2, m3, pb[gi / 4].x, pb[gi / 4].y);
            if constexpr (PP == 3) {
              mma_u8u8(accr3[gi], a0, a1, a2, a3, pb3[gi / 4].x, pb3[gi / 4].y);
              mma_u8u8(accm3[gi], m0, m1, m2, m3, pb3[gi / 4].x, pb3[gi / 4].y);
            }
          }
        }
      }
    }
    stage = stage == kStages - 1 ? 0 : stage + 1;
    --left;
    const bool last = cur.unit + 1 == cur.units;
    if (last || left == 0) {  // the segment, or this worker's share, ends here
      const long long seg0 = end - left - 1 - cur.unit;  // place of the segment's first unit
      const bool whole = last && seg0 >= begin;
      flush();
      l = warp_sum(l);
      const int qh = cur.seg / a.tq, tok = cur.seg - qh * a.tq;
      T* op = out + (((long long)cur.b * a.tq + tok) * a.QH + qh) * p.D;
      float* wp = a.ws + (w * 2 + (seg0 <= begin ? 0 : 1)) * (4 + 32 * G);
      if (!whole && lane == 0) {
        wp[0] = m;
        wp[1] = l;
      }
      const float inv = 1.0f / l;
      const bool store = !whole || row_keys <= cur.keys;
#pragma unroll
      for (int gi = 0; gi < G; ++gi) {
        const float z = warp_sum(zacc[gi]);
        float4 f;
        f.x = o[gi][0] + __shfl_xor_sync(0xffffffffu, o[gi][0], 2) + z;
        f.y = o[gi][1] + __shfl_xor_sync(0xffffffffu, o[gi][1], 2) + z;
        f.z = o[gi][2] + __shfl_xor_sync(0xffffffffu, o[gi][2], 2) + z;
        f.w = o[gi][3] + __shfl_xor_sync(0xffffffffu, o[gi][3], 2) + z;
        if (t == (gi & 3) >> 1 && store) {
          const int c = 32 * gi + 4 * g;
          if (!whole) {
            *reinterpret_cast<float4*>(wp + 4 + c) = f;
          } else {
            if (c < p.D) op[c] = from_f32<T>(f.x * inv);
            if (c + 1 < p.D) op[c + 1] = from_f32<T>(f.y * inv);
            if (c + 2 < p.D) op[c + 2] = from_f32<T>(f.z * inv);
            if (c + 3 < p.D) op[c + 3] = from_f32<T>(f.w * inv);
          }
        }
      }
      fresh = true;
    }
    cur.next(p, a);
    __syncwarp();
  }
  cp_async_wait<0>();
}

// Joins the workers' shares of a segment that more than one of them holds, in
// the workers' order.  One CTA per worker: the one whose share begins inside a
// segment, the first to do so, joins that segment.  Its threads take the
// channels (times slices of the shares, so that a segment of hundreds of
// shares is not one long chain of loads).
constexpr int kJoinThreads = 256;
constexpr int kJoinShares = 256;  // shares weighted at once

template <typename T, int G>
__global__ void __launch_bounds__(kJoinThreads) attn_join_kernel(const Pool p, const Problem a, long long W) {
  pdl_wait();
  pdl_trigger();
  constexpr int CH = 32 * G, SL = kJoinThreads / CH;  // channels, slices
  __shared__ float weight[kJoinShares], sum_x[SL > 1 ? SL : 1][CH], red[kJoinThreads / 32];
  __shared__ uint32_t place[kJoinShares];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int segs = a.QH * a.tq;
  const long long total = all_units(p, a, segs);
  W = min(W, total);
  const long long mid = blockIdx.x + 1;  // the worker whose begin is looked at
  if (mid >= W) return;
  const Cursor c = seek(p, a, segs, total * mid / W);
  const long long u0 = total * mid / W - c.unit, u1 = u0 + c.units;
  if (c.unit == 0 || total * (mid - 1) / W > u0) return;
  const long long w0 = mid - 1, w1 = (u1 * W - 1) / total;  // the worker of a unit u: the last with total * w / W <= u
  const int qh = c.seg / a.tq, tok = c.seg - qh * a.tq;
  if (a.start_pos[c.b] + tok >= p.max_seq) return;  // zeros already
  T* op = static_cast<T*>(a.out) + (((long long)c.b * a.tq + tok) * a.QH + qh) * p.D;
  constexpr int stride = 4 + CH;
  float m = -INFINITY, l = 0.f, x = 0.f;  // x: this thread's channel over its slice of the shares
  const int ch = tid % CH, sl = tid / CH;
  for (long long base = w0; base <= w1; base += kJoinShares) {
    const int n = (int)min((long long)kJoinShares, w1 + 1 - base);
    float mine = -INFINITY, ml = 0.f;
    if (tid < n) {
      const long long w = base + tid;
      const uint32_t at = (uint32_t)(w * 2 + (total * w / W >= u0 ? 0 : 1));
      place[tid] = at;
      mine = a.ws[(long long)at * stride];
      ml = a.ws[(long long)at * stride + 1];
    }
    float mx = warp_max(mine);
    __syncthreads();  // the previous round's weights are read
    if (lane == 0) red[warp] = mx;
    __syncthreads();
    mx = m;
#pragma unroll
    for (int i = 0; i < kJoinThreads / 32; ++i) mx = fmaxf(mx, red[i]);
    const float alpha = m == -INFINITY ? 0.f : ex2(m - mx);
    m = mx;
    // a share whose units are all masked has maximum -inf and counts nothing
    const float f = tid < n && !(mine == -INFINITY && ml == 0.f) ? ex2(mine - m) : 0.f;
    weight[tid] = f;
    const float part = warp_sum(tid < n ? f * ml : 0.f);
    __syncthreads();
    if (lane == 0) red[warp] = part;
    __syncthreads();
    l *= alpha;
#pragma unroll
    for (int i = 0; i < kJoinThreads / 32; ++i) l += red[i];
    x *= alpha;
    if (sl < SL) {
#pragma unroll 4
      for (int i = sl; i < n; i += SL) x = fmaf(weight[i], a.ws[(long long)place[i] * stride + 4 + ch], x);
    }
  }
  if (SL > 1) {
    if (sl < SL) sum_x[sl][ch] = x;
    __syncthreads();
    x = 0.f;
#pragma unroll
    for (int i = 0; i < SL; ++i) x += sum_x[i][ch];
  }
  if (sl == 0 && ch < p.D) op[ch] = from_f32<T>(x / l);
}

template <typename T, int G>
static int launch_row(const Pool& p, const Problem& a, int grid, cudaStream_t st) {
  constexpr int smem = kWarps * Unit<T, G>::warp_bytes;
  static bool attr_set[64] = {};
  const int dev = current_device();
  if (dev >= 0 && dev < 64 && !attr_set[dev]) {
    const cudaError_t e =
        cudaFuncSetAttribute(attn_row_kernel<T, G>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return check_cuda(e, "neb_kv4_attention smem attribute");
    attr_set[dev] = true;
  }
  cudaError_t e = launch_pdl(attn_row_kernel<T, G>, dim3((unsigned)grid), dim3(kWarps * 32), smem, st, 1, p, a);
  count_launch();
  if (e != cudaSuccess) return check_cuda(e, "neb_kv4_attention launch");
  const long long W = (long long)grid * kWarps;
  if (W < 2) return FML_OK;
  e = launch_pdl(attn_join_kernel<T, G>, dim3((unsigned)(W - 1)), dim3(kJoinThreads), 0, st, 1, p, a, W);
  count_launch();
  return check_cuda(e, "neb_kv4_attention join launch");
}

// The row kernel's grid: a whole number of resident CTAs per SM, no more
// workers than the longest batch has units.
template <typename T, int G>
static int row_grid(const Pool& p, long long segments) {
  const long long units = segments * ((p.max_seq + kUnit - 1) / kUnit);
  return (int)std::min<long long>((long long)Unit<T, G>::resident * num_sms(current_device()), (units + kWarps - 1) / kWarps);
}

#define KV4_GROUPS(CALL) \
  switch (p.G) {         \
    case 1: CALL(1);     \
    case 2: CALL(2);     \
    case 3: CALL(3);     \
    case 4: CALL(4);     \
    case 5: CALL(5);     \
    case 6: CALL(6);     \
    case 7: CALL(7);     \
    default: CALL(8);    \
  }

template <typename T>
static int grid_of(const Pool& p, long long segments) {
#define CALL(G) return row_grid<T, G>(p, segments)
  KV4_GROUPS(CALL)
#undef CALL
}

static size_t workspace_bytes(const Pool& p, int dtype, int64_t batch, int64_t t, int64_t q_heads) {
  const long long segs = batch * t * q_heads;
  const int grid = dtype == FML_F32 ? grid_of<float>(p, segs)
                   : dtype == FML_F16 ? grid_of<__half>(p, segs) : grid_of<__nv_bfloat16>(p, segs);
  return (size_t)grid * kWarps * 2 * (4 + 32 * p.G) * sizeof(float);
}

template <typename T>
static int attention(const Pool& p, const Problem& a, cudaStream_t st) {
  const int grid = grid_of<T>(p, (long long)a.B * a.tq * a.QH);
#define CALL(G) return launch_row<T, G>(p, a, grid, st)
  KV4_GROUPS(CALL)
#undef CALL
}

}  // namespace kv4
}  // namespace fml

using namespace fml;

extern "C" size_t neb_kv4_attention_workspace_size(const neb_kv4_pool* pool, int64_t batch, int64_t t,
                                                   int64_t q_heads) {
  kv4::Pool p;
  if (kv4::pool_from(pool, "neb_kv4_attention_workspace_size", &p) || batch <= 0 || t <= 0 || q_heads <= 0) return 0;
  return kv4::workspace_bytes(p, pool->dtype, batch, t, q_heads);
}

extern "C" int neb_kv4_attention(const void* q, const int64_t q_strides[4], const neb_kv4_pool* pool,
                                 const int32_t* slot_of, const int32_t* start_pos, void* out, int64_t batch,
                                 int64_t t, int64_t q_heads, float scale, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  kv4::Pool p;
  if (const int rc = kv4::pool_from(pool, "neb_kv4_attention", &p)) return rc;
  if (!q || !q_strides || !slot_of || !start_pos || !out) return fail(FML_EINVAL, "neb_kv4_attention: null pointer");
  if (batch <= 0 || t <= 0 || q_heads <= 0) return fail(FML_EINVAL, "neb_kv4_attention: sizes must be positive");
  if (q_heads % p.H != 0) return fail(FML_EINVAL, "neb_kv4_attention: q_heads must be a multiple of the pool's heads");
  if (q_strides[3] != 1) return fail(FML_EUNSUPPORTED, "neb_kv4_attention: q innermost stride must be 1");
  if (t > p.max_seq) return fail(FML_EINVAL, "neb_kv4_attention: t exceeds max_seq");
  if (batch > (1 << 24) || q_heads > (1 << 20) || batch * t > (1ll << 31) / q_heads / 8)
    return fail(FML_EUNSUPPORTED, "neb_kv4_attention: too many queries");
  const size_t need = kv4::workspace_bytes(p, pool->dtype, batch, t, q_heads);
  if (workspace_bytes < need || (need && !workspace))
    return fail(FML_EWORKSPACE, "neb_kv4_attention: workspace of " + std::to_string(need) + " bytes needed");
  if (reinterpret_cast<uintptr_t>(workspace) & 15)
    return fail(FML_EINVAL, "neb_kv4_attention: workspace must be 16-byte aligned");
  kv4::Problem a = {};
  a.slot_of = slot_of;
  a.start_pos = start_pos;
  a.B = (int)batch;
  a.tq = (int)t;
  a.QH = (int)q_heads;
  a.group = (int)(q_heads / p.H);
  a.qs0 = q_strides[0];
  a.qs1 = q_strides[1];
  a.qs2 = q_strides[2];
  a.scale_log2 = scale * 1.4426950408889634f;
  a.q = q;
  a.out = out;
  a.ws = static_cast<float*>(workspace);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (pool->dtype == FML_F32) return kv4::attention<float>(p, a, st);
  if (pool->dtype == FML_BF16) return kv4::attention<__nv_bfloat16>(p, a, st);
  return kv4::attention<__half>(p, a, st);
}
