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
// so eight codes cost one logic instruction for the keys.  Spreading them into
// bfloat16 operands costs seven, and the integer ALU was what bounded that form:
// 44 us for 64 requests of 128 .. 2303 positions (8 heads of 128, bf16), 30 us now.
//
// Measured (bf16, heads of 128, device time):
//   32 requests x 16 heads x 512 .. 639    18.3 us   2.6 TB/s of cache
//   64 requests x  8 heads x 128 .. 2303   30.2 us   3.3
//    1 request  x 16 heads x 100001        50.4 us   5.1
// Long streams come near the memory's rate; what is left of the shorter ones is
// latency: about 2 us until the first copies are issued, 1 to 2 us for a segment's
// query, flush and output, and the join where segments are split.
//
// What is rounded: q to 27 bits below its largest channel (four 8-bit digits;
// the 16-bit types and all but the smallest channels of fp32 are exact), the
// weights p s to 16 bits below their running bound (two digits; three, 23
// bits, for fp16 and fp32, whose outputs keep more bits than bf16's).  What a lane
// rounds off it adds to the weight of its next position: of many weights below a
// whole step none would count otherwise, beside a large one, while the sum of
// weights and the minima's share count them all.  Scores, maxima, sums and outputs
// are fp32.  An fp32 cache's scores, whose errors the
// exponentials pass on whole, are put together from the integers in 64 bits, and
// its values' codes count from 8: p (z + 8 s) + p s (c - 8) keeps the bits that
// p z + p s c, two sums of a group's whole range that all but cancel, loses.
#include <algorithm>
#include <atomic>
#include <string>
#include <type_traits>

#include "kv4_attention.cuh"

namespace fml {
namespace kv4 {

// The batch's segments (a request's query rows) are laid end to end and counted
// in units of 32 positions; one CTA per SM takes an equal, contiguous share of
// them and every warp an equal part of that, so the work is even whatever the
// lengths are and no warp waits for another one while it streams.  (Where no
// segment is long, a CTA takes the whole segments that begin in its share.)  A
// warp copies its units into its own stages of shared memory (a bulk copy each:
// four small ones a unit bound the kernel to 30 ns apiece per SM) and keeps a
// running maximum, sum and output; a segment that it holds
// whole is written out.  At its end the CTA joins the segments that several of
// its warps hold, and a segment that several CTAs hold is finished by the last
// of them to arrive: each leaves (maximum, sum, output) in the workspace and
// takes a ticket, and the one that takes the last ticket joins them, in the
// shares' order, so the result does not depend on who that was.  Nobody waits
// for another CTA.  (A second kernel for this took 5 to 15 us.)
constexpr int kUnit = kTile;
// Longest segment (units) for which the CTAs take whole segments: their unequal
// ends then cost less than the join through memory (about 3 us, in which a CTA
// streams some 25 units).
constexpr int kWholeUnits = 24;

template <typename T> struct Parts { static constexpr int p = 3; };
template <> struct Parts<__nv_bfloat16> { static constexpr int p = 2; };

template <typename T, int G>
struct Unit {
  static constexpr int SETS = (G + 3) / 4;           // groups are handled four at a time
  static constexpr int CR = 16 * G;                  // bytes of a row's codes
  static constexpr int PR = 2 * G * (int)sizeof(T);  // bytes of a row's parameters
  static constexpr int kc = 0, kp = kUnit * CR, vc = kUnit * (CR + PR), vp = vc + kUnit * CR;
  static constexpr int bytes = 2 * vc;
  // A warp's shared memory beside its stages: the scores' parts [set][8][36]
  // fp32 (36: distinct banks), the weights' digits [set][8 or 16][32], an mbarrier
  // per stage, the fp32 output [4 G][32 lanes] that the integer sums are taken over
  // into, its shares of the segments
  // that it holds in part (the first and the last).
  static constexpr int share = 4 + 32 * G;
  static constexpr int dots = 0;
  static constexpr int digits = dots + SETS * 8 * 36 * 4;
  static constexpr int bars = digits + SETS * (Parts<T>::p == 3 ? 16 : 8) * 32;
  static constexpr int out = bars + 64;
  static constexpr int parts = out + 4 * G * 32 * 4;
  static constexpr int stages_at = (parts + 2 * share * 4 + 127) / 128 * 128;
  static constexpr int room = 227 * 1024 - 2048;
  // Warps: by registers (the sums of every group, of three digits twice, beside
  // the query: 168 for twelve warps) and by shared memory for two stages.
  static constexpr int by_regs = G > 4 || (G == 4 && Parts<T>::p == 3) ? 8 : 12;
  static constexpr int by_smem = room / (stages_at + 2 * bytes);
  static constexpr int warps = by_regs < by_smem ? by_regs : by_smem;
  static constexpr int fit = (room / warps - stages_at) / bytes;
  static constexpr int stages = fit < 4 ? fit : 4;
  static constexpr int warp_bytes = stages_at + stages * bytes;
  static constexpr int cta_bytes = warps * warp_bytes;
  static_assert(stages >= 2, "shared memory");
};

// d = a b + c: a 16 x 32 signed or unsigned bytes, b 32 x 8 unsigned bytes.
__device__ __forceinline__ void mma_s8u8(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8u8_zero(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));
}
__device__ __forceinline__ void mma_u8u8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.u8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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
// A row's parameters, (s, z) per group; zeros unless ok (looked at where the
// unit is `part`ial).
template <typename T, int G>
__device__ __forceinline__ void lds_params(const uint8_t* s, bool part, bool ok, float (&step)[G], float (&low)[G]) {
  constexpr int N = 2 * G * (int)sizeof(T) / 4;
  uint32_t w[N];
  lds_words<N>(s, w);
  if (part) {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = ok ? w[i] : 0u;
  }
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

// The four balanced base-256 digits of x, |x| <= 127 (2^24 + 2^16 + 2^8 + 1), a
// signed byte each: adding 128 to the lower three carries into the ones above
// as needed, and the 128s are taken off again modulo 256.
__device__ __forceinline__ uint32_t digits_of(int x) { return ((uint32_t)x + 0x00808080u) ^ 0x00808080u; }

// Eight consecutive channels of a row as they lie; channels past D give 0.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int c0, int D, bool vec, uint4 (&raw)[sizeof(T) / 2]) {
  constexpr int N = (int)sizeof(T) / 2;
  if (vec) {  // D a multiple of 8, rows 16-byte aligned
#pragma unroll
    for (int i = 0; i < N; ++i)
      raw[i] = c0 < D ? reinterpret_cast<const uint4*>(p + c0)[i] : make_uint4(0, 0, 0, 0);
  } else {
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = c0 + i < D ? p[c0 + i] : from_f32<T>(0.f);
#pragma unroll
    for (int i = 0; i < N; ++i) raw[i] = reinterpret_cast<const uint4*>(e)[i];
  }
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
// A running (maximum, sum, output) of a warp, V float4s of channels a lane, and
// another share of the same segment.  One that saw no position counts nothing.
template <int V>
struct Running {
  float m = -INFINITY, l = 0.f;
  float4 x[V];
  __device__ __forceinline__ Running() {
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __device__ __forceinline__ void add(float om, float ol, const float4 (&y)[V]) {
    if (om == -INFINITY && ol == 0.f) return;
    const float mn = fmaxf(m, om), fa = m == -INFINITY ? 0.f : ex2(m - mn), fb = ex2(om - mn);
    m = mn;
    l = fmaf(l, fa, fb * ol);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      x[v].x = fmaf(x[v].x, fa, fb * y[v].x);
      x[v].y = fmaf(x[v].y, fa, fb * y[v].y);
      x[v].z = fmaf(x[v].z, fa, fb * y[v].z);
      x[v].w = fmaf(x[v].w, fa, fb * y[v].w);
    }
  }
};
// Four channels of an output row.
template <typename T>
__device__ __forceinline__ void store4(T* op, int c, int D, bool vec, float4 f) {
  if (vec && sizeof(T) == 2) {  // D a multiple of 4, rows 8-byte aligned
    if (c < D) {
      T e[4] = {from_f32<T>(f.x), from_f32<T>(f.y), from_f32<T>(f.z), from_f32<T>(f.w)};
      *reinterpret_cast<uint2*>(op + c) = *reinterpret_cast<const uint2*>(e);
    }
  } else {
    if (c < D) op[c] = from_f32<T>(f.x);
    if (c + 1 < D) op[c + 1] = from_f32<T>(f.y);
    if (c + 2 < D) op[c + 2] = from_f32<T>(f.z);
    if (c + 3 < D) op[c + 3] = from_f32<T>(f.w);
  }
}

constexpr int kFlush = 1000;
// The integers' scale to_int stays finite: with kToIntMax the weights p s have all
// their digits down to 2^-110 (two digits) or 2^-103 (three).  Where those of every
// group are below kTiny, weights and sums are taken kLift times larger, which keeps the
// digits of the smallest steps.
constexpr float kToIntMax = 8.507059e37f;  // 2^126; a fast division by more gives 0
constexpr float kTiny = 5.42101086e-20f, kLift = 1.1529215e18f;  // 2^-64, 2^60
constexpr float kQMax = 1.2e8f;  // |16 q0 - q1| stays within four digits

template <typename T, int G>
__global__ void __launch_bounds__(Unit<T, G>::warps * 32, 1) attn_row_kernel(const Pool p, const Problem a) {
  using U = Unit<T, G>;
  constexpr int PP = Parts<T>::p, SETS = U::SETS, kWarps = U::warps, kStages = U::stages;
  constexpr float kPMax = PP == 3 ? 8388600.f : 65530.f;
  constexpr bool kWide = std::is_same<T, float>::value;
  constexpr bool kLifts = !std::is_same<T, __half>::value;  // fp16's smallest step is 2^-24
  using Score = typename std::conditional<kWide, double, float>::type;
  extern __shared__ __align__(128) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  uint8_t* mem = smem + warp * U::warp_bytes;
  uint8_t* ring = mem + U::stages_at;
  const uint32_t ring_u32 = smem_u32(ring);
  float* dots = reinterpret_cast<float*>(mem + U::dots);
  uint8_t* digits = mem + U::digits;
  T* const out = static_cast<T*>(a.out);
  pdl_wait();
  pdl_trigger();

  const Plan<kUnit> plan(p, a);
  const unsigned total = plan.total;
  const bool by_segment = plan.longest <= kWholeUnits;
  // a share of a few units at least: an empty one could not be joined
  const Shares shares(total, by_segment ? gridDim.x : min(gridDim.x, (total + 3) / 4));
  unsigned cta_begin = total, cta_end = total;
  if (blockIdx.x < shares.W) {
    cta_begin = shares.begin(blockIdx.x);
    cta_end = shares.begin(blockIdx.x + 1);
  }
  Cursor<kUnit> cur = plan.seek(p, a, min(cta_begin, max(total, 1u) - 1));
  if (by_segment && total > 0) {  // the segments that begin in the share
    const Cursor<kUnit> tail = plan.seek(p, a, min(cta_end, total - 1));
    if (cta_begin < total && cur.unit > 0) {
      cta_begin += cur.units - cur.unit;
      cur.next_segment(p, a);
    }
    if (cta_end < total && tail.unit > 0) cta_end += tail.units - tail.unit;
    cta_end = max(cta_end, cta_begin);
  }
  const unsigned cta_units = cta_end - cta_begin;
  const unsigned begin = cta_begin + cta_units * warp / kWarps;
  int left = (int)(cta_begin + cta_units * (warp + 1) / kWarps - begin), ahead = left;
  const int share_units = left;
  const unsigned end = begin + left;
  const bool busy = left > 0;
  const Cursor<kUnit> cta_cur = cur;
  if (busy) cur.skip(p, a, begin - cta_begin);
  Cursor<kUnit> pre = cur;
  const uint32_t bars = smem_u32(mem + U::bars);
  const uint8_t* pre_head = nullptr;  // tiles of the head that `pre` is in
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(bars + 8 * i, 1);
    fence_mbar_init();
  }
  __syncwarp();
  // Copies the next unit's tile (rows past the last one are masked).
  auto copy = [&](int stage) {
    if (ahead == 0) return;
    if (lane == 0) {
      mbar_arrive_expect_tx(bars + 8 * stage, U::bytes);
      bulk_load(ring_u32 + stage * U::bytes, pre_head + (long long)pre.unit * U::bytes, U::bytes, bars + 8 * stage);
    }
    --ahead;
    if (pre.next(p, a) && ahead > 0) pre_head = head_tiles(p, a.slot_of[pre.b], pre.seg / (a.group * a.tq));
  };
  // The first stages at once, a lane each.
  if (busy) pre_head = head_tiles(p, a.slot_of[pre.b], pre.seg / (a.group * a.tq));
  {
    const uint8_t* first = nullptr;
#pragma unroll 1
    for (int i = 0; i < kStages && ahead > 0; ++i) {
      if (lane == i) first = pre_head + (long long)pre.unit * U::bytes;
      --ahead;
      if (pre.next(p, a) && ahead > 0) pre_head = head_tiles(p, a.slot_of[pre.b], pre.seg / (a.group * a.tq));
    }
    if (first != nullptr) {
      mbar_arrive_expect_tx(bars + 8 * lane, U::bytes);
      bulk_load(ring_u32 + lane * U::bytes, first, U::bytes, bars + 8 * lane);
    }
  }
  __syncwarp();

  // The segments that the share begins and ends in are other CTAs' too where they
  // reach past it: their tickets' words.
  if (!by_segment && cta_units > 0 && warp == 0) {
    Cursor<kUnit> c = cta_cur;
    unsigned at = cta_begin;
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
      const unsigned seg0 = at - c.unit;
      if (seg0 < cta_begin || seg0 + c.units > cta_end) {
        const unsigned word = shares.holder(seg0, blockIdx.x);
        if (lane == 0) open_tickets(a.tickets + word, a.launch);
      }
      c.skip(p, a, cta_units - 1);
      at += cta_units - 1;
    }
  }
  // Zeros for queries without a place in the pool.
  for (int b = blockIdx.x * kWarps + warp; b < a.B; b += gridDim.x * kWarps) {
    const int keys = keys_of(p, a, b), good = keys == 0 ? 0 : min(a.tq, keys - a.start_pos[b]);
    if (good == a.tq) continue;
    if (lane == 0) raise_device_error(DEV_ERR_ATTN_RANGE);
    const long long n = (long long)(a.tq - good) * a.QH * p.D;
    T* bad = out + ((long long)b * a.tq + good) * a.QH * p.D;
    for (long long i = lane; i < n; i += 32) bad[i] = from_f32<T>(0.f);
  }

  // Offsets of this lane's reads within a stage.
  const int krow = (g & 1) ? 4 + ((g >> 1) ^ 1) : (g >> 1);  // position (of 8) that column g of a product stands for
  const int k_off = U::kc + krow * U::CR + t * 4 * G;
  const int v_off0 = U::vc + t * U::CR + ((g * 2 * G) ^ v_swizzle(G, t));
  const int v_off1 = U::vc + (4 + (t ^ 1)) * U::CR + ((g * 2 * G) ^ v_swizzle(G, t ^ 1));
  // the position that this lane turns into a weight: number `lane` of the order (t, i)
  const int lt = lane >> 3, li = lane & 7;
  const int my_pos = 16 * (li >> 2) + 4 * (li & 3) + ((li & 1) ? lt ^ 1 : lt);

  uint32_t qa[G][4];  // A: this lane's bytes, zero outside its row's group
  Score qsum[G], unit_q = 0;
  int accm[G][4], accr[G][4];                                // sums of P lo and of P (lo + 16 hi)
  int accm3[PP == 3 ? G : 1][4], accr3[PP == 3 ? G : 1][4];  // third digits
  int ones[kWide ? SETS : 1][4], ones3[kWide ? SETS : 1][4];  // sums of P: the codes count from 8 then
  float zacc[G], to_int[G], carry[G], lift = 1.f, m = -INFINITY, l = 0.f;
  float* const o = reinterpret_cast<float*>(mem + U::out) + lane;  // channel 32 gi + 4 g + i: o[(4 gi + i) * 32]
  int stage = 0, since = 0;
  uint32_t parity = 0;
  bool live = true;
  // The segments that this warp holds in part: the first and last of its share.
  float* const parts = reinterpret_cast<float*>(mem + U::parts);
  __shared__ unsigned part_seg0[kWarps][2];  // place of the segment's first unit
  __shared__ int part_units[kWarps][2];      // its units; 0: none
  __shared__ T* part_op[kWarps][2];
  if (lane < 2) part_units[warp][lane] = 0;
  __syncwarp();

  // Takes the integer sums over into the output, times `scale` (channels 32 gi +
  // 4 g .. + 3, valid in the lanes whose columns are group gi's).
  auto flush = [&](float scale) {
#pragma unroll
    for (int gi = 0; gi < G; ++gi) {
      const float u = __fdividef(scale, to_int[gi]);
      const float d1 = t < 2 ? (PP == 3 ? 65536.f : 256.f) * u : (PP == 3 ? 256.f : 1.f) * u;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int e = 2 * h + (gi & 1);
        float* const x = o + (4 * gi + 2 * h) * 32;
        const int w = kWide ? ones[gi / 4][e] : 0;
        float x0 = fmaf((float)(accm[gi][e] - 8 * w), d1, x[0] * scale);
        float x1 = fmaf((float)(accr[gi][e] - accm[gi][e] - 128 * w), d1 * 0.0625f, x[32] * scale);
        if constexpr (PP == 3) {
          if (t < 2) {
            const int w3 = kWide ? ones3[gi / 4][e] : 0;
            x0 = fmaf((float)(accm3[gi][e] - 8 * w3), u, x0);
            x1 = fmaf((float)(accr3[gi][e] - accm3[gi][e] - 128 * w3), u * 0.0625f, x1);
          }
        }
        x[0] = x0;
        x[32] = x1;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        accm[gi][e] = accr[gi][e] = 0;
        if constexpr (PP == 3) accm3[gi][e] = accr3[gi][e] = 0;
      }
    }
    if constexpr (kWide) {
#pragma unroll
      for (int s = 0; s < SETS; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e) ones[s][e] = ones3[s][e] = 0;
    }
  };

  // A segment's query, as it lies: lane (g, t) holds channels 8 t .. 8 t + 7 of
  // its own groups, every channel of the row in two lanes.  The next segment's
  // is loaded a segment ahead.
  uint4 q_raw[SETS][sizeof(T) / 2];
  T* op = nullptr;
  int row_keys = 0;
  auto load_query = [&](const Cursor<kUnit>& c) {
    int qh = c.seg, tok = 0;
    if (a.tq > 1) {
      qh = c.seg / a.tq;
      tok = c.seg - qh * a.tq;
    }
    op = out + (((long long)c.b * a.tq + tok) * a.QH + qh) * p.D;
    row_keys = a.start_pos[c.b] + tok + 1;
    const T* qp = static_cast<const T*>(a.q) + c.b * a.qs0 + tok * a.qs1 + qh * a.qs2;
#pragma unroll
    for (int s = 0; s < SETS; ++s) load8<T>(qp, (4 * s + (g & 3)) * 32 + 8 * t, p.D, a.q_vec, q_raw[s]);
  };
  if (busy) load_query(cur);

  while (left > 0) {  // the share's segments
    const int n_units = min(cur.units - cur.unit, left);
    T* const seg_op = op;
    const int seg_keys = row_keys;
    float big = 0.f, x[SETS][8];
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
      const T* e = reinterpret_cast<const T*>(q_raw[s]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[s][i] = to_f32<T>(e[i]);
        big = fmaxf(big, fabsf(x[s][i]));
        if (!(fabsf(x[s][i]) <= 3.402823466e38f)) big = INFINITY;
      }
    }
    Cursor<kUnit> nxt = cur;
    nxt.next_segment(p, a);
    if (n_units < left) load_query(nxt);
    big = warp_max(big);
    const bool sound = big <= 3.402823466e38f;
    const float to_q = big > 0.f && sound ? fminf(__fdividef(kQMax, big), 1e37f) : 0.f;
    // scores = (integer sums / 16) * unit_q + minima's share, in log2 units
    if constexpr (kWide) unit_q = sound ? (to_q > 0.f ? 0.0625 / to_q * a.scale_log2_wide : 0.0) : (double)NAN;
    else unit_q = sound ? (to_q > 0.f ? __fdividef(0.0625f, to_q) * a.scale_log2 : 0.f) : NAN;
    const int hi = g < 4 ? 3 : 1;
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
      Score sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += x[s][i];
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      if constexpr (kWide) sum *= a.scale_log2_wide;
      else sum *= a.scale_log2;
      uint32_t r[4] = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int q0 = __float2int_rn(x[s][2 * i] * to_q), q1 = __float2int_rn(x[s][2 * i + 1] * to_q);
        const uint32_t d0 = digits_of(16 * q0 - q1), d1 = digits_of(q1);
        r[0] |= (d0 >> (8 * hi) & 0xffu) << (8 * i);
        r[1] |= (d0 >> (8 * hi - 8) & 0xffu) << (8 * i);
        r[2] |= (d1 >> (8 * hi) & 0xffu) << (8 * i);
        r[3] |= (d1 >> (8 * hi - 8) & 0xffu) << (8 * i);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int gi = 4 * s + k;
        if (gi < G) {
          qsum[gi] = __shfl_sync(0xffffffffu, sum, 4 * k);
#pragma unroll
          for (int i = 0; i < 4; ++i) qa[gi][i] = (g & 3) == k ? r[i] : 0u;
        }
      }
    }
#pragma unroll
    for (int gi = 0; gi < G; ++gi) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        accm[gi][i] = accr[gi][i] = 0;
        if constexpr (PP == 3) accm3[gi][i] = accr3[gi][i] = 0;
        o[(4 * gi + i) * 32] = 0.f;
      }
      zacc[gi] = 0.f;
      to_int[gi] = kToIntMax;
      carry[gi] = 0.5f;
    }
    if constexpr (kWide) {
#pragma unroll
      for (int s = 0; s < SETS; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e) ones[s][e] = ones3[s][e] = 0;
    }
    m = -INFINITY;
    l = 0.f;
    lift = 1.f;
    since = -1;
    for (int i = 0; i < n_units && live; ++i) {
    live = __all_sync(0xffffffffu, wait_copies(bars + 8 * stage, parity >> stage & 1));
    if (!live) break;
    const uint8_t* st = ring + stage * U::bytes;
    const int nk = seg_keys - (cur.unit + i) * kUnit;  // positions of the unit that the row attends
    if (nk > 0) {
      // The values' codes, loaded ahead of the scores: the exchange of their bytes
      // fills the scores' waits.
      uint32_t vw[8][(G + 1) / 2];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        lds_halves<G>(st + ((i & 1) ? v_off1 : v_off0) + (16 * (i >> 2) + 8 * ((i >> 1) & 1)) * U::CR, vw[i]);
      // ---- scores
      int c[SETS][4][4];
#pragma unroll
      for (int nt = 0; nt < 4; ++nt) {
        uint32_t kw[G];
        lds_words<G>(st + k_off + nt * 8 * U::CR, kw);
#pragma unroll
        for (int gi = 0; gi < G; ++gi) {
          if (gi % 4 == 0) mma_s8u8_zero(c[gi / 4][nt], qa[gi], kw[gi] & 0x0f0f0f0fu, kw[gi]);
          else mma_s8u8(c[gi / 4][nt], qa[gi], kw[gi] & 0x0f0f0f0fu, kw[gi]);
        }
      }
#pragma unroll
      for (int s = 0; s < SETS; ++s)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int4 f = make_int4(c[s][2 * i][0] * 256 + c[s][2 * i][2], c[s][2 * i][1] * 256 + c[s][2 * i][3],
                                   c[s][2 * i + 1][0] * 256 + c[s][2 * i + 1][2],
                                   c[s][2 * i + 1][1] * 256 + c[s][2 * i + 1][3]);
          float* const at = dots + s * 8 * 36 + g * 36 + t * 8 + 4 * i;
          if constexpr (kWide) *reinterpret_cast<int4*>(at) = f;
          else *reinterpret_cast<float4*>(at) = make_float4((float)f.x, (float)f.y, (float)f.z, (float)f.w);
        }
      __syncwarp();
      const bool part = nk < kUnit, valid = my_pos < nk;
      float step[G], low[G];
      lds_params<T, G>(st + U::kp + my_pos * U::PR, part, valid, step, low);
      Score codes = 0, lows = 0;
#pragma unroll
      for (int gi = 0; gi < G; ++gi) {
        const float* d = dots + (gi / 4) * 8 * 36 + (gi & 3) * 36 + lane;
        if constexpr (kWide) {
          const int* e = reinterpret_cast<const int*>(d);
          codes = fma((double)step[gi], fma((double)e[0], 65536.0, (double)e[4 * 36]), codes);
          lows = fma((double)low[gi], qsum[gi], lows);
        } else {
          // (the steps' products with the integers may overflow: unit_q goes with the steps)
          codes = fmaf(step[gi] * unit_q, fmaf(d[0], 65536.f, d[4 * 36]), codes);
          lows = fmaf(low[gi], qsum[gi], lows);
        }
      }
      if constexpr (kWide) codes *= unit_q;
      const Score sc = valid ? codes + lows : (Score)-INFINITY;
      // In 32 bits; a score that has more is rounded up, so that no weight passes 1.
      float near;
      if constexpr (kWide) near = __double2float_ru(sc);
      else near = sc;
      const float mx = warp_max(near);
      lds_params<T, G>(st + U::vp + my_pos * U::PR, part, valid, step, low);
      // ---- weights, as integers up to kPMax
      const float mn = fmaxf(m, mx);
      float away = (float)(sc - mn);
      // Scores that 32 bits do not keep apart from the largest one count, however large.
      if (kWide && near == mn) away = fmaxf(away, -16.f);
      const float pr = valid ? ex2(away) : 0.f;
      float x[G], n[G];
      bool over = false;
#pragma unroll
      for (int gi = 0; gi < G; ++gi) {
        x[gi] = fmaf(pr * lift * step[gi], to_int[gi], carry[gi]);
        n[gi] = __fadd_rz(x[gi], 8388608.f);
        over |= n[gi] > 8388608.f + kPMax;
      }
      over = __any_sync(0xffffffffu, over);
      if (mx > m || over || since == kFlush) {  // the same in every lane
        const float alpha = ex2(m - mn);
        m = mn;
        // The bounds of p s.  What went before counts alpha times as much now, for its
        // bound too: a large step whose weight vanishes must not leave the later weights
        // without digits.  A quarter of headroom, so that they rise seldom.
        float bound[G], most = 0.f;
#pragma unroll
        for (int gi = 0; gi < G; ++gi) {
          const float past = __fdividef(kPMax * alpha, to_int[gi]) * (lift == 1.f ? 1.f : 1.f / kLift);
          bound[gi] = fmaxf(1.25f * warp_max(pr * step[gi]), since < 0 ? 0.f : past);
          most = fmaxf(most, bound[gi]);
        }
        const float was = lift;
        lift = kLifts && most < kTiny ? kLift : 1.f;
        if (since >= 0) {  // not the segment's first unit
          flush(lift == was ? alpha : lift == 1.f ? alpha * (1.f / kLift) : alpha * kLift);
          l *= alpha;
#pragma unroll
          for (int gi = 0; gi < G; ++gi) zacc[gi] *= alpha;
        }
        since = 0;
#pragma unroll
        for (int gi = 0; gi < G; ++gi) {
          to_int[gi] = __fdividef(kPMax, fmaxf(bound[gi] * lift, kPMax / kToIntMax));
          x[gi] = fmaf(pr * lift * step[gi], to_int[gi], 0.5f);
          n[gi] = __fadd_rz(x[gi], 8388608.f);
        }
      }
      ++since;
      l += pr;
#pragma unroll  // (cut off, from half a step on: 0 <= carry < 1)
      for (int gi = 0; gi < G; ++gi) carry[gi] = x[gi] - (n[gi] - 8388608.f);
#pragma unroll
      for (int gi = 0; gi < G; ++gi) zacc[gi] = fmaf(pr, kWide ? fmaf(8.f, step[gi], low[gi]) : low[gi], zacc[gi]);
#pragma unroll
      for (int gi = 0; gi < G; ++gi) {
        const uint32_t w = __float_as_uint(n[gi]);
        uint8_t* d = digits + (gi / 4) * (PP == 3 ? 16 : 8) * 32 + (gi & 3) * 32 + lane;
        if constexpr (PP == 3) {
          d[0] = (uint8_t)((w >> 16) & 0x7f);
          d[4 * 32] = (uint8_t)(w >> 8);
          d[8 * 32] = (uint8_t)w;
        } else {
          d[0] = (uint8_t)(w >> 8);
          d[4 * 32] = (uint8_t)w;
        }
      }
      __syncwarp();
      uint2 pb[SETS], pb3[SETS];
#pragma unroll
      for (int s = 0; s < SETS; ++s) {
        const uint8_t* d = digits + s * (PP == 3 ? 16 : 8) * 32 + t * 8;
        pb[s] = *reinterpret_cast<const uint2*>(d + g * 32);
        if constexpr (PP == 3) pb3[s] = *reinterpret_cast<const uint2*>(d + (8 + (g & 3)) * 32);
        if constexpr (kWide) {
          constexpr uint32_t k1 = 0x01010101u;
          mma_u8u8(ones[s], k1, k1, k1, k1, pb[s].x, pb[s].y);
          mma_u8u8(ones3[s], k1, k1, k1, k1, pb3[s].x, pb3[s].y);
        }
      }

      // ---- output: per word (two groups) the bytes of four rows change places
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
    __syncwarp();  // the stage is read
    copy(stage);
    parity ^= 1u << stage;
    stage = stage == kStages - 1 ? 0 : stage + 1;
    }

    // ---- the segment, or this share of it, ends.  (Where a wait gave up, with NaN, and so do
    // the share's other ones: whoever joins a segment counts every part's ticket.)
    flush(1.f);
    l = live ? warp_sum(l) : NAN;
    const bool whole = n_units == cur.units;
    const int which = left == share_units ? 0 : 1;
    float* own = parts + which * U::share;
    if (!whole && lane == 0) {
      own[0] = m;
      own[1] = l;
      part_seg0[warp][which] = end - left - cur.unit;
      part_units[warp][which] = cur.units;
      part_op[warp][which] = seg_keys <= cur.keys ? seg_op : nullptr;  // null: a token outside the pool, zeros already
    }
    const float inv = __frcp_rn(l), drop = lift == 1.f ? 1.f : 1.f / kLift;
#pragma unroll
    for (int gi = 0; gi < G; ++gi) {
      const float z = warp_sum(zacc[gi]);
      float4 f;
      f.x = o[(4 * gi + 0) * 32];
      f.x = fmaf(f.x + __shfl_xor_sync(0xffffffffu, f.x, 2), drop, z);
      f.y = o[(4 * gi + 1) * 32];
      f.y = fmaf(f.y + __shfl_xor_sync(0xffffffffu, f.y, 2), drop, z);
      f.z = o[(4 * gi + 2) * 32];
      f.z = fmaf(f.z + __shfl_xor_sync(0xffffffffu, f.z, 2), drop, z);
      f.w = o[(4 * gi + 3) * 32];
      f.w = fmaf(f.w + __shfl_xor_sync(0xffffffffu, f.w, 2), drop, z);
      if (t == (gi & 3) >> 1) {
        const int c = 32 * gi + 4 * g;
        if (!whole) {
          *reinterpret_cast<float4*>(own + 4 + c) = f;
        } else if (seg_keys <= cur.keys) {
          f.x *= inv;
          f.y *= inv;
          f.z *= inv;
          f.w *= inv;
          store4<T>(seg_op, c, p.D, a.out_vec, f);
        }
      }
    }
    left -= n_units;
    cur = nxt;
  }
  // a wait gave up: let the copies in flight land before the warp exits
  if (!live)
    for (int i = 0; i < kStages; ++i) wait_copies(bars + 8 * i, parity >> i & 1);

  // ---- segments held in part.  A warp joins those whose first share in this CTA
  // is its own.
  __syncthreads();
  constexpr int V = (G + 3) / 4;  // float4s of a share per lane
  // a share's float4 number v of this lane
  auto in_share = [&](int v) { return v * 128 + lane * 4 < 32 * G; };
#pragma unroll 1
  for (int mine = 0; mine < 2; ++mine) {
    const int units = part_units[warp][mine];
    if (units == 0) continue;
    const unsigned seg0 = part_seg0[warp][mine];
    // begun in an earlier warp's part of the share: joined there
    if (seg0 < begin && begin > cta_begin) continue;
    T* const dest = part_op[warp][mine];
    Running<V> run;
    for (int w = warp; w < kWarps; ++w) {
      const int k = w == warp ? mine : 0;
      if (part_units[w][k] == 0 || part_seg0[w][k] != seg0) continue;
      const float* sh = reinterpret_cast<const float*>(smem + w * U::warp_bytes + U::parts) + k * U::share;
      float4 y[V];
#pragma unroll
      for (int v = 0; v < V; ++v)
        y[v] = in_share(v) ? reinterpret_cast<const float4*>(sh + 4)[v * 32 + lane] : make_float4(0.f, 0.f, 0.f, 0.f);
      run.add(sh[0], sh[1], y);
    }
    if (seg0 < cta_begin || seg0 + units > cta_end) {  // other CTAs hold parts of it
      const unsigned w0 = shares.holder(seg0, blockIdx.x), w1 = shares.holder(seg0 + units - 1, blockIdx.x);
      float* sh = a.ws + ((long long)blockIdx.x * 2 + (seg0 <= cta_begin ? 0 : 1)) * U::share;
      if (lane == 0) __stcg(reinterpret_cast<float4*>(sh), make_float4(run.m, run.l, 0.f, 0.f));
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (in_share(v)) __stcg(reinterpret_cast<float4*>(sh + 4) + v * 32 + lane, run.x[v]);
      __syncwarp();
      unsigned taken = 0;
      if (lane == 0) {
        taken = take_ticket(a.tickets + w0);
        if (taken == w1 - w0 + 1) a.tickets[w0] = 0;  // clean for the next launch
      }
      taken = __shfl_sync(0xffffffffu, taken, 0);
      if (taken != w1 - w0 + 1) continue;
      constexpr int kBatch = G > 4 ? 6 : 12;  // shares in flight
      run = Running<V>();
      for (unsigned w = w0; w <= w1; w += kBatch) {
        float4 ml[kBatch], y[kBatch][V];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const unsigned wk = w + k;
          // the segment is the last of the share that it starts in, the first of the others
          const float* o2 = a.ws + ((long long)wk * 2 + (wk == w0 && shares.begin(wk) < seg0 ? 1 : 0)) * U::share;
          const bool in = wk <= w1;
          ml[k] = in ? __ldcg(reinterpret_cast<const float4*>(o2)) : make_float4(-INFINITY, 0.f, 0.f, 0.f);
#pragma unroll
          for (int v = 0; v < V; ++v)
            y[k][v] = in && in_share(v) ? __ldcg(reinterpret_cast<const float4*>(o2 + 4) + v * 32 + lane)
                                        : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) run.add(ml[k].x, ml[k].y, y[k]);
      }
    }
    if (dest == nullptr) continue;
    const float inv = 1.0f / run.l;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      run.x[v].x *= inv;
      run.x[v].y *= inv;
      run.x[v].z *= inv;
      run.x[v].w *= inv;
      store4<T>(dest, v * 128 + lane * 4, p.D, a.out_vec, run.x[v]);
    }
  }
}

template <typename T, int G>
static int launch_row(const Pool& p, const Problem& a, int grid, cudaStream_t st) {
  static std::atomic<bool> ready[64] = {};
  const int dev = current_device();
  if (dev < 0 || dev >= 64) return fail(FML_EUNSUPPORTED, "neb_kv4_attention: device index out of range");
  if (!ready[dev].load()) {
    const cudaError_t e = cudaFuncSetAttribute(attn_row_kernel<T, G>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               Unit<T, G>::cta_bytes);
    if (e != cudaSuccess) return check_cuda(e, "neb_kv4_attention smem attribute");
    ready[dev].store(true);
  }
  const cudaError_t e = launch_pdl(attn_row_kernel<T, G>, dim3((unsigned)grid), dim3(Unit<T, G>::warps * 32),
                                   Unit<T, G>::cta_bytes, st, 1, p, a);
  count_launch();
  return check_cuda(e, "neb_kv4_attention launch");
}

// The row kernel's CTAs: one per SM.  The workspace holds the shares of every
// CTA, then the tickets.
static int row_grid() { return num_sms(current_device()); }
static size_t shares_bytes(const Pool& p) { return (size_t)row_grid() * 2 * (4 + 32 * p.G) * sizeof(float); }
static size_t workspace_bytes(const Pool& p) {
  return shares_bytes(p) + (size_t)row_grid() * sizeof(unsigned long long);
}

template <typename T>
static int attention(const Pool& p, Problem a, cudaStream_t st) {
  const int grid = row_grid();
  a.tickets = reinterpret_cast<unsigned long long*>(reinterpret_cast<uint8_t*>(a.ws) + shares_bytes(p));
  a.launch = launch_number();
  switch (p.G) {
    case 1: return launch_row<T, 1>(p, a, grid, st);
    case 2: return launch_row<T, 2>(p, a, grid, st);
    case 3: return launch_row<T, 3>(p, a, grid, st);
    case 4: return launch_row<T, 4>(p, a, grid, st);
    case 5: return launch_row<T, 5>(p, a, grid, st);
    case 6: return launch_row<T, 6>(p, a, grid, st);
    case 7: return launch_row<T, 7>(p, a, grid, st);
    default: return launch_row<T, 8>(p, a, grid, st);
  }
}

}  // namespace kv4
}  // namespace fml

using namespace fml;

extern "C" size_t neb_kv4_attention_workspace_size(const neb_kv4_pool* pool, int64_t batch, int64_t t,
                                                   int64_t q_heads) {
  kv4::Pool p;
  if (kv4::pool_from(pool, "neb_kv4_attention_workspace_size", &p) || batch <= 0 || t <= 0 || q_heads <= 0) return 0;
  if (q_heads % p.H == 0 && kv4::tc_covers(p, pool->dtype, t, q_heads / p.H))
    return kv4::tc_workspace_bytes(p, batch, t, q_heads / p.H);
  return kv4::workspace_bytes(p);
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
  if (!(scale > 0.f && scale <= 3.402823466e38f))
    return fail(FML_EINVAL, "neb_kv4_attention: scale must be positive and finite");
  if (batch > (1 << 24) || q_heads > (1 << 20) || batch * t > (1ll << 31) / q_heads / 8)
    return fail(FML_EUNSUPPORTED, "neb_kv4_attention: too many queries");
  const bool tc = kv4::tc_covers(p, pool->dtype, t, q_heads / p.H);
  const size_t need = tc ? kv4::tc_workspace_bytes(p, batch, t, q_heads / p.H) : kv4::workspace_bytes(p);
  if (workspace_bytes < need || (need && !workspace))
    return fail(FML_EWORKSPACE, "neb_kv4_attention: workspace of " + std::to_string(need) + " bytes needed");
  if (reinterpret_cast<uintptr_t>(workspace) & 15)
    return fail(FML_EINVAL, "neb_kv4_attention: workspace must be 16-byte aligned");
  kv4::Problem a = {};
  a.tq = (int)t;
  a.QH = (int)q_heads;
  a.group = (int)(q_heads / p.H);
  a.segs = (int)(t * q_heads);
  a.qs0 = q_strides[0];
  a.qs1 = q_strides[1];
  a.qs2 = q_strides[2];
  a.scale_log2 = scale * 1.4426950408889634f;
  a.scale_log2_wide = (double)scale * 1.4426950408889634;
  const size_t es = dtype_size(pool->dtype);
  a.q_vec = p.D % 8 == 0 && reinterpret_cast<uintptr_t>(q) % 16 == 0 && q_strides[0] * es % 16 == 0 &&
            q_strides[1] * es % 16 == 0 && q_strides[2] * es % 16 == 0;
  a.out_vec = p.D % 4 == 0 && reinterpret_cast<uintptr_t>(out) % 8 == 0;
  a.ws = static_cast<float*>(workspace);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (tc) {
    a.B = (int)batch;
    a.slot_of = slot_of;
    a.start_pos = start_pos;
    a.q = q;
    a.out = out;
    a.out_vec = p.D % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
    return kv4::tc_attention(p, a, pool->dtype, st);
  }
  // Units are counted in 31 bits: a larger batch goes in slices of requests.
  const int64_t per_request = t * q_heads * ((p.max_seq + kv4::kUnit - 1) / kv4::kUnit);
  const int64_t slice = std::min<int64_t>(batch, ((1ll << 31) - 1) / per_request);
  if (slice == 0) return fail(FML_EUNSUPPORTED, "neb_kv4_attention: too many queries");
  for (int64_t b = 0; b < batch; b += slice) {
    a.B = (int)std::min(slice, batch - b);
    a.slot_of = slot_of + b;
    a.start_pos = start_pos + b;
    a.q = static_cast<const uint8_t*>(q) + b * q_strides[0] * (int64_t)es;
    a.out = static_cast<uint8_t*>(out) + b * t * q_heads * p.D * (int64_t)es;
    const int rc = pool->dtype == FML_F32    ? kv4::attention<float>(p, a, st)
                   : pool->dtype == FML_BF16 ? kv4::attention<__nv_bfloat16>(p, a, st)
                                             : kv4::attention<__half>(p, a, st);
    if (rc != FML_OK) return rc;
  }
  return FML_OK;
}
