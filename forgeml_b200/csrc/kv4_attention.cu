// Attention over the 4-bit key/value cache (neb_kv4_attention).
//
//   out[b,t,h,:] = sum_j p_j v_j,  p = softmax_j(scale * q[b,t,h,:] . k_j),
//   j = 0 .. start_pos[b] + t,     k_j, v_j = z + c s per group (kv4.cuh)
//
// Per group of 32 channels the row's step and minimum leave the sums:
//   q . k_j = sum_g s_g[j] (q_g . c_g[j]) + z_g[j] sum(q_g)
//   out_g   = sum_j (p_j s_g[j]) c_g[j] + sum_j p_j z_g[j]
// so the matrix instructions multiply the codes themselves, which bfloat16
// holds exactly as 128 + c: one logic instruction turns two codes into two
// operands.  The 128s are taken off again by starting the score sums at
// -128 sum(q_g) and by one product of the weights with ones.
//
// Nothing else is rounded below fp32: q enters as a sum of bfloat16 parts (one
// for bf16, two for fp16, three for fp32: exact), p s as two (2^-17 of it;
// three for fp32).
#include <algorithm>
#include <string>

#include "kv4.cuh"

namespace fml {
namespace kv4 {

// One query row: each warp is a worker with its own contiguous share of all
// (request, head) rows of the batch, counted in units of 32 positions, so the
// work is even whatever the lengths are.  A worker streams its units through
// its own ring of shared memory with cp.async and keeps a running maximum,
// sum and output; a segment that it holds whole is written out, the others
// leave (maximum, sum, output) in the workspace for the join kernel.
constexpr int kUnit = 32;
constexpr int kWarps = 4;
constexpr int kStages = 2;

template <typename T, int G>
struct Unit {
  static constexpr int CR = 16 * G;                  // bytes of a row's codes
  static constexpr int PR = 2 * G * (int)sizeof(T);  // bytes of a row's parameters
  static constexpr int kc = 0, vc = kUnit * CR, kp = 2 * kUnit * CR, vp = kp + kUnit * PR;
  static constexpr int bytes = vp + kUnit * PR;
};

struct Problem {
  const int32_t *slot_of, *start_pos;
  int B, tq, QH, group;  // group: query heads of a key/value head
  long long qs0, qs1, qs2;
  float scale_log2;  // softmax scale * log2(e)
  const void* q;
  void* out;
  float* ws;  // [worker][first / last segment][rows][2 + 32 G]: maximum, sum, output
};

// Positions that request b's last query attends; 0 for a bad slot or position.
__device__ __forceinline__ int keys_of(const Pool& p, const Problem& a, int b) {
  const int slot = a.slot_of[b], start = a.start_pos[b];
  if (slot < 0 || slot >= p.slots || start < 0 || start >= p.max_seq) return 0;
  return min(start + a.tq, p.max_seq);
}
__device__ __forceinline__ int units_of(int keys) { return (keys + kUnit - 1) / kUnit; }

// Units of all requests before `b` (of one head); the whole warp calls.
__device__ __forceinline__ long long units_before(const Pool& p, const Problem& a, int b) {
  long long n = 0;
  for (int i = threadIdx.x & 31; i < b; i += 32) n += units_of(keys_of(p, a, i));
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) n += __shfl_xor_sync(0xffffffffu, n, off);
  return n;
}

// Where a worker is: request, head (times row tiles), unit of the segment.
struct Cursor {
  int b, seg, unit, keys, units;
  const Pool* p;
  const Problem* a;
  int segs;  // segments of a request
  __device__ __forceinline__ void request(int nb) {
    b = nb;
    keys = units = 0;
    while (b < a->B) {
      keys = keys_of(*p, *a, b);
      units = units_of(keys);
      if (units > 0) break;
      ++b;
    }
  }
  // The unit at place `at` of the batch's order (request, segment, unit).
  __device__ __forceinline__ void seek(long long at) {
    const int lane = threadIdx.x & 31;
    long long before = 0;
    for (int base = 0; base < a->B; base += 32) {
      const int i = base + lane;
      const long long mine = i < a->B ? (long long)units_of(keys_of(*p, *a, i)) * segs : 0;
      long long incl = mine;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const long long o = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += o;
      }
      const unsigned past = __ballot_sync(0xffffffffu, before + incl > at);
      if (past) {
        const int l = __ffs(past) - 1;
        const long long first = before + __shfl_sync(0xffffffffu, incl - mine, l);
        request(base + l);
        seg = (int)((at - first) / units);
        unit = (int)((at - first) % units);
        return;
      }
      before += __shfl_sync(0xffffffffu, incl, 31);
    }
  }
  __device__ __forceinline__ void next() {
    if (++unit < units) return;
    unit = 0;
    if (++seg < segs) return;
    seg = 0;
    request(b + 1);
  }
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Copies a unit's rows (those before `keys`; the rest of the stage keeps what
// it held and is masked) into a stage.
template <typename T, int G>
__device__ __forceinline__ void load_unit(const Pool& p, long long row, int nk, uint32_t dst) {
  using U = Unit<T, G>;
  const int lane = threadIdx.x & 31;
  const uint8_t* kc = p.kc + row * U::CR;
  const uint8_t* vc = p.vc + row * U::CR;
  const uint8_t* kp = static_cast<const uint8_t*>(p.kp) + row * U::PR;
  const uint8_t* vp = static_cast<const uint8_t*>(p.vp) + row * U::PR;
#pragma unroll
  for (int i = 0; i < G; ++i) {
    const int c = (i * 32 + lane) * 16;
    if (c < nk * U::CR) {
      cp_async16(dst + U::kc + c, kc + c);
      cp_async16(dst + U::vc + c, vc + c);
    }
  }
#pragma unroll
  for (int i = 0; i < (kUnit * U::PR + 511) / 512; ++i) {
    const int c = (i * 32 + lane) * 16;
    if (c < nk * U::PR) {
      cp_async16(dst + U::kp + c, kp + c);
      cp_async16(dst + U::vp + c, vp + c);
    }
  }
}

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float low_bf16(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_bf16(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// Codes i and i + 4 of a word as two bfloat16 numbers 128 + c.
template <int I>
__device__ __forceinline__ uint32_t codes2(uint32_t w) {
  return ((w >> (4 * I)) & 0x000f000fu) | 0x43004300u;
}

// N consecutive words / half words of shared memory, in the widest loads that
// their alignment (their own size's largest power of two) allows.
template <int N>
__device__ __forceinline__ void lds_words(const uint8_t* s, uint32_t (&w)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) *reinterpret_cast<uint4*>(&w[i]) = *reinterpret_cast<const uint4*>(s + 4 * i);
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) *reinterpret_cast<uint2*>(&w[i]) = *reinterpret_cast<const uint2*>(s + 4 * i);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = *reinterpret_cast<const uint32_t*>(s + 4 * i);
  }
}
// Pairs of half words (two groups a word); an odd last one sits alone.
template <int G>
__device__ __forceinline__ void lds_halves(const uint8_t* s, uint32_t (&w)[(G + 1) / 2]) {
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
template <typename T>
__device__ __forceinline__ float2 lds_param(const uint8_t* s) {
  if constexpr (sizeof(T) == 4) {
    return *reinterpret_cast<const float2*>(s);
  } else {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(s);
    const T* e = reinterpret_cast<const T*>(&w);
    return make_float2(to_f32<T>(e[0]), to_f32<T>(e[1]));
  }
}

template <typename T> struct Parts;
template <> struct Parts<__nv_bfloat16> { static constexpr int q = 1, p = 2; };
template <> struct Parts<__half> { static constexpr int q = 2, p = 2; };
template <> struct Parts<float> { static constexpr int q = 3, p = 3; };

// ---------------------------------------------------------------------------
// One query row per segment (a key/value head with one query head, one token).
//
// Scores, 8 positions a product (m16n8k16, A = query, B = codes): row j of A
// holds q restricted to group j (and j + 4 in a second product for D > 128),
// rows 4-7 its second bfloat16 part, rows 8-11 its third, so lane (g, t) gets
// the sums of group g & 3 for two positions, scales them and adds the groups
// up by shuffles.  For bf16, rows 4-7 repeat rows 0-3: one shuffle less.
// Output (A = codes: 16 channels, B = weights): column j of B holds p s of
// group j, column 4 + j the remainder of its rounding to bfloat16, and a tile
// of channels of group j takes its column j (+ 4 + j) at the end.
// Lane (g, t) = (lane / 4, lane % 4) handles the positions
//   t, 4 + (t ^ 1), 8 + t, 12 + (t ^ 1)
// of every 16: the scores' columns and the weights' rows are then the same
// positions (the weights need no exchange), and the rows that a quarter or half
// of the warp reads at once lie in distinct banks (kv4.cuh).
// ---------------------------------------------------------------------------
template <typename T, int G>
__global__ void __launch_bounds__(kWarps * 32, G <= 4 ? 4 : 2) attn_row_kernel(const Pool p, const Problem a) {
  using U = Unit<T, G>;
  constexpr int QP = Parts<T>::q, PP = Parts<T>::p;
  constexpr int SETS = (G + 3) / 4;
  extern __shared__ __align__(128) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * (kStages * U::bytes);
  const uint32_t ring_u32 = smem_u32(ring);
  pdl_wait();
  pdl_trigger();

  const long long total = units_before(p, a, a.B) * p.H;
  const long long W = min((long long)gridDim.x * kWarps, total), w = (long long)blockIdx.x * kWarps + warp;
  if (w >= W) return;  // every worker holds a unit
  const long long begin = total * w / W, end = total * (w + 1) / W;
  Cursor cur, pre;
  cur.p = &p;
  cur.a = &a;
  cur.segs = p.H;
  cur.seek(begin);
  pre = cur;
  long long left = end - begin, ahead = end - begin;
  auto prefetch = [&](int stage) {
    if (ahead > 0) {
      const long long row = head_row(p, a.slot_of[pre.b], pre.seg) + pre.unit * kUnit;
      load_unit<T, G>(p, row, min(kUnit, pre.keys - pre.unit * kUnit), ring_u32 + stage * U::bytes);
      pre.next();
      --ahead;
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) prefetch(i);

  const int col = g & 3;  // this lane's group within a set
  int krow[4];
  krow[0] = t;
  krow[1] = 4 + (t ^ 1);
  krow[2] = 8 + t;
  krow[3] = 12 + (t ^ 1);
  const int brow = (g & 1) ? 4 + ((g >> 1) ^ 1) : (g >> 1);  // position of column g of the scores' products

  uint32_t qa[G][2][2], qb[QP == 3 ? G : 1][2][2];  // A: rows g (and 8 + g), two products of 16 channels a group
  float qsum[SETS], qsum3[SETS];
  float o[2 * G][4], ones[SETS][4], zacc[SETS], m = -INFINITY, l = 0.f;
  int stage = 0;
  bool fresh = true;
  while (left > 0) {
    if (fresh) {  // a segment begins: its query, empty sums
      const T* qp = static_cast<const T*>(a.q) + cur.b * a.qs0 + cur.seg * a.qs2;
#pragma unroll
      for (int s = 0; s < SETS; ++s) {
        qsum[s] = qsum3[s] = zacc[s] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) ones[s][i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < 2 * G; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
      m = -INFINITY;
      l = 0.f;
#pragma unroll
      for (int gi = 0; gi < G; ++gi) {
        const bool own = (gi & 3) == col;
        float part[8], third[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int c = gi * 32 + 8 * t + i;
          const float x = own && c < p.D ? to_f32<T>(qp[c]) : 0.f;
          const float p1 = __bfloat162float(__float2bfloat16_rn(x));
          const float p2 = __bfloat162float(__float2bfloat16_rn(x - p1));
          part[i] = QP == 1 || g < 4 ? p1 : p2;
          third[i] = g < 4 ? x - p1 - p2 : 0.f;
          qsum[gi / 4] += part[i];
          qsum3[gi / 4] += third[i];
        }
        // pairs of a product: codes i and i + 4 share a register
        qa[gi][0][0] = pack_bf16(part[0], part[4]);
        qa[gi][0][1] = pack_bf16(part[1], part[5]);
        qa[gi][1][0] = pack_bf16(part[2], part[6]);
        qa[gi][1][1] = pack_bf16(part[3], part[7]);
        if constexpr (QP == 3) {
          qb[gi][0][0] = pack_bf16(third[0], third[4]);
          qb[gi][0][1] = pack_bf16(third[1], third[5]);
          qb[gi][1][0] = pack_bf16(third[2], third[6]);
          qb[gi][1][1] = pack_bf16(third[3], third[7]);
        }
      }
#pragma unroll
      for (int s = 0; s < SETS; ++s) {
#pragma unroll
        for (int off = 1; off <= 2; off <<= 1) {
          qsum[s] += __shfl_xor_sync(0xffffffffu, qsum[s], off);
          qsum3[s] += __shfl_xor_sync(0xffffffffu, qsum3[s], off);
        }
      }
      fresh = false;
    }
    cp_async_wait<kStages - 2>();
    __syncwarp();
    prefetch(stage == 0 ? kStages - 1 : stage - 1);
    const uint8_t* st = ring + stage * U::bytes;
    const int nk = min(kUnit, cur.keys - cur.unit * kUnit);

    // ---- scores of the unit's positions: sc[i] for krow[i & 3] + 16 (i >> 2)
    float sc[8];
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
      float c[2][SETS][4];
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        uint32_t kw[G];
        lds_words<G>(st + U::kc + (sub * 16 + nt * 8 + brow) * U::CR + t * 4 * G, kw);
#pragma unroll
        for (int s = 0; s < SETS; ++s) {
          c[nt][s][0] = c[nt][s][1] = -128.f * qsum[s];
          c[nt][s][2] = c[nt][s][3] = QP == 3 ? -128.f * qsum3[s] : 0.f;
        }
#pragma unroll
        for (int gi = 0; gi < G; ++gi) {
          const uint32_t b3 = QP == 3 ? qb[QP == 3 ? gi : 0][0][0] : 0u, b4 = QP == 3 ? qb[QP == 3 ? gi : 0][0][1] : 0u;
          const uint32_t b5 = QP == 3 ? qb[QP == 3 ? gi : 0][1][0] : 0u, b6 = QP == 3 ? qb[QP == 3 ? gi : 0][1][1] : 0u;
          mma_bf16(c[nt][gi / 4], qa[gi][0][0], b3, qa[gi][0][1], b4, codes2<0>(kw[gi]), codes2<1>(kw[gi]));
          mma_bf16(c[nt][gi / 4], qa[gi][1][0], b5, qa[gi][1][1], b6, codes2<2>(kw[gi]), codes2<3>(kw[gi]));
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x = 0.f;
#pragma unroll
        for (int s = 0; s < SETS; ++s) {
          const int gi = col + 4 * s;
          if (gi < G) {
            const float2 sz = lds_param<T>(st + U::kp + (sub * 16 + krow[i]) * U::PR + gi * 2 * (int)sizeof(T));
            const float dot = QP == 3 ? c[i >> 1][s][i & 1] + c[i >> 1][s][2 + (i & 1)] : c[i >> 1][s][i & 1];
            x = fmaf(sz.x, dot, fmaf(sz.y, QP == 3 ? qsum[s] + qsum3[s] : qsum[s], x));
          }
        }
        sc[sub * 4 + i] = x;
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sc[i] += __shfl_xor_sync(0xffffffffu, sc[i], 4);
      sc[i] += __shfl_xor_sync(0xffffffffu, sc[i], 8);
      if (QP > 1) sc[i] += __shfl_xor_sync(0xffffffffu, sc[i], 16);
      sc[i] *= a.scale_log2;
      if (krow[i & 3] + 16 * (i >> 2) < nk) mx = fmaxf(mx, sc[i]);
    }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    if (mx > m) {  // the same in every lane
      const float alpha = ex2(m - mx);
      m = mx;
      l *= alpha;
#pragma unroll
      for (int s = 0; s < SETS; ++s) {
        zacc[s] *= alpha;
#pragma unroll
        for (int e = 0; e < 4; ++e) ones[s][e] *= alpha;
      }
#pragma unroll
      for (int i = 0; i < 2 * G; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] *= alpha;
    }

    // ---- weights and output
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
      if (sub == 1 && nk <= 16) break;
      float pr[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        pr[i] = krow[i] + 16 * sub < nk ? ex2(sc[sub * 4 + i] - m) : 0.f;
        l += pr[i];
      }
      uint32_t b[SETS][2], b3[SETS][2];
#pragma unroll
      for (int s = 0; s < SETS; ++s) {
        const int gi = col + 4 * s;
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = 0.f;
          if (gi < G && krow[i] + 16 * sub < nk) {
            const float2 sz = lds_param<T>(st + U::vp + (sub * 16 + krow[i]) * U::PR + gi * 2 * (int)sizeof(T));
            x[i] = pr[i] * sz.x;
            zacc[s] = fmaf(pr[i], sz.y, zacc[s]);
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t h = pack_bf16(x[2 * i], x[2 * i + 1]);
          const float r0 = x[2 * i] - low_bf16(h), r1 = x[2 * i + 1] - high_bf16(h);
          const uint32_t r = pack_bf16(r0, r1);
          b[s][i] = g < 4 ? h : r;
          if constexpr (PP == 3) b3[s][i] = g < 4 ? 0u : pack_bf16(r0 - low_bf16(r), r1 - high_bf16(r));
        }
        mma_bf16(ones[s], 0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u, b[s][0], b[s][1]);
        if constexpr (PP == 3)
          mma_bf16(ones[s], 0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u, b3[s][0], b3[s][1]);
      }
      uint32_t vw[4][(G + 1) / 2];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        lds_halves<G>(st + U::vc + (sub * 16 + krow[i]) * U::CR + ((g * 2 * G) ^ v_swizzle(G, krow[i])), vw[i]);
#pragma unroll
      for (int gi = 0; gi < G; ++gi) {
        const uint32_t sel = (gi & 1) ? 0x7632u : 0x5410u;  // this group's half of both words
        const uint32_t u = __byte_perm(vw[0][gi / 2], vw[1][gi / 2], sel);
        const uint32_t v = __byte_perm(vw[2][gi / 2], vw[3][gi / 2], sel);
        mma_bf16(o[2 * gi], codes2<0>(u), codes2<1>(u), codes2<0>(v), codes2<1>(v), b[gi / 4][0], b[gi / 4][1]);
        mma_bf16(o[2 * gi + 1], codes2<2>(u), codes2<3>(u), codes2<2>(v), codes2<3>(v), b[gi / 4][0], b[gi / 4][1]);
        if constexpr (PP == 3) {
          mma_bf16(o[2 * gi], codes2<0>(u), codes2<1>(u), codes2<0>(v), codes2<1>(v), b3[gi / 4][0], b3[gi / 4][1]);
          mma_bf16(o[2 * gi + 1], codes2<2>(u), codes2<3>(u), codes2<2>(v), codes2<3>(v), b3[gi / 4][0], b3[gi / 4][1]);
        }
      }
    }
    stage = stage == kStages - 1 ? 0 : stage + 1;
    --left;
    const bool last = cur.unit + 1 == cur.units;
    if (last || left == 0) {  // the segment, or this worker's share, ends here
      const long long done = end - left;          // place just past this unit
      const long long seg0 = done - cur.unit - 1;  // the segment's first unit
      const bool whole = last && seg0 >= begin;
      float lt = l;
      lt += __shfl_xor_sync(0xffffffffu, lt, 1);
      lt += __shfl_xor_sync(0xffffffffu, lt, 2);
#pragma unroll
      for (int s = 0; s < SETS; ++s) {
        zacc[s] += __shfl_xor_sync(0xffffffffu, zacc[s], 1);
        zacc[s] += __shfl_xor_sync(0xffffffffu, zacc[s], 2);
      }
      T* op = static_cast<T*>(a.out) + ((long long)cur.b * a.QH + cur.seg) * p.D;
      float* wp = a.ws + (w * 2 + (seg0 <= begin ? 0 : 1)) * (2 + 32 * G);
      if (!whole && lane == 0) {
        wp[0] = m;
        wp[1] = lt;
      }
      const float inv = 1.0f / lt;
#pragma unroll
      for (int gi = 0; gi < G; ++gi) {
        const float z = __shfl_sync(0xffffffffu, zacc[gi / 4], (gi & 3) * 4);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // channels 32 gi + 4 g + 2 h, + 1: rows g and g + 8 of the tile
          float x0 = fmaf(-128.f, ones[gi / 4][gi & 1], o[2 * gi + h][gi & 1]);
          float x1 = fmaf(-128.f, ones[gi / 4][gi & 1], o[2 * gi + h][2 + (gi & 1)]);
          x0 += __shfl_xor_sync(0xffffffffu, x0, 2);
          x1 += __shfl_xor_sync(0xffffffffu, x1, 2);
          x0 += z;
          x1 += z;
          if (t == (gi & 3) >> 1) {
            const int c = 32 * gi + 4 * g + 2 * h;
            if (whole) {
              if (c < p.D) op[c] = from_f32<T>(x0 * inv);
              if (c + 1 < p.D) op[c + 1] = from_f32<T>(x1 * inv);
            } else {
              *reinterpret_cast<float2*>(wp + 2 + c) = make_float2(x0, x1);
            }
          }
        }
      }
      fresh = true;
    }
    cur.next();
    __syncwarp();
  }
  cp_async_wait<0>();
}

// Joins the workers' shares of the segments that more than one of them holds,
// in the workers' order; zeros for bad requests.  One CTA per segment: its
// threads take the channels (times slices of the shares, so that a segment of
// hundreds of shares is not one long chain of loads).
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
  const int b = blockIdx.x / p.H, seg = blockIdx.x % p.H;
  const int keys = keys_of(p, a, b), units = units_of(keys);
  T* op = static_cast<T*>(a.out) + ((long long)b * a.QH + seg) * p.D;
  if (keys == 0) {
    if (tid == 0) raise_device_error(DEV_ERR_ATTN_RANGE);
    for (int d = tid; d < p.D; d += kJoinThreads) op[d] = from_f32<T>(0.f);
    return;
  }
  const long long total = units_before(p, a, a.B) * p.H;
  const long long u0 = units_before(p, a, b) * p.H + (long long)seg * units, u1 = u0 + units;
  W = min(W, total);
  // worker of a unit u: the largest w with total * w / W <= u
  const long long w0 = ((u0 + 1) * W - 1) / total, w1 = (u1 * W - 1) / total;
  if (w0 == w1) return;
  constexpr int stride = 2 + CH;
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
    float mx = mine;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
    __syncthreads();  // the previous round's weights are read
    if (lane == 0) red[warp] = mx;
    __syncthreads();
    mx = m;
#pragma unroll
    for (int i = 0; i < kJoinThreads / 32; ++i) mx = fmaxf(mx, red[i]);
    const float alpha = m == -INFINITY ? 0.f : ex2(m - mx);
    m = mx;
    const float f = tid < n ? ex2(mine - m) : 0.f;
    weight[tid] = f;
    float part = f * ml;
    if (tid >= n) part = 0.f;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) part += __shfl_xor_sync(0xffffffffu, part, off);
    __syncthreads();
    if (lane == 0) red[warp] = part;
    __syncthreads();
    l *= alpha;
#pragma unroll
    for (int i = 0; i < kJoinThreads / 32; ++i) l += red[i];
    x *= alpha;
    if (sl < SL) {
#pragma unroll 4
      for (int i = sl; i < n; i += SL) x = fmaf(weight[i], a.ws[(long long)place[i] * stride + 2 + ch], x);
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
  constexpr int smem = kWarps * kStages * Unit<T, G>::bytes;
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
  e = launch_pdl(attn_join_kernel<T, G>, dim3((unsigned)(a.B * p.H)), dim3(kJoinThreads), 0, st, 1, p, a,
                 (long long)grid * kWarps);
  count_launch();
  return check_cuda(e, "neb_kv4_attention join launch");
}

constexpr int kSimpleWarps = 8;
// One CTA per (request, token, query head), a warp per row; lane l holds
// channels 32 g + l.
template <typename T>
__global__ void __launch_bounds__(kSimpleWarps * 32)
    attn_simple_kernel(const T* __restrict__ q, long long qs0, long long qs1, long long qs2, const Pool p,
                const int32_t* __restrict__ slot_of, const int32_t* __restrict__ start_pos, T* __restrict__ out,
                int tq, int QH, float scale) {
  pdl_wait();
  pdl_trigger();
  __shared__ float sm_o[kSimpleWarps][kMaxD], sm_m[kSimpleWarps], sm_l[kSimpleWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int qh = blockIdx.x % QH, t = (blockIdx.x / QH) % tq, b = blockIdx.x / QH / tq;
  const int h = qh / (QH / p.H);
  const int slot = slot_of[b], start = start_pos[b];
  const bool bad = slot < 0 || slot >= p.slots || start < 0 || start > p.max_seq - 1 - t;
  T* op = out + (((long long)b * tq + t) * QH + qh) * p.D;
  if (bad) {
    if (threadIdx.x == 0) raise_device_error(DEV_ERR_ATTN_RANGE);
    for (int d = threadIdx.x; d < p.D; d += blockDim.x) op[d] = from_f32<T>(0.f);
    return;
  }
  const long long r0 = head_row(p, slot, h);
  constexpr int MG = kMaxD / kGroup;
  float qv[MG], o[MG];
#pragma unroll
  for (int g = 0; g < MG; ++g) {
    const int c = g * 32 + lane;
    qv[g] = c < p.D ? to_f32<T>(q[b * qs0 + t * qs1 + qh * qs2 + c]) * scale : 0.f;
    o[g] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int pos = warp; pos <= start + t; pos += kSimpleWarps) {
    const long long r = r0 + pos;
    float s = 0.f;
#pragma unroll
    for (int g = 0; g < MG; ++g) {
      if (g >= p.G) break;
      const int c = g * 32 + lane;
      const T* pr = static_cast<const T*>(p.kp) + (r * p.G + g) * 2;
      const int code = p.kc[r * 16 * p.G + k_byte(p.G, c)] >> (4 * (c & 1)) & 15;
      if (c < p.D) s = fmaf(qv[g], fmaf((float)code, to_f32<T>(pr[0]), to_f32<T>(pr[1])), s);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    const float mn = fmaxf(m, s), alpha = expf(m - mn), pr_ = expf(s - mn);
    l = l * alpha + pr_;
    m = mn;
#pragma unroll
    for (int g = 0; g < MG; ++g) {
      if (g >= p.G) break;
      const int c = g * 32 + lane;
      const T* pr = static_cast<const T*>(p.vp) + (r * p.G + g) * 2;
      const int code = p.vc[r * 16 * p.G + v_byte(p.G, c, pos)] >> (4 * (c & 1)) & 15;
      o[g] = fmaf(pr_, fmaf((float)code, to_f32<T>(pr[0]), to_f32<T>(pr[1])), o[g] * alpha);
    }
  }
#pragma unroll
  for (int g = 0; g < MG; ++g) sm_o[warp][g * 32 + lane] = o[g];
  if (lane == 0) {
    sm_m[warp] = m;
    sm_l[warp] = l;
  }
  __syncthreads();
  float mm = -INFINITY, ll = 0.f, w[kSimpleWarps];
  for (int i = 0; i < kSimpleWarps; ++i) mm = fmaxf(mm, sm_m[i]);
  for (int i = 0; i < kSimpleWarps; ++i) {
    w[i] = sm_m[i] == -INFINITY ? 0.f : expf(sm_m[i] - mm);
    ll += w[i] * sm_l[i];
  }
  for (int d = threadIdx.x; d < p.D; d += blockDim.x) {
    float acc = 0.f;
    for (int i = 0; i < kSimpleWarps; ++i) acc += w[i] * sm_o[i][d];
    op[d] = from_f32<T>(acc / ll);
  }
}


// Workers' grid of the row kernel: a whole number of resident CTAs per SM, no
// more workers than the longest batch has units.
template <typename T, int G>
static int row_grid(const Pool& p, long long segments) {
  const int smem = kWarps * kStages * Unit<T, G>::bytes;
  const int per_sm = std::max(1, std::min(G <= 4 ? 4 : 2, (227 * 1024) / (smem + 1024)));
  const long long units = segments * ((p.max_seq + kUnit - 1) / kUnit);
  return (int)std::min<long long>((long long)per_sm * num_sms(current_device()), (units + kWarps - 1) / kWarps);
}

template <typename T>
static int grid_of(const Pool& p, long long segments) {
  switch (p.G) {
#define KV4_CASE(G) case G: return row_grid<T, G>(p, segments);
    KV4_CASE(1) KV4_CASE(2) KV4_CASE(3) KV4_CASE(4) KV4_CASE(5) KV4_CASE(6) KV4_CASE(7)
#undef KV4_CASE
    default: return row_grid<T, 8>(p, segments);
  }
}

static size_t workspace_bytes(const Pool& p, int dtype, int64_t batch, int64_t t, int64_t q_heads) {
  if (t != 1 || q_heads != p.H) return 0;
  const long long segs = batch * p.H;
  const int grid = dtype == FML_F32 ? grid_of<float>(p, segs) : grid_of<__half>(p, segs);
  return (size_t)grid * kWarps * 2 * (2 + 32 * p.G) * sizeof(float);
}

template <typename T>
static int attention(const Pool& p, const Problem& a, cudaStream_t st) {
  if (a.tq == 1 && a.group == 1) {
    const int grid = grid_of<T>(p, (long long)a.B * p.H);
    switch (p.G) {
#define KV4_CASE(G) case G: return launch_row<T, G>(p, a, grid, st);
      KV4_CASE(1) KV4_CASE(2) KV4_CASE(3) KV4_CASE(4) KV4_CASE(5) KV4_CASE(6) KV4_CASE(7)
#undef KV4_CASE
      default: return launch_row<T, 8>(p, a, grid, st);
    }
  }
  const cudaError_t e =
      launch_pdl(attn_simple_kernel<T>, dim3((unsigned)((long long)a.B * a.tq * a.QH)), dim3(kSimpleWarps * 32), 0, st, 1,
                 static_cast<const T*>(a.q), a.qs0, a.qs1, a.qs2, p, a.slot_of, a.start_pos, static_cast<T*>(a.out),
                 a.tq, a.QH, a.scale_log2 * 0.6931471805599453f);
  count_launch();
  return check_cuda(e, "neb_kv4_attention launch");
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
