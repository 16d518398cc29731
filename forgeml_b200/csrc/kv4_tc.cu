// Attention of several query rows over the 4-bit key/value cache on the tcgen05
// tensor cores: a prompt's tokens, a few drafted ones, query heads that share a
// key/value head (16-bit types).
//
// A segment is a request's key/value head with up to 128 of its query rows (row =
// token * group + query head within the group: UMMA M, the TMEM lanes).  Its
// positions go by in blocks of 128, a running maximum and sum, warp-specialised:
//
//   warps 8-11  turn the cache's codes into fp16 operands: a lane takes a position's
//               key and value, loaded a block ahead, and writes z + c s, rounded once,
//               into the swizzled blocks (two of each).  A code under the exponent of
//               1024 is a 16-bit number, two at a time; the channels of every eight
//               stay in the order 0 4 1 5 2 6 3 7 that this leaves, in the queries too,
//               and are put right where the output is written;
//   warp 12     TMEM owner and single-thread UMMA issuer: S = Q K^T of block j + 1
//               into the other of two TMEM score blocks while block j's softmax
//               runs, O += P V into TMEM;
//   warps 0-7   queries, softmax and epilogue: two threads a row, half of a block's
//               positions (and of the output's channels) each, the scores read from
//               TMEM once (blocks of numbers of very different sizes: position by
//               position, see power_to_12).
//
// Rounded below fp32: the operands (keys, values) and P, to fp16, whose 11 bits cost
// the output no more than its own rounding to the cache's type.
//
// Measured: 8 x 1000 tokens after 0 .. 1048 others, 16 heads of 128, bf16: 224.6 us,
// 299 TFLOP/s; 16 requests of 4000 .. 8190 positions, 8 heads of 128 with 4 query
// heads each, go through the row kernel (tc_covers).  A block of 128 positions takes
// about 4600 cycles, bound by the softmax warps' chain (scores from TMEM, maximum,
// exponentials, P to TMEM), with the dequantisation hidden behind it.
//
// Work: either one segment per CTA (prompts: enough segments), or, for few
// segments, equal shares of all blocks per CTA with the split segments joined by
// the last CTA to arrive (kv4_attention.cuh).
//
// Every wait is bounded (DEV_ERR_ATTN_TIMEOUT); a CTA that gives up lets its
// products finish and frees its TMEM before it exits.
#include <string>
#include <type_traits>

#include "kv4_tc_walk.cuh"

namespace fml {
namespace kv4 {
namespace tc {

constexpr int kThreads = 416;
constexpr int kDequant = 8, kMma = 12;  // first warps of the roles
// TMEM columns: two score blocks, the output, P and the queries (fp16 pairs).  P and
// the queries as operands from TMEM halve what the products read of shared memory,
// whose bandwidth the operands' writes and reads are bound by.  Above 128 channels
// there is room for one block of operands and of scores, and P takes the place of
// the scores that it is made of: a block's softmax then waits for the block before.
constexpr uint32_t kTmemCols = 512;

template <int G>
struct Smem {
  static constexpr int D = 32 * G, kSlabs = (G + 1) / 2;  // 128-byte slabs along the head dim
  static constexpr uint32_t kTileBytes = 2 * kTile * G * (16 + 4);
  static constexpr uint32_t kOperand = kRows * 128 * kSlabs;
  static constexpr uint32_t stages = G > 4 ? 1 : 2;
  static constexpr uint32_t tm_o = stages * kBlock, tm_p = G > 4 ? 0 : 384, tm_q = G > 4 ? 384 : 448;
  static_assert(tm_o + D <= (G > 4 ? tm_q : tm_p) && tm_q + D / 2 <= kTmemCols, "TMEM");
  static constexpr uint32_t k = 0, v = stages * kOperand;
  static constexpr uint32_t bars = 2 * stages * kOperand;
  static constexpr uint32_t rows = bars + 512;  // what a row's two threads tell each other: [2][2][128] fp32 pairs
  static constexpr uint32_t factors = rows + 4096;  // the tiles' keys' powers of two and values' exponents: [4 blocks][2][4]
  static constexpr uint32_t nans = factors + 128;   // first position whose value is NaN: [4 parts][4 tiles][8 groups]
  static constexpr uint32_t own = nans + 512;  // wide tiles' positions' factors of their scores, values' exponents: [4 blocks][2][128] fp32
  static constexpr uint32_t total = own + 4096 + 1024;  // 1024: alignment of the base
  static_assert(total <= 227 * 1024, "shared memory");
};
enum Bar : int {
  kQFull = 0, kKFull = 1, kKEmpty = kKFull + 2,
  kVFull = kKEmpty + 2, kVEmpty = kVFull + 2, kSFull = kVEmpty + 2, kPFull = kSFull + 2, kOFull, kTogether, kPair, kNumBars = kPair + 4
};

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void sts4(uint32_t at, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
// 64 consecutive fp32 columns of the warp's 32 TMEM lanes; complete on return.
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, float (&v)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
      "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63"
      "}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
        "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
        "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31]),
        "=f"(v[32]), "=f"(v[33]), "=f"(v[34]), "=f"(v[35]), "=f"(v[36]), "=f"(v[37]), "=f"(v[38]), "=f"(v[39]),
        "=f"(v[40]), "=f"(v[41]), "=f"(v[42]), "=f"(v[43]), "=f"(v[44]), "=f"(v[45]), "=f"(v[46]), "=f"(v[47]),
        "=f"(v[48]), "=f"(v[49]), "=f"(v[50]), "=f"(v[51]), "=f"(v[52]), "=f"(v[53]), "=f"(v[54]), "=f"(v[55]),
        "=f"(v[56]), "=f"(v[57]), "=f"(v[58]), "=f"(v[59]), "=f"(v[60]), "=f"(v[61]), "=f"(v[62]), "=f"(v[63])
      : "r"(taddr)
      : "memory");
}

// 16 columns of 32 bits (32 fp16 numbers of a row); tmem_st_wait() completes them.
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&w)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]), "r"(w[8]), "r"(w[9]),
      "r"(w[10]), "r"(w[11]), "r"(w[12]), "r"(w[13]), "r"(w[14]), "r"(w[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 8 fp32 columns; complete on return.
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, float (&v)[8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const float (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n\ttcgen05.wait::st.sync.aligned;" ::"r"(taddr),
               "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st4(uint32_t taddr, const uint32_t (&w)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};\n\ttcgen05.wait::st.sync.aligned;" ::"r"(taddr),
               "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
               : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
// D[tmem] (+)= A[tmem] * B[smem desc]^T: A's row is its TMEM lane, two fp16 numbers a
// column.
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// The tensor cores multiply fp16 numbers whatever the cache's type: bf16 numbers,
// rounded to 8 bits once more, would double the output's error.  bf16's range is
// kept by powers of two: of a query row, of a tile's keys and of a tile's values,
// each chosen so that the largest number lies near 2^12 (numbers 2^-26 of that are
// still whole).  They are taken off the scores.  On the values' side a row's weights
// become P = p 2^(14 - e - w): e the exponent of the position's tile, w the running
// maximum of (log2 of the tile's largest p) - e over the tiles that the row attends.
// So P is at most 2^14, and near it where weight times value is largest, whatever a
// value of vanishing weight, or one that the row does not attend, is; the output is
// in units of 2^(w - 14).  w is kept against the scores' running maximum.
//
// A tile whose positions' largest keys, or values, differ by more than kWide is a wide
// one: its positions have powers of their own, so that none takes the others' bits,
// attended or not, and a block with such a tile has its weights formed position by
// position.  (None of the usual caches has any.)
//
// 2^12 over the power of two at or below x (positive, not NaN); 2^126 at most (a
// fast division by more gives 0).
__device__ __forceinline__ float power_to_12(float x) {
  const int e = __float_as_int(x) >> 23;
  return __int_as_float(max(1, min(253, 266 - e)) << 23);
}
__device__ __forceinline__ float exponent_of(float power) { return (float)((__float_as_int(power) >> 23) - 127); }
constexpr float kTop = 14.f;  // log2 of the largest weight as the tensor cores get it
constexpr float kWide = 1024.f;  // (of fp16's 27 binades that leaves every position 17)
// Scores from which on the rounding of their maximum shows in the weights.
constexpr float kFar = 4194304.f;  // 2^22
// What fp16's weights and their sum are taken against, for a maximum m: they go up to
// 2^14 as well where m keeps its ones (up to 1 they would end at 2^-25, and of many small
// ones beside a large one none would count).
template <typename T>
__device__ __forceinline__ float base_of(float m) {
  return std::is_same<T, __half>::value && fabsf(m) < kFar ? m - kTop : m;
}

// A word of eight codes as eight fp16 numbers z + c s (s, z in `sz`), in the order
// 0 4 1 5 2 6 3 7, within the finite range that a rounded-up step could leave.
__device__ __forceinline__ uint4 operand8(uint32_t w, uint32_t sz) {
  const uint32_t exponent = 0x64006400u, top = 0x7bff7bffu;
  const uint32_t ss = __byte_perm(sz, sz, 0x1010), zz = __byte_perm(sz, sz, 0x3232);
  uint32_t e[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t c = ((w >> (4 * i)) & 0x000f000fu) | exponent;
    const __half2 x =
        __hmin2_nan(__hfma2(__hsub2(*reinterpret_cast<const __half2*>(&c), *reinterpret_cast<const __half2*>(&exponent)),
                            *reinterpret_cast<const __half2*>(&ss), *reinterpret_cast<const __half2*>(&zz)),
                    *reinterpret_cast<const __half2*>(&top));
    e[i] = *reinterpret_cast<const uint32_t*>(&x);
  }
  return make_uint4(e[0], e[1], e[2], e[3]);
}
// (s, z) of the cache's type times a power of two, in fp16; and the largest
// number that a group can stand for.
template <typename T>
__device__ __forceinline__ uint32_t scaled_params(uint32_t sz, float f) {
  if constexpr (std::is_same<T, __half>::value) {
    return sz;
  } else {
    return pack2<__half>(__uint_as_float(sz << 16) * f, __uint_as_float(sz & 0xffff0000u) * f);
  }
}
__device__ __forceinline__ float largest_of(uint32_t sz) {  // bf16
  const float s = __uint_as_float(sz << 16), z = __uint_as_float(sz & 0xffff0000u);
  return fmaxf(fabsf(z), fabsf(fmaf(15.f, s, z)));
}

// Whether a group's numbers are NaN, as its parameters are: an exponent of ones, plus
// one, carries into the sign's place.
template <typename T>
__device__ __forceinline__ uint32_t reads_nan(uint32_t sz) {
  constexpr bool half = std::is_same<T, __half>::value;
  return ((sz & (half ? 0x7c007c00u : 0x7f807f80u)) + (half ? 0x04000400u : 0x00800080u)) & 0x80008000u;
}

template <typename T, int G>
__global__ void __launch_bounds__(kThreads, 1)
    attn_tc_kernel(const Pool p, const Problem a, const int row_tiles, const int shared_blocks) {
  using L = Smem<G>;
  constexpr int D = L::D;  // channels of whole groups; the row has p.D of them
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  constexpr unsigned NS = L::stages;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const mem = smem_raw + (base - smem_u32(smem_raw));
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  auto bar = [&](int i) { return base + L::bars + 8u * (uint32_t)i; };
  const uint32_t tmem_holder = base + L::bars + 8u * kNumBars;
  if (threadIdx.x == 0) {
    mbar_init(bar(kQFull), 8);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(kKFull + i), 4);
      mbar_init(bar(kKEmpty + i), 1);
      mbar_init(bar(kVFull + i), 4);
      mbar_init(bar(kVEmpty + i), 1);
      mbar_init(bar(kSFull + i), 1);
    }
    mbar_init(bar(kPFull), 8);
    mbar_init(bar(kTogether), 8);
    for (int i = 0; i < 4; ++i) mbar_init(bar(kPair + i), 2);
    mbar_init(bar(kOFull), 1);
    fence_mbar_init();
  }
  if (warp == kMma) {
    tmem_alloc(tmem_holder, kTmemCols);
    tmem_relinquish();
  }
  pdl_wait();
  pdl_trigger();
  // ---- this CTA's work
  __shared__ unsigned taken_sh, took_sh, total_sh;  // tickets of a word; this CTA's parts that took theirs; the batch's units
  __shared__ bool gave_up_sh;
  if (threadIdx.x == 0) {
    took_sh = 0;
    gave_up_sh = false;
  }
  Walk walk;
  walk.shared = shared_blocks != 0;
  walk.row_tiles = row_tiles;
  walk.begin = walk.at = 0;
  Shares shares(1, 1);
  if (walk.shared) {
    const Plan<kBlock> plan(p, a);
    // a share of a few blocks at least: an empty one could not be joined
    shares = Shares(plan.total, min(gridDim.x, (plan.total + 1) / 2));
    if (threadIdx.x == 0) total_sh = plan.total;
    walk.left = 0;
    if (plan.total > 0 && blockIdx.x < shares.W) {
      walk.begin = walk.at = shares.begin(blockIdx.x);
      walk.left = (int)(shares.begin(blockIdx.x + 1) - walk.begin);
      walk.cur = plan.seek(p, a, walk.begin);
    }
  } else {
    // one segment; the longest (a head's last rows) of every request first
    const int per_tile = gridDim.x / row_tiles, tile = blockIdx.x / per_tile, bh = blockIdx.x - tile * per_tile;
    walk.cur.b = bh / p.H;
    walk.cur.seg = (bh - walk.cur.b * p.H) * row_tiles + (row_tiles - 1 - tile);
    walk.cur.unit = 0;
    walk.cur.keys = keys_of(p, a, walk.cur.b);
    walk.cur.units = 1;
    walk.left = walk.cur.keys > 0 ? 1 : 0;
  }
  // Zeros for queries without a place in the pool.
  for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
    const int keys = keys_of(p, a, b), good = keys == 0 ? 0 : min(a.tq, keys - a.start_pos[b]);
    if (good == a.tq) continue;
    if (threadIdx.x == 0) raise_device_error(DEV_ERR_ATTN_RANGE);
    const long long n = (long long)(a.tq - good) * a.QH * p.D;
    T* bad = static_cast<T*>(a.out) + ((long long)b * a.tq + good) * a.QH * p.D;
    for (long long i = threadIdx.x; i < n; i += kThreads) bad[i] = from_f32<T>(0.f);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(tmem_holder) : "memory");

  Part part;
  if (warp == kMma) {
    // ------------------------------------------------------------ UMMA issuer
    // The whole warp walks along (its values are then the same in every lane, which
    // the products' operands must be); one lane issues.  It polls: its answer to P is
    // on the blocks' critical path.
    const uint32_t id_s = umma_idesc(0, 0, 0, kBlock);  // fp16: Q (TMEM) x K (K-major)
    const uint32_t id_o = umma_idesc(0, 0, 1, D);       // P (TMEM) x V (MN-major along the head dim)
    const bool leader = elect_one();
    const uint64_t dk0 = umma_desc_sw128(base + L::k, 16u, 1024u);
    const uint64_t dv0 = umma_desc_sw128(base + L::v, (uint32_t)(kBlock * 128), 1024u);
    bool live = true;
    unsigned blk = 0, parts = 0, s_issued = 0, o_issued = 0;
    auto await = [&](int b, uint32_t parity) {
      live = __all_sync(0xffffffffu, live && mbar_wait(bar(b), parity, DEV_ERR_ATTN_TIMEOUT));
      return live;
    };
    auto scores = [&](unsigned n) {
      if (!await(kKFull + n % NS, (n / NS) & 1)) return;
      tc_fence_after();
      if (leader) {
        const uint64_t dk = dk0 + (n % NS) * (L::kOperand >> 4);
        const uint32_t to = tmem + (n % NS) * kBlock;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          umma_f16_ts(to, tmem + L::tm_q + k * 8, dk + (uint32_t)(((k / 4) * kBlock * 128 + (k % 4) * 32) >> 4), id_s, k != 0);
        umma_commit(bar(kSFull + n % NS));
        umma_commit(bar(kKEmpty + n % NS));
      }
      __syncwarp();
      s_issued = n + 1;
    };
    while (live && walk.next(p, a, part)) {
      const int nb = part.hi - part.lo;
      if (nb == 0) continue;
      if (!await(kQFull, parts & 1)) break;
      ++parts;
      scores(blk);
      for (int j = 0; j < nb && live; ++j, ++blk) {
        if (NS == 2 && j + 1 < nb) scores(blk + 1);
        if (!await(kVFull + blk % NS, (blk / NS) & 1) || !await(kPFull, blk & 1)) break;
        tc_fence_after();
        if (leader) {
          const uint64_t dv = dv0 + (blk % NS) * (L::kOperand >> 4);
#pragma unroll
          for (int k = 0; k < kBlock / 16; ++k)
            umma_f16_ts(tmem + L::tm_o, tmem + L::tm_p + k * 8, dv + (uint32_t)((k * 16 * 128) >> 4), id_o, (j | k) != 0);
          umma_commit(bar(kOFull));
          umma_commit(bar(kVEmpty + blk % NS));
        }
        __syncwarp();
        o_issued = blk + 1;
        if (NS == 1 && j + 1 < nb) {  // the next scores go where P is
          if (!await(kOFull, blk & 1)) break;
          scores(blk + 1);
        }
      }
    }
    // every UMMA issued completes before TMEM is released
    if (s_issued > 0) mbar_wait(bar(kSFull + (s_issued - 1) % NS), ((s_issued - 1) / NS) & 1, DEV_ERR_ATTN_TIMEOUT);
    if (o_issued > 0) mbar_wait(bar(kOFull), (o_issued - 1) & 1, DEV_ERR_ATTN_TIMEOUT);
    __syncwarp();
  } else if (warp >= kDequant) {
    // ------------------------------------------------------------ codes to operands
    const int dw = warp - kDequant, row = dw * 32 + lane;  // tile, row of the block
    const uint32_t out_row = (uint32_t)row * 128u;
    float* const factors = reinterpret_cast<float*>(mem + L::factors);
    int* const nans = reinterpret_cast<int*>(mem + L::nans);
    bool live = true;
    unsigned blk = 0, parts = 0;  // blocks so far, parts with blocks
    // A position's key and value: 16 G bytes of codes, (s, z) of its groups.
    uint4 codes[2][G];
    uint32_t sz[2][G];
    while (live && walk.next(p, a, part)) {
      const uint8_t* const rows = head_tiles(p, a.slot_of[part.b], part.h) + dw * L::kTileBytes;
      auto load = [&](int kv, int j) {
        if (j >= part.hi || j * kBlock + row >= part.kend) return;
        const uint8_t* const half = rows + (long long)j * (kBlock / kTile) * L::kTileBytes + kv * (L::kTileBytes / 2);
#pragma unroll
        for (int i = 0; i < G; ++i) codes[kv][i] = __ldcg(reinterpret_cast<const uint4*>(half + lane * 16 * G) + i);
        if constexpr (G % 2 != 0) {
#pragma unroll
          for (int i = 0; i < G; ++i)
            sz[kv][i] = __ldcg(reinterpret_cast<const uint32_t*>(half + kTile * 16 * G + lane * G * 4) + i);
        } else {
#pragma unroll
          for (int i = 0; i < G; i += 2) {
            const uint2 x = __ldcg(reinterpret_cast<const uint2*>(half + kTile * 16 * G + lane * G * 4) + i / 2);
            sz[kv][i] = x.x;
            sz[kv][i + 1] = x.y;
          }
        }
      };
      load(0, part.lo);
      load(1, part.lo);
      int nan = 0x7fffffff;  // lane i: the part's first position where group i's value is NaN
      for (int j = part.lo; j < part.hi && live; ++j, ++blk) {
        const bool ok = j * kBlock + row < part.kend;
        // A weight of zero does not undo a value of NaN: it counts as 0 here, and the rows
        // that attend it are told.
        uint32_t bad = 0;
#pragma unroll
        for (int i = 0; i < G; ++i) bad |= reads_nan<T>(sz[1][i]);
        if (__any_sync(0xffffffffu, ok && bad != 0)) {
#pragma unroll
          for (int i = 0; i < G; ++i) {
            const bool mine = ok && reads_nan<T>(sz[1][i]) != 0;
            const uint32_t who = __ballot_sync(0xffffffffu, mine);
            if (mine) sz[1][i] = 0;
            if (who != 0 && lane == i) nan = min(nan, j * kBlock + dw * 32 + __ffs((int)who) - 1);
          }
        }
        // bf16: powers of two of the tile, or of the lane's position
        bool wide = false;
        float own[2], powers[2];
        float mine = 1.f;  // lane 0: the keys' power of two (-1: a wide tile), lane 1: the values' exponent
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            float big = 0.f;
#pragma unroll
            for (int i = 0; i < G; ++i) big = fmaxf(big, ok ? largest_of(sz[kv][i]) : 0.f);
            const float most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(big)));
            wide |= big > 0.f && big * kWide < most;
            own[kv] = big;
            powers[kv] = power_to_12(most);
          }
          wide = __any_sync(0xffffffffu, wide);
          if (wide) {
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) powers[kv] = power_to_12(own[kv]);
          }
#pragma unroll
          for (int kv = 0; kv < 2; ++kv)
#pragma unroll
            for (int i = 0; i < G; ++i) sz[kv][i] = scaled_params<T>(sz[kv][i], powers[kv]);
          mine = lane != 0 ? exponent_of(powers[1]) : wide ? -1.f : powers[0];
        }
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          if (blk >= NS) live = wait_copies(bar((kv ? kVEmpty : kKEmpty) + blk % NS), (blk / NS - 1) & 1);
          if (!__all_sync(0xffffffffu, live)) {
            live = false;
            break;
          }
          // The powers of two, for this block's softmax.  Four blocks' lie side by side: the
          // keys' place is free once S of the block two before is done, which was issued
          // after the softmax of the block four before.
          if (kv == 0 && lane < 2) factors[(blk & 3) * 8 + 4 * lane + dw] = mine;
          if (kv == 0 && wide) {
            float* const at = reinterpret_cast<float*>(mem + L::own) + (blk & 3) * 2 * kBlock + row;
            at[0] = __int_as_float((254 << 23) - __float_as_int(powers[0]));  // 1 / power
            at[kBlock] = exponent_of(powers[1]);
          }
          // likewise four parts': S of a part's first block is issued after the softmax's
          // warps have read all of the part before
          if (kv == 0 && lane < G) nans[(parts & 3) * 32 + 8 * dw + lane] = nan;
          const uint32_t dst = base + (kv ? L::v : L::k) + (blk % NS) * L::kOperand + out_row;
          // eight channels, number o8 of the row
          auto put = [&](int o8, uint32_t x, uint32_t sz8) {
            sts4(dst + (o8 / 8) * (kBlock * 128) + (((o8 & 7) ^ (row & 7)) * 16), operand8(x, sz8));
          };
          if (!ok) {  // no such position: its value must not count, and its weight is zero
            if (kv)
              for (int c = 0; c < D / 8; ++c)
                sts4(dst + (c / 8) * (kBlock * 128) + (((c % 8) ^ (row & 7)) * 16), make_uint4(0u, 0u, 0u, 0u));
          } else {
            if constexpr (G == 4) {
#pragma unroll
              for (int c = 0; c < G; ++c) {  // 16-byte chunks of the row
                uint4 x = codes[kv][c];
                int quarter = c;
                if (kv) {  // the values' order is turned by position; half words of channels 8 q .. and 8 q + 4 ..
                  quarter = c ^ (((lane >> 1) & 1) * 2);
                  x = make_uint4(__byte_perm(x.x, x.z, 0x5410), __byte_perm(x.x, x.z, 0x7632),
                                 __byte_perm(x.y, x.w, 0x5410), __byte_perm(x.y, x.w, 0x7632));
                }
                put(quarter, x.x, sz[kv][0]);
                put(4 + quarter, x.y, sz[kv][1]);
                put(8 + quarter, x.z, sz[kv][G - 2]);
                put(12 + quarter, x.w, sz[kv][G - 1]);
              }
            } else {
              const uint32_t* const w = reinterpret_cast<const uint32_t*>(codes[kv]);
#pragma unroll
              for (int i = 0; i < 4 * G; ++i) {
                const int quarter = i / G, group = i % G;
                uint32_t x = w[i];
                if (kv && G < 8) {  // half words of channels 8 q .. and 8 q + 4 ..
                  const int h0 = 2 * quarter * G + group, h1 = h0 + G;
                  x = __byte_perm(w[h0 / 2], w[h1 / 2], (h0 % 2 ? 0x32 : 0x10) | (h1 % 2 ? 0x7600 : 0x5400));
                }
                int o8 = 4 * group + quarter;
                if (kv && G == 8) {  // turned by position: a pair of 16-byte chunks is another quarter's
                  x = __byte_perm(w[8 * quarter + group / 2], w[8 * quarter + 4 + group / 2], group % 2 ? 0x7632 : 0x5410);
                  o8 = 4 * group + (quarter ^ (lane & 3));
                }
                put(o8, x, sz[kv][group]);
              }
            }
          }
          load(kv, j + 1);
          fence_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar((kv ? kVFull : kKFull) + blk % NS));
        }
      }
      if (part.lo < part.hi) ++parts;
    }
  } else {
    // ------------------------------------------------------------ queries, softmax, epilogue
    const int quad = warp & 3, hx = warp >> 2, r = quad * 32 + lane;  // row of the segment = TMEM lane; half
    const uint32_t trow = tmem + ((uint32_t)(quad * 32) << 16);
    float2* const told = reinterpret_cast<float2*>(mem + L::rows);
    // the thread's share of the channels, in groups
    constexpr int kHalf = (G + 1) / 2;
    const int group0 = hx ? kHalf : 0, group1 = hx ? G : kHalf;
    constexpr int kShare = kRows * (4 + D);  // floats of a part in the workspace
    bool live = true;
    unsigned blk = 0, parts = 0, met = 0, paired = 0;
    // What the row's other thread has to tell (the two warps of the same rows meet).
    auto exchange = [&](float x, float y = 0.f) {
      const int buf = paired & 1;
      told[(buf * 2 + hx) * kRows + r] = make_float2(x, y);
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kPair + quad));
      live = __all_sync(0xffffffffu, live && wait_copies(bar(kPair + quad), buf));
      ++paired;
      return told[(buf * 2 + (hx ^ 1)) * kRows + r];
    };
    // the eight warps meet (bounded, unlike a hardware barrier: one may have given up)
    auto together = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kTogether));
      live = __all_sync(0xffffffffu, wait_copies(bar(kTogether), met & 1));
      ++met;
      return live;
    };
    while (live && walk.next(p, a, part)) {
      const int nb = part.hi - part.lo;
      const int row = part.row0 + r, tok = row / a.group, qh = part.h * a.group + (row - tok * a.group);
      const bool mine = r < part.rows && part.start + tok < p.max_seq;
      const bool used = __any_sync(0xffffffffu, mine);  // the warp has rows at all
      const int row_keys = mine ? part.start + tok + 1 : 0;
      unsigned w0 = 0, w1 = 0;
      if (!part.whole) {
        w0 = shares.holder(part.seg0, blockIdx.x);
        w1 = shares.holder(part.seg0 + part.units - 1, blockIdx.x);
        if (threadIdx.x == 0) open_tickets(a.tickets + w0, a.launch);
      }
      float q_scale = a.scale_log2;  // of the scores, the row's power of two taken off
      // Where a block's least factor is below this, scores could pass kFar: the products of
      // bf16's operands are below 2^34 (2^26 D), fp16's below the query's sum times 65504.
      float far_below = 0.f;
      if (nb > 0) {
        uint4 w[4 * kHalf];  // the thread's groups' channels; zeros where there is no row or channel
#pragma unroll
        for (int c = 0; c < 4 * kHalf; ++c) w[c] = make_uint4(0u, 0u, 0u, 0u);
        float big = 0.f;
        if (mine) {
          const T* qp = static_cast<const T*>(a.q) + part.b * a.qs0 + tok * a.qs1 + qh * a.qs2;
#pragma unroll
          for (int c = 0; c < 4 * kHalf; ++c) {
            const int c0 = 32 * group0 + 8 * c;
            if (c0 >= p.D) continue;
            if (a.q_vec) {
              w[c] = *reinterpret_cast<const uint4*>(qp + c0);
            } else {
              T e[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) e[i] = c0 + i < p.D ? qp[c0 + i] : from_f32<T>(0.f);
              w[c] = *reinterpret_cast<const uint4*>(e);
            }
          }
        }
        if constexpr (std::is_same<T, __half>::value) {
          float sum = 0.f;
#pragma unroll
          for (int c = 0; c < 4 * kHalf; ++c) {
            const __half2* const x = reinterpret_cast<const __half2*>(&w[c]);
#pragma unroll
            for (int i = 0; i < 4; ++i) sum += fabsf(__low2float(x[i])) + fabsf(__high2float(x[i]));
          }
          sum += exchange(sum).x;
          if (!live) break;
          far_below = sum * 65504.f * q_scale > kFar ? 2.f : 0.f;  // the factors are 1
        }
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
          if (mine) {
#pragma unroll
            for (int c = 0; c < 4 * kHalf; ++c) {
              const uint32_t x[4] = {w[c].x, w[c].y, w[c].z, w[c].w};
#pragma unroll
              for (int i = 0; i < 4; ++i)
                big = fmaxf(big, fmaxf(fabsf(__uint_as_float(x[i] << 16)), fabsf(__uint_as_float(x[i] & 0xffff0000u))));
            }
          }
          big = fmaxf(big, exchange(big).x);
          if (!live) break;
          const float f = power_to_12(big);
          q_scale = __fdividef(a.scale_log2, f);
          far_below = q_scale * (1.71798692e10f / kFar);
#pragma unroll
          for (int c = 0; c < 4 * kHalf; ++c) {
            uint32_t x[4] = {w[c].x, w[c].y, w[c].z, w[c].w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
              x[i] = pack2<__half>(__uint_as_float(x[i] << 16) * f, __uint_as_float(x[i] & 0xffff0000u) * f);
            w[c] = make_uint4(x[0], x[1], x[2], x[3]);
          }
        }
        // the operands' order: 0 4 1 5 2 6 3 7
#pragma unroll
        for (int c = 0; c < 4 * kHalf; c += 4) {
          if (group0 + c / 4 >= G) break;
          uint32_t x[16];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[4 * i] = __byte_perm(w[c + i].x, w[c + i].z, 0x5410);
            x[4 * i + 1] = __byte_perm(w[c + i].x, w[c + i].z, 0x7632);
            x[4 * i + 2] = __byte_perm(w[c + i].y, w[c + i].w, 0x5410);
            x[4 * i + 3] = __byte_perm(w[c + i].y, w[c + i].w, 0x7632);
          }
          tmem_st16(trow + L::tm_q + 16 * group0 + 4 * c, x);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kQFull));
      }
      // Scores' running maximum and sum of weights; w - m (bf16: see power_to_12).
      float m = -INFINITY, l = 0.f, wm = -INFINITY;
      for (int j = 0; j < nb && live; ++j, ++blk) {
        live = wait_copies(bar(kSFull + blk % NS), (blk / NS) & 1);
        if (!__all_sync(0xffffffffu, live)) {
          live = false;
          break;
        }
        tc_fence_after();
        const uint32_t ts = trow + (blk % NS) * kBlock, to = trow + L::tm_o;
        const int lim = row_keys - (part.lo + j) * kBlock;  // positions of the block that the row attends
        const bool full = __all_sync(0xffffffffu, lim >= kBlock || !mine);
        const bool any = __any_sync(0xffffffffu, lim > 0);
        const float* const f = reinterpret_cast<const float*>(mem + L::factors) + (blk & 3) * 8;
        constexpr bool kScaled = std::is_same<T, __nv_bfloat16>::value;
        // The maximum of the row's scores moves to mn, that of weight times value to `seen`
        // against it at least; the running sum and output follow.  False where a wait gave up.
        auto move = [&](float mn, float seen) {
          float alpha = 1.f;
          if (any) {
            alpha = m == -INFINITY ? 0.f : ex2(base_of<T>(m) - base_of<T>(mn));
            l *= alpha;
            if constexpr (kScaled) {
              const float was = m == -INFINITY ? -INFINITY : wm + (m - mn);
              wm = fmaxf(was, seen);
              alpha = was == -INFINITY ? 0.f : ex2(was - wm);
            }
            m = mn;
          }
          // P and the running output are free once the block before is through
          if (j > 0) {
            live = wait_copies(bar(kOFull), (blk - 1) & 1);
            if (!__all_sync(0xffffffffu, live)) {
              live = false;
              return false;
            }
            tc_fence_after();
            if (used && !__all_sync(0xffffffffu, alpha == 1.f || !mine)) {
#pragma unroll 1
              for (int c = group0; c < group1; ++c) {
                float o[32];
                tmem_ld32(to + c * 32, o);
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] *= alpha;
                tmem_st32(to + c * 32, o);
              }
            }
          }
          return true;
        };
        auto scale_of = [&](int c) { return kScaled ? fmaxf(__fdividef(q_scale, fabsf(f[2 * hx + c])), 1.2e-38f) : q_scale; };
        const float4 f4 = *reinterpret_cast<const float4*>(f);
        if (__any_sync(0xffffffffu, fminf(fminf(f4.x, f4.y), fminf(f4.z, f4.w)) < far_below)) {
          // A block with a wide tile, or with scores that could be far: position by position,
          // the scores rounded before their maximum is taken.  (Rolled, in a branch of its own:
          // unrolled, or within the usual way, these lines cost blocks that do not take them up
          // to 9 % of their time.)
          const float* const own = reinterpret_cast<const float*>(mem + L::own) + (blk & 3) * 2 * kBlock + 64 * hx;
          float mx = -INFINITY, at = -INFINITY, mn = m;
          if (any) {
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
              const float k = scale_of(c / 4), tile = f[4 + 2 * hx + c / 4];
              const bool wide = f[2 * hx + c / 4] < 0.f;
              float x[8];
              tmem_ld8(ts + 64 * hx + 8 * c, x);
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                x[e] = 64 * hx + 8 * c + e < lim ? __fmul_rn(wide ? x[e] * own[8 * c + e] : x[e], k) : -INFINITY;
                mx = fmaxf(mx, x[e]);
                if (kScaled) at = fmaxf(at, x[e] - (wide ? own[kBlock + 8 * c + e] : tile));
              }
              tmem_st8(ts + 64 * hx + 8 * c, x);
            }
            tc_fence_before();
            const float2 other = exchange(mx, at - mx);
            if (!live) break;
            tc_fence_after();
            mn = fmaxf(m, fmaxf(mx, other.x));
            at = fmaxf(at - mx + (mx - mn), other.y + (other.x - mn));
          }
          if (!move(mn, at)) break;
          if (any) {
            const float off = m == -INFINITY ? 0.f : base_of<T>(m);
            // With one block of scores P goes over them: a thread's own go by ahead of it, those
            // of the row's first thread before its second one begins.
            if (NS == 1 && hx == 1) {
              exchange(0.f);
              tc_fence_after();
            }
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
              const float tile = f[4 + 2 * hx + c / 4];
              const bool wide = f[2 * hx + c / 4] < 0.f;
              float x[8], p[8];
              tmem_ld8(ts + 64 * hx + 8 * c, x);
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                x[e] -= off;
                p[e] = ex2(x[e]);
                l += p[e];
                if (kScaled) p[e] = ex2(fminf(x[e] - (wide ? own[kBlock + 8 * c + e] : tile) + (kTop - wm), kTop + 1.f));
              }
              tmem_st4(trow + L::tm_p + 32 * hx + 4 * c,
                       {pack2<__half>(p[0], p[1]), pack2<__half>(p[2], p[3]), pack2<__half>(p[4], p[5]), pack2<__half>(p[6], p[7])});
            }
            if (NS == 1 && hx == 0) {
              tc_fence_before();
              exchange(0.f);
            }
            if (!live) break;
          }
        } else {
          float v[64], k_scale[2], v_scale[2], mn = m, seen = -INFINITY;
          if (any) {
            tmem_ld64(ts + 64 * hx, v);
            float mt[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              // scores in log2 units: both powers of two off
              k_scale[c] = scale_of(c);
              float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
              if (full) {
#pragma unroll
                for (int e = 0; e < 32; ++e) m4[e & 3] = fmaxf(m4[e & 3], v[32 * c + e]);
              } else {
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                  if (64 * hx + 32 * c + e >= lim) v[32 * c + e] = -INFINITY;
                  m4[e & 3] = fmaxf(m4[e & 3], v[32 * c + e]);
                }
              }
              mt[c] = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * k_scale[c];
            }
            const float mx = fmaxf(mt[0], mt[1]);
            // the largest weight times value of the thread's tiles, against its own maximum
            // (NaN where it attends nothing: fmaxf passes it over)
            const float at = kScaled ? fmaxf(mt[0] - mx - f[4 + 2 * hx], mt[1] - mx - f[5 + 2 * hx]) : 0.f;
            if (NS == 1) tc_fence_before();  // the other thread's P goes over these scores
            const float2 other = exchange(mx, at);
            if (!live) break;
            if (NS == 1) tc_fence_after();
            mn = fmaxf(m, fmaxf(mx, other.x));
            seen = fmaxf(at + (mx - mn), other.y + (other.x - mn));
          }
          if (!move(mn, seen)) break;
          if (any) {
            const float off = m == -INFINITY ? 0.f : base_of<T>(m);
            float lp[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              if (kScaled) v_scale[c] = ex2(fminf(kTop - f[4 + 2 * hx + c] - wm, 126.f));
              uint32_t w[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const int x = 32 * c + 2 * e;
                const float p0 = ex2(fmaf(v[x], k_scale[c], -off)), p1 = ex2(fmaf(v[x + 1], k_scale[c], -off));
                if constexpr (!kScaled) {
                  w[e] = pack2<__half>(p0, p1);
                  const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
                  lp[e & 3] += g.x + g.y;  // the sum of what the tensor core multiplies
                } else {
                  w[e] = pack2<__half>(p0 * v_scale[c], p1 * v_scale[c]);
                  lp[e & 3] += p0 + p1;
                }
              }
              tmem_st16(trow + L::tm_p + 32 * hx + 16 * c, w);
            }
            tmem_st_wait();
            l += (lp[0] + lp[1]) + (lp[2] + lp[3]);
          }
        }
        if (!any && used) {  // all masked: weights of zero
          const uint32_t w[16] = {};
          tmem_st16(trow + L::tm_p + 32 * hx, w);
          tmem_st16(trow + L::tm_p + 32 * hx + 16, w);
          tmem_st_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kPFull));
      }
      if (nb > 0 && live) {
        live = wait_copies(bar(kOFull), (blk - 1) & 1);
        live = __all_sync(0xffffffffu, live);
        tc_fence_after();
      }
      if (!live) break;
      l += exchange(l).x;
      if (!live) break;
      // the output's unit, in two factors: their product may pass the range of numbers
      const float unit = std::is_same<T, __half>::value ? 1.f : 1.f / (float)(1 << (int)kTop);
      const float scale = std::is_same<T, __half>::value || wm == -INFINITY ? 1.f : ex2(wm);
      // whether the row attends a value of NaN in the channels of group c
      const int* const nans = reinterpret_cast<const int*>(mem + L::nans) + (parts & 3) * 32;
      auto nan_in = [&](int c) {
        return nb > 0 && min(min(nans[c], nans[8 + c]), min(nans[16 + c], nans[24 + c])) < row_keys;
      };
      if (nb > 0) ++parts;
      T* const op = static_cast<T*>(a.out) + (((long long)part.b * a.tq + tok) * a.QH + qh) * p.D;
      // a row's 32 columns, in the operands' order, as the output's channels
      auto store = [&](int c, const float (&v)[32], float f, float f2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float* x = v + 8 * i;
          auto two = [&](int i0, int i1) { return pack2<T>(x[i0] * f * f2, x[i1] * f * f2); };
          const uint4 w = make_uint4(two(0, 2), two(4, 6), two(1, 3), two(5, 7));
          const int c0 = c * 32 + 8 * i;
          if (a.out_vec) {
            if (c0 < p.D) *reinterpret_cast<uint4*>(op + c0) = w;
          } else {
            const T* e = reinterpret_cast<const T*>(&w);
            for (int k = 0; k < 8; ++k)
              if (c0 + k < p.D) op[c0 + k] = e[k];
          }
        }
      };
      if (part.whole) {
        if (used) {
          const float inv = __fdividef(unit, l);
#pragma unroll 1
          for (int c = group0; c < group1; ++c) {
            float v[32];
            tmem_ld32(trow + L::tm_o + c * 32, v);
            if (mine) store(c, v, nan_in(c) ? NAN : inv, scale);
          }
        }
        continue;
      }
      // ---- other CTAs hold parts of the segment
      float* own = a.ws + ((long long)blockIdx.x * 2 + part.which) * kShare + r * (4 + D);
      if (used) {
        if (mine && hx == 0) __stcg(reinterpret_cast<float4*>(own), make_float4(base_of<T>(m), l, 0.f, 0.f));
#pragma unroll 1
        for (int c = group0; c < group1; ++c) {
          float v[32];
          if (nb > 0) tmem_ld32(trow + L::tm_o + c * 32, v);
          const float f = nan_in(c) ? NAN : unit;
          if (mine && nb > 0)
#pragma unroll
            for (int i = 0; i < 8; ++i)
              __stcg(reinterpret_cast<float4*>(own + 4 + c * 32) + i,
                     make_float4(v[4 * i] * f * scale, v[4 * i + 1] * f * scale, v[4 * i + 2] * f * scale,
                                 v[4 * i + 3] * f * scale));
        }
      }
      if (!together()) break;
      if (threadIdx.x == 0) {
        const unsigned taken = take_ticket(a.tickets + w0);
        if (taken == w1 - w0 + 1) a.tickets[w0] = 0;  // clean for the next launch
        taken_sh = taken;
        took_sh |= 1u << part.which;
      }
      if (!together()) break;
      if (taken_sh == w1 - w0 + 1 && mine) {
        const float* at = a.ws + r * (4 + D);
        // the segment is the last part of the share that it starts in, the first of the others
        auto share = [&](unsigned w) {
          return at + ((long long)w * 2 + (w == w0 && shares.begin(w) < part.seg0 ? 1 : 0)) * kShare;
        };
        float mx = -INFINITY, ls = 0.f;
        for (unsigned w = w0; w <= w1; ++w) mx = fmaxf(mx, __ldcg(share(w)));
        for (unsigned w = w0; w <= w1; ++w) {
          const float2 ml = __ldcg(reinterpret_cast<const float2*>(share(w)));
          if (!(ml.x == -INFINITY && ml.y == 0.f)) ls = fmaf(ex2(ml.x - mx), ml.y, ls);
        }
#pragma unroll 1
        for (int c = group0; c < group1; ++c) {
          float x[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) x[e] = 0.f;
          for (unsigned w = w0; w <= w1; ++w) {
            const float* s = share(w);
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(s));
            if (ml.x == -INFINITY && ml.y == 0.f) continue;  // all masked: no output left
            const float f = ex2(ml.x - mx);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float4 y = __ldcg(reinterpret_cast<const float4*>(s + 4 + c * 32) + i);
              x[4 * i] = fmaf(f, y.x, x[4 * i]);
              x[4 * i + 1] = fmaf(f, y.y, x[4 * i + 1]);
              x[4 * i + 2] = fmaf(f, y.z, x[4 * i + 2]);
              x[4 * i + 3] = fmaf(f, y.w, x[4 * i + 3]);
            }
          }
          store(c, x, 1.0f / ls, 1.f);
        }
      }
      together();  // taken_sh is read
    }
    if (!live && threadIdx.x == 0) gave_up_sh = true;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMma) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
  if (shared_blocks != 0 && threadIdx.x == 0 && gave_up_sh) {
    // NaN for the CTA that joins what is missing; the error word is set
    give_up(p, a, Shares(total_sh, min(gridDim.x, (total_sh + 1) / 2)), row_tiles, blockIdx.x, took_sh,
            [&](const Part& o, unsigned w0) {
              float* const own = a.ws + ((long long)blockIdx.x * 2 + o.which) * (kRows * (4 + D));
              for (int i = 0; i < kRows; ++i) __stcg(reinterpret_cast<float4*>(own + i * (4 + D)), make_float4(NAN, NAN, 0.f, 0.f));
              open_tickets(a.tickets + w0, a.launch);
              return take_ticket(a.tickets + w0);
            },
            [&](unsigned w0) { a.tickets[w0] = 0; });
  }
}

template <typename T, int G>
static int launch(const Pool& p, const Problem& a, int row_tiles, bool shared, cudaStream_t st) {
  static std::atomic<bool> ready[64] = {};
  const int dev = current_device();
  if (dev < 0 || dev >= 64) return fail(FML_EUNSUPPORTED, "neb_kv4_attention: device index out of range");
  if (!ready[dev].load()) {
    const cudaError_t e = cudaFuncSetAttribute(attn_tc_kernel<T, G>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)Smem<G>::total);
    if (e != cudaSuccess) return check_cuda(e, "neb_kv4_attention smem attribute");
    ready[dev].store(true);
  }
  const long long grid = shared ? num_sms(dev) : (long long)a.B * p.H * row_tiles;
  const cudaError_t e = launch_pdl(attn_tc_kernel<T, G>, dim3((unsigned)grid), dim3(kThreads), Smem<G>::total, st, 1, p, a,
                                   row_tiles, shared ? 1 : 0);
  count_launch();
  return check_cuda(e, "neb_kv4_attention launch");
}

template <typename T>
static int launch_groups(const Pool& p, const Problem& a, int row_tiles, bool shared, cudaStream_t st) {
  switch (p.G) {
    case 1: return launch<T, 1>(p, a, row_tiles, shared, st);
    case 2: return launch<T, 2>(p, a, row_tiles, shared, st);
    case 3: return launch<T, 3>(p, a, row_tiles, shared, st);
    case 4: return launch<T, 4>(p, a, row_tiles, shared, st);
    case 5: return launch<T, 5>(p, a, row_tiles, shared, st);
    case 6: return launch<T, 6>(p, a, row_tiles, shared, st);
    case 7: return launch<T, 7>(p, a, row_tiles, shared, st);
    default: return launch<T, 8>(p, a, row_tiles, shared, st);
  }
}

}  // namespace tc

// Whether the tensor-core kernel takes the call: more than 8 query rows of a
// key/value head.  Up to there the row kernel, which goes over the cache once per
// row (from L2 after the first), is the faster one or near it.  Measured, row kernel
// against this one, at 2 / 4 / 8 / 16 rows, head dim 128, bf16:
//   16 requests x 8 heads x 6000 positions   47 / 78 / 141 / 267 against 127 .. 130 us
//    2 requests x 8 heads x 6000             17 / 21 /  32 /  46 against  49 ..  53 us
//    4 requests x 8 heads x 300               9 /  9 /  10 /  13 against  25 ..  26 us
// and at 4 / 8 / 16 rows, other head dims, 16 requests x 8 heads:
//   32 x 6000 positions  44 /  75 / 137 against  92 ..  93 us
//   96 x 6000            68 / 119 / 221 against 106 .. 109
//   256 x 3000           89 / 158 / 301 against 177 .. 183
// (The lengths, which decide where exactly the two meet, lie on the device.)
bool tc_covers(const Pool& p, int dtype, int64_t t, int64_t group) {
  return (dtype == FML_BF16 || dtype == FML_F16) && t * group > 8;
}
static bool tc_shared(const Pool& p, int64_t segments, int64_t requests_units) {
  return segments < 2 * num_sms(current_device()) && requests_units < (1ll << 31);
}
size_t tc_workspace_bytes(const Pool& p, int64_t batch, int64_t t, int64_t group) {
  const int64_t tiles = (t * group + tc::kRows - 1) / tc::kRows, segs = batch * p.H * tiles;
  if (!tc_shared(p, segs, segs * ((p.max_seq + tc::kBlock - 1) / tc::kBlock))) return 0;
  const size_t sms = (size_t)num_sms(current_device());
  return sms * 2 * tc::kRows * (4 + 32 * p.G) * sizeof(float) + sms * sizeof(unsigned long long);
}
int tc_attention(const Pool& p, Problem a, int dtype, cudaStream_t st) {
  const int tiles = (int)(((int64_t)a.tq * a.group + tc::kRows - 1) / tc::kRows);
  const int64_t segs = (int64_t)a.B * p.H * tiles;
  if (segs >= (1ll << 31)) return fail(FML_EUNSUPPORTED, "neb_kv4_attention: too many queries");
  const bool shared = tc_shared(p, segs, segs * ((p.max_seq + tc::kBlock - 1) / tc::kBlock));
  a.segs = p.H * tiles;
  const size_t sms = (size_t)num_sms(current_device());
  a.tickets = reinterpret_cast<unsigned long long*>(reinterpret_cast<uint8_t*>(a.ws) +
                                                    sms * 2 * tc::kRows * (4 + 32 * p.G) * sizeof(float));
  a.launch = launch_number();
  return dtype == FML_BF16 ? tc::launch_groups<__nv_bfloat16>(p, a, tiles, shared, st)
                           : tc::launch_groups<__half>(p, a, tiles, shared, st);
}

}  // namespace kv4
}  // namespace fml
