// The 4-bit key/value cache: format and addressing, shared by the kernels that
// write it, read it back and attend over it.
//
// A row is one position of one key/value head: D numbers of type T in G =
// ceil(D / 32) groups of 32 channels (the last may be shorter).  A group keeps
//   z = min x,   s = T((max x - min x) / 15),   c = rint((x - z) / s) in 0..15
// (ties to even; c = 0 where s = 0) and stands for z + c * s: at most s / 2
// from x as long as s is a normal number of type T.  z is one of the group's
// own numbers, so storing it in T loses nothing; s is the one rounding besides
// the codes, and the codes are taken against the rounded s.  A group that
// holds an infinity or a NaN has s = z = NaN and reads back as NaN, as loudly
// as a 16-bit cache would.  Unused channels of a short group hold code 0.
//
// Memory of a layer: [slots][heads][tiles], a tile being 32 positions of one
// head in one piece, so that a kernel fetches it with one copy:
//   keys' codes [32][16 G bytes], keys' parameters [32][G][2] (s, z) in T,
//   values' codes, values' parameters.
//
// Order of the codes within a row.  The row kernel feeds bytes of codes to
// mma.sync m16n8k32 operands as they lie; the order makes a thread's codes of
// all groups one contiguous chunk, for keys and for values.
//   keys:   chunk t (of 4, 4 G bytes) holds for each group one 32-bit word,
//           its channels 8 t .. 8 t + 7;
//   values: chunk l (of 8, 2 G bytes) holds for each group one 16-bit word,
//           its channels 4 l .. 4 l + 3.  For G = 4 and 8 the byte offset is
//           XORed with a function of the position (32 * bits of it), so that
//           the four rows a quarter of a warp reads at once sit in distinct
//           shared-memory banks.
#pragma once

#include "common.cuh"

namespace fml {
namespace kv4 {

constexpr int kGroup = 32;
constexpr int kMaxD = 256;
constexpr int kTile = 32;  // positions of a tile

struct Pool {
  uint8_t* data;
  long long tiles;  // of one (slot, head)
  int slots, H, max_seq, D, G;
  int half;  // bytes of a tile's keys (and of its values)
};

__host__ __device__ __forceinline__ int groups_of(int d) { return (d + kGroup - 1) / kGroup; }

// The first tile of a (slot, head).
__device__ __forceinline__ uint8_t* head_tiles(const Pool& p, int slot, int h) {
  return p.data + ((long long)slot * p.H + h) * p.tiles * (2 * p.half);
}

__device__ __forceinline__ int v_swizzle(int G, int pos) {
  return G == 4 ? ((pos >> 1) & 1) * 32 : G == 8 ? (pos & 3) * 32 : 0;
}
// Byte of channel c within a row (the nibble is c & 1, low first).
__device__ __forceinline__ int k_byte(int G, int c) {
  return ((c & 31) >> 3) * 4 * G + (c >> 5) * 4 + ((c & 7) >> 1);
}
__device__ __forceinline__ int v_byte(int G, int c, int pos) {
  return (((c & 31) >> 2) * 2 * G + (c >> 5) * 2 + ((c & 3) >> 1)) ^ v_swizzle(G, pos);
}

// Host: checks shared by the entry points; fills `p`.
int pool_from(const neb_kv4_pool* pool, const char* who, Pool* p);

}  // namespace kv4
}  // namespace fml
