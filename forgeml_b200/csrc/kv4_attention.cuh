// What the kernels that attend over the 4-bit cache share: the problem, how a
// batch's work is counted and divided, and the tickets by which a segment that
// several CTAs hold is finished.
#pragma once

#include <algorithm>
#include <atomic>
#include <chrono>

#include "kv4.cuh"

namespace fml {
namespace kv4 {

struct Problem {
  const int32_t *slot_of, *start_pos;
  int B, tq, QH, group;  // group: query heads of a key/value head
  int segs;              // segments of a request: tq * QH
  long long qs0, qs1, qs2;
  bool q_vec, out_vec;  // 16-byte loads of q, 8-byte stores of the output
  float scale_log2;  // softmax scale * log2(e)
  double scale_log2_wide;
  const void* q;
  void* out;
  // Workspace: the CTAs' shares of the segments that they hold in part, then a
  // ticket word per CTA for the segment that starts in its share and ends in
  // another's: 48 bits that name the launch (a word of any other launch counts as
  // empty; the last taker clears it) and the tickets taken.
  float* ws;
  unsigned long long* tickets;
  unsigned long long launch;
};

// kv4_tc.cu: several query rows of a key/value head on the tensor cores.
bool tc_covers(const Pool& p, int dtype, int64_t t, int64_t group);
size_t tc_workspace_bytes(const Pool& p, int64_t batch, int64_t t, int64_t group);
int tc_attention(const Pool& p, Problem a, int dtype, cudaStream_t st);

// Positions that request b's last query attends; 0 for a bad slot or position.
__host__ __device__ __forceinline__ int keys_of(const Pool& p, const Problem& a, int b) {
  const int slot = a.slot_of[b], start = a.start_pos[b];
  if (slot < 0 || slot >= p.slots || start < 0 || start >= p.max_seq) return 0;
  return min(start + a.tq, p.max_seq);
}


// Where a warp is: a request, one of its segments (query rows: head, then the
// head's rows, tokens innermost), a unit of it.  Every segment of a request has
// all of the request's units (an earlier token's last ones may be masked whole).
template <int UNIT>
struct Cursor {
  int b, seg, unit, keys, units;
  __host__ __device__ __forceinline__ void request(const Pool& p, const Problem& a, int nb) {
    b = nb;
    keys = units = 0;
    while (b < a.B) {
      keys = keys_of(p, a, b);
      units = (keys + UNIT - 1) / UNIT;
      if (units > 0) break;
      ++b;
    }
  }
  __host__ __device__ __forceinline__ void next_segment(const Pool& p, const Problem& a) {
    unit = 0;
    if (++seg == a.segs) {
      seg = 0;
      request(p, a, b + 1);
    }
  }
  // The next unit; true when it opens another segment.
  __host__ __device__ __forceinline__ bool next(const Pool& p, const Problem& a) {
    if (unit + 1 < units) {
      ++unit;
      return false;
    }
    next_segment(p, a);
    return true;
  }
  // n units on.
  __host__ __device__ __forceinline__ void skip(const Pool& p, const Problem& a, unsigned n) {
    n += unit;
    while (b < a.B) {
      const unsigned here = (unsigned)(a.segs - seg) * units;
      if (n < here) {
        const unsigned k = n / (unsigned)units;
        seg += k;
        unit = n - k * units;
        return;
      }
      n -= here;
      seg = 0;
      request(p, a, b + 1);
    }
  }
};

// Contiguous shares of `total` units: part w of W begins at unit total * w / W.
struct Shares {
  unsigned total, each, W, extra;
  __host__ __device__ __forceinline__ Shares(unsigned total_, unsigned parts) : total(total_), W(parts) {
    each = total / W;
    extra = total - each * W;
  }
  // extra * w stays below W * W
  __host__ __device__ __forceinline__ unsigned begin(unsigned w) const { return each * w + extra * w / W; }
  // The part that holds unit u, from part w on up or down.
  __host__ __device__ __forceinline__ unsigned holder(unsigned u, unsigned w) const {
    while (begin(w) > u) --w;
    while (w + 1 < W && begin(w + 1) <= u) ++w;
    return w;
  }
};

// The batch in front of a warp: its units, and the place of any of them.
template <int UNIT>
struct Plan {
  unsigned total;
  int longest;
  unsigned units, incl;  // of the request of this lane's number: units, units up to its end
  __device__ __forceinline__ static unsigned units_of(const Pool& p, const Problem& a, int b) {
    return (keys_of(p, a, b) + UNIT - 1) / UNIT;
  }
  __device__ __forceinline__ static unsigned scan(unsigned u) {
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const unsigned o = __shfl_up_sync(0xffffffffu, u, off);
      if ((int)(threadIdx.x & 31) >= off) u += o;
    }
    return u;
  }
  __device__ __forceinline__ Plan(const Pool& p, const Problem& a) {
    const int lane = threadIdx.x & 31;
    units = lane < a.B ? units_of(p, a, lane) : 0;
    incl = scan(units);
    unsigned sum = 0, most = units;
    for (int i = lane + 32; i < a.B; i += 32) {
      const unsigned u = units_of(p, a, i);
      sum += u;
      most = max(most, u);
    }
    if (a.B > 32) sum = __reduce_add_sync(0xffffffffu, sum);
    total = (sum + __shfl_sync(0xffffffffu, incl, 31)) * a.segs;
    longest = __reduce_max_sync(0xffffffffu, most);
  }
  // The unit at place `at` < total of the batch's order.
  __device__ __forceinline__ Cursor<UNIT> seek(const Pool& p, const Problem& a, unsigned at) const {
    const int lane = threadIdx.x & 31;
    Cursor<UNIT> c;
    c.b = c.seg = c.unit = c.keys = c.units = 0;
    unsigned mine = units, upto = incl;
    for (int base = 0; base < a.B; base += 32) {
      if (base > 0) {
        mine = base + lane < a.B ? units_of(p, a, base + lane) : 0;
        upto = scan(mine);
      }
      const unsigned past = __ballot_sync(0xffffffffu, upto * a.segs > at);
      if (past) {
        const int l = __ffs(past) - 1;
        at -= (__shfl_sync(0xffffffffu, upto, l) - __shfl_sync(0xffffffffu, mine, l)) * a.segs;
        c.request(p, a, base + l);
        c.seg = at / (unsigned)c.units;
        c.unit = at - c.seg * c.units;
        return c;
      }
      at -= __shfl_sync(0xffffffffu, upto, 31) * a.segs;
    }
    return c;
  }
};

// A ticket word of this launch: zero (clean) or whatever another launch or other
// use of the memory left becomes this launch's, with no tickets taken.  Every
// CTA that will take a ticket calls this first, early on.
__device__ __forceinline__ void open_tickets(unsigned long long* word, unsigned long long launch) {
  unsigned long long seen = *reinterpret_cast<volatile unsigned long long*>(word);
  if (seen >> 16 != launch) atomicCAS(word, seen, launch << 16);  // fails only where another CTA did it
}
// Takes a ticket; returns the tickets taken so far.  What the warp wrote before is
// visible to whoever takes a later one.
__device__ __forceinline__ unsigned take_ticket(unsigned long long* word) {
  unsigned long long was;
  asm volatile("atom.acq_rel.gpu.global.add.u64 %0, [%1], 1;" : "=l"(was) : "l"(word) : "memory");
  return (unsigned)(was & 0xffff) + 1;
}
// Waits for a phase of an mbarrier; try_wait suspends the warp for a while, which
// leaves the issue slots to the others.  Bounded (a few seconds): false and the
// device error word when it gives up.
__device__ __forceinline__ bool wait_copies(uint32_t bar, uint32_t parity) {
  const long long t0 = clock64();
  while (true) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    if (ok) return true;
    if (clock64() - t0 > kWaitBudgetCycles) break;
  }
  raise_device_error(DEV_ERR_ATTN_TIMEOUT);
  return false;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A number that no other launch of this process uses, 48 bits, never 0; they
// start at a place that memory written by others will hardly hold.
inline unsigned long long launch_number() {
  static std::atomic<unsigned long long> next{
      (unsigned long long)std::chrono::steady_clock::now().time_since_epoch().count() * 0x9e3779b97f4a7c15ull};
  unsigned long long n;
  do n = next.fetch_add(1, std::memory_order_relaxed) & 0xffffffffffffull;
  while (n == 0);
  return n;
}

}  // namespace kv4
}  // namespace fml
