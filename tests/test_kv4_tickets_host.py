"""Tickets of the tensor-core attention over the 4-bit cache, on the CPU: the kernel's own
walk over a batch's parts (csrc/kv4_tc_walk.cuh), compiled for the host, with CTAs that
give up somewhere.  Whatever they leave out, every ticket word has to be clean for the
next launch, a replayed graph's with the same launch number among them."""

import subprocess

from forgeml_b200 import build

PROGRAM = r"""
#include <cstdio>
#include <random>
#include <vector>
#include "kv4_tc_walk.cuh"
using namespace fml::kv4;
using fml::kv4::tc::Part;
using fml::kv4::tc::Walk;

int main() {
  std::mt19937 rng(1);
  auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
  int split = 0, gave_up = 0;
  for (int round = 0; round < 2000; ++round) {
    Pool p = {};
    p.slots = 4;
    p.H = pick(1, 3);
    p.max_seq = pick(1, 3000);
    Problem a = {};
    a.B = pick(1, 5);
    a.tq = pick(1, p.max_seq < 300 ? p.max_seq : 300);
    a.group = pick(1, 4);
    a.QH = p.H * a.group;
    const int tiles = (a.tq * a.group + tc::kRows - 1) / tc::kRows;
    a.segs = p.H * tiles;
    std::vector<int32_t> slot(a.B), start(a.B);
    unsigned total = 0;
    a.slot_of = slot.data();
    a.start_pos = start.data();
    for (int b = 0; b < a.B; ++b) {
      slot[b] = pick(0, 9) == 0 ? 7 : pick(0, 3);
      start[b] = pick(-1, p.max_seq);
      total += (keys_of(p, a, b) + tc::kBlock - 1) / tc::kBlock * a.segs;
    }
    if (total == 0) continue;
    const unsigned grid = pick(1, 148);
    const Shares shares(total, std::min(grid, (total + 1) / 2));
    std::vector<int> words(shares.W, 0);
    for (int launch = 0; launch < 2; ++launch) {  // the second one is whole
      std::vector<unsigned> order(shares.W), joined(shares.W, 0);
      for (unsigned c = 0; c < shares.W; ++c) order[c] = c;
      std::shuffle(order.begin(), order.end(), rng);
      std::vector<int> due(shares.W, 0);  // tickets that a word is still to give
      for (int pass = 0; pass < 2; ++pass)
        for (unsigned c : order) {
          Walk w = tc::walk_from(p, a, tiles, shares.begin(c), shares.begin(c + 1));
          const bool fails = launch == 0 && pass == 1 && pick(0, 4) == 0;
          int until = pick(0, 3);
          const bool owed = pick(0, 1) != 0;
          unsigned took = 0;
          gave_up += fails;
          auto take = [&](unsigned w0) { --due[w0]; return (unsigned)++words[w0]; };
          auto clean = [&](unsigned w0) {
            if (due[w0] != 0 || joined[w0]++) { std::printf("joined early or twice\n"); std::exit(1); }
            words[w0] = 0;
          };
          Part part;
          while (w.next(p, a, part)) {
            const unsigned w0 = shares.holder(part.seg0, c), w1 = shares.holder(part.seg0 + part.units - 1, c);
            if (pass == 0) {
              due[w0] += !part.whole;
              continue;
            }
            split += !part.whole;
            const bool now = fails && until-- == 0;
            if (!(now && owed) && !part.whole) {
              took |= 1u << part.which;
              if (take(w0) == w1 - w0 + 1) clean(w0);
            }
            if (now) {
              tc::give_up(p, a, shares, tiles, c, took, [&](const Part&, unsigned x) { return take(x); }, clean);
              break;
            }
          }
        }
      for (unsigned c = 0; c < shares.W; ++c)
        if (words[c] != 0 || due[c] != 0) { std::printf("word %u of %u left at %d\n", c, shares.W, words[c]); return 1; }
    }
  }
  std::printf("split %d gave_up %d\n", split, gave_up);
  return 0;
}
"""


def test_ctas_that_give_up_leave_clean_tickets(tmp_path):
    src, exe = tmp_path / "tickets.cu", tmp_path / "tickets"
    src.write_text(PROGRAM)
    r = subprocess.run([build.nvcc_path(), *build.ARCH, "-std=c++17", "--expt-relaxed-constexpr", "-rdc=true",
                        f"-I{build.CSRC}", f"-I{build.PKG.parent / 'include'}", str(src), "-o", str(exe)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
    words = r.stdout.split()
    assert int(words[1]) > 1000 and int(words[3]) > 1000  # both were met
