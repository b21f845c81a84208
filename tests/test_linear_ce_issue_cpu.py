"""The order of waits, products and commits of the head loss's tensor-core kernel (csrc/cuda/linear_ce_issue.h), run on the host: behind a wait that
expires no accumulator is handed to the epilogues, so that what they store is NaN and not a sum that lacks blocks."""
import os
import subprocess
from pathlib import Path

import oxibonsai_b200

SOURCE = Path(oxibonsai_b200.__file__).parent / "csrc" / "cuda"
PROGRAM = r"""
#include <cstdio>
#include <vector>
#include "linear_ce_issue.h"

struct Ops {
  int expires, waits = 0, products = 0, fresh = 0, buffer = -1;      // which wait expires; products since the last accumulator
  bool gone = false, bad = false;
  std::vector<int> committed, parity;
  bool wait() { bad |= gone; gone = waits++ == expires; return !gone; }
  bool wait_acc(int ab, unsigned phase) {
    buffer = ab; fresh = 0;
    parity.push_back((int)phase);
    return wait();
  }
  bool wait_full() { return wait(); }
  void product(int ab, bool first) { bad |= gone || ab != buffer || first != (fresh == 0); ++fresh; ++products; }
  void commit_acc(int ab) { bad |= gone || ab != buffer; committed.push_back(fresh); }
};

template <int kBufs, int kSegment> int check(int tiles, int blocks, int terms) {
  const int segments = kSegment == 0 ? 1 : (blocks + kSegment - 1) / kSegment, waits = tiles * (segments + blocks * terms);
  for (int expires = -1; expires < waits; ++expires) {
    Ops ops;
    ops.expires = expires;
    int seg = 0, done = 0;
    bool ok = true;
    for (int t = 0; t < tiles && ok; ++t) ok = bonsai::ce_issue<kBufs, kSegment>(ops, 5, 5 + blocks, terms, &seg);
    if (ok != (expires < 0) || ops.bad || (int)ops.committed.size() != seg) return 1;
    for (int i = 0; i < (int)ops.committed.size(); ++i) {
      const int at = i % segments, k0 = at * kSegment, want = (kSegment != 0 && k0 + kSegment < blocks ? kSegment : blocks - k0) * terms;
      if (ops.committed[i] != want) return 2;      // an accumulator that lacks products
      done += want;
    }
    for (int i = 0; i < (int)ops.parity.size(); ++i)
      if (ops.parity[i] != ((i / kBufs) & 1 ^ 1)) return 3;
    if (expires < 0 && (seg != tiles * segments || done != tiles * blocks * terms)) return 4;
    if (expires >= 0 && done >= tiles * blocks * terms) return 5;
  }
  return 0;
}

int main() {
  int r = 0;
  for (int tiles = 1; tiles <= 3; ++tiles)
    for (int blocks = 1; blocks <= 9; ++blocks)
      for (int terms = 1; terms <= 6; terms += 5) r |= check<2, 0>(tiles, blocks, terms) | check<2, 2>(tiles, blocks, terms) | check<4, 4>(tiles, blocks, terms);
  Ops ops;
  ops.expires = -1;
  int seg = 3;
  if (!bonsai::ce_issue<2, 0>(ops, 4, 4, 1, &seg) || seg != 3 || ops.waits) r |= 8;      // an empty part of a sum
  std::printf("%d\n", r);
  return r;
}
"""


def test_expired_waits_hand_over_no_accumulator(tmp_path):
    (tmp_path / "issue.cpp").write_text(PROGRAM)
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-O1", "-I", str(SOURCE), str(tmp_path / "issue.cpp"), "-o", str(tmp_path / "issue")], check=True)
    done = subprocess.run([str(tmp_path / "issue")], capture_output=True, text=True)
    assert done.returncode == 0, f"check {done.stdout.strip()} failed"
