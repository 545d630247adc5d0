"""The exchange between the two warps that share a tile's rows
(theria_b200/csrc/pair_exchange.cuh), compiled for the host: two threads run the
loop of the width-128 forward kernels with every order of waits that run out or
return late.  A meeting that only one of them comes to would hang the kernel, so
here each meeting has a limit and reports it."""

import pathlib
import shutil
import subprocess

import pytest

CSRC = pathlib.Path(__file__).resolve().parents[1] / "theria_b200" / "csrc"

PROGRAM = r"""
#include <chrono>
#include <condition_variable>
#include <cstdio>
#include <mutex>
#include <thread>
#include "pair_exchange.cuh"

struct Alone {};

struct Barrier {  // of two threads
  std::mutex m;
  std::condition_variable c;
  int here = 0, round = 0;
  void meet() {
    std::unique_lock<std::mutex> l(m);
    const int r = round;
    if (++here == 2) { here = 0; ++round; c.notify_all(); return; }
    if (!c.wait_for(l, std::chrono::seconds(5), [&] { return round != r; })) throw Alone{};
  }
};

struct Result { bool ok = true, alone = false; float m = -1.f, l = 0.f; };

// A warp's loop: waits[j] is what its wait of tile j returns, j + 1 (one half) and
// 10 (j + 1) (the other) the maxima, 1 and 2 the sums.
void warp(int h, int tiles, unsigned waits, float (*red)[2], Barrier& b, Result& r) {
  auto meet = [&] { b.meet(); };
  try {
    for (int j = 0; j < tiles; ++j) {
      float other;
      if (!(waits >> j & 1)) {
        r.ok = false;
        theria::tc::pair_exchange(&red[j & 1][h], &red[j & 1][h ^ 1], false, 0.f, other, meet);
        break;
      }
      const float mt = (h ? 10.f : 1.f) * (j + 1);
      if (!theria::tc::pair_exchange(&red[j & 1][h], &red[j & 1][h ^ 1], true, mt, other, meet)) {
        r.ok = false;
        break;
      }
      r.m = mt > other ? mt : other;
    }
    if (r.ok) {
      red[tiles & 1][h] = h ? 2.f : 1.f;
      meet();
      r.l = red[tiles & 1][h] + red[tiles & 1][h ^ 1];
    }
  } catch (Alone) { r.alone = true; }
}

int main() {
  int bad = 0, runs = 0;
  for (int tiles = 1; tiles <= 4; ++tiles)
    for (unsigned a = 0; a < 1u << tiles; ++a)
      for (unsigned c = 0; c < 1u << tiles; ++c, ++runs) {
        float red[2][2] = {};
        Barrier b;
        Result r[2];
        std::thread x(warp, 0, tiles, a, red, std::ref(b), std::ref(r[0]));
        std::thread y(warp, 1, tiles, c, red, std::ref(b), std::ref(r[1]));
        x.join();
        y.join();
        const bool all = (a & c) + 1 == 1u << tiles;
        for (const Result& e : r)
          if (e.alone || e.ok != all || (all && (e.m != 10.f * tiles || e.l != 3.f))) {
            std::printf("tiles %d waits %u %u: ok %d alone %d m %g l %g\n", tiles, a, c, e.ok,
                        e.alone, e.m, e.l);
            if (++bad > 4) return 1;
          }
      }
  std::printf("runs %d\n", runs);
  return bad != 0;
}
"""


def test_no_warp_is_left_at_a_meeting(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host compiler")
    (tmp_path / "pair.cpp").write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-O1", "-pthread", "-x", "c++", "-D__device__=",
                    "-D__forceinline__=inline", f"-I{CSRC}", str(tmp_path / "pair.cpp"), "-o",
                    str(tmp_path / "pair")], check=True)
    run = subprocess.run([str(tmp_path / "pair")], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stdout
    assert run.stdout == f"runs {sum(4 ** n for n in range(1, 5))}\n"


@pytest.mark.parametrize("name", ["ragged_tc_fwd.cuh", "sdpa_tc_fwd.cuh"])
def test_the_forward_kernels_meet_nowhere_else(name):
    """The only barrier of part of a block that these kernels have is the pair's: met
    in pair_exchange, and once at the end by pairs whose loops ended well."""
    text = (CSRC / name).read_text()
    assert text.count("named_bar(") == 1
    assert text.count("tc::pair_exchange(") == 2
    assert text.count("      meet();") == 1
    before = text[:text.index("      meet();")].rstrip().splitlines()
    assert before[-2].strip() == "if (ok) {"
