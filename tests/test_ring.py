"""The stage ring of the delta rule's recurrences (csrc/qrb_ring.cuh), run on the host: every order in which a
loader, a thread that issues products and the threads that compute can take their steps.  The kernels' waits use
the same two functions for stages and parities."""
import shutil
import subprocess

import pytest

from conftest import PKG

MODEL = r"""
#include <cstdio>
#include <set>
#include <tuple>
#include "qrb_ring.cuh"

constexpr int kItems = 9;

// A barrier is the number of phases it has completed; a wait by parity passes when the current phase's parity is
// not the one waited for.
struct State {
  int load = 0, issue = 0, issued = 0, work = 0;   // items begun / ended by each role; issued: first products
  int full[2] = {0, 0}, empty[2] = {0, 0};
  auto key() const { return std::make_tuple(load, issue, issued, work, full[0], full[1], empty[0], empty[1]); }
};
bool passes(int phases, unsigned parity) { return ((unsigned)phases & 1u) != parity; }

// SHARED: one `empty` barrier for all stages, waited for by the parity of the item (what must not be).
template <int S, bool SHARED>
struct Model {
  using R = qrb::Ring<S>;
  std::set<decltype(State().key())> seen;
  int stuck = 0, overwritten = 0, ended = 0;

  static int bar(int i) { return SHARED ? 0 : R::stage(i); }
  static unsigned parity(int i) { return SHARED ? (unsigned)i & 1u : R::phase(i); }

  void go(const State& s) {
    if (!seen.insert(s.key()).second) return;
    bool moved = false;
    if (s.load < kItems && (s.load < S || passes(s.empty[bar(s.load - S)], parity(s.load - S)))) {
      State t = s;
      if (t.load >= S && t.work < t.load - S + 1) ++overwritten;   // the stage's last item is still in use
      ++t.full[R::stage(t.load++)];
      moved = true;
      go(t);
    }
    // the issuer: an item's first products when it is loaded, the others when the item before is done with
    if (s.issue < kItems && s.issued == s.issue && passes(s.full[R::stage(s.issue)], R::phase(s.issue))) {
      State t = s;
      ++t.issued;
      moved = true;
      go(t);
    }
    if (s.issue < kItems && s.issued == s.issue + 1 &&
        (s.issue == 0 || passes(s.empty[bar(s.issue - 1)], parity(s.issue - 1)))) {
      State t = s;
      if (t.issue > 0 && t.work < t.issue) ++overwritten;
      ++t.issue;
      moved = true;
      go(t);
    }
    // the computing threads: an item ends when all its products are there
    if (s.work < kItems && s.work < s.issue && passes(s.full[R::stage(s.work)], R::phase(s.work))) {
      State t = s;
      ++t.empty[bar(t.work++)];
      moved = true;
      go(t);
    }
    if (!moved) (s.work == kItems ? ended : stuck) += 1;
  }
};

template <int S, bool SHARED>
void run(const char* name) {
  Model<S, SHARED> m;
  m.go(State());
  std::printf("%s %d %d %d\n", name, m.stuck, m.overwritten, m.ended);
}

int main() {
  run<1, false>("one");
  run<2, false>("two");
  run<2, true>("shared");
}
"""


@pytest.fixture(scope="module")
def outcomes(tmp_path_factory):
    where = tmp_path_factory.mktemp("ring")
    src, exe = where / "model.cpp", where / "model"
    src.write_text(MODEL)
    cxx = shutil.which("g++") or "c++"
    subprocess.run([cxx, "-std=c++17", "-O1", f"-I{PKG / 'csrc'}", str(src), "-o", str(exe)], check=True)
    text = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    return {name: tuple(map(int, rest)) for name, *rest in map(str.split, text.splitlines())}


@pytest.mark.parametrize("stages", ["one", "two"])
def test_every_order_ends(outcomes, stages):
    stuck, overwritten, ended = outcomes[stages]
    assert (stuck, overwritten, ended) == (0, 0, 1)


def test_one_barrier_for_two_stages_can_stop(outcomes):
    """The model finds what a shared barrier allows: the loader two phases behind, waiting for good."""
    assert outcomes["shared"][0] > 0


@pytest.mark.parametrize("source", ["qrb_delta_scan.cu", "qrb_delta_rscan.cu"])
def test_recurrences_wait_by_stage(source):
    """Each stage has barriers of its own, and every wait for one takes stage and parity from the ring."""
    import re
    text = (PKG / "csrc" / source).read_text()
    assert "full[2], empty[2]" in text
    waits = re.findall(r"_wait(?:_abort)?\(&bars\.(full|empty)\[([^\]]+)\], ([^,]+(?:\([^)]*\))?)", text)
    assert {w[0] for w in waits} == {"full", "empty"}
    for name, stage, parity in waits:
        assert parity.startswith("R::phase("), (name, stage, parity)
