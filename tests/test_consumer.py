"""What happens to memory whose consumer lets go of it: the decision, compiled with a stand-in for the queries of its
stream (a stream that is gone is not made on a GPU)."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
#include <cstdio>
#include <cstdlib>
#include "rx_consumer.h"
using namespace rx;
struct Fake {
  Query capture, identity;
  bool active;
  unsigned long long now;
  Query capturing(int, bool* a) const { *a = active; return capture; }
  Query id(int, unsigned long long* i) const { *i = now; return identity; }
};
int main(int, char** v) {
  const Fake f{(Query)atoi(v[1]), (Query)atoi(v[3]), atoi(v[2]) != 0, strtoull(v[4], nullptr, 10)};
  printf("%d", (int)consumer_state(f, 0, 7ull));
}
"""
OK, IMPLICIT, FAILED = range(3)
PRESENT, CAPTURED, GONE = range(3)


@pytest.fixture(scope="module")
def decide(tmp_path_factory):
    where = tmp_path_factory.mktemp("consumer")
    (where / "p.cpp").write_text(PROGRAM)
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-I", os.path.join(ROOT, "reactant.jl_b200", "csrc"), "-o", str(where / "p"), str(where / "p.cpp")], check=True)
    return lambda *a: int(subprocess.run([str(where / "p")] + [str(int(v)) for v in a], check=True, capture_output=True, text=True).stdout)


@pytest.mark.parametrize("capture,active,identity,now,want", [
    (OK, False, OK, 7, PRESENT),
    (OK, True, OK, 7, CAPTURED),
    (IMPLICIT, False, OK, 7, CAPTURED),
    (FAILED, False, OK, 7, GONE),      # the handle is no stream any more: not to be asked again and again
    (FAILED, True, FAILED, 0, GONE),
    (OK, False, OK, 8, GONE),          # the handle has been given to another stream
    (OK, False, FAILED, 7, GONE),
])
def test_consumers_that_let_go(decide, capture, active, identity, now, want):
    assert decide(capture, active, identity, now) == want
