"""The converter warps' order of work in the prompt attention kernel, run on the
host with waits that succeed and waits that run out."""

import ctypes
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "mlir-cim22_b200" / "csrc"

# Event codes: 0 index wait, 1 slot wait, 2 load, 3 store, 4 used. The
# `stop`-th wait and, as in the kernel, all waits after it run out.
DRIVER = r"""
#include "kv_convert.h"
extern "C" int run(int parts, int stop, int *events, int capacity) {
  int n = 0, waits = 0;
  auto note = [&](int code, int side, int part) {
    if (n < capacity) {
      events[3 * n] = code;
      events[3 * n + 1] = side;
      events[3 * n + 2] = part;
    }
    ++n;
  };
  auto wait = [&] { return waits++ < stop; };
  cim::convert_parts(
      parts, [&](int j) { note(0, 0, j); return wait(); },
      [&](int side, int j) { note(1, side, j); return wait(); },
      [&](int j, int side) { note(2, side, j); }, [&](int side, int j) { note(3, side, j); },
      [&](int j) { note(4, 0, j); });
  return n;
}
"""
INDEX, SLOT, LOAD, STORE, USED = range(5)


@pytest.fixture(scope="module")
def run(tmp_path_factory):
    at = tmp_path_factory.mktemp("convert")
    (at / "driver.cpp").write_text(DRIVER)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", str(CSRC), "-o",
                    str(at / "driver.so"), str(at / "driver.cpp")], check=True)
    lib = ctypes.CDLL(str(at / "driver.so"))

    def run(parts, stop=10 ** 6):
        events = (ctypes.c_int * 3000)()
        n = lib.run(parts, stop, events, 1000)
        assert n <= 1000
        return [tuple(events[3 * i:3 * i + 3]) for i in range(n)]

    return run


@pytest.mark.parametrize("parts", [0, 2, 4, 6, 10, 34])
def test_every_part_is_loaded_and_stored_in_order(run, parts):
    events = run(parts)
    for side in range(2):
        assert [p for c, s, p in events if c == LOAD and s == side] == list(range(parts))
        assert [p for c, s, p in events if c == STORE and s == side] == list(range(parts))
        # Four parts' slots: a fifth waits until its slot has been read.
        assert [p for c, s, p in events if c == SLOT and s == side] == list(range(4, parts))
    assert [p for c, _, p in events if c == INDEX] == list(range(parts))
    assert [p for c, _, p in events if c == USED] == list(range(parts))


def test_a_negative_count_is_no_work(run):
    assert run(-3) == []


@pytest.mark.parametrize("parts", [2, 6, 34])
def test_nothing_relies_on_a_wait_that_ran_out(run, parts):
    waits = sum(c in (INDEX, SLOT) for c, _, _ in run(parts))
    for stop in range(waits):
        events, passed = run(parts, stop), 0
        indexed, emptied = set(), {(s, p) for s in range(2) for p in range(4)}
        for code, side, part in events:
            if code in (INDEX, SLOT):
                if passed < stop and code == INDEX:
                    indexed.add(part)
                elif passed < stop:
                    emptied.add((side, part))
                passed += 1
            elif code in (LOAD, USED):
                assert part in indexed, (stop, events)
            else:
                assert (side, part) in emptied, (stop, events)
