"""The turn of a plan's device-resident runs (csrc/turn.h) where a CUDA call
fails, with a fake of the calls: an order that could not be made is an error,
never a run without it."""
import subprocess
from pathlib import Path

PKG = Path(__file__).resolve().parent.parent / "bafe-basic-algibra-fusion-engine-_b200"

SOURCE = r"""
#include "turn.h"
#include <cstdio>
#include <string>

std::string calls;
int fail_capturing, fail_wait, fail_make, fail_record;
bool in_capture;

struct Fake {
    typedef int Stream;
    typedef int* Event;
    int capturing(int, bool& is) { calls += "c"; is = in_capture; return fail_capturing; }
    int wait(int st, int*) { calls += "w" + std::to_string(st); return fail_wait; }
    int make(int*& e) {
        calls += "m";
        static int event;
        e = fail_make ? nullptr : &event;
        return fail_make;
    }
    int record(int*, int st) { calls += "r" + std::to_string(st); return fail_record; }
};
typedef bafe_cuda::Turn<Fake> Turn;

int* last = nullptr;
// begin, a run with the result `rc`, end; -1 in place of the result where the run was not reached
int run(int st, bool needed, int rc, int& reached) {
    calls.clear();
    reached = 0;
    Turn t(Fake(), last, st);
    if (int e = t.begin(needed)) return e;
    reached = 1;
    calls += "R";
    return t.end(rc);
}
#define EXPECT(st, needed, rc, result, was_reached, log) \
    do { \
        int reached = 0, got = run(st, needed, rc, reached); \
        if (got != (result) || reached != (was_reached) || calls != (log)) { \
            std::printf("line %d: %d, reached %d, %s\n", __LINE__, got, reached, calls.c_str()); \
            return 1; \
        } \
    } while (0)

int main() {
    EXPECT(1, false, 0, 0, 1, "R");                       // no scratch: no calls
    EXPECT(1, false, 5, 5, 1, "R");
    fail_make = 7;
    EXPECT(1, true, 0, 7, 0, "cm");                       // no event: no run
    fail_make = 0;
    EXPECT(1, true, 0, 0, 1, "cmw1Rr1");                  // and the next one tries again
    EXPECT(2, true, 0, 0, 1, "cw2Rr2");
    EXPECT(2, true, 5, 5, 1, "cw2Rr2");                   // what a failed run enqueued is waited for too
    fail_wait = 7;
    EXPECT(3, true, 0, 7, 0, "cw3");                      // no order: no run, and nothing recorded over the last end
    fail_wait = 0;
    fail_record = 7;
    EXPECT(4, true, 0, 7, 1, "cw4Rr4");                   // the next run's order would be lost: reported
    EXPECT(4, true, 5, 5, 1, "cw4Rr4");                   // the run's own error comes first
    fail_record = 0;
    in_capture = true;
    EXPECT(5, true, 0, 0, 1, "cR");                       // a captured run's order is its graph's
    in_capture = false;
    fail_capturing = 7;
    EXPECT(5, true, 0, 7, 0, "c");
    std::puts("in turn");
}
"""


def test_failed_calls_are_reported(tmp_path):
    src, exe = tmp_path / "turn.cpp", tmp_path / "turn"
    src.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", f"-I{PKG / 'csrc'}", str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "in turn" in r.stdout, r.stdout
