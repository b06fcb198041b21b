"""Calls of the library from several host threads at once (ctypes releases
the GIL for their length): refusals here, without a GPU, and kernels' calls
on one."""
import subprocess
import sys
import textwrap
from pathlib import Path

import pytest

PKG = Path(__file__).resolve().parent.parent / "bafe-basic-algibra-fusion-engine-_b200"


def run(code, timeout=300):
    """In a process of its own: memory that two threads write would end this one."""
    return subprocess.run([sys.executable, "-c", textwrap.dedent(code), str(PKG)], capture_output=True, text=True,
                          timeout=timeout)


def test_threads_that_are_refused_read_their_own_message():
    r = run("""
        import ctypes, sys, threading
        sys.path.insert(0, sys.argv[1])
        from bafe_b200 import _binding
        from bafe_b200._binding import DTYPE_BF16, lib
        P = ctypes.c_void_p(256)
        wrong = []

        def norms():
            for _ in range(20000):
                if lib.bafe_cuda_rms_norm(None, 64, None, 0, P, P, 64, None, None, 0, 4, 64, DTYPE_BF16, DTYPE_BF16,
                                          DTYPE_BF16, 1e-6, None) != 8:
                    wrong.append("norm")
                code, msg = _binding.last_error()
                if code != 8 or msg != "rms_norm: null operand":
                    wrong.append(msg)

        def products():
            for _ in range(20000):
                if lib.bafe_cuda_grouped_matmul_workspace(P, 64, P, 64, 2048, 1, 8, 0, 32, 64, DTYPE_BF16) != -1:
                    wrong.append("grouped")
                code, msg = _binding.last_error()
                if code != 8 or not msg.startswith("grouped_matmul: sizes out of range"):
                    wrong.append(msg)

        threads = [threading.Thread(target=f) for f in (norms, products) * 3]
        for t in threads: t.start()
        for t in threads: t.join()
        assert not wrong, (len(wrong), wrong[:3])
        print("apart")
    """)
    assert r.returncode == 0 and "apart" in r.stdout, (r.returncode, r.stderr[-1500:])


def test_a_thread_without_an_error_reads_the_last_one():
    r = run("""
        import ctypes, sys, threading
        sys.path.insert(0, sys.argv[1])
        from bafe_b200 import _binding
        from bafe_b200._binding import lib
        seen = []
        other = lambda f: (lambda t: (t.start(), t.join()))(threading.Thread(target=f))
        other(lambda: lib.bafe_cuda_rms_norm_grad_workspace(-1, 64, 5))
        other(lambda: seen.append(_binding.last_error()))
        assert _binding.last_error() == seen[0] and seen[0][0] == 8 and "rms_norm" in seen[0][1]
        lib.bafe_cuda_clear_error()
        assert _binding.last_error() == (0, "")
        print("read")
    """)
    assert r.returncode == 0 and "read" in r.stdout, r.stderr[-1500:]
