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


def test_first_callers_of_a_device_share_what_is_made(tmp_path):
    """The device's error word: one is made however many ask at once, and a failure is not kept."""
    src = tmp_path / "once.cpp"
    src.write_text("""
        #include "once_per_device.h"
        #include <chrono>
        #include <cstdio>
        #include <thread>
        #include <vector>
        bafe_cuda::OncePerDevice<unsigned, 4> words;
        int main() {
            if (words.get(-1, [] { return new unsigned(0); }) || words.get(4, [] { return new unsigned(0); })) return 1;
            if (words.peek(2) || words.get(2, []() -> unsigned* { return nullptr; }) || words.peek(2)) return 2;
            std::atomic<int> made{0};
            std::vector<unsigned*> got(32);
            std::vector<std::thread> threads;
            for (int i = 0; i < 32; ++i)
                threads.emplace_back([&, i] {
                    got[i] = words.get(2, [&] {
                        std::this_thread::sleep_for(std::chrono::milliseconds(20));
                        ++made;
                        return new unsigned(7);
                    });
                });
            for (auto& t : threads) t.join();
            for (unsigned* p : got) if (!p || p != got[0] || *p != 7) return 3;
            if (made != 1 || words.peek(2) != got[0] || words.peek(1) || words.peek(9)) return 4;
            std::puts("one");
        }
    """)
    exe = tmp_path / "once"
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", f"-I{PKG / 'csrc'}", str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "one" in r.stdout, r.returncode


@pytest.mark.gpu
def test_first_grouped_call_in_a_capture_on_a_blocking_stream(cuda):
    """A stream that the legacy default stream waits for, as a C caller's cudaStreamCreate makes it."""
    r = run("""
        import ctypes, sys
        sys.path.insert(0, sys.argv[1])
        import torch
        import bafe_b200
        from bafe_b200 import lm
        x, w = torch.randn(64, 128, device="cuda").bfloat16(), torch.randn(2, 64, 128, device="cuda").bfloat16()
        off = torch.tensor([0, 10, 64], dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        rt = ctypes.CDLL(next(l.split()[-1] for l in open("/proc/self/maps") if "libcudart" in l))
        raw = ctypes.c_void_p()
        assert rt.cudaStreamCreate(ctypes.byref(raw)) == 0
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=torch.cuda.ExternalStream(raw.value)):
            y = lm.grouped_matmul(x, w, off)
        g.replay()
        bafe_b200.synchronize()
        got = y.clone()
        assert torch.equal(got, lm.grouped_matmul(x, w, off))
        bafe_b200.synchronize()
        print("same")
    """)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


@pytest.mark.gpu
def test_first_grouped_calls_of_several_threads(cuda):
    r = run("""
        import sys, threading
        sys.path.insert(0, sys.argv[1])
        import torch
        import bafe_b200
        from bafe_b200 import lm
        x, w = torch.randn(300, 128, device="cuda").bfloat16(), torch.randn(2, 64, 128, device="cuda").bfloat16()
        off = torch.tensor([0, 100, 300], dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        go, out = threading.Barrier(8), [None] * 8

        def call(i):
            stream = torch.cuda.Stream()
            go.wait()
            out[i] = lm.grouped_matmul(x, w, off, stream=stream)

        threads = [threading.Thread(target=call, args=(i,)) for i in range(8)]
        for t in threads: t.start()
        for t in threads: t.join()
        bafe_b200.synchronize()
        want = lm.grouped_matmul(x, w, off)
        bafe_b200.synchronize()
        assert all(torch.equal(y, want) for y in out)
        print("same")
    """)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


@pytest.mark.gpu
def test_launches_of_several_threads_are_all_counted(cuda):
    r = run("""
        import sys, threading
        sys.path.insert(0, sys.argv[1])
        import torch
        import bafe_b200
        from bafe_b200 import lm
        from bafe_b200._binding import DTYPE_F32, lib
        x, w = torch.randn(1, 8, device="cuda"), torch.ones(8, device="cuda")
        outs = [torch.empty_like(x) for _ in range(6)]
        torch.cuda.synchronize()
        before, each = bafe_b200.launch_count(), 3000

        def call(y):
            s = torch.cuda.Stream().cuda_stream
            for _ in range(each):
                assert lib.bafe_cuda_rms_norm(x.data_ptr(), 8, None, 0, w.data_ptr(), y.data_ptr(), 8, None, None, 0,
                                              1, 8, DTYPE_F32, DTYPE_F32, DTYPE_F32, 1e-6, s) == 0

        threads = [threading.Thread(target=call, args=(y,)) for y in outs]
        for t in threads: t.start()
        for t in threads: t.join()
        torch.cuda.synchronize()
        assert bafe_b200.launch_count() - before == each * 6, bafe_b200.launch_count() - before
        assert all(torch.equal(y, lm.rms_norm(x, w)) for y in outs)
        print("all")
    """)
    assert r.returncode == 0 and "all" in r.stdout, r.stderr[-2000:]


@pytest.mark.gpu
def test_a_product_from_a_thread_without_a_context(cuda):
    """A host thread whose first CUDA call is the product itself (nothing to allocate)."""
    r = run("""
        import sys, threading
        sys.path.insert(0, sys.argv[1])
        import torch
        import bafe_b200
        from bafe_b200 import lm
        x, w = torch.randn(64, 128, device="cuda").bfloat16(), torch.randn(2, 64, 128, device="cuda").bfloat16()
        off, y = torch.tensor([0, 10, 64], dtype=torch.int32, device="cuda"), torch.empty(64, 64, device="cuda", dtype=torch.bfloat16)
        dw = torch.empty_like(w)
        lm.grouped_matmul(x, w, off)                     # all that the library makes once is made
        torch.cuda.synchronize()
        failed = []

        def call():
            try:
                lm.grouped_matmul(x, w, off, out=y)
                lm.grouped_matmul_grad_weight(y, x, off, out=dw)
            except RuntimeError as e:
                failed.append(str(e))

        t = threading.Thread(target=call)
        t.start()
        t.join()
        assert not failed, failed
        bafe_b200.synchronize()
        assert torch.equal(y, lm.grouped_matmul(x, w, off)) and torch.equal(dw, lm.grouped_matmul_grad_weight(y, x, off))
        print("same")
    """)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


@pytest.mark.gpu
def test_first_products_of_many_threads_at_once(cuda):
    """What the first product looks up in the driver is there for all of them."""
    for _ in range(4):
        r = run("""
            import sys, threading
            sys.path.insert(0, sys.argv[1])
            import torch
            import bafe_b200
            from bafe_b200 import lm
            from bafe_b200._binding import DTYPE_BF16, last_error, lib
            x, w = torch.randn(64, 128, device="cuda").bfloat16(), torch.randn(2, 64, 128, device="cuda").bfloat16()
            off = torch.tensor([0, 10, 64], dtype=torch.int32, device="cuda")
            lm.grouped_matmul_grad_weight(x[:0], x[:0], off)        # no product: the error word only
            outs, failed = [torch.empty(64, 64, device="cuda", dtype=torch.bfloat16) for _ in range(32)], []
            torch.cuda.synchronize()
            args = [(x.data_ptr(), 128, w.data_ptr(), 128, 64 * 128, 1, off.data_ptr(), None, None, 0, y.data_ptr(), 64, 64, 2,
                     64, 128, DTYPE_BF16, DTYPE_BF16, None, 0, None) for y in outs]
            ready, go = threading.Semaphore(0), []

            def call(a):
                torch.cuda.Stream()                      # the thread has a context
                ready.release()
                while not go:
                    pass
                if lib.bafe_cuda_grouped_matmul(*a):
                    failed.append(last_error())

            sys.setswitchinterval(1e-5)
            threads = [threading.Thread(target=call, args=(a,)) for a in args]
            for t in threads: t.start()
            for t in threads: ready.acquire()
            go.append(1)
            for t in threads: t.join()
            bafe_b200.synchronize()
            assert not failed, (len(failed), failed[0])
            want = lm.grouped_matmul(x, w, off)
            bafe_b200.synchronize()
            assert all(torch.equal(y, want) for y in outs)
            print("all")
        """)
        assert r.returncode == 0 and "all" in r.stdout, r.stderr[-2000:]
