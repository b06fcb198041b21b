"""Whether operands share memory, against the sets of bytes themselves (no GPU)."""
import itertools

import torch

from bafe_b200 import lm


def places(t):
    at = t.data_ptr() + t.element_size() * sum(
        torch.arange(n).view([-1 if j == i else 1 for j in range(t.dim())]) * s
        for i, (n, s) in enumerate(zip(t.shape, t.stride())))
    return {int(a) + b for a in at.reshape(-1) for b in range(t.element_size())}


def test_rows_of_any_stride():
    """One row of a broadcast tensor has stride 0; a row's stride says nothing where there is one row."""
    buf = torch.zeros(400, dtype=torch.bfloat16)
    views = [buf[a:a + (r - 1) * s + w].as_strided((r, w), (s, 1))
             for r, w, s, a in itertools.product((1, 3), (1, 16, 40), (0, 1, 8, 50), (0, 7, 16, 40, 57)) if r == 1 or s >= w]
    views += [buf.view(8, 50)[:, 10:20], buf.view(8, 50)[2:, 20:50], buf[:100].view(torch.float32).view(2, 25), buf[5:5]]
    views += [buf[:64].expand(4, 64)[:1, :32], buf[:64].expand(4, 64)[:1, 16:48]]
    shared = 0
    for a, b in itertools.product(views, views):
        if places(a) & places(b) if a.numel() and b.numel() else False:
            assert lm._overlap(a, b), (a.shape, a.stride(), a.storage_offset(), b.shape, b.stride(), b.storage_offset())
            shared += 1
    assert shared > 500
