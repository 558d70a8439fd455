"""Sizes next to 2^31, where a kernel's counters would pass the end of their type: refused before anything is launched, and left to the plain operators by Python."""
import ctypes as C

import torch

import mini_nccl_b200 as mn
from mini_nccl_b200.ops import distill


def test_tokens_and_classes():
    L = mn.lib()
    p = C.c_void_p(4096)   # never looked at: every call below is refused before anything is launched
    f = [p, 9, 2**31, 4, 64, p, p, 8, 1.0, p, p, p, p, p, p, p, None]
    b = [p, 9, 2**31, 4, 64, p, p, 8, 1.0, p, p, p, 0, None, p, 2**31, None]
    for call, args in ((L.mncclDistillForward, f), (L.mncclDistillBackward, b)):
        for at in (3, 4):
            for n in (2**31 - 2**12 + 1, 2**31 - 1):
                bad = list(args)
                bad[at] = n
                assert call(*bad) == -2, (at, n)


def test_python_goes_by_the_same_limit(monkeypatch):
    class Shaped:
        """What the question looks at, of sizes that no test could hold."""
        is_cuda, dtype = True, torch.bfloat16

        def __init__(self, *shape):
            self.shape = shape

        def numel(self):
            return self.shape[0] * self.shape[1]

    monkeypatch.setattr(distill, "_plain", lambda t: True)
    monkeypatch.setattr(distill, "no_tangent", lambda t: True)
    for n, takes in ((2**31 - 2**12, True), (2**31 - 2**12 + 1, False), (2**31 - 1, False)):
        assert distill._native(Shaped(n, 8), Shaped(n, 3), Shaped(n, 3)) is takes
        assert distill._native(Shaped(8, n), Shaped(8, 3), Shaped(8, 3)) is takes
