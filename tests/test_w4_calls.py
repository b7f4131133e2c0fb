"""What the calls of 4-bit products do with memory, arguments and devices, beside their numbers (tests/test_w4_ops.py)."""
import weakref

import pytest
import torch

from pie_b200 import ops
from pie_b200.ops import w4


class Rows:
    """bf16 rows as a call on a GPU looks at them, in host memory, that remember the scratch made of them."""

    dtype = torch.bfloat16

    def __init__(self, t):
        self.t, self.made = t, []
        self.shape, self.stride, self.dim, self.data_ptr = t.shape, t.stride, t.dim, t.data_ptr

    def get_device(self):
        return -1

    def new_empty(self, *shape):
        scratch = self.t.new_empty(*shape)
        self.made.append(weakref.ref(scratch))
        return scratch


class Launchers:
    """The place of a weight's launchers. A launcher runs without the interpreter's lock: another thread may be given whatever is free by then."""

    def __init__(self, q, rows, most):
        self.weight, self.n, self.k, self.pitch, self.device = 0, q.shape[-2], q.shape[-1], (q.shape[-1] + 63) // 64 * 64, -1
        self.rows, self.status, self.sms, self.alive, self.of, self.most = most, 0, 148, [], rows, most
        self.few = self.many = self.few_tiles = self.all_tiles = self.launch
        self.few_rows = lambda e, k, n: n <= most

    def launch(self, *args):
        self.alive.append([ref() is not None for ref in self.of.made])
        return 0


@pytest.mark.parametrize("most", [0, 1 << 30])
def test_scratch_lives_until_the_launches_are_made(monkeypatch, most):
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: -1, raising=False)
    monkeypatch.setattr(w4, "stream_ptr", lambda: 0)
    q = ops.quantize_w4(torch.randn(2, 64, 128))
    a, out = Rows(torch.zeros(256, 128, dtype=torch.bfloat16)), torch.zeros(256, 64, dtype=torch.bfloat16)
    q._gpu = at = Launchers(q, a, most)
    ops.grouped_gemm(a, q, torch.zeros(2, dtype=torch.int32), out, 2, ops.EPI_STORE, torch.zeros(3, dtype=torch.int32), 4)
    assert at.alive == ([[]] if most else [[True]])
    x = Rows(torch.zeros(3, 128, dtype=torch.bfloat16))
    one = ops.quantize_w4(torch.randn(64, 128))
    one._gpu = at = Launchers(one, x, most)
    ops.gemm_w4(x, one)
    assert at.alive == ([[True]] if most else [[True, True]])          # the output is made of the rows too
