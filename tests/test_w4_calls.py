"""What the calls of 4-bit products do with memory, arguments and devices, beside their numbers (tests/test_w4_ops.py)."""
import weakref

import pytest
import torch

from pie_b200 import ops
from pie_b200.ops import w4

from test_w4_ops import FORMS, close, expected, expert_case, product_case


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


@pytest.mark.gpu
@pytest.mark.parametrize("form", [FORMS[0], FORMS[2], FORMS[5]], ids=["int4", "int4z", "fp4"])
def test_lanes_that_part_ahead_of_instructions_of_whole_warps(form):
    """Batches of which a part of a warp has a turn more before a cluster joins, features past the last inside a warp between reads of
    tensor memory, experts' steps that few lanes store: right, and the same every time."""
    for m, n, k in ((1, 64, 16384), (3, 64, 16384), (1, 4096, 14336), (7, 264, 8192), (40, 40, 128), (200, 24, 128), (130, 1000, 256)):
        k = k // form[3] * form[3]
        x, w, _, want, room = product_case(m, n, k, form)
        first = ops.gemm_w4(x, w)
        close(first, want, room)
        for _ in range(20):
            assert torch.equal(ops.gemm_w4(x, w), first)
    for counts in ([1, 0, 3], [2] * 40, [300, 9, 40]):
        for n, k in ((8, 128), (40, 1024)):
            a, w, buf, mt, want, room, used = expert_case(counts, n, k, form, ops.EPI_STORE)
            for rows in (1, 1 << 40):
                out = torch.full(want.shape, 3.0, device="cuda").bfloat16()
                ops.grouped_gemm(a, w, buf.tile_expert, out, mt, ops.EPI_STORE, buf.tile_list, rows)
                close(out, want, room)
                again = torch.full(want.shape, 3.0, device="cuda").bfloat16()
                ops.grouped_gemm(a, w, buf.tile_expert, again, mt, ops.EPI_STORE, buf.tile_list, rows)
                assert torch.equal(again, out)
    ops.check_kernel_status()


@pytest.mark.parametrize("preset", ["tiny-llama", "tiny-qwen3-moe"])
def test_the_cpu_driver_that_a_configuration_makes_has_its_weights_in_4_bits(preset):
    from pie_b200.server import config as cfgmod
    from pie_b200.server.serve import _build_drivers_direct
    text = f'[[model]]\nname = "m"\npreset = "{preset}"\n[model.driver]\ntype = "cpu"\n'
    held = []
    for key in ("", 'weight_dtype = "int4"\n'):
        (drv,), _, _, _ = _build_drivers_direct(cfgmod.parse(text + key).model[0])
        held.append([isinstance(lw["wqkv"], ops.W4Linear) for lw in drv.model.w["layers"]])
    assert not any(held[0]) and all(held[1])


def test_layers_in_fp16_are_quantised():
    from pie_b200.models.config import preset
    from pie_b200.models.weights import quantize_layers, random_weights
    cfg = preset("tiny-llama")
    for lw in quantize_layers(random_weights(cfg, "cpu", torch.float16), cfg, "int4")["layers"]:
        assert isinstance(lw["wqkv"], ops.W4Linear) and isinstance(lw["wo"], ops.W4Linear)


@pytest.mark.gpu
def test_an_expert_alone_is_taken_without_waiting_and_in_a_graph(monkeypatch):
    gen = torch.Generator("cuda").manual_seed(2)
    q = ops.quantize_w4(torch.randn(3, 64, 256, generator=gen, device="cuda"), 64, asymmetric=True)
    x = torch.randn(5, 256, generator=gen, device="cuda").bfloat16()
    want, room = expected(x, q[1].dequant(torch.float64))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.gemm_w4(x, q[1])
    g.replay()
    close(y, want, room)

    def stop(device=None):
        raise AssertionError("the device is waited for")
    monkeypatch.setattr(torch.cuda, "synchronize", stop)
    assert torch.equal(ops.gemm_w4(x, q[-2]), y)
    with pytest.raises(AssertionError):                                # a weight of its own does wait for what wrote it
        ops.W4Linear.from_packed(q.packed[:1], q.scale[:1], q.zero[:1], q.factor[:1], (64, 256), 64, "int4")
