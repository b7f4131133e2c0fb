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


@pytest.mark.gpu
def test_rows_past_32_bits():
    """Batches of more than 2^31 elements: their first and last rows' products, norms and experts' products."""
    gen = torch.Generator("cuda").manual_seed(3)
    m, n, k = 270000, 64, 8192
    q = ops.quantize_w4(torch.randn(n, k, generator=gen, device="cuda"), 128)
    x = torch.randn(512, k, generator=gen, device="cuda").bfloat16().repeat(528, 1)[:m]
    assert x.numel() > 2 ** 31
    ends = torch.tensor([0, 1, 511, m - 70, m - 1], device="cuda")
    y = ops.gemm_w4(x, q)
    close(y[ends], *expected(x[ends], q.dequant(torch.float64)))
    assert torch.equal(y[:512], y[512 * 400:512 * 401])                # the same rows in other places
    w = torch.ones(k, device="cuda").bfloat16()
    x8, sx = ops.rmsnorm_fp8(x, w, 1e-6)
    want8, want = ops.rmsnorm_fp8(x[ends].clone(), w, 1e-6)
    assert torch.equal(sx[ends], want) and torch.equal(x8[ends].view(torch.uint8), want8.view(torch.uint8))
    e, mt = 2, m // 128
    twice = lambda t: torch.cat([t, t]) if t is not None else None
    experts = ops.W4Experts.from_packed(twice(q.packed), twice(q.scale), twice(q.zero), twice(q.factor), (e, n, k), 128, "int4")
    buf = ops.MoeBuffers(m, 8, 8, e, 1, "cuda")
    for counts in ([m // 256 * 128, 100], [3, (mt - 2) * 128 + 5]):
        buf.counts.copy_(torch.tensor(counts, dtype=torch.int32))
        ops.moe_align(buf, mt)
        first = -(-counts[0] // 128) * 128                             # the second expert's first row
        at = torch.tensor([0, counts[0] - 1, first, first + counts[1] - 1], device="cuda")
        for rows in (1, 1 << 40):
            out = torch.zeros(mt * 128, n, device="cuda").bfloat16()
            ops.grouped_gemm(x, experts, buf.tile_expert, out, mt, ops.EPI_STORE, buf.tile_list, rows)
            close(out[at], *expected(x[at], q.dequant(torch.float64)))
            assert not out[first + counts[1]:].any() and not out[counts[0]:first].any()
    ops.check_kernel_status()


@pytest.mark.gpu
def test_calls_of_several_threads():
    """Threads that share weights, each on a stream of its own and all on one: every result is what the call alone gives."""
    import threading
    cases = [product_case(m, 512, 2048, FORMS[i]) for m, i in ((1, 0), (5, 2), (40, 5), (300, 3))]
    mixed = [expert_case([3, 0, 200, 40], 320, 576 // FORMS[i][3] * FORMS[i][3], FORMS[i], ops.EPI_STORE, seed=i) for i in (0, 5)]
    torch.cuda.synchronize()
    runs = [lambda c=c: ops.gemm_w4(c[0], c[1]) for c in cases]
    for c in mixed:
        for rows in (1, 1 << 40):
            runs.append(lambda c=c, rows=rows: ops.grouped_gemm(c[0], c[1], c[2].tile_expert, torch.full(c[4].shape, 3.0, device="cuda").bfloat16(),
                                                                c[3], ops.EPI_STORE, c[2].tile_list, rows))
    first = [f() for f in runs]
    torch.cuda.synchronize()
    for own in (False, True):
        wrong, shared = [], torch.cuda.Stream()

        def work(i):
            with torch.cuda.stream(torch.cuda.Stream() if own else shared):
                for _ in range(30):
                    y = runs[i]()
                    if not torch.equal(y, first[i]):
                        wrong.append(i)
        threads = [threading.Thread(target=work, args=(i,)) for i in range(len(runs))]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert not wrong, wrong
    ops.check_kernel_status()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 6, 40])
def test_rows_that_share_memory_or_have_odd_strides(m):
    x, w, r, want, room = product_case(m, 128, 384, FORMS[0], ops.EPI_RESIDUAL)
    one = x[:1].expand(m, -1)
    close(ops.gemm_w4(one, w, r, ops.EPI_RESIDUAL), *expected(one, w.dequant(torch.float64), r, ops.EPI_RESIDUAL))
    close(ops.gemm_w4(x, w, r[:1].expand(m, -1), ops.EPI_RESIDUAL), *expected(x, w.dequant(torch.float64), r[:1].expand(m, -1), ops.EPI_RESIDUAL))
    flat = torch.randn(384 + 5 * m, device="cuda").bfloat16()
    near = flat.as_strided((m, 384), (5, 1))                           # rows that begin five elements after one another
    close(ops.gemm_w4(near, w), *expected(near, w.dequant(torch.float64)))
    near = flat.as_strided((m, 384), (8 if m < 6 else 0, 1))
    close(ops.gemm_w4(near, w), *expected(near, w.dequant(torch.float64)))
    gain = torch.ones(384, device="cuda").bfloat16()
    a, b = ops.rmsnorm_fp8(near, gain, 1e-6), ops.rmsnorm_fp8(near.clone(), gain, 1e-6)
    assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and torch.equal(a[1], b[1])
