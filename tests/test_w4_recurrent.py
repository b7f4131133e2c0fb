"""Layers with a recurrent state (Gated DeltaNet, Mamba-2) whose projections are held in 4 bits, through the driver: chunked prompts and
decode steps against the dense fp32 forward over the same weights expanded."""
import numpy as np
import pytest
import torch

from pie_b200 import ops
from pie_b200.driver.executor import TorchDriver
from pie_b200.driver.schema import ForwardRequest, SamplerKind, SamplerSpec
from pie_b200.models.config import preset
from pie_b200.models.transformer import dense_reference_forward
from pie_b200.models.weights import dequantized, random_weights

from test_w4_model import cosine, to_cpu

RAW = SamplerSpec(SamplerKind.RAW_LOGITS)
NAMES = {"tiny-qwen3.5": ("w_gdn_in", "w_gdn_out"), "tiny-mamba2": ("w_mamba_in", "w_mamba_out")}


def run(drv, tokens, cuts):
    """Logits after each of the chunks that `cuts` make of one context's tokens."""
    i32 = lambda *a: np.asarray(a, dtype=np.int32)
    out = []
    for a, b in zip((0,) + cuts, cuts):
        req = ForwardRequest(tokens=np.asarray(tokens[a:b], np.int32), positions=np.arange(a, b, dtype=np.int32), qo_indptr=i32(0, b - a),
                             kv_page_indices=np.arange(-(-b // 16), dtype=np.int32), kv_page_indptr=i32(0, -(-b // 16)),
                             kv_last_page_lens=i32((b - 1) % 16 + 1), slot_req=i32(0), slot_row=i32(b - a - 1), slot_samplers=[RAW],
                             rs_slots=i32(1), rs_reset=i32(int(a == 0)))
        out.append(np.frombuffer(drv.fire_batch(req).slots[0].logits, dtype=np.float32).copy())
    return out


def build(name, device, dtype, **over):
    cfg = preset(name, dtype=dtype, **over)
    w = random_weights(cfg, device, torch.bfloat16 if dtype == "bfloat16" else torch.float32, seed=4)
    drv = TorchDriver(cfg, device, weights=w, num_pages=32, page_size=16, max_requests=4, max_tokens=128, weight_dtype="int4")
    held = [key for lw in w["layers"] for key, v in lw.items() if isinstance(v, ops.W4Linear)]
    assert set(NAMES[name]) <= set(held), held
    return cfg, w, drv


@pytest.mark.parametrize("name", NAMES)
def test_cpu_driver(name):
    cfg, w, drv = build(name, "cpu", "float32")
    tokens, cuts = list(range(60, 81)), (9, 20, 21)
    want = dense_reference_forward(cfg, to_cpu(dequantized(w)), torch.tensor(tokens)).numpy()
    for b, got in zip(cuts, run(drv, tokens, cuts)):
        assert np.abs(got - want[b - 1]).max() < 1e-4


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_driver(name):
    """Chunks of a few rows, of some ten and of some hundred, decode steps as graphs."""
    cfg, w, drv = build(name, "cuda", "bfloat16")
    tokens, cuts = list(range(60, 190)), (3, 23, 123, 124, 125, 126, 130)
    want = dense_reference_forward(cfg, to_cpu(dequantized(w)), torch.tensor(tokens)).numpy()
    for b, got in zip(cuts, run(drv, tokens, cuts)):
        assert cosine(got, want[b - 1]) > 0.995, (b, cosine(got, want[b - 1]))
    ops.check_kernel_status(drv.device)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("rows", [1, 7, 40, 130])
def test_projections(name, rows):
    """A layer's two products against their expanded weights, within what tests/test_w4_ops.py derives."""
    from test_w4_ops import close, expected
    cfg, w, drv = build(name, "cuda", "bfloat16")
    gen = torch.Generator("cuda").manual_seed(rows)
    for key in NAMES[name]:
        q = next(lw[key] for lw in w["layers"] if key in lw)
        x = torch.randn(rows, q.shape[1], generator=gen, device="cuda").bfloat16()
        close(drv.model._gemm(x, q), *expected(x, q.dequant(torch.float64)))
        r = torch.randn(rows, q.shape[0], generator=gen, device="cuda").bfloat16()
        close(drv.model._gemm(x, q, residual=r), *expected(x, q.dequant(torch.float64), r, ops.EPI_RESIDUAL))
    ops.check_kernel_status()
