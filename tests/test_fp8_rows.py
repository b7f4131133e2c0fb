"""Block-scaled fp8 products over rows that come in 8 bits: what they refuse, and residuals of any layout."""
import pytest
import torch

from pie_b200 import ops

from test_w4_ops import close, expected


def case(m, n, k, device):
    gen = torch.Generator().manual_seed(m + n + k)
    q = ops.quantize_fp8_block((torch.randn(n, k, generator=gen) * 0.03).to(device))
    rows = ops.rmsnorm_fp8(torch.randn(m, k, generator=gen).to(device, torch.bfloat16 if device == "cuda" else torch.float32),
                           torch.ones(k, device=device, dtype=torch.bfloat16 if device == "cuda" else torch.float32), 1e-6)
    return q, rows, torch.randn(m, n, generator=gen).to(device, torch.bfloat16)


def refused(q, rows, r):
    x8, sx = rows
    return (lambda: ops.gemm_fp8w(rows, q, epilogue=ops.EPI_RESIDUAL), lambda: ops.gemm_fp8w(rows, q, residual=r),
            lambda: ops.gemm_fp8w(rows, q, residual=r[:2], epilogue=ops.EPI_RESIDUAL),
            lambda: ops.gemm_fp8w(rows, q, residual=r[:, :16], epilogue=ops.EPI_RESIDUAL),
            lambda: ops.gemm_fp8w(rows, q, epilogue=ops.EPI_GEGLU), lambda: ops.gemm_fp8w(rows, q, epilogue=99))


def test_refused():
    q, rows, r = case(3, 32, 128, "cpu")
    ops.gemm_fp8w(rows, q, residual=r, epilogue=ops.EPI_RESIDUAL)
    for bad in refused(q, rows, r):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(3, 32, 128), (40, 512, 1024), (200, 256, 512)])
def test_refused_on_the_gpu_and_residuals_of_any_layout(m, n, k):
    q, rows, r = case(m, n, k, "cuda")
    other = ops.Fp8Linear(q.w8.cpu(), q.scale.cpu())
    for bad in refused(q, rows, r) + (lambda: ops.gemm_fp8w(rows, other), lambda: ops.gemm_fp8w(rows, q, residual=r.cpu(), epilogue=ops.EPI_RESIDUAL),
                                      lambda: ops.gemm_fp8w(rows, q, residual=r.float(), epilogue=ops.EPI_RESIDUAL)):
        with pytest.raises(ValueError):
            bad()
    x64, w64 = (a.double() * s.double().repeat_interleave(128, -1)[:, :a.shape[1]] for a, s in (rows, (q.w8, q.scale)))
    want, room = expected(x64, w64, r, ops.EPI_RESIDUAL)
    wide = torch.zeros(2 * m, n + 24, device="cuda").bfloat16()
    for at in (wide[:m, 8:8 + n], wide[:m, 3:3 + n], wide[::2, 16:16 + n], wide.new_zeros(n, m).t()):
        at.copy_(r)
        close(ops.gemm_fp8w(rows, q, residual=at, epilogue=ops.EPI_RESIDUAL), want, room)
    assert ops.gemm_fp8w((rows[0][:0], rows[1][:0]), q).shape == (0, n)
    ops.check_kernel_status()


@pytest.mark.parametrize("k,rows8", [(4096, True), (16384, True), (16400, False)])
def test_norms_of_rows_that_are_too_long_for_8_bits_stay_in_bf16(monkeypatch, k, rows8):
    """A model's choice between its two norms, by the sizes that each of them takes."""
    from types import SimpleNamespace

    from pie_b200.models.transformer import Transformer
    said = []
    monkeypatch.setattr(ops, "rmsnorm_fp8", lambda h, w, eps: said.append(8))
    monkeypatch.setattr(ops, "rmsnorm", lambda h, w, eps: said.append(16))
    model = SimpleNamespace(fp8_norm=True, gemm_backend="tcgen05", cfg=SimpleNamespace(rms_norm_eps=1e-6))
    h = SimpleNamespace(is_cuda=True, dtype=torch.bfloat16, shape=(5, k))
    q = ops.Fp8Linear(torch.zeros(16, k).to(torch.float8_e4m3fn), torch.ones(16, -(-k // 128)))
    Transformer._norm_rows(model, h, None, q)
    assert said == [8 if rows8 else 16]
