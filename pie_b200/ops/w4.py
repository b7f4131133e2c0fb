"""Weights in 4-bit codes with one 16-bit scale per row and group of columns, and the products that read them.

W[n, k] = scale[n, k // group] * v(codes[n, k]) with v(q) = q - 8 (`kind` "int4"), q - zero[n, k // group] (the same with zero points: GPTQ and
AWQ checkpoints) or the e2m1 number of q ("fp4": MXFP4 blocks, whose scales are powers of two). A weight is laid out once, when it is
made, in the order the kernels read (csrc/kernels/gemm_w4.cu has the layout).

Counterpart of the reference's W4A16 path (driver/cuda/src/kernels/dequant_wna16.cu).
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _lib, reference
from ._lib import check, fn, ptr, stream_ptr

W4_GROUPS = (32, 64, 128)
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


class _Weight(C.Structure):            # W4Weight of gemm_w4.cu
    _fields_ = [("codes", C.c_void_p), ("scale", C.c_void_p), ("zero", C.c_void_p), ("factor", C.c_void_p), ("experts", C.c_int),
                ("n", C.c_int), ("k", C.c_int), ("group", C.c_int), ("fp4", C.c_int)]


def _tiles(t: torch.Tensor, fill: int) -> torch.Tensor:
    """[E, N, G] -> [E, panels, G, 8, 8, 2]: per panel of 128 rows and group the row tiles' rows g beside their rows g + 8."""
    e, n, g = t.shape
    ps = -(-n // 128)
    if ps * 128 != n:
        pad = torch.full((e, ps * 128, g), fill, dtype=t.dtype, device=t.device)
        pad[:, :n] = t
        t = pad
    return t.view(e, ps, 8, 2, 8, g).permute(0, 1, 5, 2, 4, 3).contiguous()


class _OnGpu:
    """What a product needs of a weight on a GPU, looked up once."""

    __slots__ = ("weight", "n", "k", "pitch", "device", "rows", "status", "sms", "few", "many", "few_rows", "few_tiles", "all_tiles")

    def __init__(self, q):
        from . import ensure_pdl, kernel_status, num_sms
        ensure_pdl()
        self.weight, self.n, self.k, self.pitch = q._at, q.shape[-2], q.shape[-1], (q.shape[-1] + 63) // 64 * 64
        self.device = q.packed.get_device()
        self.status, self.sms = ptr(kernel_status(q.device)), num_sms(q.device)
        self.few, self.many = fn("pie_gemm_w4"), fn("pie_gemm_w4_tiles")
        self.few_rows, self.few_tiles, self.all_tiles = fn("pie_grouped_gemm_w4_rows"), fn("pie_grouped_gemm_w4_few"), fn("pie_grouped_gemm_w4")
        self.rows = fn("pie_gemm_w4_rows")(self.n, self.k, int(q.kind == "fp4"), self.sms)


class W4Linear:
    """Weight [N, K] in 4-bit codes. `codes` [N, K] uint8 (0..15), `scale` [N, K / group] bf16 or fp16, `zero` [N, K / group] uint8 (0..15,
    "int4" only; 8 without it), group = 32, 64 or 128. A scale is held exactly down to 2^-24 of its row's largest, with fewer bits below, and as zero
    below 2^-39 of it (e2m1: 2^-35). The tensors it holds are not to be changed: products read them while the kernel ahead of them in the
    stream is still running."""

    dims = 2

    def __init__(self, codes: torch.Tensor, scale: torch.Tensor, zero: Optional[torch.Tensor] = None, kind: str = "int4"):
        if kind not in ("int4", "fp4"):
            raise ValueError(f"4-bit weight: unknown kind {kind!r} (int4 | fp4)")
        if codes.dim() != self.dims or codes.dtype != torch.uint8:
            raise ValueError(f"4-bit weight: codes must be uint8 with {self.dims} dimensions, not {codes.dtype} {tuple(codes.shape)}")
        if scale.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"4-bit weight: scales must be bf16 or fp16, not {scale.dtype}")
        k, groups = codes.shape[-1], scale.shape[-1] if scale.dim() == self.dims else 0
        group = k // groups if groups and k % groups == 0 else 0
        if group not in W4_GROUPS or scale.shape[:-1] != codes.shape[:-1] or 0 in codes.shape[-2:]:
            raise ValueError(f"4-bit weight: scales {tuple(scale.shape)} do not give codes {tuple(codes.shape)} groups of 32, 64 or 128 columns")
        if zero is not None and (kind != "int4" or zero.dtype != torch.uint8 or zero.shape != scale.shape):
            raise ValueError("4-bit weight: zero points are uint8, one per scale, of integer codes")
        if any(t is not None and t.device != codes.device for t in (scale, zero)):
            raise ValueError("4-bit weight: codes, scales and zero points must be on one device")
        if not bool(torch.isfinite(scale).all()):
            raise ValueError("4-bit weight: scales must be finite")
        for name, t in (("codes", codes), ("zero points", zero)):
            if t is not None and t.numel() and int(t.max()) > 15:
                raise ValueError(f"4-bit weight: {name} above 15")
        e = codes.shape[0] if self.dims == 3 else 1
        n = codes.shape[-2]
        c, s, z = codes.reshape(e, n, k), scale.reshape(e, n, groups), zero.reshape(e, n, groups) if zero is not None else None
        ps, kb = -(-n // 128), -(-k // 64)
        if ps * 128 != n or kb * 64 != k:
            pad = torch.full((e, ps * 128, kb * 64), 0 if kind == "fp4" else 8, dtype=torch.uint8, device=c.device)
            pad[:, :n, :k] = c
            c = pad
        padded = kb * 64 // group if group < 128 else groups
        if padded != groups:
            more = lambda t, v: torch.cat([t, torch.full((e, n, padded - groups), v, dtype=t.dtype, device=t.device)], -1)
            s, z = more(s, 0), more(z, 8) if z is not None else None
        # [e, panel, row tile, half, row, block, j / 2, t, j % 2, pair, which] -> bytes [e, panel, block, row tile, row, t, j, which, half] of two
        # nibbles (pairs), or for e2m1 [.., half, pair] (which)
        c = c.view(e, ps, 8, 2, 8, kb, 2, 4, 2, 2, 2).permute(0, 1, 5, 2, 4, 7, 6, 8, *((3, 9, 10) if kind == "fp4" else (10, 3, 9)))
        packed = (c[..., 0] | (c[..., 1] << 4)).contiguous().view(e, ps, kb, 8, 512)
        # scales in fp16 times a power of two per row that brings the largest to [2^14, 2^15) (integers), [2^10, 2^11) (e2m1)
        s = s.double()
        top = s.abs().amax(-1)
        shift = torch.where(top > 0, (11 if kind == "fp4" else 15) - torch.frexp(top.clamp_min(2.0 ** -200)).exponent, 0)
        factor = torch.zeros(e, ps * 128, dtype=torch.float32, device=c.device)
        factor[:, :n] = torch.exp2(-shift.double())
        s = (s * torch.exp2(shift.double())[..., None]).half()
        if kind == "int4" and z is None and bool(((s != 0) & (s.abs() < 512)).any()):
            # scales of one row far apart: the kernels' way for zero points has the range
            z = torch.full(s.shape, 8, dtype=torch.uint8, device=s.device)
        self._hold(packed, _tiles(s, 0), _tiles(z, 8) if z is not None else None, factor, tuple(codes.shape), group, kind)

    @classmethod
    def from_packed(cls, packed, scale, zero, factor, shape, group: int, kind: str):
        """A weight whose tensors are laid out already (`packed`, `scale`, `zero` and `factor` of another one)."""
        shape = tuple(shape)
        if kind not in ("int4", "fp4") or group not in W4_GROUPS or len(shape) != cls.dims or min(shape[-2:]) < 1 or shape[-1] % group:
            raise ValueError(f"4-bit weight: no layout for {kind} codes {shape} in groups of {group}")
        e, ps, kb = shape[0] if cls.dims == 3 else 1, -(-shape[-2] // 128), -(-shape[-1] // 64)
        groups = shape[-1] // group if group == 128 else kb * 64 // group
        for name, t, dtype, dims in (("packed", packed, torch.uint8, (e, ps, kb, 8, 512)), ("scale", scale, torch.float16, (e, ps, groups, 8, 8, 2)),
                                     ("zero", zero, torch.uint8, (e, ps, groups, 8, 8, 2)), ("factor", factor, torch.float32, (e, ps * 128))):
            if t is None and name == "zero":
                continue
            if t.dtype != dtype or tuple(t.shape) != dims or not t.is_contiguous() or t.data_ptr() % 16 or t.device != packed.device:
                raise ValueError(f"4-bit weight: {name} must be {dtype} {dims}, dense and on the codes' device, not {t.dtype} {tuple(t.shape)}")
        if zero is not None and kind != "int4":
            raise ValueError("4-bit weight: zero points are of integer codes")
        q = cls.__new__(cls)
        q._hold(packed, scale, zero, factor, tuple(shape), group, kind)
        return q

    def _hold(self, packed, scale, zero, factor, shape, group, kind, written: bool = False):
        """`written`: what wrote the tensors is done."""
        self.packed, self.scale, self.zero, self.factor = packed, scale, zero, factor
        self.shape, self.group, self.kind = torch.Size(shape), group, kind
        e = shape[0] if self.dims == 3 else 1
        self._struct = _Weight(ptr(packed), ptr(scale), ptr(zero), ptr(factor), e, shape[-2], shape[-1], group, int(kind == "fp4"))
        self._at = C.addressof(self._struct)
        self._gpu = None
        if packed.is_cuda:
            # the products request weights before the kernel ahead of them in the stream is done
            if not written:
                torch.cuda.synchronize(packed.device)
            self._gpu = _OnGpu(self)

    @property
    def device(self):
        return self.packed.device

    @property
    def is_cuda(self):
        return self.packed.is_cuda

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.packed, self.scale, self.zero, self.factor) if t is not None)

    def to(self, device):
        move = lambda t: t.to(device) if t is not None else None
        return type(self).from_packed(move(self.packed), move(self.scale), move(self.zero), move(self.factor), self.shape, self.group, self.kind)

    def float(self) -> torch.Tensor:
        return self.dequant(torch.float32)

    def dequant(self, dtype=torch.bfloat16) -> torch.Tensor:
        """The weight in `dtype`, each value rounded once. `gemm` over it right away wants `fresh_w=True`, as over any weight just written."""
        if not self.is_cuda or dtype != torch.bfloat16:
            return self._plain(dtype)
        out = torch.empty(self.shape, dtype=torch.bfloat16, device=self.device)
        with torch.cuda.device(self.device):
            check(fn("pie_w4_expand")(self._at, ptr(out), stream_ptr()), "w4_expand")
        return out

    def _plain(self, dtype) -> torch.Tensor:
        e, ps, kb, _, _ = self.packed.shape
        n, k = self.shape[-2], self.shape[-1]
        b = self.packed.view(e, ps, kb, 8, 8, 4, 2, 2, 2, 2)              # row tile, row, t, j / 2, j % 2, then which, half (e2m1: half, pair)
        c = torch.stack([b & 15, b >> 4], dim=-1)                        # pair (e2m1: which)
        order = (0, 1, 3, 8, 4, 2, 6, 5, 7, 9, 10) if self.kind == "fp4" else (0, 1, 3, 9, 4, 2, 6, 5, 7, 10, 8)
        c = c.permute(*order).reshape(e, ps * 128, kb * 64)
        flat = lambda t: t.permute(0, 1, 3, 5, 4, 2).reshape(e, ps * 128, -1).repeat_interleave(self.group, dim=-1)
        if self.kind == "fp4":
            v = torch.tensor(E2M1, device=self.device)[c.int()]
        else:
            v = c.float() - (flat(self.zero).float() if self.zero is not None else 8.0)
        v = v.double() * flat(self.scale).double() * self.factor.double()[..., None]
        return v[:, :n, :k].reshape(self.shape).to(dtype)


class W4Experts(W4Linear):
    """Weights [E, N, K] of E experts in 4-bit codes (see `W4Linear`), for `grouped_gemm`."""

    dims = 3

    def is_contiguous(self) -> bool:
        return True

    def __getitem__(self, e: int) -> W4Linear:
        """Expert e's weight, in the same memory: no wait, and usable while a graph is captured."""
        if not -self.shape[0] <= e < self.shape[0]:
            raise IndexError(f"expert {e} of {self.shape[0]}")
        part = lambda t: t[e % self.shape[0]][None] if t is not None else None
        q = W4Linear.__new__(W4Linear)
        q._hold(part(self.packed), part(self.scale), part(self.zero), part(self.factor), self.shape[1:], self.group, self.kind, written=True)
        return q


def quantize_w4(w: torch.Tensor, group: int = 128, kind: str = "int4", asymmetric: bool = False, scale_dtype=torch.bfloat16):
    """Round-to-nearest quantisation of a weight [N, K] (`W4Linear`) or [E, N, K] (`W4Experts`). "int4": scale = absmax / 7.5 per group,
    or (max - min) / 15 with a zero point where `asymmetric`; "fp4": the power of two that brings the group's absmax into e2m1's range,
    which gives MXFP4 weights that were expanded back exactly. A group whose scale is zero (in `scale_dtype`) has weights of zero."""
    if group not in W4_GROUPS or w.shape[-1] % group:
        raise ValueError(f"4-bit weight: {w.shape[-1]} columns are no multiple of a group of {group} (32, 64 or 128)")
    cls = W4Experts if w.dim() == 3 else W4Linear
    g = w.float().reshape(*w.shape[:-1], w.shape[-1] // group, group)
    amax = g.abs().amax(-1)
    if kind not in ("int4", "fp4") or (asymmetric and kind == "fp4"):
        raise ValueError(f"4-bit weight: no {'asymmetric ' if asymmetric else ''}quantisation to {kind!r}")
    if kind == "fp4":
        s = torch.exp2(torch.ceil(torch.log2(amax.clamp_min(2.0 ** -100) / 6.0))).to(scale_dtype)
        a = (g / s.float()[..., None]).abs()
        q = torch.zeros_like(a, dtype=torch.uint8)
        for i, (lo, hi) in enumerate(zip(E2M1[:7], E2M1[1:8])):           # a tie goes to the even code
            q += (a > (lo + hi) / 2 if i % 2 == 0 else a >= (lo + hi) / 2).to(torch.uint8)
        return cls((q + (g < 0).to(torch.uint8) * 8).view(w.shape), s, kind="fp4")
    lo, hi = (g.amin(-1).clamp_max(0.0), g.amax(-1).clamp_min(0.0)) if asymmetric else (-amax, amax)
    s = ((hi - lo) / 15).to(scale_dtype)
    d = torch.where(s > 0, s.float(), 1.0)
    z = torch.round(-lo / d).clamp(0, 15) if asymmetric else torch.full_like(d, 8)
    q = (torch.round(g / d[..., None]) + z[..., None]).clamp(0, 15).to(torch.uint8).view(w.shape)
    return cls(q, s, zero=z.to(torch.uint8) if asymmetric else None)


def _check_product(x, q, residual, epilogue, out):
    from . import EPI_GEGLU, EPI_RESIDUAL, EPI_STORE, EPI_SWIGLU
    if type(q) is not W4Linear:
        raise TypeError(f"gemm_w4: the weight must be a W4Linear, not {type(q).__name__}")
    n, k = q.shape
    if epilogue not in (EPI_STORE, EPI_RESIDUAL, EPI_SWIGLU, EPI_GEGLU):
        raise ValueError(f"gemm_w4: unknown epilogue {epilogue}")
    glu = epilogue in (EPI_SWIGLU, EPI_GEGLU)
    if x.dim() != 2 or x.shape[1] != k:
        raise ValueError(f"gemm_w4: rows {tuple(x.shape)} do not fit a weight of {n} x {k}")
    if (residual is not None) != (epilogue == EPI_RESIDUAL):
        raise ValueError("gemm_w4: a residual comes with EPI_RESIDUAL and with nothing else")
    cols = n // 2 if glu else n
    if residual is not None and tuple(residual.shape) != (x.shape[0], n):
        raise ValueError(f"gemm_w4: residual {tuple(residual.shape)} for outputs of {x.shape[0]} x {n}")
    if out is not None and tuple(out.shape) != (x.shape[0], cols):
        raise ValueError(f"gemm_w4: out {tuple(out.shape)} for outputs of {x.shape[0]} x {cols}")
    if glu and n % 2:
        raise ValueError("gemm_w4: gate and up rows come in pairs")
    if any(t is not None and t.device != q.device for t in (x, residual, out)):
        raise ValueError("gemm_w4: rows, weight, residual and output must be on one device")
    return cols


def _rows16(t):
    """t with rows that 16-byte loads can walk, copied if need be."""
    fits = t.stride(1) == 1 and t.stride(0) % 8 == 0 and t.stride(0) < 2 ** 31 and t.data_ptr() % 16 == 0
    return t if fits else t.clone(memory_format=torch.contiguous_format)


def _apart(t, out, same: bool):
    """t, or a copy of it where `out` shares its memory (`same`: unless they are the same elements)."""
    if t is None or out is None or t.untyped_storage().data_ptr() != out.untyped_storage().data_ptr():
        return t
    return t if same and t.data_ptr() == out.data_ptr() and t.stride() == out.stride() else t.clone(memory_format=torch.contiguous_format)


def gemm_w4(x, q: W4Linear, residual=None, epilogue: int = 0, out=None):
    """y = x @ W.T for a weight in 4-bit codes, with the epilogues of `gemm`: EPI_STORE, EPI_RESIDUAL (+ residual), EPI_SWIGLU / EPI_GEGLU over
    interleaved gate / up rows. x [M, K] bf16 (up to 2^100), any strides; y [M, N] or [M, N / 2] bf16, sums in 32 bits. On the GPU N is a
    multiple of 8 (32 for the GLUs). `out` may be the residual, or share memory with the rows."""
    at = q._gpu if type(q) is W4Linear else None
    # the common call, checked in one go: a product takes less time than a careful look at its arguments
    if at is not None and out is None and x.dtype is torch.bfloat16 and x.dim() == 2 and x.get_device() == at.device == torch._C._cuda_getDevice():
        m, k = x.shape
        ldx, last = x.stride()
        xp = x.data_ptr()
        glu = epilogue == 2 or epilogue == 7
        if k == at.k and m > 0 and last == 1 and not (ldx & 7 or ldx >> 31 or xp & 15 or at.n & (31 if glu else 7)):
            if epilogue == 1:
                ok = residual is not None and residual.dtype is torch.bfloat16 and residual.shape == (m, at.n) and residual.get_device() == at.device
                if ok:
                    ldr, last = residual.stride()
                    rp = residual.data_ptr()
                    ok = last == 1 and not (ldr & 7 or ldr >> 31 or rp & 15)
            else:
                ok, rp, ldr = residual is None and (epilogue == 0 or glu), 0, 0
            if ok:
                cols = at.n >> 1 if glu else at.n
                y = x.new_empty((m, cols))
                _product(at, m, xp, ldx, y.data_ptr(), cols, rp, ldr, epilogue, x)
                return y
    return _gemm_w4(x, q, residual, epilogue, out)


def _product(at, m, xp, ldx, yp, ldy, rp, ldr, epilogue, x):
    if m <= at.rows:
        check(at.few(at.weight, xp, ldx, yp, ldy, rp, ldr, m, epilogue, at.status, at.sms, stream_ptr()), "gemm_w4")
    else:
        scratch = x.new_empty(m * at.pitch + 2 * m + 8)               # the rows in fp16, their factors in 32 bits
        p = scratch.data_ptr()
        check(at.many(at.weight, xp, ldx, p, p + 2 * m * at.pitch, yp, ldy, rp, ldr, m, epilogue, at.status, at.sms, stream_ptr()), "gemm_w4")


def _gemm_w4(x, q, residual, epilogue, out):
    from . import EPI_GEGLU, EPI_RESIDUAL, EPI_SWIGLU
    cols = _check_product(x, q, residual, epilogue, out)
    if not x.is_cuda:
        y = reference.gemm(x, q.dequant(torch.float32), residual if epilogue == EPI_RESIDUAL else None)
        y = reference.swiglu_interleaved(y) if epilogue == EPI_SWIGLU else reference.glu_interleaved(y, "gelu_tanh") if epilogue == EPI_GEGLU else y
        return y if out is None else out.copy_(y)
    if any(t is not None and t.dtype != torch.bfloat16 for t in (x, residual, out)):
        raise ValueError("gemm_w4: rows, residual and output are bf16 on the GPU")
    m, n = x.shape[0], q.shape[0]
    if n % (32 if cols != n else 8):
        raise ValueError(f"gemm_w4: {n} weight rows are no multiple of {32 if cols != n else 8}")
    if x.get_device() != torch.cuda.current_device():
        with torch.cuda.device(x.device):
            return _gemm_w4(x, q, residual, epilogue, out)
    if m == 0:
        return out if out is not None else x.new_empty(0, cols)
    x = _rows16(_apart(x, out, False))
    residual = _rows16(_apart(residual, out, True)) if residual is not None else None
    y = out if out is not None and out.stride(0) >= cols and _rows16(out) is out else x.new_empty(m, cols)
    _product(q._gpu, m, ptr(x), x.stride(0), ptr(y), y.stride(0), ptr(residual), residual.stride(0) if residual is not None else 0, epilogue, x)
    return y if out is None or y is out else out.copy_(y)


def _tile_rows(t, rows: int, width: int, device: int):
    """(address, row stride) of bf16 rows [rows or more, width] that the kernels can walk, or None."""
    if t.dtype is not torch.bfloat16 or t.dim() != 2 or t.get_device() != device:
        return None
    m, k = t.shape
    ld, last = t.stride()
    p = t.data_ptr()
    return (p, ld) if k == width and m >= rows and last == 1 and width <= ld < 2 ** 31 and not (ld & 7 or p & 15) else None


def _table(t, least: int, device: int):
    """Address of an int32 table with so many entries, or None."""
    return t.data_ptr() if t.dtype is torch.int32 and t.get_device() == device and t.is_contiguous() and t.numel() >= least else None


def grouped_gemm_w4(a, q: W4Experts, tile_expert, out, max_mtiles: int, epilogue: int = 0, tile_list=None, rows_in_use=None):
    """`grouped_gemm` for experts in 4-bit codes: out[tile rows] = a[tile rows] @ W[tile_expert[tile]].T, EPI_STORE or EPI_SWIGLU."""
    at = q._gpu if type(q) is W4Experts else None
    if at is not None and at.device == torch._C._cuda_getDevice() and (epilogue == 0 or epilogue == 2) and max_mtiles > 0 and q.shape[0]:
        # the common call, checked in one go
        rows, n = max_mtiles * 128, at.n
        ap = _tile_rows(a, rows, at.k, at.device)
        yp = _tile_rows(out, rows, n >> 1 if epilogue else n, at.device)
        te = _table(tile_expert, max_mtiles, at.device)
        tl = None if tile_list is None else _table(tile_list, 1 + max_mtiles, at.device)
        if ap and yp and te and (tl or tile_list is None) and not n & (31 if epilogue else 7):
            e = q.shape[0]
            if rows_in_use is None:            # as many as `moe_max_mtiles` makes room for
                rows_in_use = (max_mtiles - e) * 128 if max_mtiles > e else rows
            if tl and at.few_rows(e, at.k, min(rows_in_use, rows)):
                check(at.few_tiles(at.weight, *ap, *yp, te, tl, max_mtiles, epilogue, at.status, at.sms, stream_ptr()), "grouped_gemm_w4")
                return out
            # the rows in fp16, their factors in 32 bits, the list of items; held until both launches are made: the call lets other threads
            # run, which may be given what is free
            scratch = a.new_empty(rows * at.pitch + 2 * rows + 8 + 64 * max_mtiles)
            p = scratch.data_ptr()
            back = p + 2 * rows * at.pitch
            check(at.all_tiles(at.weight, *ap, p, back, back + 4 * rows, *yp, te, tl, max_mtiles, epilogue, at.status, at.sms, stream_ptr()),
                  "grouped_gemm_w4")
            return out
    return _grouped_gemm_w4(a, q, tile_expert, out, max_mtiles, epilogue, tile_list, rows_in_use)


def _grouped_gemm_w4(a, q, tile_expert, out, max_mtiles, epilogue, tile_list, rows_in_use):
    """Why a call is not the common one: an error, another device, nothing to do."""
    from . import EPI_STORE, EPI_SWIGLU, MOE_TILE
    if type(q) is not W4Experts:
        raise TypeError(f"grouped_gemm_w4: the weights must be W4Experts, not {type(q).__name__}")
    e, n, k = q.shape
    if epilogue not in (EPI_STORE, EPI_SWIGLU):
        raise ValueError(f"grouped_gemm_w4: unknown epilogue {epilogue}")
    if any(t is not None and (t.device != a.device or not t.is_cuda) for t in (q, out, tile_expert, tile_list)):
        raise ValueError("grouped_gemm_w4: rows, weights, output and tiles must be on one GPU")
    rows, device = max_mtiles * MOE_TILE, a.get_device()
    for name, t, width in (("rows", a, k), ("out", out, n // 2 if epilogue == EPI_SWIGLU else n)):
        if _tile_rows(t, rows, width, device) is None:
            raise ValueError(f"grouped_gemm_w4: {name} must be bf16 [{rows} or more, {width}] with dense rows on 16-byte boundaries, "
                             f"not {t.dtype} {tuple(t.shape)}")
    for name, t, least in (("tile_expert", tile_expert, max_mtiles), ("tile_list", tile_list, 1 + max_mtiles)):
        if t is not None and _table(t, least, device) is None:
            raise ValueError(f"grouped_gemm_w4: {name} must be int32 with {least} entries or more")
    if n % (32 if epilogue == EPI_SWIGLU else 8):
        raise ValueError(f"grouped_gemm_w4: {n} weight rows are no multiple of {32 if epilogue == EPI_SWIGLU else 8}")
    if max_mtiles <= 0 or e == 0:
        return out
    with torch.cuda.device(a.device):
        return grouped_gemm_w4(a, q, tile_expert, out, max_mtiles, epilogue, tile_list, rows_in_use)
