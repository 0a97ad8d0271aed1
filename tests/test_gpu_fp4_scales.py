"""4-bit rows under row scales of any value, as other programs' rows have them: what the
rows stand for, and their products.
"""
import numpy as np
import pytest
import torch

import test_gpu_fp4 as P
from reflex_b200 import kernels as K

pytestmark = pytest.mark.gpu
BF, F32, MX, NV = P.BF, P.F32, P.MX, P.NV


def rounded(v, dtype):
    """The nearest number of the type, ties to even, of doubles (which a cast to bf16 would
    round twice, by way of fp32)."""
    if dtype == F32:
        with np.errstate(over="ignore"):
            return torch.from_numpy(v.astype(np.float32))
    _, e = np.frexp(v)
    step = np.ldexp(1.0, np.maximum(e - 8, -133))
    y = np.rint(v / step) * step
    return torch.from_numpy(np.where(np.abs(y) >= 2.0 ** 128, np.copysign(np.inf, y), y)).to(BF)


SCALES = [1 / 3, 0.1, 7e-5, -0.3, 1.9999999, 5.877472e-39, 1e-44, 3.3e37, -2.0 ** 127, 2.0 ** 127, 2.0 ** 119, 2.0 ** -126,
          1.1754942e-38, 3.4028235e38, 448.0, 0.0]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,Kc", [(64, 4304), (300, 1000), (16, 31), (700, 513), (48, 16384)])
def test_any_row_scale_is_rounded_once(dtype, T, Kc):
    """code x block scale x row scale with one rounding, for row scales that are no powers of two
    and those at the ends of fp32."""
    r = P.gen(T + Kc)
    out = P.quantized(r(T, Kc) * torch.exp(r(T, 1)), NV)
    scale = torch.from_numpy(np.exp(np.random.default_rng(T).uniform(-9, 9, T)).astype(np.float32))
    scale[:len(SCALES)] = torch.tensor(SCALES)[:T]
    out.row_scale.copy_(scale)
    y = torch.empty(T, Kc, dtype=dtype, device="cuda")
    K.dequant_fp4(x=out, out=y)
    P.done()
    want = rounded(P.values(out), dtype)
    assert torch.equal(y.cpu(), want), (int((y.cpu() != want).sum()), y.numel())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_every_product_near_a_tie_is_rounded_once(dtype):
    """All codes under all block scales, with row scales whose products lie at and one fp32 step
    beside the middle of two bf16 numbers."""
    middle = 1 + (np.arange(0, 128, 5) * 2 + 1) * 2.0 ** -8
    by = np.array([1.0, 3.0, 5.0, 7.0, 9.0, 11.0, 13.0, 15.0, 27.0, 33.0, 39.0, 45.0])  # (what codes times e4m3 numbers are)
    near = (middle[:, None] / by).astype(np.float32).ravel().view(np.uint32)
    scale = torch.from_numpy(np.concatenate([near - 1, near, near + 1]).view(np.float32).copy())
    T, Kc = len(scale), 16 * 127
    out = K.Fp4Rows.allocate(T, Kc, NV)
    k = torch.arange(Kc // 2)
    out.q.copy_((((2 * k) % 16) | (((2 * k + 1) % 16) << 4)).to(torch.uint8).expand(T, -1))
    out.row_scale.copy_(scale)
    t, j = np.arange(T), np.arange(128)
    at = ((t // 128)[:, None] * 32 + j // 4) * 512 + ((t % 128 % 32) * 16 + t % 128 // 32 * 4)[:, None] + j % 4
    byte = np.zeros(out.scale.numel(), np.uint8)
    byte[at.ravel()] = np.tile(np.where(j < 127, j, 0), T)
    out.scale.copy_(torch.from_numpy(byte))
    y = torch.empty(T, Kc, dtype=dtype, device="cuda")
    K.dequant_fp4(x=out, out=y)
    P.done()
    assert torch.equal(y.cpu(), rounded(P.values(out), dtype))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,Kc", [(1, 192), (50, 192), (128, 192), (129, 192), (300, 192), (60, 9000), (129, 9000)])
@pytest.mark.parametrize("epi", [P.STORE, P.GEGLU])
@pytest.mark.parametrize("ex,ew", [(74, 74), (-65, -65), (120, -90), (-90, 120), (110, -126), (-75, -60), (60, 60), (-126, 125)])
def test_row_scales_whose_product_leaves_fp32(ex, ew, T, Kc, epi, dtype):
    """x and w of such sizes (2^ex, 2^ew) that the product of two row scales, or of one and the
    sum, is beyond fp32 or below it: the outputs are the formula's all the same, sums of 0 (rows
    that share no places) are 0, and what is too large is infinite; in few tokens and in many, and
    where K is in parts."""
    O = 96
    r = P.gen(T + ex)
    x, w = r(T, Kc), r(O, Kc)
    x[::2, Kc // 2:] = 0
    w[::3, :Kc // 2] = 0
    xq = P.quantized(x.mul(2.0 ** ex) if ex > -120 else x, NV)
    wq = P.quantized(w.mul(2.0 ** ew) if ew > -120 else w, NV, 2 if epi == P.GEGLU else 1)
    for q, e in ((xq, ex), (wq, ew)):  # (smaller than the quantizer makes them)
        if e <= -120:
            q.row_scale.fill_(2.0 ** e)
    y = torch.empty(T, O // 2 if epi == P.GEGLU else O, dtype=dtype, device="cuda")
    K.linear_fp4(w=wq, x=xq, y=y, epilogue=epi)
    P.done()
    got = y.double().cpu().numpy()
    with np.errstate(over="ignore", invalid="ignore"):
        want, tol = P.ref_linear(P.values(xq), P.values(wq), None, P.STORE)
        sure = np.ones(want.shape, bool)
        if epi == P.GEGLU:  # (of gates and ups that are fp32 numbers: what infinities give is another test's)
            sure = (np.abs(want) < 1e37)[:, :O // 2] & (np.abs(want) < 1e37)[:, O // 2:]
            least = 2.0 ** -148 * (np.abs(want[:, :O // 2]) + np.abs(want[:, O // 2:]) + 1)
            want, tol = P.ref_linear(P.values(xq), P.values(wq), None, P.GEGLU)
            tol = tol + least
        top = float(torch.finfo(dtype).max)
        tol = tol + P.HALF[dtype] * (np.abs(want) + tol) + (2.0 ** -133 if dtype == BF else 2.0 ** -148)
        close = np.abs(got - want) <= tol
        over = (np.abs(want) >= top * (1 - 2.0 ** -7)) & (got == np.copysign(np.inf, want))
    bad = ~(close | over) & sure
    assert not bad.any(), (int(bad.sum()), bad.size, got[bad][:4], want[bad][:4], np.argwhere(bad)[:4].tolist())
    nothing = (P.values(xq) @ P.values(wq).T == 0) & sure if epi == P.STORE else np.zeros_like(sure)
    assert (got[nothing] == 0).all() and (epi == P.GEGLU or nothing.sum() >= (T + 1) // 2 * (O // 3))
