"""The 4-bit layer operators on the GPU against plain restatements: rows bit for
bit, products in 64 bits.

Tolerances count roundings: u = 2^-24 is half a step of fp32 (2^-8 of bf16).
"""
import numpy as np
import pytest
import torch

from reflex_b200 import _lib as L
from reflex_b200 import kernels as K

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24
BF, F32 = torch.bfloat16, torch.float32
HALF = {BF: 2.0 ** -8, F32: U32}
MX, NV = L.RFX_FP4_MX, L.RFX_FP4_NV
BLOCK = {MX: 32, NV: 16}
E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E4M3 = np.concatenate([np.arange(8) * 2.0 ** -9] + [(8 + np.arange(8)) * 2.0 ** (e - 3) for e in range(-6, 9)])[:127]


def gen(seed):
    g = torch.Generator().manual_seed(seed)
    return lambda *shape, std=1.0: torch.randn(*shape, generator=g) * std


def done():
    torch.cuda.synchronize()
    assert K.device_status() == 0


def nearest(a, grid):
    """Place of the nearest of the ascending numbers `grid` (ties to the even place)."""
    hi = np.clip(np.searchsorted(grid, a), 1, len(grid) - 1)
    up, down = grid[hi] - a, a - grid[hi - 1]
    return np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, hi - 1)


def ref_quant(x, fmt):
    """(codes [T, K], scale bytes [T, blocks], row scales): fp32 numpy, IEEE division."""
    x = x.float().cpu().numpy()
    T, n = x.shape
    b = np.pad(x, ((0, 0), (0, -n % BLOCK[fmt]))).reshape(T, -1, BLOCK[fmt])
    most = np.abs(b).max(axis=2)
    if fmt == MX:
        _, e = np.frexp(most)
        byte = np.where(most > 0, np.maximum(e - 1 - 2, -127), -127) + 127
        step = np.ldexp(np.float64(1), byte - 127)
        row = None
    else:
        _, e = np.frexp(most.max(axis=1))
        row = np.ldexp(np.float32(1), np.maximum(np.where(most.max(axis=1) > 0, e - 1 - 10, -100), -100)).astype(np.float32)
        ratio = ((most / np.float32(6)).astype(np.float32) / row[:, None]).astype(np.float32)
        byte = nearest(ratio.astype(np.float64), E4M3)
        step = E4M3[byte] * row[:, None]
    with np.errstate(divide="ignore", invalid="ignore"):
        y = (b / step[:, :, None].astype(np.float32 if fmt == NV else np.float64)).astype(np.float32)
    y = np.where(step[:, :, None] > 0, y, 0).astype(np.float64)
    code = nearest(np.minimum(np.abs(y), 6.0), E2M1) + 8 * np.signbit(y)
    return code.reshape(T, -1)[:, :n], byte.astype(np.uint8), row


def unpack(r):
    """(codes [T, K], scale bytes [T, blocks]) of Fp4Rows, byte by byte."""
    q, s = r.q.cpu().numpy(), r.scale.cpu().numpy().reshape(-1)
    T = q.shape[0]
    k = np.arange(r.K)
    code = (q[:, k // 2] >> (4 * (k % 2)).astype(np.uint8)) & 15
    if r.K % 2:
        assert (q[:, -1] >> 4 == 0).all()
    n = -(-r.K // BLOCK[r.fmt])
    kt = -(-n // 4)
    per = T // r.parts
    t, j = np.arange(T), np.arange(kt * 4)
    tile = (t // per) * -(-per // 128) + (t % per) // 128
    u = t % per % 128
    at = (tile[:, None] * kt + j // 4) * 512 + ((u % 32) * 16 + u // 32 * 4)[:, None] + j % 4
    byte = s[at]
    return code, byte[:, :n], byte[:, n:]


def values(r):
    """What Fp4Rows stand for, in 64 bits."""
    code, byte, _ = unpack(r)
    scale = np.ldexp(1.0, byte.astype(np.int64) - 127) if r.fmt == MX else E4M3[np.minimum(byte, 126)]
    v = np.where(code > 7, -1.0, 1.0) * E2M1[code & 7] * np.repeat(scale, BLOCK[r.fmt], axis=1)[:, :r.K]
    return v if r.row_scale is None else v * r.row_scale.double().cpu().numpy()[:, None]


def framed(T, Kc, dtype, ld, fill):
    """A [T, Kc] view with row stride ld inside a buffer filled with `fill`,
    and a check that nothing but the view was written."""
    buf = torch.full((T + 2, ld), fill, dtype=dtype, device="cuda")
    view = buf[1:T + 1, :Kc]

    def untouched():
        assert (buf[0] == fill).all() and (buf[T + 1] == fill).all() and (buf[1:T + 1, Kc:] == fill).all()
    return view, untouched


def rows_for(T, Kc, fmt, parts=1, fill=0xA5):
    """Fp4Rows whose memory holds `fill` everywhere, and a check of what lies around the rows."""
    r = K.Fp4Rows.allocate(T, Kc, fmt, parts)
    view, clean = framed(T, (Kc + 1) // 2, torch.uint8, -(-Kc // 32) * 16 + 16, fill)
    r.scale.fill_(fill)
    return K.Fp4Rows(view, r.scale, r.row_scale, Kc, fmt, parts), clean


def quantized(x, fmt, parts=1):
    r = K.Fp4Rows.allocate(x.shape[0], x.shape[1], fmt, parts)
    K.quant_fp4(x=x.cuda(), out=r)
    return r


# -------------------------------------------------------- quant, dequant ---
LENGTHS = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 128, 513, 1024, 1025, 2047, 2048, 2056, 4304, 8192, 16384]


@pytest.mark.parametrize("fmt", [MX, NV])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("Kc", LENGTHS)
def test_quant_is_exact(fmt, dtype, Kc):
    """Bit for bit the fp32 formula at any length, for rows of very different
    sizes with small blocks among them; nothing outside the rows is written, and
    a row's last scale group is filled up with zeros."""
    T = 3 if Kc > 3000 else 131
    r = gen(Kc + fmt)
    x = (r(T, Kc) * torch.exp(3 * r(T, 1)) * torch.exp2(torch.randint(-12, 3, (1, Kc), generator=torch.Generator().manual_seed(Kc)).float())).to(dtype)
    x[0, 0] = 0.0
    out, clean = rows_for(T, Kc, fmt)
    K.quant_fp4(x=x.cuda(), out=out)
    y = torch.full((T, Kc), -1.0, dtype=dtype, device="cuda")
    K.dequant_fp4(x=out, out=y)
    done()
    code, byte, row = ref_quant(x, fmt)
    got_code, got_byte, rest = unpack(out)
    if row is not None:
        assert np.array_equal(out.row_scale.cpu().numpy(), row)
    assert np.array_equal(got_byte, byte)
    assert (rest == 0).all()
    assert np.array_equal(got_code & 7, code & 7)
    assert np.array_equal(got_code[got_code & 7 > 0] >> 3, code[code & 7 > 0] >> 3)
    clean()
    want = torch.from_numpy(values(out)).to(dtype)
    assert torch.equal(y.cpu(), want)


@pytest.mark.parametrize("fmt", [MX, NV])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,Kc,pad,off", [(5, 200, 3, 0), (600, 70, 0, 1), (300, 600, 2, 1), (2, 4099, 8, 0), (700, 2048, 0, 0),
                                          (300, 8000, 16, 0), (2, 16385, 0, 0), (3, 40000, 8, 0), (2, 65536, 0, 1)])
def test_quant_of_any_rows(fmt, dtype, T, Kc, pad, off):
    """Rows off the 16-byte boundaries, of any stride, many of them, and rows too
    long for a CTA's registers."""
    x = gen(T + Kc)(T, Kc).to(dtype)
    buf = torch.full((T * (Kc + pad) + off + 8,), 1e30, dtype=dtype, device="cuda")
    xv = buf[off:off + T * (Kc + pad)].view(T, Kc + pad)[:, :Kc]
    xv.copy_(x)
    out, clean = rows_for(T, Kc, fmt)
    K.quant_fp4(x=xv, out=out)
    yb, y_clean = framed(T, Kc, dtype, Kc + pad + off, 7.0)
    K.dequant_fp4(x=out, out=yb)
    done()
    code, byte, row = ref_quant(x, fmt)
    got_code, got_byte, rest = unpack(out)
    assert np.array_equal(got_byte, byte) and (rest == 0).all()
    assert np.array_equal(got_code & 7, code & 7)
    clean()
    y_clean()
    assert torch.equal(yb.cpu(), torch.from_numpy(values(out)).to(dtype))


@pytest.mark.parametrize("fmt", [MX, NV])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_quant_special_rows(fmt, dtype):
    """Zeros, ties, the smallest and largest numbers; an infinity or a NaN makes
    its block (NV: its row) NaN and no other."""
    Kc = 96
    x = torch.zeros(8, Kc)
    x[1] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 12)  # ties, on a scale of 1 (MX)
    x[2] = -x[1] * 4
    x[3] = 1e-39
    x[4, 5] = 1e-45
    x[5] = 3e38
    x[6] = 1.0
    x[6, 40] = float("inf")
    x[7] = 1.0
    x[7, 95] = float("nan")
    x = x.to(dtype)
    out = quantized(x, fmt)
    y = torch.empty(8, Kc, dtype=dtype, device="cuda")
    K.dequant_fp4(x=out, out=y)
    done()
    code, byte, row = ref_quant(x[:6], fmt)
    got_code, got_byte, _ = unpack(out)
    assert np.array_equal(got_byte[:6], byte) and np.array_equal(got_code[:6] & 7, code & 7)
    assert torch.equal(y[:6].cpu(), torch.from_numpy(values(out)[:6]).to(dtype))
    bad = torch.isnan(y[6:]).cpu()
    if fmt == MX:
        assert bad[0, 32:64].all() and bad[1, 64:].all() and int(bad.sum()) == 64
        assert got_byte[6, 1] == 255 and got_byte[7, 2] == 255
    else:
        assert bad.all() and torch.isnan(out.row_scale[6:]).all()
    assert (got_code[6:][np.isnan(values(out)[6:])] == 0).all() if fmt == NV else (got_code[6, 32:64] == 0).all()


def test_quant_in_parts():
    """A weight of two parts has each part's scale tiles from their own beginning."""
    for fmt in (MX, NV):
        x = gen(5)(2 * 200, 130).to(BF)
        out = quantized(x, fmt, parts=2)
        alone = [quantized(p, fmt) for p in x.chunk(2)]
        done()
        assert torch.equal(out.q, torch.cat([a.q for a in alone]))
        keep = [torch.from_numpy(unpack(a)[1]) for a in alone]
        assert np.array_equal(unpack(out)[1], torch.cat(keep).numpy())
        assert out.scale.numel() == 2 * alone[0].scale.numel()


# ----------------------------------------------------------------- linear ---
def ref_linear(x, w, bias, epi):
    """(y, tol) in 64 bits.  The tensor cores add K products in fp32; with a whole
    step (2 u) lost at each of one addition per 16 products and 2 more, that is (K
    / 16 + 2) 2u of the sum of magnitudes.  Row scales are powers of two; the bias
    adds one rounding, an activation an argument error of 3 u per unit of its
    exponent and 2^-20 of its own; the slope of GELU and SiLU is below 1.2."""
    a = x @ w.T
    d = (x.shape[1] / 16 + 2) * 2 * U32 * (np.abs(x) @ np.abs(w).T)
    if bias is not None:
        b = bias.double().numpy()
        a = a + b
        d = d + U32 * (np.abs(a) + np.abs(b))

    def gelu(v, dv):
        u2 = 1.5957691216057308 * (v + 0.044715 * v ** 3)
        with np.errstate(over="ignore"):
            y = v / (1 + np.exp(-u2))
        return y, 1.2 * dv + np.abs(y) * (3 * U32 * np.abs(u2) * 1.5 + 2.0 ** -20) + 1e-30

    if epi == L.RFX_EPI_SILU:
        with np.errstate(over="ignore"):
            y = a / (1 + np.exp(-a))
        return y, 1.2 * d + np.abs(y) * (3 * U32 * np.abs(a) + 2.0 ** -20) + 1e-30
    if epi == L.RFX_EPI_GELU:
        return gelu(a, d)
    if epi == L.RFX_EPI_GEGLU:
        F = a.shape[1] // 2
        g, dg = gelu(a[:, :F], d[:, :F])
        up, du = a[:, F:], d[:, F:]
        return g * up, np.abs(up) * dg + np.abs(g) * du + dg * du + 2 * U32 * np.abs(g * up)
    return a, d


def check_linear(T, O, Kc, fmt, epi, dtype, bias, pad=0, off=0, seed=0):
    r = gen(seed + T * 31 + O * 7 + Kc)
    x = quantized(r(T, Kc) * torch.exp(0.5 * r(T, 1)), fmt)
    w = quantized(r(O, Kc) * Kc ** -0.5, fmt, 2 if epi == L.RFX_EPI_GEGLU else 1)
    F = O // 2 if epi == L.RFX_EPI_GEGLU else O
    b = r(O) * 0.5 if bias else None
    buf = torch.full((T + 2, F + pad), -77.0, dtype=dtype, device="cuda")
    flat = buf.view(-1)
    y = flat[F + pad + off:F + pad + off + T * (F + pad)].view(T, F + pad)[:, :F]
    K.linear_fp4(w=w, x=x, y=y, epilogue=epi, bias=None if b is None else b.cuda())
    done()
    want, tol = ref_linear(values(x), values(w), b, epi)
    got = y.double().cpu().numpy()
    tol = tol + HALF[dtype] * (np.abs(want) + tol) + 1e-38
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), bad.size, float(np.max(np.abs(got - want) / tol)), np.argwhere(bad)[:4].tolist())
    inside = torch.zeros_like(flat, dtype=torch.bool)
    inside[F + pad + off:F + pad + off + T * (F + pad)].view(T, F + pad)[:, :F] = True
    assert (flat[~inside] == -77.0).all()
    return y


STORE, SILU, GELU, GEGLU = L.RFX_EPI_STORE, L.RFX_EPI_SILU, L.RFX_EPI_GELU, L.RFX_EPI_GEGLU


@pytest.mark.parametrize("fmt", [MX, NV])
@pytest.mark.parametrize("T", [1, 2, 5, 16, 17, 50, 64, 65, 100, 127, 128])
@pytest.mark.parametrize("O,Kc,epi", [(256, 512, STORE), (130, 100, GELU), (512, 1024, GEGLU), (300, 4304, SILU)])
def test_linear_few_tokens(fmt, T, O, Kc, epi):
    check_linear(T, O, Kc, fmt, epi, BF if T % 2 else F32, epi != GEGLU)


@pytest.mark.parametrize("fmt", [MX, NV])
@pytest.mark.parametrize("T,O,Kc,epi", [(129, 64, 256, STORE), (256, 192, 64, STORE), (257, 200, 320, GELU), (300, 1153, 1000, SILU),
                                        (511, 384, 2048, GEGLU), (768, 1000, 96, GEGLU), (1000, 250, 4096, STORE),
                                        (2048, 2048, 512, GEGLU), (1537, 3000, 130, STORE)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_linear_many_tokens(fmt, T, O, Kc, epi, dtype):
    check_linear(T, O, Kc, fmt, epi, dtype, epi == STORE)


@pytest.mark.parametrize("fmt", [MX, NV])
@pytest.mark.parametrize("T", [3, 200])
@pytest.mark.parametrize("Kc", [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 255, 257, 511, 16384])
def test_linear_any_length(fmt, T, Kc):
    check_linear(T, 96, Kc, fmt, STORE, F32, False)


@pytest.mark.parametrize("fmt", [MX, NV])
@pytest.mark.parametrize("T", [1, 60, 300])
@pytest.mark.parametrize("O,pad,off", [(1, 0, 0), (7, 0, 1), (33, 2, 0), (129, 1, 1), (1024, 8, 0), (65, 4, 2)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_linear_any_output(fmt, T, O, pad, off, dtype):
    """Output rows of any length, stride and alignment; nothing beside them is written."""
    check_linear(T, O, 160, fmt, STORE, dtype, True, pad, off)
