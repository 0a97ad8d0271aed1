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


@pytest.mark.parametrize("fmt", [MX, NV])
@pytest.mark.parametrize("T,O,Kc,epi", [(129, 300, 9000, GELU), (200, 128, 16384, STORE), (700, 130, 5000, GEGLU),  # K in parts
                                        (300, 2048, 4096, SILU), (2048, 2600, 512, STORE), (4000, 1100, 300, GELU),
                                        (1300, 7000, 256, GEGLU), (600, 9000, 128, STORE)])                       # tiles of two widths
def test_linear_as_it_is_cut_up(fmt, T, O, Kc, epi):
    check_linear(T, O, Kc, fmt, epi, F32, epi != GEGLU)


@pytest.mark.parametrize("fmt", [MX, NV])
@pytest.mark.parametrize("T,O,Kc,epi", [(1, 300, 4096, STORE), (50, 512, 2048, GEGLU), (129, 300, 9000, GELU), (700, 2600, 512, STORE)])
def test_same_bits_every_time(fmt, T, O, Kc, epi):
    r = gen(3)
    x, w = quantized(r(T, Kc), fmt), quantized(r(O, Kc) * Kc ** -0.5, fmt, 2 if epi == GEGLU else 1)
    y = [torch.empty(T, O // 2 if epi == GEGLU else O, device="cuda") for _ in range(8)]
    for t in y:
        K.linear_fp4(w=w, x=x, y=t, epilogue=epi)
    done()
    assert all(torch.equal(t, y[0]) for t in y[1:])


@pytest.mark.parametrize("fmt", [MX, NV])
@pytest.mark.parametrize("T", [1, 40, 300])
def test_nan_stays_in_its_row_and_column(fmt, T):
    """A row of x or w that holds an infinity is NaN from quantizing on, and
    reaches no other row's or column's products (in MX: its block)."""
    r = gen(4)
    x, w = r(T, 500), r(200, 500)
    clean = torch.empty(T, 200, device="cuda")
    K.linear_fp4(w=quantized(w, fmt), x=quantized(x, fmt), y=clean)
    w[77, 499] = float("inf")
    x[T - 1, 3] = float("nan")
    y = torch.empty(T, 200, device="cuda")
    xq, wq = quantized(x, fmt), quantized(w, fmt)
    K.linear_fp4(w=wq, x=xq, y=y)
    back = torch.empty(T, 500, device="cuda")
    K.dequant_fp4(x=xq, out=back)
    done()
    assert y[T - 1].isnan().all() and y[:, 77].isnan().all()
    keep = [c for c in range(200) if c != 77]
    assert torch.equal(y[:T - 1][:, keep], clean[:T - 1][:, keep])
    assert back[T - 1, :32].isnan().all() and not back[:T - 1].isnan().any()


def test_no_rows():
    for fmt in (MX, NV):
        none, w = K.Fp4Rows.allocate(0, 64, fmt), quantized(gen(1)(8, 64), fmt)
        e = torch.empty(0, 64, device="cuda")
        K.quant_fp4(x=e, out=none)
        K.dequant_fp4(x=none, out=e)
        K.linear_fp4(w=w, x=none, y=torch.empty(0, 8, device="cuda"))
    done()


def test_wrong_sizes_are_refused():
    r = gen(2)
    x, w = quantized(r(4, 64), MX), quantized(r(8, 64), MX)
    y = torch.empty(4, 8, device="cuda")
    for kw in (dict(x=quantized(r(4, 96), MX)), dict(x=quantized(r(4, 64), NV)), dict(w=quantized(r(8, 64), MX, 2)),
               dict(epilogue=GEGLU), dict(y=y[:3]), dict(y=y[:, :7]), dict(y=y.half()), dict(y=y.t().contiguous().t()),
               dict(bias=torch.zeros(7, device="cuda")), dict(bias=torch.zeros(8, device="cuda").double()), dict(bias=torch.zeros(8)),
               dict(y=y.cpu())):
        with pytest.raises(ValueError):
            K.linear_fp4(**{**dict(w=w, x=x, y=y), **kw})
    for kw in (dict(x=r(5, 64).cuda()), dict(x=r(4, 63).cuda()), dict(x=r(4, 64).cuda().half()), dict(x=r(256).cuda())):
        with pytest.raises(ValueError):
            K.quant_fp4(**{**dict(x=r(4, 64).cuda(), out=x), **kw})
    with pytest.raises(ValueError):
        K.dequant_fp4(x=x, out=torch.empty(4, 65, device="cuda"))
    with pytest.raises(L.RfxError):
        K.linear_fp4(w=w, x=x, y=y, epilogue=L.RFX_EPI_RESIDUAL)
    done()


def test_rows_past_32_bits():
    """Rows so far apart that an element's offset passes 2^31, one operand at a time
    (rows of different pitches that interleave are refused)."""
    r = gen(8)
    big = torch.empty((1 << 32) + (1 << 20), dtype=torch.uint8, device="cuda")
    x = r(2, 64).to(BF).cuda()
    want = quantized(x, NV)
    near = K.Fp4Rows.allocate(2, 64, NV)
    far = K.Fp4Rows(big.as_strided((2, 32), ((1 << 32) + 64, 1)), near.scale, near.row_scale, 64, NV)
    w = quantized(r(96, 64), NV)
    y, back = torch.empty(2, 96, device="cuda"), torch.empty(2, 64, device="cuda")
    K.quant_fp4(x=x, out=far)
    K.linear_fp4(w=w, x=far, y=y)
    K.dequant_fp4(x=far, out=back)
    done()
    assert torch.equal(far.q, want.q) and torch.equal(far.scale, want.scale)
    v, tol = ref_linear(values(want), values(w), None, STORE)
    assert (np.abs(y.double().cpu().numpy() - v) <= tol + HALF[F32] * np.abs(v)).all()
    assert np.array_equal(back.double().cpu().numpy(), values(want))
    wide = big.view(BF).as_strided((2, 64), ((1 << 31) + 64, 1))
    wide.copy_(x)
    K.quant_fp4(x=wide, out=near)
    done()
    assert torch.equal(near.q, want.q) and torch.equal(near.row_scale, want.row_scale)
    K.dequant_fp4(x=near, out=wide.zero_())
    done()
    assert torch.equal(wide.double(), back.to(BF).double())
    for T in (2, 5, 200):
        xs = quantized(r(T, 64), NV)
        ys = big.view(F32).as_strided((T, 96), ((1 << 30) // (T - 1) + 64, 1))
        flat = torch.empty(T, 96, device="cuda")
        K.linear_fp4(w=w, x=xs, y=ys)
        K.linear_fp4(w=w, x=xs, y=flat)
        done()
        assert torch.equal(ys, flat)


@pytest.mark.parametrize("T", [1, 50, 300])
def test_captured_calls_follow_their_inputs(T):
    """Captured into a graph and replayed on another stream over changed
    inputs: what the eager calls give, bit for bit; so does a plan."""
    r = gen(12)
    Kc, O = 1000, 700
    x, b = r(T, Kc).to(BF).cuda(), r(O).cuda()
    w = quantized(r(O, Kc) * Kc ** -0.5, NV)
    xq, y, back = K.Fp4Rows.allocate(T, Kc, NV), torch.empty(T, O, dtype=BF, device="cuda"), torch.empty(T, Kc, device="cuda")

    def step():
        K.quant_fp4(x=x, out=xq)
        K.linear_fp4(w=w, x=xq, y=y, epilogue=SILU, bias=b)
        K.dequant_fp4(x=xq, out=back)
        return [t.clone() for t in (xq.q, xq.scale, xq.row_scale, y, back)]
    step()
    g, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g):
        captured = step()
    plan = K.Plan()
    for d in (K.quant_fp4_desc(x=x, out=xq), K.linear_fp4_desc(w=w, x=xq, y=y, epilogue=SILU, bias=b), K.dequant_fp4_desc(x=xq, out=back)):
        plan.add(d)
    assert plan.num_launches == 3
    for _ in range(3):
        x.copy_(r(T, Kc))
        want = step()
        done()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            g.replay()
        done()
        assert all(torch.equal(a, c) for a, c in zip(captured, want))
        y.zero_()
        back.zero_()
        plan.run()
        done()
        assert torch.equal(y, want[3]) and torch.equal(back, want[4])


def test_two_streams_at_once():
    cases = []
    for i, (T, O, Kc) in enumerate([(50, 1024, 4096), (300, 300, 9000)]):
        r = gen(20 + i)
        x, w, y = quantized(r(T, Kc), NV), quantized(r(O, Kc), NV), torch.empty(T, O, device="cuda")
        K.linear_fp4(w=w, x=x, y=y)
        cases.append((w, x, y.clone(), y, torch.cuda.Stream()))
    done()
    for *_, y, st in cases:
        y.zero_()
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for w, x, want, y, st in cases:
            with torch.cuda.stream(st):
                K.linear_fp4(w=w, x=x, y=y)
    done()
    for *_, want, y, st in cases:
        assert torch.equal(want, y)


@pytest.mark.parametrize("fmt", [MX, NV])
@pytest.mark.parametrize("T,O,Kc", [(128, 8192, 4096), (120, 8192, 9000), (128, 2048, 16384), (97, 600, 8192)])
def test_rings_of_one_stage(fmt, T, O, Kc):
    """Many tokens and K steps beside the sums of a split K in shared memory: rings of a
    stage or two, filled again many times."""
    check_linear(T, O, Kc, fmt, GEGLU, F32, False)


@pytest.mark.parametrize("epi", [GELU, SILU])
@pytest.mark.parametrize("T", [2, 200])
def test_activations_of_any_size(epi, T):
    """Outputs from -1e30 to 1e30 side by side, infinities and NaN among them."""
    big = torch.tensor([0.0, -1e-3, -0.5, -3.0, -9.0, -15.0, -40.0, -1e4, -1e30, 1e30, 1e4, 40.0, 9.0, 3.0, 0.5, 1e-3])
    O = 16 * 12
    b = big.repeat(12)
    b[5 * 16 + 3], b[7 * 16 + 4], b[9 * 16 + 8] = float("nan"), float("inf"), float("-inf")
    x, w = quantized(torch.zeros(T, 64), MX), quantized(torch.zeros(O, 64), MX)
    y = torch.empty(T, O, device="cuda")
    K.linear_fp4(w=w, x=x, y=y, epilogue=epi, bias=b.cuda())
    done()
    got, v = y.double().cpu().numpy(), b.double().numpy()
    with np.errstate(over="ignore", invalid="ignore"):
        e = v if epi == SILU else 1.5957691216057308 * (v + 0.044715 * v ** 3)
        want = v / (1 + np.exp(-e))  # (-inf: NaN, as the formula's 0 times infinity)
        want[v == -np.inf] = np.nan
        tol = np.abs(want) * (3 * U32 * np.abs(e) * 1.5 + 2.0 ** -20) + 2.0 ** -58 * np.minimum(np.abs(v), 64)
    assert np.array_equal(np.isnan(got), np.broadcast_to(np.isnan(want), got.shape))
    ok = np.isfinite(want)
    assert (np.abs(got[:, ok] - want[ok]) <= tol[ok]).all(), np.abs(got[:, ok] - want[ok]).max()
    assert (got[:, v == np.inf] == np.inf).all()


@pytest.mark.parametrize("fmt", [MX, NV])
@pytest.mark.parametrize("T,O,Kc", [(594, 40, 9598), (300, 200, 16384), (200, 256, 12000), (1024, 20, 8000)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_geglu_in_many_parts(fmt, T, O, Kc, dtype):
    """Few outputs of a long K: what the parts of K send one another fits beside the scales."""
    check_linear(T, O, Kc, fmt, GEGLU, dtype, True)
