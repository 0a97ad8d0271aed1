"""The int8 layer operators on the GPU against plain 64-bit restatements.

Tolerances count roundings: u = 2^-24 is half a step of fp32 (2^-8 of bf16).
"""
import math

import numpy as np
import pytest
import torch

from reflex_b200 import _lib as L
from reflex_b200 import kernels as K

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: U32}
BF, F32 = torch.bfloat16, torch.float32


def gen(seed):
    g = torch.Generator().manual_seed(seed)
    return lambda *shape, std=1.0: torch.randn(*shape, generator=g) * std


def done():
    torch.cuda.synchronize()
    assert K.device_status() == 0


def within(got, want, tol, what=""):
    """|got - want| <= tol element by element (want and tol fp64 numpy)."""
    got = got.double().cpu().numpy()
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (what, int(bad.sum()), float(np.max(np.abs(got - want) / np.maximum(tol, 1e-300))))


def framed(T, Kc, dtype, ld, fill):
    """A [T, Kc] view with row stride ld inside a buffer filled with `fill`,
    and a check that nothing but the view was written."""
    buf = torch.full((T + 2, ld), fill, dtype=dtype, device="cuda")
    view = buf[1:T + 1, :Kc]

    def untouched():
        assert (buf[0] == fill).all() and (buf[T + 1] == fill).all() and (buf[1:T + 1, Kc:] == fill).all()
    return view, untouched


def ref_quant(x):
    """scale = fl(absmax / 127), q = clamp(rne(fl(x / scale))): fp32 numpy, IEEE division."""
    x = x.float().cpu().numpy()
    scale = (np.abs(x).max(axis=1) / np.float32(127.0)).astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.rint((x / scale[:, None]).astype(np.float32))
    q = np.where(scale[:, None] > 0, np.clip(q, -127, 127), 0).astype(np.int8)
    return q, scale


# ------------------------------------------------------------- quant_rows ---
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,Kc", [(1, 1), (1, 4096), (3, 7), (5, 8), (6, 31), (9, 256), (4, 257), (50, 1024), (7, 1025),
                                  (3, 2048), (2, 4304), (2, 8191), (3, 16384), (130, 16383), (2000, 64)])
@pytest.mark.parametrize("pad", [0, 24])
def test_quant_rows_is_exact(dtype, T, Kc, pad):
    """Bit for bit the IEEE fp32 formula, at any length and row stride, for
    rows of very different sizes; nothing outside the rows is written."""
    r = gen(T * 7 + Kc)
    x = (r(T, Kc) * torch.exp(3 * r(T, 1))).to(dtype)
    x[0, 0] = 0.0
    xb, _ = framed(T, Kc, dtype, Kc + pad, 3.0)
    xb.copy_(x)
    q, clean = framed(T, Kc, torch.int8, Kc + pad, 77)
    scale = torch.full((T,), -1.0, device="cuda")
    K.quant_rows(x=xb, q=q, scale=scale)
    done()
    want_q, want_s = ref_quant(x)
    assert np.array_equal(scale.cpu().numpy(), want_s)
    assert np.array_equal(q.cpu().numpy(), want_q)
    clean()


@pytest.mark.parametrize("Kc", [64, 1000, 4096])
def test_quant_rows_special_rows(Kc):
    """Zeros, a row of one value, ties, the smallest numbers, and rows with an
    infinity or a NaN: scale inf / NaN and q 0."""
    x = torch.zeros(8, Kc)
    x[1] = -2.5
    x[2] = torch.arange(Kc) % 255 - 127.0  # scale 1: whole numbers
    x[3] = (torch.arange(Kc) % 253 - 126.0) + 0.5  # ties, once a 127 sets the scale
    x[3, 0] = 127.0
    x[4] = 1e-42  # a denormal scale
    x[5] = 1e-45  # absmax / 127 underflows to 0
    x[6] = 1.0
    x[6, Kc - 1] = float("inf")
    x[7] = 1.0
    x[7, Kc // 2] = float("nan")
    q = torch.full((8, Kc), 9, dtype=torch.int8, device="cuda")
    scale = torch.empty(8, device="cuda")
    K.quant_rows(x=x.cuda(), q=q, scale=scale)
    done()
    want_q, want_s = ref_quant(x[:6])
    assert np.array_equal(scale[:6].cpu().numpy(), want_s)
    assert np.array_equal(q[:6].cpu().numpy(), want_q)
    assert torch.isinf(scale[6]) and torch.isnan(scale[7]) and (q[6:] == 0).all()


# -------------------------------------------------------------- linear_i8 ---
def ints(seed, rows, cols, ld=None):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-127, 128, (rows, cols), generator=g, dtype=torch.int8)
    ld = ld or (cols + 15) // 16 * 16
    buf = torch.full((rows, ld), 111, dtype=torch.int8)  # the padding must not be read
    buf[:, :cols] = q
    return q, buf.cuda()[:, :cols]


def ref_linear(q, w, sx, sw, bias, epi):
    """(y, tol): fp64 value, and what fp32 roundings can move it by.  A
    pre-activation carries 4 of them (conversion, two scales, bias), the
    exponential an argument error of 3 u per unit of 2u and 2^-21 of its own
    with the division; the slope of GELU and SiLU is below 1.2."""
    a = q.double().numpy() @ w.double().numpy().T * sx.double().numpy()[:, None] * sw.double().numpy()
    mag = np.abs(a) + (np.abs(bias.double().numpy()) if bias is not None else 0)
    if bias is not None:
        a = a + bias.double().numpy()
    d = 5 * U32 * mag

    def gelu(v):
        u2 = 1.5957691216057308 * (v + 0.044715 * v ** 3)
        with np.errstate(over="ignore"):
            y = v / (1 + np.exp(-u2))
        return y, 1.2 * d + np.abs(y) * ((3 * U32) * np.abs(u2) * 1.5 + 2.0 ** -20) + 1e-30

    if epi == L.RFX_EPI_STORE:
        return a, d
    if epi == L.RFX_EPI_SILU:
        with np.errstate(over="ignore"):
            y = a / (1 + np.exp(-a))
        return y, 1.2 * d + np.abs(y) * ((3 * U32) * np.abs(a) + 2.0 ** -20) + 1e-30
    if epi == L.RFX_EPI_GELU:
        return gelu(a)
    F = a.shape[1] // 2
    full, dfull = gelu(a)
    g, dg, up, du = full[:, :F], dfull[:, :F], a[:, F:], d[:, F:]
    return g * up, np.abs(up) * dg + np.abs(g) * du + dg * du + U32 * np.abs(g * up)


def check_linear(T, O, Kc, epi, dtype, bias, ldy_pad=0, seed=0):
    r = gen(seed + T + O)
    q, x = ints(seed + 1, T, Kc)
    w, wd = ints(seed + 2, O, Kc)
    sx, sw = torch.exp(r(T)) * 1e-2, torch.exp(r(O) * 0.5) / math.sqrt(Kc) * 1e-1
    b = r(O) if bias else None
    cols = O // 2 if epi == L.RFX_EPI_GEGLU else O
    y, clean = framed(T, cols, dtype, cols + ldy_pad, 5.0)
    K.linear_i8(w=wd, w_scale=sw.cuda(), x=x, x_scale=sx.cuda(), y=y, epilogue=epi,
                bias=b.cuda() if bias else None)
    done()
    want, tol = ref_linear(q, w, sx, sw, b, epi)
    within(y, want, tol + (1.01 * HALF[dtype]) * np.abs(want) + (1e-38 if dtype == F32 else 0), (T, O, Kc, epi))
    clean()


@pytest.mark.parametrize("T,O,Kc", [
    (1, 1, 1), (1, 2560, 2048), (2, 8, 16), (3, 31, 33), (7, 129, 127), (8, 128, 128), (16, 256, 129), (50, 8192, 1024),
    (50, 1024, 4096), (64, 100, 200), (65, 2048, 640), (127, 300, 1152), (128, 1152, 4304), (129, 130, 255),
    (200, 4304, 1152), (256, 512, 16384), (300, 2050, 511), (768, 2560, 2048), (771, 1153, 4304), (1600, 1024, 128),
    (4, 260, 1040), (5, 260, 1040), (8, 3000, 2100), (9, 3000, 48), (2000, 6000, 128), (2047, 5001, 64),
])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_linear_i8_store(T, O, Kc, dtype):
    """Few and many tokens, K and O off every tile, one value alone; with and
    without bias and an output inside wider rows."""
    check_linear(T, O, Kc, L.RFX_EPI_STORE, dtype, bias=(T + O) % 2 == 0, ldy_pad=(O * T) % 3, seed=T)


@pytest.mark.parametrize("epi", [L.RFX_EPI_SILU, L.RFX_EPI_GELU, L.RFX_EPI_GEGLU])
@pytest.mark.parametrize("T,O,Kc", [(1, 2, 16), (1, 8192, 1024), (5, 66, 100), (50, 8192, 1024), (130, 258, 700),
                                    (513, 1154, 1152), (768, 4608, 2048), (1000, 300, 64), (4, 66, 272), (2000, 9002, 64)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_linear_i8_activations(epi, T, O, Kc, dtype):
    check_linear(T, O, Kc, epi, dtype, bias=T % 2 == 1, seed=epi * 100 + T)


@pytest.mark.parametrize("epi", [L.RFX_EPI_STORE, L.RFX_EPI_GEGLU])
@pytest.mark.parametrize("T,O,Kc", [(50, 74, 256), (333, 1178, 300), (129, 526, 8192)])
def test_linear_i8_aligned_rows_of_odd_length(epi, T, O, Kc):
    """Outputs of 37, 589, 263 or twice as many columns in rows of a multiple
    of 16 bytes: the wide stores stop at the last column and the last row."""
    for dtype in (BF, F32):
        cols = O // 2 if epi == L.RFX_EPI_GEGLU else O
        check_linear(T, O, Kc, epi, dtype, bias=False, ldy_pad=-cols % 8 + 8, seed=3)


@pytest.mark.parametrize("epi", [L.RFX_EPI_STORE, L.RFX_EPI_GELU, L.RFX_EPI_GEGLU])
@pytest.mark.parametrize("T,O,Kc", [
    (1, 20002, 64), (2, 9000, 333), (3, 2050, 9000), (5, 128, 128), (6, 130, 129), (15, 1026, 4096), (16, 256, 1100),
    (17, 2560, 1024), (31, 126, 2000), (33, 2050, 3333), (48, 60002, 100), (49, 1152, 4304), (63, 514, 16384),
    (64, 40000, 200), (65, 700, 512), (80, 300, 2049), (96, 5002, 700), (97, 64, 30000), (112, 4096, 2048),
    (113, 2, 2048), (127, 20000, 72), (128, 2050, 5000),
])
def test_linear_i8_up_to_128_tokens(epi, T, O, Kc):
    """One and several parts of K and rounds of tiles, tiles of one row and of
    all but one, tokens at and around the multiples of 16."""
    check_linear(T, O, Kc, epi, BF if (T + O) % 4 else F32, bias=T % 2 == 0, ldy_pad=T % 3, seed=T + 7)


@pytest.mark.parametrize("T", [8, 100])
def test_linear_i8_largest_sums_of_some_tokens(T):
    """As the test below, with K in parts that are joined."""
    Kc = 65536
    x = torch.full((T, Kc), -128, dtype=torch.int8, device="cuda")
    w = torch.full((40, Kc), -128, dtype=torch.int8, device="cuda")
    w[1] = 127
    y = torch.empty(T, 40, device="cuda")
    K.linear_i8(w=w, w_scale=torch.ones(40, device="cuda"), x=x, x_scale=torch.ones(T, device="cuda"), y=y)
    done()
    assert (y[:, 0] == 2.0 ** 30).all() and (y[:, 2:] == 2.0 ** 30).all()
    assert (y[:, 1] == float(-128 * 127 * Kc)).all()


def test_linear_i8_rows_do_not_depend_on_the_others():
    """A token's outputs are the same bits in any batch: the forms that a call
    may take differ in no rounding."""
    q, x = ints(8, 300, 2304)
    w, wd = ints(9, 1536, 2304)
    sx, sw, b = torch.rand(300).cuda(), torch.rand(1536).cuda() * 1e-4, torch.randn(1536).cuda()
    for epi in (L.RFX_EPI_STORE, L.RFX_EPI_SILU, L.RFX_EPI_GELU, L.RFX_EPI_GEGLU):
        F = 768 if epi == L.RFX_EPI_GEGLU else 1536
        whole = None
        for T in (300, 128, 64, 50, 16, 5, 4, 2, 1):
            y = torch.empty(T, F, device="cuda")
            K.linear_i8(w=wd, w_scale=sw, x=x[:T], x_scale=sx[:T], y=y, epilogue=epi, bias=b)
            done()
            whole = y if whole is None else whole
            assert torch.equal(y, whole[:T]), (epi, T)


def test_linear_i8_largest_sums():
    """Every product at its extreme (-128 * -128 over K = 65536, a sum of
    2^30): the s32 accumulators hold it."""
    Kc = 65536
    x = torch.full((3, Kc), -128, dtype=torch.int8, device="cuda")
    w = torch.full((40, Kc), -128, dtype=torch.int8, device="cuda")
    w[1] = 127
    y = torch.empty(3, 40, device="cuda")
    K.linear_i8(w=w, w_scale=torch.ones(40, device="cuda"), x=x, x_scale=torch.ones(3, device="cuda"), y=y)
    done()
    assert (y[:, 0] == 2.0 ** 30).all() and (y[:, 2:] == 2.0 ** 30).all()
    assert (y[:, 1] == float(-128 * 127 * Kc)).all()


def test_linear_i8_nonfinite_scale_shows():
    """A token whose row could not be quantized (scale NaN or infinity, q 0)
    comes out as NaN; the other tokens are not touched by it."""
    r = gen(3)
    x = r(4, 256)
    x[1, 5], x[2, 9] = float("nan"), float("inf")
    q = torch.empty(4, 256, dtype=torch.int8, device="cuda")
    s = torch.empty(4, device="cuda")
    K.quant_rows(x=x.cuda(), q=q, scale=s)
    w, wd = ints(4, 64, 256)
    y = torch.empty(4, 64, dtype=BF, device="cuda")
    K.linear_i8(w=wd, w_scale=torch.ones(64, device="cuda"), x=q, x_scale=s, y=y)
    done()
    assert torch.isnan(y[1]).all() and torch.isnan(y[2]).all() and torch.isfinite(y[[0, 3]]).all()


def test_linear_i8_is_deterministic():
    q, x = ints(5, 50, 4096)
    w, wd = ints(6, 1024, 4096)
    sx, sw = torch.rand(50).cuda(), torch.rand(1024).cuda()
    ys = [torch.empty(50, 1024, dtype=F32, device="cuda") for _ in range(3)]
    for y in ys:
        K.linear_i8(w=wd, w_scale=sw, x=x, x_scale=sx, y=y)
    done()
    assert torch.equal(ys[0], ys[1]) and torch.equal(ys[0], ys[2])


# ------------------------------------------------------------- block_norm ---
def check_norm(T, S, Kc, dtype, post, gate, mod, out, a1=True, y=True, pad=0, in_place=False, shared=False, seed=0):
    r = gen(seed + T * 3 + Kc)
    B = -(-T // S)
    hb, h_clean = framed(T, Kc, dtype, Kc + pad, 2.0)
    hb.copy_((r(T, Kc) * torch.exp(r(T, 1))).to(dtype))
    yv = r(T, Kc).to(dtype) if y else None
    vec = lambda on, *s: (1 + 0.3 * r(*s)) if on else None  # noqa: E731
    per = (Kc,) if shared else (B, Kc)
    pw, g, v1 = vec(post, Kc), vec(gate, *per), vec(a1, Kc)
    v2, vb = vec(mod, *per), vec(mod, *per)
    rs, eps = 0.7, 1e-6
    h0 = hb.double().cpu().numpy()
    cuda = lambda t: t.cuda() if t is not None else None  # noqa: E731
    ho, ho_clean = (hb, h_clean) if in_place else framed(T, Kc, dtype, Kc + pad, 4.0)
    kw = {}
    if out == "z":
        kw["z"], z_clean = framed(T, Kc, dtype, Kc + pad, 6.0)
    elif out == "q":
        kw["z_q"], z_clean = framed(T, Kc, torch.int8, Kc + pad, 99)
        kw["z_scale"] = torch.empty(T, device="cuda")
    K.block_norm(h=hb, S=S, y=cuda(yv), post_w=cuda(pw), gate=cuda(g), residual_scale=rs, h_out=ho if y else None,
                 norm_a1=cuda(v1), norm_a2=cuda(v2), norm_b2=cuda(vb), eps=eps, **kw)
    done()
    # rows of a sum of squares: at most 33 fused steps a thread, 5 shuffles and
    # 16 warps, half of that in its root, 2 steps of rsqrt
    dr = (0.5 * (33 + 5 + 16) + 4) * U32
    n = lambda t: 1.0 if t is None else t.double().numpy()  # noqa: E731
    rows = lambda t, none: none if t is None else (t.double().numpy()[None].repeat(T, 0) if t.dim() == 1  # noqa: E731
                                                   else t.double().numpy().repeat(S, 0)[:T])
    held = h0
    if y:
        u = yv.double().numpy()
        if post:
            u = u / np.sqrt((u * u).mean(1, keepdims=True) + eps) * n(pw)
        u = rs * u * rows(g, 1.0)
        want = h0 + u
        within(ho, want, np.abs(u) * (dr + 5 * U32) + np.abs(want) * 1.01 * HALF[dtype] + 2 * U32 * np.abs(want), "h")
        ho_clean()
        held = ho.double().cpu().numpy()
    if out is None:
        return
    z = held / np.sqrt((held * held).mean(1, keepdims=True) + eps) * n(v1) * rows(v2, 1.0)
    b2 = rows(vb, 0.0)
    tol = np.abs(z) * (dr + 5 * U32) + U32 * np.abs(b2)
    z = z + b2
    tol = tol + U32 * np.abs(z)
    if out == "z":
        within(kw["z"], z, tol + 1.01 * HALF[dtype] * np.abs(z), "z")
    else:
        s = kw["z_scale"].double().cpu().numpy()
        top = np.argmax(np.abs(z), 1)
        # the scale follows the largest magnitude, whichever element that is
        assert (np.abs(s * 127 - np.abs(z).max(1)) <= tol.max(1) + 2 * U32 * np.abs(z).max(1)).all(), top
        q = kw["z_q"].double().cpu().numpy()
        assert np.abs(q).max() <= 127
        within(torch.from_numpy(q * s[:, None]), z, s[:, None] * (0.5 + 128 * 2 * U32) + tol, "z_q")
    z_clean()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,S,Kc", [(1, 1, 1), (1, 1, 1024), (2, 1, 8), (7, 3, 33), (50, 50, 1024), (100, 50, 1024),
                                    (5, 7, 257), (12, 4, 1152), (9, 9, 2048), (6, 2, 2047), (3, 3, 4096), (4, 2, 8192),
                                    (3, 1, 16384), (2, 2, 16383), (1700, 50, 256)])
@pytest.mark.parametrize("out", ["z", "q"])
def test_block_norm_full(dtype, T, S, Kc, out):
    """Norm after the block, gate, residual scale, norm before the next one
    with scale and shift per stream; any length, the last stream cut short."""
    check_norm(T, S, Kc, dtype, True, True, True, out)


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("mod", [False, True])
@pytest.mark.parametrize("out", ["z", "q", None])
@pytest.mark.parametrize("Kc,pad", [(1024, 0), (200, 3)])
def test_block_norm_parts(post, gate, mod, out, Kc, pad):
    """Every part left out in turn, rows inside wider buffers, in place."""
    vecs = out is not None
    check_norm(13, 5, Kc, BF, post, gate, mod and vecs, out, a1=vecs and not mod, pad=pad, in_place=post)


@pytest.mark.parametrize("Kc", [64, 1024, 1030])
def test_block_norm_without_block_output(Kc):
    """y = None: the norm alone (the first layer's), over h as it is."""
    for out in ("z", "q"):
        check_norm(10, 10, Kc, BF, False, False, True, out, y=False)


def test_block_norm_shared_vectors():
    """One gate, scale and shift for all streams ([K] instead of [B, K])."""
    check_norm(20, 5, 512, F32, True, True, True, "z", shared=True)


@pytest.mark.parametrize("Kc", [200, 1024, 1031])
def test_block_norm_nonfinite_rows_show(Kc):
    """A NaN or an infinity in the stream or the block's output leaves its row's
    scale not finite and its int8 values 0; the other rows are not touched."""
    r = gen(Kc)
    h, y = r(6, Kc).cuda(), r(6, Kc).cuda()
    a1 = torch.ones(Kc, device="cuda")
    out = []
    for bad in (False, True):
        hb, yb = h.clone(), y.clone()
        if bad:
            hb[1, 3], yb[4, Kc - 1] = float("nan"), float("inf")
        q, s = torch.full((6, Kc), 5, dtype=torch.int8, device="cuda"), torch.empty(6, device="cuda")
        K.block_norm(h=hb, y=yb, S=3, h_out=hb, norm_a1=a1, z_q=q, z_scale=s)
        out.append((hb, q, s))
    done()
    (h0, q0, s0), (h1, q1, s1) = out
    keep, bad = [0, 2, 3, 5], [1, 4]
    assert torch.equal(h0[keep], h1[keep]) and torch.equal(q0[keep], q1[keep]) and torch.equal(s0[keep], s1[keep])
    assert not torch.isfinite(s1[bad]).any() and (q1[bad] == 0).all()


@pytest.mark.parametrize("Kc", [1024, 1027, 6000])
def test_block_norm_output_over_an_input(Kc):
    """z over y, or over h (with the stream written elsewhere): the same as apart."""
    r = gen(Kc + 1)
    h, y = r(40, Kc).to(BF).cuda(), r(40, Kc).to(BF).cuda()
    w = (1 + 0.1 * r(Kc)).cuda()
    kw = dict(S=8, post_w=w, norm_a1=w)
    h0, z0 = torch.empty_like(h), torch.empty_like(h)
    K.block_norm(h=h, y=y, h_out=h0, z=z0, **kw)
    y1, h1 = y.clone(), h.clone()
    K.block_norm(h=h1, y=y1, h_out=h1, z=y1, **kw)
    h2, hz = torch.empty_like(h), h.clone()
    K.block_norm(h=hz, y=y, h_out=h2, z=hz, **kw)
    done()
    assert torch.equal(h1, h0) and torch.equal(y1, z0) and torch.equal(h2, h0) and torch.equal(hz, z0)


def test_block_norm_matches_rms_norm():
    """The norm alone agrees with rfx_rms_norm to one rounding of bf16."""
    r = gen(11)
    x, a1 = r(50, 1024).to(BF).cuda(), (1 + 0.1 * r(1024)).cuda()
    a2, b2 = (1 + 0.1 * r(1, 1024)).cuda(), (0.1 * r(1, 1024)).cuda()
    z, z0 = torch.empty_like(x), torch.empty_like(x)
    K.block_norm(h=x, S=50, norm_a1=a1, norm_a2=a2, norm_b2=b2, z=z)
    K.rms_norm(x=x, y=z0, S=50, norm_a1=a1, norm_a2=a2, norm_b2=b2, norm_ab_stride=1024)
    done()
    assert ((z.float() - z0.float()).abs() <= 2 * HALF[BF] * z0.float().abs() + 1e-6).all()


# ------------------------------------------------------------------- rope ---
def check_rope(B, S, Hq, Hkv, D, rot, pairs, dtype, first, v=True, pad=0, head_major=True, in_place=False, mag=1.25,
               positions=None):
    r = gen(B * 100 + S + D + rot)
    T, heads = B * S, Hq + Hkv * (2 if v else 1)
    xb, x_clean = framed(T, heads * D, dtype, heads * D + pad, 3.0)
    xb.copy_(r(T, heads * D).to(dtype))
    x0 = xb.double().cpu().numpy().reshape(B, S, heads, D).transpose(0, 2, 1, 3)
    pos = positions if positions is not None else (first + torch.arange(S)).repeat(B).to(torch.int32)
    freq, _ = K.rope_frequencies(rot, device="cuda")
    if in_place:
        v4 = xb.unflatten(1, (heads, D)).unflatten(0, (B, S)).transpose(1, 2)  # [B, heads, S, D] over x
        q, k, vo = v4[:, :Hq], v4[:, Hq:Hq + Hkv], v4[:, Hq + Hkv:]
    else:
        make = lambda H: (torch.empty(B, H, S, D, dtype=dtype, device="cuda") if head_major else  # noqa: E731
                          torch.empty(B, S, H, D, dtype=dtype, device="cuda").transpose(1, 2))
        q, k, vo = make(Hq), make(Hkv), make(Hkv)
    K.rope(x=xb, positions=pos.cuda(), inv_freq=freq, q_out=q, k_out=k if Hkv else None, v_out=vo if v and Hkv else None,
           pairs=pairs, magnitude=mag)
    done()
    ang = pos.double().numpy().reshape(B, 1, S, 1) * freq.cpu().numpy()
    c, s = mag * np.cos(ang), mag * np.sin(ang)
    i0 = np.arange(rot // 2) if pairs == L.RFX_ROPE_HALF else np.arange(0, rot, 2)
    i1 = i0 + (rot // 2 if pairs == L.RFX_ROPE_HALF else 1)
    want, tol = x0.copy(), np.zeros_like(x0)
    R = Hq + Hkv
    a, b = x0[:, :R][..., i0], x0[:, :R][..., i1]
    want[:, :R][..., i0], want[:, :R][..., i1] = a * c - b * s, b * c + a * s
    # fraction of a turn to fp32 and sine / cosine: 2 pi 2^-25 + 2 steps; 3 products and sums
    d = mag * (np.abs(a) + np.abs(b)) * (2.0 ** -22 + 4 * U32)
    tol[:, :R][..., i0] = tol[:, :R][..., i1] = d
    tol = tol + 1.01 * HALF[dtype] * np.abs(want) * (tol > 0)
    within(q, want[:, :Hq], tol[:, :Hq], "q")
    if Hkv:
        within(k, want[:, Hq:R], tol[:, Hq:R], "k")
        if v:
            within(vo, want[:, R:], tol[:, R:], "v")
    x_clean()


@pytest.mark.parametrize("pairs", [L.RFX_ROPE_HALF, L.RFX_ROPE_INTERLEAVED])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,S,Hq,Hkv,D,rot", [
    (1, 1, 1, 0, 2, 2), (1, 1, 8, 1, 256, 256), (1, 50, 8, 1, 256, 256), (3, 17, 4, 2, 64, 32), (2, 5, 3, 1, 72, 72),
    (1, 300, 8, 1, 256, 64), (2, 9, 2, 2, 72, 40), (1, 7, 5, 1, 250, 10), (1, 3, 2, 1, 256, 2), (4, 700, 1, 1, 128, 128),
    (2, 3, 16, 4, 128, 96), (2, 700, 16, 4, 128, 74), (1, 60, 4, 1, 256, 250), (1, 2, 64, 16, 256, 74),
])
def test_rope(pairs, dtype, B, S, Hq, Hkv, D, rot):
    """Both layouts, part of the head and all of it, head dims off the vector
    width, one head alone, several KV heads."""
    check_rope(B, S, Hq, Hkv, D, rot, pairs, dtype, first=818, v=Hkv > 0)


@pytest.mark.parametrize("rot", [48, 44])
@pytest.mark.parametrize("pairs", [L.RFX_ROPE_HALF, L.RFX_ROPE_INTERLEAVED])
@pytest.mark.parametrize("in_place,head_major,pad,v", [(True, True, 0, True), (True, True, 5, True), (False, False, 0, True),
                                                       (False, True, 8, False), (False, False, 1, False)])
def test_rope_layouts(pairs, in_place, head_major, pad, v, rot):
    """Over its own input, token-major outputs, wider rows, no v heads; halves
    on and off 16-byte boundaries."""
    check_rope(2, 33, 4, 2, 64, rot, pairs, BF, first=0, v=v, pad=pad, head_major=head_major, in_place=in_place)


def test_rope_far_and_negative_positions():
    """Angles stay right at any int32 position: a fp32 angle would be off by
    radians at 2^31 (fp64 turns leave 2^-53 * 2^31 / 2 pi of one)."""
    pos = torch.tensor([0, 1, -1, -5000, 10 ** 6, 10 ** 9, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)
    check_rope(1, 8, 2, 1, 64, 64, L.RFX_ROPE_HALF, F32, 0, positions=pos)


# ---------------------------------------------------------- together ---
def test_refusals_with_gpu_tensors():
    """Shapes and types that would be read out of bounds are refused before a launch."""
    q8 = torch.zeros(4, 64, dtype=torch.int8, device="cuda")
    x, s4 = torch.zeros(4, 64, dtype=BF, device="cuda"), torch.zeros(4, device="cuda")
    with pytest.raises(ValueError):
        K.quant_rows(x=x.half(), q=q8, scale=s4)
    with pytest.raises(ValueError):
        K.quant_rows(x=x, q=q8[:3], scale=s4)
    with pytest.raises(ValueError):
        K.quant_rows(x=x, q=q8, scale=s4[:3])
    with pytest.raises(ValueError):
        K.quant_rows(x=x.t(), q=q8.t(), scale=torch.zeros(64, device="cuda"))
    with pytest.raises(ValueError):
        K.quant_rows(x=x[:1].expand(4, 64), q=q8, scale=s4)
    y = torch.zeros(4, 4, dtype=BF, device="cuda")
    with pytest.raises(ValueError):
        K.linear_i8(w=q8, w_scale=s4, x=q8[:, :32], x_scale=s4, y=y)
    with pytest.raises(ValueError):
        K.linear_i8(w=q8, w_scale=s4[:2], x=q8, x_scale=s4, y=y)
    with pytest.raises(ValueError):
        K.linear_i8(w=q8, w_scale=s4, x=q8, x_scale=s4, y=y, epilogue=L.RFX_EPI_GEGLU)
    with pytest.raises(L.RfxError):
        K.linear_i8(w=q8, w_scale=s4, x=q8, x_scale=s4, y=y, epilogue=L.RFX_EPI_RESIDUAL)
    odd = torch.zeros(4, 72, dtype=torch.int8, device="cuda")[:, :64]
    with pytest.raises(L.RfxError):
        K.linear_i8(w=odd, w_scale=s4, x=q8, x_scale=s4, y=y)
    with pytest.raises(ValueError):
        K.block_norm(h=x, S=1, norm_a2=torch.zeros(3, 64, device="cuda"), z=torch.empty_like(x))
    with pytest.raises(ValueError):
        K.block_norm(h=x, S=4, y=x.float(), h_out=x)
    with pytest.raises(L.RfxError):
        K.block_norm(h=x, S=4, y=x.clone())
    f = torch.ones(33, dtype=torch.float64, device="cuda")
    p = torch.zeros(4, dtype=torch.int32, device="cuda")
    qo = torch.empty(1, 1, 4, 64, dtype=BF, device="cuda")
    with pytest.raises(L.RfxError):
        K.rope(x=x, positions=p, inv_freq=f, q_out=qo)
    with pytest.raises(ValueError):
        K.rope(x=x, positions=p[:3], inv_freq=f[:8], q_out=qo)
    with pytest.raises(ValueError):
        K.rope(x=x, positions=p, inv_freq=f[:8].float(), q_out=qo)
    with pytest.raises(ValueError):
        K.rope(x=x, positions=p, inv_freq=f[:8], q_out=qo[:, :, :1].expand(1, 1, 4, 64))
    done()


def test_empty_calls():
    e8, eb, es = (torch.empty(0, 64, dtype=d, device="cuda") for d in (torch.int8, BF, F32))
    s = torch.empty(0, device="cuda")
    w = torch.zeros(16, 64, dtype=torch.int8, device="cuda")
    K.quant_rows(x=eb, q=e8, scale=s)
    K.linear_i8(w=w, w_scale=torch.ones(16, device="cuda"), x=e8, x_scale=s, y=es[:, :16])
    K.block_norm(h=eb, S=1, z=eb.clone())
    K.rope(x=eb, positions=torch.empty(0, dtype=torch.int32, device="cuda"),
           inv_freq=torch.ones(8, dtype=torch.float64, device="cuda"), q_out=torch.empty(1, 1, 0, 64, dtype=BF, device="cuda"))
    done()


def int8_rows(rows, cols):
    """int8 [rows, cols] whose rows begin on 16-byte boundaries, as linear_i8 takes them."""
    return torch.zeros(rows, -(-cols // 16) * 16, dtype=torch.int8, device="cuda")[:, :cols]


class Int8Layer:
    """One prefix-shaped layer (MQA, GeGLU, norms before and after each block)
    on the int8 operators and the library's attention, as a launch list."""

    def __init__(self, B, S, W, H, F, seed):
        D = 256
        r = gen(seed)
        self.dims = (B, S, W, H, D, F)
        T = B * S
        self.r = r
        self.h0 = r(T, W).to(BF)
        self.wf = {"qkv": r((H + 2) * D, W) / math.sqrt(W), "o": r(W, H * D) / math.sqrt(H * D),
                   "gu": r(2 * F, W) / math.sqrt(W), "down": r(W, F) / math.sqrt(F)}
        self.n = {k: (1 + 0.1 * r(W)).cuda() for k in ("in", "post1", "mid", "post2", "next")}
        self.wq, self.ws = {}, {}
        for k, w in self.wf.items():
            q, s = int8_rows(*w.shape), torch.empty(w.shape[0], device="cuda")
            K.quant_rows(x=w.cuda(), q=q, scale=s)
            self.wq[k], self.ws[k] = q, s
        e = lambda *s, dt=BF: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
        self.h, self.z = self.h0.cuda(), e(T, W)
        self.xq, self.xs = e(T, W, dt=torch.int8), e(T, dt=F32)
        self.qkv, self.q = e(T, (H + 2) * D), e(B, H, S, D)
        self.k, self.v, self.att = e(T, D), e(T, D), e(T, H * D)
        self.aq, self.as_ = e(T, H * D, dt=torch.int8), e(T, dt=F32)
        self.y = e(T, W)
        self.act, self.fq, self.fs = e(T, F), int8_rows(T, F), e(T, dt=F32)
        self.pos = torch.arange(S, dtype=torch.int32).repeat(B).cuda()
        self.freq, _ = K.rope_frequencies(D)
        self.ws_attn = torch.zeros(1 << 24, dtype=torch.uint8, device="cuda")

    def descs(self):
        B, S, W, H, D, F = self.dims
        tok = lambda t: t.view(B, S, 1, D).transpose(1, 2)  # noqa: E731
        lin = lambda k, x, s, y, **kw: K.linear_i8_desc(w=self.wq[k], w_scale=self.ws[k], x=x, x_scale=s, y=y, **kw)  # noqa: E731
        ad = K.attention_desc(q=self.q, k_new=self.k, v_new=self.v, ring=None, n_ctx=0, out=self.att,
                              softmax_scale=D ** -0.5)
        need = K.attention_workspace_bytes(ad)
        assert need + 1024 <= self.ws_attn.numel()
        if need:
            ad.workspace, ad.workspace_bytes = K.aligned_ptr(self.ws_attn, 1024), need
        return [
            K.block_norm_desc(h=self.h, S=S, norm_a1=self.n["in"], z_q=self.xq, z_scale=self.xs),
            lin("qkv", self.xq, self.xs, self.qkv),
            K.rope_desc(x=self.qkv, positions=self.pos, inv_freq=self.freq, q_out=self.q, k_out=tok(self.k),
                        v_out=tok(self.v)),
            ad,
            K.quant_rows_desc(x=self.att, q=self.aq, scale=self.as_),
            lin("o", self.aq, self.as_, self.y),
            K.block_norm_desc(h=self.h, y=self.y, S=S, post_w=self.n["post1"], h_out=self.h, norm_a1=self.n["mid"],
                              z_q=self.xq, z_scale=self.xs),
            lin("gu", self.xq, self.xs, self.act, epilogue=L.RFX_EPI_GEGLU),
            K.quant_rows_desc(x=self.act, q=self.fq, scale=self.fs),
            lin("down", self.fq, self.fs, self.y),
            K.block_norm_desc(h=self.h, y=self.y, S=S, post_w=self.n["post2"], h_out=self.h, norm_a1=self.n["next"],
                              z=self.z),
        ]

    def reference(self):
        """The layer in fp64 with the weights as quantized and activations not."""
        B, S, W, H, D, F = self.dims
        c = lambda t: t.double().cpu()  # noqa: E731
        w = {k: c(self.wq[k]) * c(self.ws[k])[:, None] for k in self.wq}
        n = {k: c(v) for k, v in self.n.items()}
        rms = lambda v: v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6)  # noqa: E731
        h = c(self.h0)
        x = (rms(h) * n["in"]) @ w["qkv"].t()
        x = x.view(B, S, H + 2, D).transpose(1, 2)
        ang = torch.arange(S, dtype=torch.float64)[:, None] * c(self.freq)
        rot = x[:, :H + 1]
        a, b = rot[..., :D // 2], rot[..., D // 2:]
        rot = torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1)
        p = torch.softmax(rot[:, :H] @ rot[:, H:].transpose(-1, -2) * D ** -0.5, -1)
        att = (p @ x[:, H + 1:]).transpose(1, 2).reshape(B * S, H * D)
        h = h + rms(att @ w["o"].t()) * n["post1"]
        gu = (rms(h) * n["mid"]) @ w["gu"].t()
        act = torch.nn.functional.gelu(gu[:, :F], approximate="tanh") * gu[:, F:]
        h = h + rms(act @ w["down"].t()) * n["post2"]
        return h, rms(h) * n["next"]


@pytest.mark.parametrize("B,S,W,H,F", [(1, 1, 512, 2, 1024), (2, 50, 1024, 8, 4096), (1, 300, 1024, 4, 2050)])
def test_layer_run_together(B, S, W, H, F):
    """A whole layer on the operators, eagerly and as a captured plan replayed
    on another stream: replays are bit-identical to the eager run, and the
    residual stream agrees with the fp64 layer.  Each of the four activation
    quantizations moves a value by at most half a step of 1/127 of its row's
    absmax (about 4.5 times the rms of a row of 4096 normal values), an rms
    error of 4.5 / 127 / sqrt(12) = 1 %; with the bf16 roundings between them
    the branches stay within 4 % in the 2-norm."""
    lay = Int8Layer(B, S, W, H, F, seed=B * 10 + S)
    for d in lay.descs():
        K.Plan.run_direct(d)
    done()
    eager_h, eager_z = lay.h.clone(), lay.z.clone()
    want_h, want_z = lay.reference()
    for got, want in ((eager_h, want_h), (eager_z, want_z)):
        rel = ((got.double().cpu() - want).norm() / want.norm()).item()
        assert rel < 4e-2, rel
    plan = K.Plan()
    for d in lay.descs():
        plan.add(d)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        plan.capture(stream)
        for _ in range(3):
            lay.h.copy_(lay.h0)
            lay.z.zero_()
            plan.replay()
    stream.synchronize()
    assert K.device_status() == 0
    assert torch.equal(lay.h, eager_h) and torch.equal(lay.z, eager_z)
    assert plan.num_launches >= 11


def test_calls_on_two_streams_at_once():
    """Calls on two streams with buffers of their own do not disturb each
    other (the operators share no workspace)."""
    cases = []
    for i, (T, O, Kc) in enumerate([(50, 1024, 4096), (300, 2560, 2048)]):
        q, x = ints(20 + i, T, Kc)
        w, wd = ints(30 + i, O, Kc)
        sx, sw = torch.rand(T).cuda(), torch.rand(O).cuda()
        y = torch.empty(T, O, dtype=F32, device="cuda")
        K.linear_i8(w=wd, w_scale=sw, x=x, x_scale=sx, y=y)
        cases.append((wd, sw, x, sx, y.clone(), y, torch.cuda.Stream()))
    done()
    for *_, y, st in cases:
        y.zero_()
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for wd, sw, x, sx, want, y, st in cases:
            with torch.cuda.stream(st):
                K.linear_i8(w=wd, w_scale=sw, x=x, x_scale=sx, y=y)
    done()
    for *_, want, y, st in cases:
        assert torch.equal(want, y)


def test_offsets_past_32_bits():
    """Rows so far apart that an element's offset passes 2^31: every operator's
    outputs land where the stride says."""
    big = torch.empty((1 << 31) + (1 << 20), dtype=BF, device="cuda")  # 4.3 GB
    r = gen(8)
    x = r(2, 64).cuda()
    q = big.view(torch.int8).as_strided((2, 64), ((1 << 32) + 64, 1))
    s = torch.empty(2, device="cuda")
    K.quant_rows(x=x, q=q, scale=s)
    done()
    assert np.array_equal(q.cpu().numpy(), ref_quant(x)[0])
    for T in (2, 5):
        ld = (1 << 31) // (T - 1) + 64
        xq, xd = ints(1, T, 256)
        w, wd = ints(2, 96, 256)
        y = big.as_strided((T, 96), (ld, 1))
        K.linear_i8(w=wd, w_scale=torch.ones(96, device="cuda"), x=xd, x_scale=torch.ones(T, device="cuda"), y=y)
        done()
        want = xq.double() @ w.double().t()
        assert ((y.double().cpu() - want).abs() <= HALF[BF] * want.abs()).all()
    far = (1 << 31) + 64
    h = big.as_strided((2, 64), (far, 1))
    h.copy_(x)
    z = torch.empty(2, 64, dtype=BF, device="cuda")
    K.block_norm(h=h, S=2, z=z)
    want = x.to(BF).double()
    want = (want / torch.sqrt((want * want).mean(1, keepdim=True) + 1e-6)).cpu()
    done()
    assert ((z.double().cpu() - want).abs() <= 1.1 * HALF[BF] * want.abs()).all()
    x1 = torch.empty(2, 64, dtype=BF, device="cuda")
    x1.copy_(x)
    out = big.as_strided((1, 1, 2, 64), (far, far, far, 1))
    K.rope(x=x1, positions=torch.zeros(2, dtype=torch.int32, device="cuda"),
           inv_freq=torch.ones(32, dtype=torch.float64, device="cuda"), q_out=out)
    done()
    assert torch.equal(out[0, 0], x1)  # position 0 turns nothing


def test_captured_direct_calls_follow_their_inputs():
    """The four calls captured into a torch CUDA graph (after one eager run)
    and replayed over changed inputs give what the eager calls give."""
    r = gen(12)
    T, W, O = 50, 1024, 1536
    h, y = r(T, W).to(BF).cuda(), r(T, W).to(BF).cuda()
    w = torch.empty(O, W, dtype=torch.int8, device="cuda")
    ws = torch.empty(O, device="cuda")
    K.quant_rows(x=r(O, W).cuda(), q=w, scale=ws)
    a1 = (1 + 0.1 * r(W)).cuda()
    zq, zs = torch.empty(T, W, dtype=torch.int8, device="cuda"), torch.empty(T, device="cuda")
    h_out, qkv = torch.empty_like(h), torch.empty(T, O, dtype=BF, device="cuda")
    aq, as_ = torch.empty(T, O, dtype=torch.int8, device="cuda"), torch.empty(T, device="cuda")
    q = torch.empty(1, 4, T, 256, dtype=BF, device="cuda")
    k, v = torch.empty(1, 1, T, 256, dtype=BF, device="cuda"), torch.empty(1, 1, T, 256, dtype=BF, device="cuda")
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    freq, _ = K.rope_frequencies(256)

    def step():
        K.block_norm(h=h, y=y, S=T, h_out=h_out, norm_a1=a1, z_q=zq, z_scale=zs)
        K.linear_i8(w=w, w_scale=ws, x=zq, x_scale=zs, y=qkv)
        K.quant_rows(x=qkv, q=aq, scale=as_)
        K.rope(x=qkv, positions=pos, inv_freq=freq, q_out=q, k_out=k, v_out=v)
        return [t.clone() for t in (h_out, zq, zs, qkv, aq, as_, q, k, v)]

    step()
    done()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = step()
    for seed in (1, 2):
        r = gen(seed)
        h.copy_(r(T, W))
        y.copy_(r(T, W))
        pos.add_(100)
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        want = step()
        done()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_rope_packed_without_strides():
    """A descriptor whose strides are all 0 writes packed [B][heads][S][D] outputs."""
    r = gen(40)
    x = r(2 * 5, 8 * 64).to(BF).cuda()
    freq, _ = K.rope_frequencies(64)
    pos = torch.arange(10, dtype=torch.int32, device="cuda")
    q, k, v = (torch.empty(2, H, 5, 64, dtype=BF, device="cuda") for H in (4, 2, 2))
    d = K.rope_desc(x=x, positions=pos, inv_freq=freq, q_out=q, k_out=k, v_out=v)
    K.Plan.run_direct(d)
    done()
    want = [t.clone() for t in (q, k, v)]
    for t in (q, k, v):
        t.zero_()
    for s in ("qs", "ks", "vs"):
        for c in "bhs":
            setattr(d, f"{s}_{c}", 0)
    K.Plan.run_direct(d)
    done()
    assert all(torch.equal(a, b) for a, b in zip((q, k, v), want))


FAR = 1 << 31  # elements


@pytest.fixture(scope="module")
def far_buffer():
    """4.3 GB whose rows can lie 2^31 elements of bf16 (2^32 of int8) apart."""
    return torch.empty(FAR + (1 << 20), dtype=BF, device="cuda")


@pytest.mark.parametrize("epi", [L.RFX_EPI_STORE, L.RFX_EPI_GEGLU])
@pytest.mark.parametrize("T,off", [(129, 0), (129, 1), (129, 2), (129, 4), (300, 0), (300, 1)])
def test_linear_i8_pair_tiles_past_32_bits(far_buffer, T, off, epi):
    """Pair tiles (more than 128 tokens) into output rows whose offsets pass
    2^31 elements: by the copy where rows lie on 16 bytes, in units of 2, 4 and
    8 bytes where they do not."""
    F, Kc = 96, 256
    O = 2 * F if epi == L.RFX_EPI_GEGLU else F
    ld = FAR // (T - 1) // 8 * 8 + 64 + off
    q, x = ints(T, T, Kc)
    w, wd = ints(T + 1, O, Kc)
    sx, sw = torch.full((T,), 1e-2), torch.full((O,), 1e-2)
    y = far_buffer.as_strided((T, F), (ld, 1))
    y.fill_(7.0)
    K.linear_i8(w=wd, w_scale=sw.cuda(), x=x, x_scale=sx.cuda(), y=y, epilogue=epi)
    done()
    want, tol = ref_linear(q, w, sx, sw, None, epi)
    within(y, want, tol + 1.01 * HALF[BF] * np.abs(want))


@pytest.mark.parametrize("T", [2, 50, 200])
@pytest.mark.parametrize("which", ["x", "w"])
def test_linear_i8_operands_past_32_bits(far_buffer, T, which):
    """Token or weight rows whose offsets pass 2^32 bytes, in each of the three
    forms: integer units, weights on the M side, pair tiles."""
    O, Kc = 96, 272
    q, x = ints(T, T, Kc)
    w, wd = ints(T + 1, O, Kc)
    n = T if which == "x" else O
    ld = ((1 << 32) // (n - 1) // 16 + 4) * 16
    far = far_buffer.view(torch.int8).as_strided((n, Kc), (ld, 1))
    far.copy_(q if which == "x" else w)
    sx, sw = torch.full((T,), 1e-2), torch.full((O,), 1e-2)
    y = torch.empty(T, O, device="cuda")
    K.linear_i8(w=far if which == "w" else wd, w_scale=sw.cuda(), x=far if which == "x" else x, x_scale=sx.cuda(), y=y)
    done()
    want, tol = ref_linear(q, w, sx, sw, None, L.RFX_EPI_STORE)
    within(y, want, tol + 1.01 * U32 * np.abs(want))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("epi", [L.RFX_EPI_STORE, L.RFX_EPI_SILU, L.RFX_EPI_GELU, L.RFX_EPI_GEGLU])
@pytest.mark.parametrize("T,Kc", [(4, 256), (50, 256), (50, 4096), (300, 256), (300, 16384)])
def test_linear_i8_nonfinite_rows_and_channels_show(T, Kc, epi, dtype):
    """In every form and with every activation a token, and an output channel,
    whose scale is NaN or infinite with q 0 comes out as NaN; everything else
    has the bits that it has without them."""
    O = 128
    F = O // 2 if epi == L.RFX_EPI_GEGLU else O
    r = gen(T + Kc)
    x, w = r(T, Kc).cuda(), (r(O, Kc) / math.sqrt(Kc)).cuda()
    ys = []
    for bad in (False, True):
        xb, wb = x.clone(), w.clone()
        if bad:
            xb[1, 5], xb[T - 1, Kc - 1] = float("nan"), float("inf")
            wb[3, 0], wb[F - 1, 7] = float("-inf"), float("nan")
        q, s = torch.empty(T, Kc, dtype=torch.int8, device="cuda"), torch.empty(T, device="cuda")
        wq, ws = torch.empty(O, Kc, dtype=torch.int8, device="cuda"), torch.empty(O, device="cuda")
        K.quant_rows(x=xb, q=q, scale=s)
        K.quant_rows(x=wb, q=wq, scale=ws)
        y = torch.empty(T, F, dtype=dtype, device="cuda")
        K.linear_i8(w=wq, w_scale=ws, x=q, x_scale=s, y=y, epilogue=epi)
        ys.append(y)
    done()
    gone = torch.zeros(T, F, dtype=torch.bool, device="cuda")
    gone[[1, T - 1]] = True
    gone[:, [3, F - 1]] = True
    assert torch.isfinite(ys[0]).all()
    assert torch.isnan(ys[1][gone]).all() and torch.equal(ys[1][~gone], ys[0][~gone])
