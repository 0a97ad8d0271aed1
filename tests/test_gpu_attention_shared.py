"""Attention over a shared context on the GPU against the formula in 64 bits.

Tolerances count roundings: u = 2^-24 is half a step of fp32, 2^-8 of bf16, 2^-11
of f16.
"""
import numpy as np
import pytest
import torch

from reflex_b200 import _lib as L
from reflex_b200 import kernels as K

pytestmark = pytest.mark.gpu
D = 256
I8, U8 = L.RFX_QUANT_I8_SYM, L.RFX_QUANT_U8_REF


def gen(seed):
    g = torch.Generator().manual_seed(seed)
    return lambda *shape, std=1.0: torch.randn(*shape, generator=g) * std


def done():
    torch.cuda.synchronize()
    assert K.device_status() == 0


def make_ring(r, B, Hkv, n, mode=I8, capacity=None):
    """A ring whose first n slots hold quantized rows; the others hold what no
    row may use: huge values under NaN scales."""
    cap = capacity or max(n, 1)
    if mode == I8:
        ring = K.KVRing.allocate(B, Hkv, cap, D, mode)
    else:
        ring = K.KVRing.allocate(B, Hkv, cap, D, mode, scale_dtype=torch.bfloat16)
    ring.k_q.fill_(125)
    ring.v_q.fill_(125)
    for t in (ring.k_scale, ring.v_scale, ring.k_zp, ring.v_zp):
        if t is not None:
            t.fill_(float("nan"))
    if n:
        k = r(B, Hkv, n, D).bfloat16().cuda()
        v = (r(B, Hkv, n, D) * torch.exp(0.5 * r(B, Hkv, n, 1))).bfloat16().cuda()
        K.kv_quant_append(k, v, ring, 0, 0, cap)
    return ring


def ring_values(ring):
    """(k, v, v's quantized magnitudes) in 64 bits, [B, H, cap, D]."""
    kq, vq = ring.k_q.double().cpu(), ring.v_q.double().cpu()
    if ring.mode == I8:
        return (kq * ring.k_scale.double().cpu()[..., None]).numpy(), (vq * ring.v_scale.double().cpu()[..., None]).numpy()
    def dq(q, s, z):  # rounded to bf16 at each step, as the reference does
        s, z = s.cpu()[..., None], z.cpu()[..., None]
        return ((q.float() - z.float()).bfloat16().float() * s.float()).bfloat16().double().numpy()
    return dq(ring.k_q.cpu(), ring.k_scale, ring.k_zp), dq(ring.v_q.cpu(), ring.v_scale, ring.v_zp)


def reference(q, shared, n_shared, scale, own=None, own_len=None, k_new=None, v_new=None, new_block=None, valid=None):
    """(out, tol) [B*S, Hq*D] in 64 bits.

    tol: scores are sums of 256 products in fp32, off by at most (256 / 16 + 2) 2u
    of the sum of magnitudes and u each for the two factors after it, which
    moves a weight by that (times the score scale) and by 2^-22 for its
    exponential; a weight (times its value scale) is rounded to f16, 2^-11 of it or
    2^-25 of the largest weight; sums over n keys in fp32 add (n / 16 + 4) 2u; the
    output is rounded to bf16."""
    q = q.double().cpu().numpy()
    B, Hq, S, _ = q.shape
    ring = shared if shared is not None else own
    Hkv = ring.k_q.shape[1] if ring is not None else k_new.shape[1]
    G = Hq // Hkv
    sk, sv = ring_values(shared) if shared is not None else (None, None)
    ok, ov = ring_values(own) if own is not None else (None, None)
    kn = None if k_new is None else k_new.double().cpu().numpy()
    vn = None if v_new is None else v_new.double().cpu().numpy()
    out, tol = np.zeros((B, S, Hq, D)), np.zeros((B, S, Hq, D))
    for b in range(B):
        for h in range(Hkv):
            k, v = [np.zeros((0, D))], [np.zeros((0, D))]
            if sk is not None:
                keep = np.ones(n_shared, bool) if valid is None else valid.cpu().numpy()[:n_shared] != 0
                k.append(sk[0, h, :n_shared][keep])
                v.append(sv[0, h, :n_shared][keep])
            if ok is not None:
                n = ok.shape[2] if own_len is None else int(min(max(int(own_len[b]), 0), ok.shape[2]))
                k.append(ok[b, h, :n])
                v.append(ov[b, h, :n])
            ctx = sum(len(x) for x in k)
            seen = np.ones((S, ctx), bool)
            if kn is not None:
                k.append(kn[b, h])
                v.append(vn[b, h])
                blk = np.zeros(S) if new_block is None else new_block.cpu().numpy()[:S]
                seen = np.concatenate([seen, blk[None, :] <= blk[:, None]], axis=1)
            k, v = np.concatenate(k), np.concatenate(v)
            if len(k) == 0:
                continue
            qq = q[b, h * G:(h + 1) * G].reshape(G * S, D)
            see = np.tile(seen, (G, 1))
            z = np.where(see, qq @ k.T * scale, -np.inf)
            mag = np.abs(qq) @ np.abs(k).T * abs(scale)
            top = z.max(axis=1, keepdims=True)
            w = np.exp(z - np.where(np.isfinite(top), top, 0))
            l = w.sum(axis=1, keepdims=True)
            ok_row = l > 0
            p = np.divide(w, l, out=np.zeros_like(w), where=ok_row)
            o = p @ v
            u = 2.0 ** -24
            ds = (18 * 2 * u + 2 * u) * mag + 4 * u * np.abs(np.where(see, z, 0)) + 2.0 ** -21
            av = np.abs(v)
            d = (p * ds) @ av + (p * ds).sum(axis=1, keepdims=True) * (p @ av)
            d += 2.0 ** -11 * (p @ av) + (2.0 ** -25 / np.maximum(l, 1e-300)) * (np.minimum(1, see) @ np.minimum(av, 127.0)) * ok_row
            d += (len(k) / 16 + 4) * 2 * u * (p @ av)
            d += 2.0 ** -8 * (np.abs(o) + d) + 1e-38
            out[b, :, h * G:(h + 1) * G] = o.reshape(G, S, D).transpose(1, 0, 2)
            tol[b, :, h * G:(h + 1) * G] = d.reshape(G, S, D).transpose(1, 0, 2)
    return out.reshape(B * S, Hq * D), tol.reshape(B * S, Hq * D)


def check(got, want, tol):
    got = got.double().cpu().numpy()
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), bad.size, float(np.nanmax(np.abs(got - want) / tol)), np.argwhere(bad)[:4].tolist())


def case(B, S, Hq, Hkv, n_shared, own, new, seed=0, mode=I8, blocks=False, holes=False, token_major=True, lens=None):
    r = gen(seed + 7 * B + 31 * S + n_shared)
    c = dict(q=(2 * r(B, Hq, S, D)).bfloat16().cuda(), n_shared=n_shared, softmax_scale=D ** -0.5,
             shared=make_ring(r, 1, Hkv, n_shared, mode, n_shared + 5) if n_shared else None)
    if own:
        c["own"] = make_ring(r, B, Hkv, own, mode, own + 3)
        c["own_max"] = own
        if lens is None:
            lens = torch.randint(0, own + 1, (B,), generator=torch.Generator().manual_seed(seed))
        c["own_len"] = torch.as_tensor(lens, dtype=torch.int32).cuda()
        ring = c["own"]  # what lies past a stream's length must not matter
        for b in range(B):
            n = min(max(int(c["own_len"][b]), 0), own)
            for t in (ring.k_scale, ring.v_scale, ring.k_zp, ring.v_zp):
                if t is not None:
                    t[b, :, n:] = float("nan")
    if new:
        mk = (lambda: r(B, S, Hkv, D).bfloat16().cuda().transpose(1, 2)) if token_major else (lambda: r(B, Hkv, S, D).bfloat16().cuda())
        c["k_new"], c["v_new"] = mk(), mk()
        if blocks:
            c["new_block"] = torch.as_tensor(np.sort(np.arange(S) * 3 // max(S, 1) - 1), dtype=torch.int32).cuda()
    if holes and n_shared:
        c["shared_valid"] = (torch.rand(n_shared, generator=torch.Generator().manual_seed(seed)) > 0.3).to(torch.uint8).cuda()
    return c


def run(c, out=None):
    B, Hq, S, _ = c["q"].shape
    if out is None:
        out = torch.full((B * S, Hq * D), 55.0, dtype=torch.bfloat16, device="cuda")
    K.attention_shared(out=out, **c)
    done()
    return out


def want_of(c):
    own = c.get("own")
    lens = None if own is None else c["own_len"].cpu().clamp(0, c["own_max"])
    return reference(c["q"], c["shared"], c["n_shared"], c["softmax_scale"], own, lens, c.get("k_new"), c.get("v_new"),
                     c.get("new_block"), c.get("shared_valid"))


SHAPES = [
    (1, 1, 8, 1, 5000, 0, False),
    (64, 50, 8, 1, 300, 0, True),
    (30, 9, 8, 1, 3000, 100, True),
    # B, S, Hq, Hkv, n_shared, own, new
    (1, 1, 1, 1, 1, 0, False),
    (1, 1, 8, 1, 100, 0, True),
    (2, 1, 8, 1, 128, 5, False),
    (3, 50, 8, 1, 818, 0, True),
    (4, 51, 8, 1, 129, 40, True),
    (16, 1, 8, 1, 1000, 200, True),
    (17, 1, 8, 1, 300, 130, False),
    (5, 3, 4, 1, 257, 64, True),
    (9, 1, 3, 1, 70, 10, True),
    (43, 1, 3, 3, 64, 3, True),
    (3, 7, 8, 2, 200, 20, True),
    (2, 130, 2, 1, 0, 0, True),
    (3, 5, 2, 1, 0, 129, False),
    (2, 16, 8, 1, 500, 128, True),
    (64, 2, 8, 4, 40, 8, True),
    (20, 50, 8, 1, 250, 0, True),
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_matches_formula(shape):
    c = case(*shape)
    check(run(c), *want_of(c))


@pytest.mark.parametrize("shape", [SHAPES[i] for i in (4, 7, 8, 13)], ids=str)
def test_uint8_scheme(shape):
    c = case(*shape, mode=U8)
    check(run(c), *want_of(c))


@pytest.mark.parametrize("shape", [SHAPES[i] for i in (1, 2, 6, 7, 10, 13, 16)], ids=str)
@pytest.mark.parametrize("holes", [False, True])
def test_masks(shape, holes):
    """Block-causal new tokens (ids from -1 on), masked shared slots."""
    c = case(*shape, blocks=True, holes=holes, token_major=False, seed=3)
    check(run(c), *want_of(c))
