"""Attention over a shared context on the GPU where a row's softmax is hard: maxima that
rise from block to block, block ids at the ends of int32, values far from 1.  Against the formula in 64 bits, with the tolerance that is
derived beside it.
"""
import numpy as np
import pytest
import torch

import test_gpu_attention_shared as A
from reflex_b200 import kernels as K

pytestmark = pytest.mark.gpu
D, I8, U8 = A.D, A.I8, A.U8


def ring_of(k, v, capacity=None, mode=I8, scale_dtype=None):
    """A ring [B, H, n, D] of these keys and values; slots past them hold what no row may use."""
    B, H, n, _ = k.shape
    ring = K.KVRing.allocate(B, H, capacity or n, D, mode, **({} if scale_dtype is None else dict(scale_dtype=scale_dtype)))
    ring.k_q.fill_(125)
    ring.v_q.fill_(125)
    for t in (ring.k_scale, ring.v_scale, ring.k_zp, ring.v_zp):
        if t is not None:
            t.fill_(float("nan"))
    t = scale_dtype or torch.bfloat16
    K.kv_quant_append(k.to(t).cuda(), v.to(t).cuda(), ring, 0, 0, ring.capacity)
    return ring


# B, S, Hq, n_shared, own: clusters, whole tiles, tiles that the last CTA joins, tiles that
# a kernel joins, few rows
RISING = [(4, 50, 8, 818, 0), (64, 50, 8, 818, 0), (64, 40, 8, 1500, 70), (16, 51, 8, 3000, 130), (64, 1, 8, 6000, 200),
          (3, 5, 8, 700, 90), (1, 1, 8, 5000, 0)]


def rising(B, S, Hq, n_shared, own, holes):
    """Keys along 16 directions whose scores rise by 17 log2 units per 64 keys up to a block
    that is another one for each, and rows of which two in three look along one of them."""
    c = A.case(B, S, Hq, 1, n_shared, own, True, seed=11, holes=holes)
    r = A.gen(B + S + n_shared)
    blocks = (n_shared + own) // 64 + 1

    def keys(B, n, first):
        k = 0.3 * r(B, 1, n, D)
        at = (first + torch.arange(n)) // 64
        for d in range(16):
            k[..., d] += 12.0 * torch.clamp(at, max=1 + (d + 1) * blocks // 16).float()
        return k
    c["shared"] = ring_of(keys(1, n_shared, 0), r(1, 1, n_shared, D), n_shared + 5)
    if own:
        c["own"] = ring_of(keys(B, own, n_shared), r(B, 1, own, D))
    q = 0.3 * r(B, Hq, S, D)
    row = torch.arange(B * Hq * S).view(B, Hq, S)
    look = torch.nn.functional.one_hot(row * 7 % 16, D).float() * 16.0
    c["q"] = torch.where((row % 3 != 0)[..., None], q + look, q).bfloat16().cuda()
    return c


@pytest.mark.parametrize("shape", RISING, ids=str)
@pytest.mark.parametrize("holes", [False, True])
def test_maxima_that_rise_in_every_block(shape, holes):
    """O is rescaled in nearly every block, for some rows of a warp and not for others: the
    formula's values, and the same bits each time."""
    c = rising(*shape, holes)
    want = A.run(c).clone()
    A.check(want, *A.want_of(c))
    for _ in range(20):
        assert torch.equal(A.run(c), want)


LOW, TOP = -0x80000000, 0x7fffffff
IDS = [[TOP], [LOW], [LOW, LOW + 1], [LOW + 1, LOW, LOW], [TOP - 1, TOP, TOP - 1], [LOW, LOW + 1, -1, 0, TOP - 1, TOP],
       [TOP] * 17, [LOW] * 9 + [TOP] * 11]


@pytest.mark.parametrize("ids", IDS, ids=lambda v: "-".join(map(str, v[:6])))
@pytest.mark.parametrize("B,n_shared,own", [(1, 0, 0), (3, 100, 20), (5, 0, 70), (70, 150, 9)])
def test_block_ids_are_any_numbers(ids, B, n_shared, own):
    """Ids from the lowest to the highest int32, in both forms: key j is seen by token i iff
    id j <= id i, ring slots by all tokens of their stream, and places without a key by none."""
    S = len(ids)
    for Hq in (1, 8):
        c = A.case(B, S, Hq, 1, n_shared, own, True, seed=S)
        c["new_block"] = torch.tensor(ids, dtype=torch.int32).cuda()
        A.check(A.run(c), *A.want_of(c))


@pytest.mark.parametrize("S", [1, 50])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_rows_without_keys_are_zero_whatever_their_query_holds(S, bad):
    """A query that is not finite makes its row NaN where the row sees a key, and leaves it 0 where
    it sees none; no other row's bits change."""
    B = 6
    c = A.case(B, S, 8, 1, 200, 70, False, lens=[0, 70, 0, 3, 70, 0], seed=2)
    c["shared_valid"] = torch.zeros(200, dtype=torch.uint8).cuda()
    want = A.run(c).view(B, S, 8, D).clone()
    assert (want[[0, 2, 5]] == 0).all()
    c["q"][0] = bad
    c["q"][2, 3, S - 1, 200] = -bad
    c["q"][4, 1, 0, 7] = bad
    got = A.run(c).view(B, S, 8, D)
    assert (got[[0, 2, 5]] == 0).all()
    assert got[4, 0, 1].isnan().all()
    got[4, 0, 1] = want[4, 0, 1]
    assert torch.equal(got, want)
    c["shared_valid"][199] = 1
    got = A.run(c).view(B, S, 8, D)
    assert got[0].isnan().all() and got[2, S - 1, 3].isnan().all() and not got[5].isnan().any()


def values_of(ring):
    """(k, v) in 64 bits, as the kernels multiply them: with fp32 scales in the uint8 scheme keys
    are rounded to bf16 and values to f16."""
    if ring.mode == I8 or ring.k_scale.dtype == torch.bfloat16:
        return A.ring_values(ring)
    dq = lambda q, s, z: (q.cpu().float() - z.cpu()[..., None]) * s.cpu()[..., None]  # noqa: E731
    return (dq(ring.k_q, ring.k_scale, ring.k_zp).bfloat16().double().numpy(),
            dq(ring.v_q, ring.v_scale, ring.v_zp).half().double().numpy())


def exact(c):
    """(out, tol) of a call without new keys, in 64 bits, for values of any size.

    As in the formula's other test, but what a weight times its value scale loses among the
    small numbers of f16: weights are relative to the row's largest (score x block's largest value
    scale, rounded up to a power of two), which is 2^15 to 2^7 there, so half a step of 2^-24 is
    at most 2^-25 * 2^-7 * 2 * (the largest value scale) of the largest weight, times an integer of
    at most 127 (times the value itself in the uint8 scheme, where the scale is 1)."""
    q = c["q"].double().cpu().numpy()
    B, Hq, S, _ = q.shape
    i8 = c["shared"].mode == I8
    n, own = c["n_shared"], c.get("own")
    sk, sv = values_of(c["shared"])
    scale = c["shared"].v_scale.double().cpu().numpy()
    ok, ov = values_of(own) if own is not None else (None, None)
    os_ = None if own is None else own.v_scale.double().cpu().numpy()
    keep = np.ones(n, bool) if "shared_valid" not in c else c["shared_valid"].cpu().numpy() != 0
    # (the shared part of all streams is one array: copies of it would be most of the time)
    first = (sk[0, 0, :n][keep], sv[0, 0, :n][keep], scale[0, 0, :n][keep])
    first_abs = np.abs(first[0]), np.abs(first[1])
    out, tol = np.zeros((B, S, Hq, D)), np.zeros((B, S, Hq, D))
    for b in range(B):
        parts = [(*first, *first_abs)]
        if own is not None:
            m = int(c["own_len"][b])
            parts.append((ok[b, 0, :m], ov[b, 0, :m], os_[b, 0, :m], np.abs(ok[b, 0, :m]), np.abs(ov[b, 0, :m])))
        qq = q[b].reshape(Hq * S, D)
        z = np.concatenate([qq @ k.T for k, *_ in parts], axis=1) * c["softmax_scale"]
        mag = np.concatenate([np.abs(qq) @ ak.T for *_, ak, _ in parts], axis=1) * c["softmax_scale"]
        w = np.exp(z - z.max(axis=1, keepdims=True))
        l = w.sum(axis=1, keepdims=True)
        p, u, keys = w / l, 2.0 ** -24, z.shape[1]
        ds = p * (38 * u * mag + 4 * u * np.abs(z) + 2.0 ** -21)

        def times(a, which):  # a [rows, keys] by the parts' values
            at = np.cumsum([0] + [len(x[0]) for x in parts])
            return sum(a[:, s:e] @ x[which] for s, e, x in zip(at, at[1:], parts))
        o, pa = times(p, 1), times(p, 4)
        d = times(ds, 4) + ds.sum(axis=1, keepdims=True) * pa + 2.0 ** -11 * pa
        top = max(x[2].max(initial=0) for x in parts)
        d += 2.0 ** -31 / l * (127.0 * keys * top if i8 else sum(x[4].sum(axis=0) for x in parts)) + (keys / 16 + 4) * 2 * u * pa
        d += 0.0 if i8 else 2.0 ** -11 * pa + 2.0 ** -25  # (V itself in f16)
        d += 2.0 ** -8 * (np.abs(o) + d)
        out[b], tol[b] = (x.reshape(Hq, S, D).transpose(1, 0, 2) for x in (o, d))
    return out.reshape(B * S, Hq * D), tol.reshape(B * S, Hq * D)


@pytest.mark.parametrize("size", [1e-7, 1e-4, 0.01, 0.03, 1.0, 1e3, 1e6, 1e15])
@pytest.mark.parametrize("shape", [(1, 1, 8, 5000, 0), (3, 5, 8, 700, 90), (64, 50, 8, 300, 40), (64, 1, 8, 32768, 70), (16, 51, 8, 3000, 0)],
                         ids=str)
def test_values_of_any_size(shape, size):
    """Values far from 1, some keys' 1000 times as large as others': as exact as values near 1."""
    B, S, Hq, n, own = shape
    c = A.case(B, S, Hq, 1, n, own, False, seed=5)
    r = A.gen(n + own)
    spread = lambda *s: size * torch.exp(1.2 * r(*s, 1)) * r(*s, D)  # noqa: E731
    c["shared"] = ring_of(r(1, 1, n, D), spread(1, 1, n), n + 5)
    if own:
        c["own"] = ring_of(r(B, 1, own, D), spread(B, 1, own))
    A.check(A.run(c), *exact(c))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [0.01, 1.0, 300.0])
@pytest.mark.parametrize("shape", [(1, 1, 8, 500, 0), (3, 5, 8, 257, 64), (64, 50, 8, 300, 40), (64, 1, 8, 6000, 70)], ids=str)
def test_uint8_scheme_with_scales_of_either_type(shape, size, dtype):
    B, S, Hq, n, own = shape
    c = A.case(B, S, Hq, 1, n, own, False, seed=6, mode=U8, holes=True)
    r = A.gen(n + own)
    c["shared"] = ring_of(r(1, 1, n, D), size * r(1, 1, n, D), n + 5, U8, dtype)
    if own:
        c["own"] = ring_of(r(B, 1, own, D), size * r(B, 1, own, D), own, U8, dtype)
    A.check(A.run(c), *exact(c))
