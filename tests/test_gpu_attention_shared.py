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
    """(k, v) in 64 bits, [B, H, cap, D]."""
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
    exponential; a weight times its value scale is rounded to f16, by 2^-11 of it or,
    among the subnormal numbers (steps of 2^-24), by 2^-25, and multiplies an integer
    of at most 127 (a ring's int8 value, which its scale does not shrink there) or the
    value itself (scale 1): (2^-25 / l) sum of those, with the largest weight 1; a bf16
    value is exact in f16 (8 of 11 bits) from 2^-14 on and off by 2^-25 below, which the
    weights' mean keeps: 2^-25; sums
    over n keys in fp32 add (n / 16 + 4) 2u; the output is rounded to bf16."""
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
            operand = av.copy()  # what the rounded weights multiply
            if ring is not None and ring.mode == I8:
                operand[:ctx] = 127.0
            d = (p * ds) @ av + (p * ds).sum(axis=1, keepdims=True) * (p @ av)
            d += 2.0 ** -11 * (p @ av) + (2.0 ** -25 / np.maximum(l, 1e-300)) * (np.minimum(1, see) @ operand) * ok_row
            d += (len(k) / 16 + 4) * 2 * u * (p @ av) + 2.0 ** -25 * ok_row
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
    (64, 40, 8, 1, 1500, 0, True),   # tiles in parts that the last CTA joins
    (70, 37, 8, 1, 1200, 30, True),
    (64, 1, 8, 1, 1000, 70, True),
    (130, 1, 4, 1, 5000, 20, True),
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


def test_rows_without_keys_are_zero():
    """No keys at all, none valid, rings of length 0: rows of zeros; a stream
    with keys beside one without."""
    c = case(2, 3, 8, 1, 0, 0, False)
    c["own"], c["own_max"] = make_ring(gen(1), 2, 1, 4), 0
    assert (run(c) == 0).all()
    for S in (1, 50):
        c = case(3, S, 8, 1, 200, 0, False, holes=True)
        c["shared_valid"].zero_()
        assert (run(c) == 0).all()
        c = case(5, S, 8, 1, 0, 70, False, lens=[0, 70, 0, 3, -5])
        out = run(c)
        check(out, *want_of(c))
        assert (out.view(5, S, -1)[[0, 2, 4]] == 0).all()


@pytest.mark.parametrize("S", [1, 40])
def test_lengths_beyond_the_ring_are_clamped(S):
    c = case(4, S, 8, 1, 100, 60, True, lens=[60, 60, 0, 10])
    want = run(c).clone()
    c["own_len"].copy_(torch.tensor([1000, 0x7fffffff, -0x80000000, 10], dtype=torch.int32))
    assert torch.equal(run(c), want)


@pytest.mark.parametrize("S", [1, 30])
def test_nan_of_one_stream_stays_there(S):
    """A NaN or an infinity in one stream's own ring or new keys (also values beyond
    f16) makes that stream's rows NaN that see it, and changes no other stream's bits."""
    c = case(6, S, 8, 1, 300, 90, True, lens=[90, 50, 90, 10, 0, 64], blocks=S > 1)
    want = run(c).view(6, S, 8, D).clone()
    c["own"].v_scale[1, :, 49] = float("nan")
    c["v_new"][3, 0, 0, 5] = float("inf")
    c["v_new"][4, 0, S - 1, 7] = 1e6
    c["k_new"][5, 0, S - 1, 9] = float("nan")
    got = run(c).view(6, S, 8, D)
    assert torch.equal(got[[0, 2]], want[[0, 2]])
    assert got[1].isnan().all() and got[3].isnan().all()
    assert got[4, S - 1].isnan().all() and got[5, S - 1].isnan().all()
    if S > 1:  # tokens of earlier blocks do not see the last block's
        assert torch.equal(got[4:, 0], want[4:, 0])


def test_masked_slots_may_hold_anything():
    for S in (1, 50):
        c = case(8, S, 8, 1, 500, 0, True, holes=True, seed=5)
        want = run(c).clone()
        off = c["shared_valid"] == 0
        c["shared"].k_scale[0, 0, :500][off] = float("nan")
        c["shared"].v_scale[0, 0, :500][off] = float("inf")
        assert torch.equal(run(c), want)


@pytest.mark.parametrize("shape", [(64, 50, 8, 1, 300, 0, True), (30, 9, 8, 1, 3000, 100, True), (16, 51, 8, 1, 2000, 48, True),
                                   (3, 1, 8, 1, 9000, 20, True), (64, 1, 8, 1, 6000, 70, False), (64, 40, 8, 1, 1500, 0, True)], ids=str)
def test_same_bits_every_time(shape):
    """Whichever CTA of a tile ends last, its parts are added in one order."""
    c = case(*shape)
    want = run(c).clone()
    for _ in range(30):
        assert torch.equal(run(c), want)


@pytest.mark.parametrize("S", [1, 20])
def test_layouts(S):
    """Strided q, keys, rings and out (rings of a larger one's slots and layers): the same bits
    as dense ones, and nothing beside out's rows is written."""
    B, Hq = 5, 8
    c = case(B, S, Hq, 1, 260, 40, True)
    want = run(c).clone()

    def spread(t, *dims):  # the same values, `dims` other strides
        big = torch.full([2 * n if i in dims else n for i, n in enumerate(t.shape)], 99, dtype=t.dtype, device="cuda")
        view = big[tuple(slice(0, 2 * n, 2) if i in dims else slice(None) for i, n in enumerate(t.shape))]
        view.copy_(t)
        return view
    c["q"] = c["q"].transpose(1, 2).contiguous().transpose(1, 2)
    c["k_new"], c["v_new"] = spread(c["k_new"], 0, 1), spread(c["v_new"], 2)
    for name in ("shared", "own"):
        ring = c[name]
        c[name] = K.KVRing(spread(ring.k_q, 0, 2), spread(ring.v_q, 0, 2), spread(ring.k_scale, 1, 2), spread(ring.v_scale, 1, 2),
                           None, None, ring.mode)
    buf = torch.full((B * S + 2, Hq * D + 24), 7.0, dtype=torch.bfloat16, device="cuda")
    out = buf[1:-1, 8:8 + Hq * D]
    assert torch.equal(run(c, out), want)
    assert (buf[0] == 7).all() and (buf[-1] == 7).all() and (buf[:, :8] == 7).all() and (buf[:, 8 + Hq * D:] == 7).all()


@pytest.mark.parametrize("S", [1, 40])
def test_slots_past_32_bits(S):
    """Slots so far apart that a byte's offset passes 2^32."""
    c = case(2, S, 8, 1, 3, 2, False, lens=[2, 1])
    want = run(c).clone()
    big = torch.empty((1 << 32) + (1 << 22), dtype=torch.int8, device="cuda")

    def far(t, n, at, step):
        view = big[at:].as_strided((t.shape[0], 1, n, D), (1 << 16, D, step, 1))
        view.copy_(t[:, :, :n])
        return view
    sh, own = c["shared"], c["own"]
    c["shared"] = K.KVRing(far(sh.k_q, 3, 0, 1 << 31), far(sh.v_q, 3, 4096, 1 << 31), sh.k_scale[:, :, :3], sh.v_scale[:, :, :3], None, None, I8)
    c["own"] = K.KVRing(far(own.k_q, 2, 8192, 1 << 32), far(own.v_q, 2, 12288, 1 << 32), own.k_scale[:, :, :2], own.v_scale[:, :, :2], None, None, I8)
    assert torch.equal(run(c), want)


@pytest.mark.parametrize("shape", [(3, 1, 8, 1, 700, 30, True), (64, 50, 8, 1, 300, 0, True), (64, 1, 8, 1, 6000, 70, True), (64, 40, 8, 1, 1500, 0, True)], ids=str)
def test_captured_calls_follow_their_inputs(shape):
    """Two graphs captured over one workspace and a plan, replayed over changed inputs
    and lengths on another stream: what the eager calls give, bit for bit."""
    full = [shape[5]] * shape[0]  # (what lies past a length is NaN)
    c, other = case(*shape, seed=1, lens=full), case(*shape, seed=2, lens=full)
    out, out2 = torch.empty_like(run(c)), torch.empty_like(run(c))
    need = K.attention_shared_workspace_bytes(K.attention_shared_desc(out=out, **c))
    ws = torch.full((need + 1024,), 0xFF, dtype=torch.uint8, device="cuda")
    K.attention_shared(out=out, workspace=ws, **c)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    with torch.cuda.graph(graphs[0]):
        K.attention_shared(out=out, workspace=ws, **c)
    with torch.cuda.graph(graphs[1]):
        K.attention_shared(out=out2, workspace=ws, **other)
    plan, out3 = K.Plan(), torch.empty_like(out)
    plan.add(K.attention_shared_desc(out=out3, workspace=ws, **c))
    st, r = torch.cuda.Stream(), gen(9)
    for i in range(3):
        c["q"].copy_(r(*c["q"].shape))
        if "k_new" in c:
            c["k_new"].copy_(r(*c["k_new"].shape))
        if "own_len" in c:
            c["own_len"].copy_(torch.randint(0, c["own_max"] + 1, c["own_len"].shape, generator=torch.Generator().manual_seed(i)))
        want, want2 = run(c).clone(), run(other).clone()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            for g in graphs * 3:
                g.replay()
        st.synchronize()
        plan.run()
        done()
        assert torch.equal(out2, want2) and torch.equal(out3, want) and torch.equal(out, want)


def test_too_small_a_workspace_is_replaced():
    c = case(64, 50, 8, 1, 300, 0, True)
    want = run(c).clone()
    assert torch.equal(run(dict(c, workspace=torch.empty(4096, dtype=torch.uint8, device="cuda"))), want)


def test_two_streams_at_once():
    cs = [case(64, 50, 8, 1, 300, 0, True), case(3, 1, 8, 1, 700, 30, True), case(64, 1, 8, 1, 6000, 70, True)]
    outs = [run(c) for c in cs]
    want = [o.clone() for o in outs]
    sts = [torch.cuda.Stream() for _ in cs]
    need = [K.attention_shared_workspace_bytes(K.attention_shared_desc(out=o, **c)) for c, o in zip(cs, outs)]
    wss = [torch.empty(n + 1024, dtype=torch.uint8, device="cuda") for n in need]
    for o, st in zip(outs, sts):
        o.zero_()
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for c, o, ws, st in zip(cs, outs, wss, sts):
            with torch.cuda.stream(st):
                K.attention_shared(out=o, workspace=ws, **c)
    done()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_wrong_sizes_are_refused():
    c = case(2, 3, 8, 1, 64, 16, True)
    out = run(c)
    bad = [dict(q=c["q"].float()), dict(q=c["q"][0]), dict(q=c["q"].transpose(2, 3)), dict(n_shared=70), dict(shared=None),
           dict(own_max=20), dict(own_len=c["own_len"].long()), dict(own_len=c["own_len"][:1]), dict(own=None),
           dict(k_new=None), dict(v_new=c["v_new"][:, :, :2]), dict(k_new=c["k_new"].float()),
           dict(new_block=torch.zeros(2, dtype=torch.int32, device="cuda")), dict(new_block=torch.zeros(3, device="cuda")),
           dict(shared_valid=torch.ones(63, dtype=torch.uint8, device="cuda")), dict(shared_valid=torch.ones(64, device="cuda")),
           dict(out=out[:5]), dict(out=out.float()), dict(out=out.cpu()), dict(workspace=torch.empty(4096, dtype=torch.uint8)),
           dict(own=make_ring(gen(1), 2, 1, 16, U8)), dict(shared=make_ring(gen(1), 1, 2, 64))]
    for kw in bad:
        with pytest.raises(ValueError):
            K.attention_shared(**{**c, "out": out, **kw})
    for kw in (dict(q=c["q"][..., :128]), dict(out=c["q"].view(-1)[:6 * 2048].view(6, 2048))):
        with pytest.raises((ValueError, L.RfxError)):
            K.attention_shared(**{**c, "out": out, **kw})
    done()


@pytest.mark.parametrize("fmt", [L.RFX_FP4_MX, L.RFX_FP4_NV])
@pytest.mark.parametrize("B,S,W,H,F", [(1, 1, 512, 2, 1024), (4, 1, 1024, 8, 2048), (6, 50, 1024, 8, 2048)])
def test_layer_run_together(fmt, B, S, W, H, F):
    """A layer of candidate streams over one prompt on the 4-bit operators and the
    attention, beside the norms and rotary positions that the library has: every stage
    against the formula of what the stage before really left, and a captured plan's
    replays on another stream bit-identical to the eager run."""
    import math
    import test_gpu_fp4 as P
    r, T, ctx = gen(B + S), B * S, 300
    e = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    w = {k: P.quantized(r(o, i) / math.sqrt(i), fmt, parts) for k, o, i, parts in
         (("qkv", (H + 2) * D, W, 1), ("o", W, H * D, 1), ("gu", 2 * F, W, 2), ("down", W, F, 1))}
    n = [(1 + 0.1 * r(W)).cuda() for _ in range(5)]
    h0 = r(T, W).bfloat16().cuda()
    h, z, qkv, att, y, act, last = h0.clone(), e(T, W), e(T, (H + 2) * D), e(T, H * D), e(T, W), e(T, F), e(T, W)
    q, kn, vn = e(B, H, S, D), e(B, 1, S, D), e(B, 1, S, D)
    zq, aq, fq = (K.Fp4Rows.allocate(T, k, fmt) for k in (W, H * D, F))
    mq = K.Fp4Rows.allocate(T, W, fmt)
    z2 = e(T, W)
    shared = make_ring(r, 1, 1, ctx)
    pos = (ctx + torch.arange(S, dtype=torch.int32)).repeat(B).cuda()
    freq, _ = K.rope_frequencies(D)
    ad = dict(q=q, shared=shared, n_shared=ctx, k_new=kn, v_new=vn, out=att, softmax_scale=D ** -0.5)
    need = K.attention_shared_workspace_bytes(K.attention_shared_desc(**ad))
    ws = torch.empty(need + 1024, dtype=torch.uint8, device="cuda")
    descs = [
        K.block_norm_desc(h=h, S=S, norm_a1=n[0], z=z),
        K.quant_fp4_desc(x=z, out=zq),
        K.linear_fp4_desc(w=w["qkv"], x=zq, y=qkv),
        K.rope_desc(x=qkv, positions=pos, inv_freq=freq, q_out=q, k_out=kn, v_out=vn),
        K.attention_shared_desc(workspace=ws, **ad),
        K.quant_fp4_desc(x=att, out=aq),
        K.linear_fp4_desc(w=w["o"], x=aq, y=y),
        K.block_norm_desc(h=h, y=y, S=S, post_w=n[1], h_out=h, norm_a1=n[2], z=z2),
        K.quant_fp4_desc(x=z2, out=mq),
        K.linear_fp4_desc(w=w["gu"], x=mq, y=act, epilogue=L.RFX_EPI_GEGLU),
        K.quant_fp4_desc(x=act, out=fq),
        K.linear_fp4_desc(w=w["down"], x=fq, y=last),
    ]
    for d in descs:
        K.Plan.run_direct(d)
    done()

    def stage(rows, weight, got, epi=L.RFX_EPI_STORE):
        want, tol = P.ref_linear(P.values(rows), P.values(weight), None, epi)
        check(got, want, tol + 2.0 ** -8 * (np.abs(want) + tol) + 1e-38)
    for x, rows in ((z, zq), (att, aq), (z2, mq), (act, fq)):
        again = P.quantized(x.cpu(), fmt)
        assert torch.equal(again.q, rows.q) and torch.equal(again.scale, rows.scale)
    stage(zq, w["qkv"], qkv)
    check(att, *reference(q, shared, ctx, D ** -0.5, None, None, kn, vn))
    stage(aq, w["o"], y)
    stage(mq, w["gu"], act, L.RFX_EPI_GEGLU)
    stage(fq, w["down"], last)
    want = [t.clone() for t in (h, att, act, last)]
    plan = K.Plan()
    for d in descs:
        plan.add(d)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        h.copy_(h0)
        plan.capture(st)
        for _ in range(3):
            h.copy_(h0)
            last.zero_()
            plan.replay()
    st.synchronize()
    assert K.device_status() == 0
    assert all(torch.equal(a, b) for a, b in zip((h, att, act, last), want))
