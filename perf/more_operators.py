"""The measured cases of the 4-bit layer operators and of the attention over a
shared context, with their plain forms.

What a batch of streams over one observation runs through in a layer whose
weights and activations are held as 4-bit floating point numbers:

* ``quant_fp4``         rows of a matrix to e2m1 values (0, 0.5, 1, 1.5, 2, 3, 4, 6
  and their negatives) with a scale per block: a power of two per 32 (``mx``),
  or an e4m3 number per 16 under a power of two per row (``nv``); and
  ``dequant_fp4`` back to what they stand for;
* ``linear_fp4``        x @ w^T over such rows, with bias and activation;
* ``attention_shared``  the attention of B streams over one context that they
  all share, each stream's own context of its own length, and its new tokens.

With ``own`` false ``run`` computes them in elementary torch operations; with
``own`` true it calls the library.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
BLOCK = {"mx": 32, "nv": 16}
D = 256  # head dim of the int8 rings


# ------------------------------------------------------------------ cases ---
def listed():
    return [
        # one token's MLP activations before its down projection: pure latency
        {"name": "quant_token", "op": "quant", "fmt": "nv", "type": "bf16", "T": 1, "K": 4096},
        # 64 streams' normed residual stream before their QKV projection
        {"name": "quant_streams", "op": "quant", "fmt": "mx", "type": "bf16", "T": 3200, "K": 1024},
        # the GeGLU output of a 768-token camera frame (2B-shape prefix layer)
        {"name": "quant_frame", "op": "quant", "fmt": "nv", "type": "bf16", "T": 768, "K": 16384},
        # one token through the prefix layer's fused QKV projection
        {"name": "linear_token_qkv", "op": "linear", "fmt": "nv", "type": "bf16", "T": 1, "K": 2048, "O": 2560,
         "epi": "store", "bias": False},
        # the action expert's gate/up projection for one stream's 50 tokens
        {"name": "linear_expert_geglu", "op": "linear", "fmt": "mx", "type": "bf16", "T": 50, "K": 1024, "O": 8192,
         "epi": "geglu", "bias": False},
        # the vision tower's fc1 over three cameras: K and O no multiple of a tile
        {"name": "linear_vision_fc1", "op": "linear", "fmt": "mx", "type": "bf16", "T": 768, "K": 1152, "O": 4304,
         "epi": "gelu", "bias": True},
        # the action expert's down projection of 64 streams of 50 tokens
        {"name": "linear_streams_down", "op": "linear", "fmt": "nv", "type": "bf16", "T": 3200, "K": 4096, "O": 1024,
         "epi": "store", "bias": False},
        # the prefix layer's gate/up projection of a frame: the largest product
        {"name": "linear_frame_geglu", "op": "linear", "fmt": "nv", "type": "bf16", "T": 768, "K": 2048, "O": 32768,
         "epi": "geglu", "bias": False},
        # four candidate chunks of one observation (818 context tokens)
        {"name": "attn_four_candidates", "op": "attn", "B": 4, "S": 50, "Hq": 8, "Hkv": 1, "shared": 818, "own": 0,
         "new": True, "blocks": False, "holes": False},
        # 64 of them
        {"name": "attn_candidates", "op": "attn", "B": 64, "S": 50, "Hq": 8, "Hkv": 1, "shared": 818, "own": 0,
         "new": True, "blocks": False, "holes": False},
        # state token and actions (block-causal) of 16 streams: a long shared context with masked slots, and
        # each stream's own few tokens
        {"name": "attn_long_blocks", "op": "attn", "B": 16, "S": 51, "Hq": 8, "Hkv": 1, "shared": 6344, "own": 48,
         "new": True, "blocks": True, "holes": True},
        # single tokens of 64 streams that branched off one long prefix
        {"name": "attn_tokens", "op": "attn", "B": 64, "S": 1, "Hq": 8, "Hkv": 1, "shared": 32768, "own": 200,
         "new": False, "blocks": False, "holes": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quant", "linear", "linear", "attn", "attn"])
    if op == "quant":
        K = _log_int(rng, 16, 16384)
        T = _log_int(rng, 1, min(4096, (1 << 23) // K))
        return {"op": op, "fmt": rng.choice(["mx", "nv"]), "type": rng.choice(["bf16", "bf16", "fp32"]), "T": T, "K": K}
    if op == "linear":
        epi = rng.choice(["store", "geglu", "gelu", "silu"])
        K = _log_int(rng, 64, 16384)
        T = _log_int(rng, 1, 3200)
        O = _log_int(rng, 64, min(32768, 50_000_000_000 // (K * T)))
        if epi == "geglu":
            O += O % 2
        return {"op": op, "fmt": rng.choice(["mx", "nv"]), "type": rng.choice(["bf16", "bf16", "fp32"]), "T": T,
                "K": K, "O": O, "epi": epi, "bias": epi != "geglu" and rng.random() < 0.5}
    Hkv = rng.choice([1, 1, 1, 2])
    Hq = Hkv * rng.choice([1, 4, 8, 8])
    S = rng.choice([1, 1, _log_int(rng, 2, 64)])
    B = _log_int(rng, 1, min(64, max(1, 25600 // (S * Hq))))
    shared = _log_int(rng, 16, min(32768, 20_000_000 // (B * S * Hq)))
    own_most = rng.choice([0, _log_int(rng, 1, 400)])
    return {"op": op, "B": B, "S": S, "Hq": Hq, "Hkv": Hkv, "shared": shared, "own": own_most,
            "new": S > 1 or rng.random() < 0.5, "blocks": S > 1 and rng.random() < 0.4, "holes": rng.random() < 0.3}


# ----------------------------------------------------------------- inputs ---
def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _activations(gen, T, K):
    """Token rows as they come out of a block: each row with a size of its own,
    and a few channels far larger than the rest."""
    x = _normal(gen, T, K) * torch.exp(0.5 * _normal(gen, T, 1))
    big = (torch.rand(K, generator=gen, device="cuda") < 0.01).float()
    return x * (1.0 + 7.0 * big)


def _codes(y):
    """e2m1 codes of fp32 values: nearest, ties to the even code, at most 6."""
    a = y.abs()
    c = (a > 0.25).to(torch.uint8)
    for edge, inclusive in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        c += (a >= edge) if inclusive else (a > edge)
    return c + 8 * (y < 0).to(torch.uint8)


def _blocks(x, n):
    """[T, K] as [T, ceil(K / n), n], zeros past K."""
    T, K = x.shape
    return torch.nn.functional.pad(x, (0, -K % n)).view(T, -1, n)


def _to_fp4(x, fmt):
    """(codes [T, blocks, n], scales as numbers [T, blocks], their bytes, row scales or None) of fp32 rows."""
    b = _blocks(x, BLOCK[fmt])
    most = b.abs().amax(dim=2)
    if fmt == "mx":
        _, e = torch.frexp(most)  # most = m 2^e with 0.5 <= m < 1
        byte = torch.where(most > 0, e - 1 - 2 + 127, torch.zeros_like(e)).clamp(0, 254)
        scale = torch.ldexp(torch.ones_like(most), byte - 127)
        return _codes(b / scale[:, :, None]), scale, byte.to(torch.uint8), None
    _, e = torch.frexp(most.amax(dim=1))
    row = torch.ldexp(torch.ones(1, device=x.device), (e - 1 - 10).clamp(min=-100))
    six = torch.full_like(most, 6.0)  # (torch multiplies by the reciprocal of a plain number)
    held = (most / six / row[:, None]).clamp(max=448.0).to(torch.float8_e4m3fn)
    scale = held.float()
    step = (scale * row[:, None])[:, :, None].expand_as(b)
    return _codes(torch.where(step > 0, b / step, torch.zeros_like(b))), scale, held.view(torch.uint8), row


def _rows_on_16(q):
    """The same rows in memory whose rows begin on 16-byte boundaries."""
    T, n = q.shape
    buf = torch.zeros(T, (n + 15) // 16 * 16, dtype=q.dtype, device=q.device)
    buf[:, :n] = q
    return buf[:, :n]


def _tiles(byte):
    """Scale bytes [T, blocks] as tiles of 128 rows x 4 blocks: tile (t / 128, j / 4) holds row t's
    byte j at (t % 32) * 16 + (t % 128) / 32 * 4 + j % 4; zeros past the matrix."""
    T, n = byte.shape
    full = torch.nn.functional.pad(byte, (0, -n % 4, 0, -T % 128))
    t = full.view(full.shape[0] // 128, 4, 32, full.shape[1] // 4, 4)
    return t.permute(0, 3, 2, 1, 4).contiguous().view(full.shape[0] // 128, full.shape[1] // 4, 512)


def _fp4_rows(x, fmt, parts=1):
    """Rows in 4 bits as a program holds them; `parts` equal parts of the rows have tiles of their own."""
    T, K = x.shape
    codes, _, byte, row = _to_fp4(x, fmt)
    codes = codes.view(T, -1)[:, :K]
    codes = torch.nn.functional.pad(codes, (0, K % 2))
    q = _rows_on_16(codes[:, 0::2] | (codes[:, 1::2] << 4))
    scale = torch.cat([_tiles(part) for part in byte.chunk(parts)])
    return {"q": q, "scale": scale, "row": row, "K": K, "T": T, "fmt": fmt, "parts": parts}


def _empty_rows(T, K, fmt):
    q = _rows_on_16(torch.zeros(T, (K + 1) // 2, dtype=torch.uint8, device="cuda"))
    scale = torch.zeros((T + 127) // 128, -(-K // (4 * BLOCK[fmt])), 512, dtype=torch.uint8, device="cuda")
    row = torch.zeros(T, device="cuda") if fmt == "nv" else None
    return {"q": q, "scale": scale, "row": row, "K": K, "T": T, "fmt": fmt, "parts": 1}


def _int8(x):
    scale = x.abs().amax(dim=-1) / 127.0
    q = torch.round(x / scale.clamp_min(1e-30)[..., None]).clamp_(-127, 127).to(torch.int8)
    return q, scale


def _ring(gen, B, Hkv, n):
    """int8 keys and values with their scales: [B, Hkv, n, D] and [B, Hkv, n]."""
    k, ks = _int8(_normal(gen, B, Hkv, n, D))
    v, vs = _int8(_normal(gen, B, Hkv, n, D) * torch.exp(0.3 * _normal(gen, B, Hkv, n, 1)))
    return {"k": k, "v": v, "ks": ks, "vs": vs}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    if case["op"] == "quant":
        s["x"] = _activations(gen, case["T"], case["K"]).to(TYPES[case["type"]])
        s["rows"] = _empty_rows(case["T"], case["K"], case["fmt"])
        s["values"] = torch.empty_like(s["x"])
    elif case["op"] == "linear":
        T, K, O = case["T"], case["K"], case["O"]
        parts = 2 if case["epi"] == "geglu" else 1
        s["x"] = _fp4_rows(_activations(gen, T, K), case["fmt"])
        s["w"] = _fp4_rows(_normal(gen, O, K) * K ** -0.5, case["fmt"], parts)
        s["bias"] = _normal(gen, O) * 0.5 if case["bias"] else None
        s["y"] = torch.empty(T, O // parts, dtype=TYPES[case["type"]], device="cuda")
    else:
        B, S, Hq, Hkv, n, m = (case[k] for k in ("B", "S", "Hq", "Hkv", "shared", "own"))
        s["q"] = (2.0 * _normal(gen, B, Hq, S, D)).bfloat16()
        s["shared"] = _ring(gen, 1, Hkv, n)
        s["valid"] = None
        if case["holes"]:
            s["valid"] = (torch.rand(n, generator=gen, device="cuda") > 0.1).to(torch.uint8)
        s["own"] = s["own_len"] = None
        if m:
            s["own"] = _ring(gen, B, Hkv, m)
            s["own_len"] = torch.randint(0, m + 1, (B,), generator=gen, device="cuda", dtype=torch.int32)
        s["k"] = s["v"] = s["block"] = None
        if case["new"]:  # token-major, as the rotary operator leaves them
            s["k"] = _normal(gen, B, S, Hkv, D).bfloat16().transpose(1, 2)
            s["v"] = _normal(gen, B, S, Hkv, D).bfloat16().transpose(1, 2)
            if case["blocks"]:  # the first token does not see the others
                s["block"] = (torch.arange(S, device="cuda") > 0).to(torch.int32)
        s["out"] = torch.empty(B * S, Hq * D, dtype=torch.bfloat16, device="cuda")
        s["scale"] = D ** -0.5
        s["workspace"] = torch.empty(128 << 20, dtype=torch.uint8, device="cuda")  # one for all of a program's calls
    return s


# ------------------------------------------------------------ plain forms ---
def _values_of(rows):
    """fp32 values of 4-bit rows, row scales left out."""
    T, K, n = rows["T"], rows["K"], BLOCK[rows["fmt"]]
    q = rows["q"]
    codes = torch.stack([q & 15, q >> 4], dim=2).view(T, -1)[:, :K].long()
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=q.device)
    v = torch.cat([table, -table])[codes]
    s = rows["scale"]
    per = T // rows["parts"]
    byte = s.view(rows["parts"], -1, s.shape[1], 32, 4, 4).permute(0, 1, 4, 3, 2, 5).reshape(rows["parts"], -1, s.shape[1] * 4)
    byte = byte[:, :per].reshape(T, -1).contiguous()
    scale = torch.ldexp(torch.ones(1, device=q.device), byte.int() - 127) if n == 32 else byte.view(torch.float8_e4m3fn).float()
    return v * scale.repeat_interleave(n, dim=1)[:, :K]


def _plain_quant(s):
    x = s["x"]
    codes, scale, _, row = _to_fp4(x.float(), s["case"]["fmt"])
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=x.device)
    step = scale if row is None else scale * row[:, None]
    values = torch.cat([table, -table])[codes.long()] * step[:, :, None]
    out = {"values": values.reshape(x.shape[0], -1)[:, :x.shape[1]].to(x.dtype)}
    if row is not None:
        out["row_scale"] = row
    return out


def _gelu(v):
    return 0.5 * v * (1.0 + torch.tanh(0.7978845608028654 * (v + 0.044715 * v * v * v)))


def _plain_linear(s):
    c = s["case"]
    v = _values_of(s["x"]) @ _values_of(s["w"]).t()
    if s["x"]["row"] is not None:
        v = v * s["x"]["row"][:, None] * s["w"]["row"]
    if s["bias"] is not None:
        v = v + s["bias"]
    if c["epi"] == "gelu":
        v = _gelu(v)
    elif c["epi"] == "silu":
        v = v / (1.0 + torch.exp(-v))
    elif c["epi"] == "geglu":
        F = c["O"] // 2
        v = _gelu(v[:, :F]) * v[:, F:]
    return v.to(TYPES[c["type"]])


def _plain_attn(s):
    c = s["case"]
    B, S, Hq, Hkv, m = (c[k] for k in ("B", "S", "Hq", "Hkv", "own"))
    q = s["q"].float().view(B, Hkv, Hq // Hkv, S, D)
    sh = s["shared"]
    ks, vs = (sh["k"].float() * sh["ks"][..., None])[0], (sh["v"].float() * sh["vs"][..., None])[0]
    z = [torch.einsum("bhgsd,hnd->bhgsn", q, ks)]
    if s["valid"] is not None:
        z[0] = z[0].masked_fill(s["valid"] == 0, -math.inf)
    values = []
    if m:
        o = s["own"]
        zo = torch.einsum("bhgsd,bhnd->bhgsn", q, o["k"].float() * o["ks"][..., None])
        past = torch.arange(m, device=q.device) >= s["own_len"][:, None]
        z.append(zo.masked_fill(past[:, None, None, None, :], -math.inf))
        values.append(o["v"].float() * o["vs"][..., None])
    if c["new"]:
        zn = torch.einsum("bhgsd,bhnd->bhgsn", q, s["k"].float())
        if s["block"] is not None:
            zn = zn.masked_fill(s["block"][None, :] > s["block"][:, None], -math.inf)
        z.append(zn)
        values.append(s["v"].float())
    z = torch.cat(z, dim=-1) * s["scale"]
    top = z.amax(dim=-1, keepdim=True)
    p = torch.exp(z - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(dim=-1, keepdim=True)
    n = c["shared"]
    out = torch.einsum("bhgsn,hnd->bhgsd", p[..., :n], vs)
    if values:
        out = out + torch.einsum("bhgsn,bhnd->bhgsd", p[..., n:], torch.cat(values, dim=2))
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    return out.view(B, Hq, S, D).transpose(1, 2).reshape(B * S, Hq * D).to(torch.bfloat16)


# -------------------------------------------------------- the library's own ---
def _handles(s):
    """The library's own views of the state's buffers, which a program makes once beside them."""
    from reflex_b200 import _lib as L
    from reflex_b200 import kernels as K

    for name in ("rows", "x", "w"):
        r = s.get(name)
        if isinstance(r, dict):
            fmt = L.RFX_FP4_MX if r["fmt"] == "mx" else L.RFX_FP4_NV
            yield name, K.Fp4Rows(q=r["q"], scale=r["scale"], row_scale=r["row"], K=r["K"], fmt=fmt, parts=r["parts"])
    for name in ("shared", "own"):
        r = s.get(name)
        if r is not None:
            yield name, K.KVRing(r["k"], r["v"], r["ks"], r["vs"], None, None, L.RFX_QUANT_I8_SYM)


def _own(s):
    from reflex_b200 import _lib as L
    from reflex_b200 import kernels as K

    c = s["case"]
    if "handles" not in s:
        s["handles"] = dict(_handles(s))
    h = s["handles"]
    if c["op"] == "quant":
        rows = h["rows"]
        K.quant_fp4(x=s["x"], out=rows)
        K.dequant_fp4(x=rows, out=s["values"])
        return {"values": s["values"]} if rows.row_scale is None else {"values": s["values"], "row_scale": rows.row_scale}
    if c["op"] == "linear":
        epi = {"store": L.RFX_EPI_STORE, "silu": L.RFX_EPI_SILU, "gelu": L.RFX_EPI_GELU, "geglu": L.RFX_EPI_GEGLU}
        K.linear_fp4(w=h["w"], x=h["x"], y=s["y"], epilogue=epi[c["epi"]], bias=s["bias"])
        return s["y"]
    K.attention_shared(q=s["q"], shared=h["shared"], n_shared=c["shared"], shared_valid=s["valid"], own=h.get("own"),
                       own_len=s["own_len"], k_new=s["k"], v_new=s["v"], new_block=s["block"], out=s["out"],
                       softmax_scale=s["scale"], workspace=s["workspace"])
    return s["out"]


_PLAIN = {"quant": _plain_quant, "linear": _plain_linear, "attn": _plain_attn}


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["case"]["op"]](state)


# --------------------------------------------------------------- the work ---
def _held_bytes(T, K, fmt):
    return T * (K + 1) // 2 + T * -(-K // BLOCK[fmt]) + (4 * T if fmt == "nv" else 0)


def work(case):
    if case["op"] == "quant":
        e = 2 if case["type"] == "bf16" else 4
        n = case["T"] * case["K"]
        return {"bytes": 2 * e * n + _held_bytes(case["T"], case["K"], case["fmt"]), "flops": 4 * n}
    if case["op"] == "linear":
        T, K, O = case["T"], case["K"], case["O"]
        e = 2 if case["type"] == "bf16" else 4
        out = T * (O // 2 if case["epi"] == "geglu" else O)
        held = _held_bytes(T, K, case["fmt"]) + _held_bytes(O, K, case["fmt"])
        return {"bytes": held + e * out + (4 * O if case["bias"] else 0), "flops": 2 * T * K * O}
    B, S, Hq, Hkv = (case[k] for k in ("B", "S", "Hq", "Hkv"))
    mean_own = case["own"] / 2  # lengths from 0 to `own`
    new = S if case["new"] else 0
    ring = 2 * (D + 4) * Hkv * (case["shared"] + B * mean_own)
    return {"bytes": 4 * B * S * Hq * D + ring + 4 * B * new * Hkv * D + (case["shared"] if case["holes"] else 0),
            "flops": 4 * B * S * Hq * D * (case["shared"] + mean_own + new)}


# ---------------------------------------------------- 64-bit definitions ---
def _np(t):
    return None if t is None else t.double().cpu().numpy()


E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def _nearest(a, grid):
    """The nearest of the ascending numbers `grid`; ties to the even place."""
    hi = np.clip(np.searchsorted(grid, a), 1, len(grid) - 1)
    lo = hi - 1
    up, down = grid[hi] - a, a - grid[lo]
    return grid[np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)]


def _e4m3_grid():
    small = np.arange(8) * 2.0 ** -9
    return np.concatenate([small] + [(8 + np.arange(8)) * 2.0 ** (e - 3) for e in range(-6, 9)])[:-1]


def _exact_rows(x, fmt):
    """(values with every scale applied, row scales) of rows in 4 bits."""
    T, K = x.shape
    n = BLOCK[fmt]
    b = np.pad(x, ((0, 0), (0, -K % n))).reshape(T, -1, n)
    most = np.abs(b).max(axis=2)
    row = None
    if fmt == "mx":
        step = np.exp2(np.maximum(np.floor(np.log2(np.where(most > 0, most, 1.0))) - 2, -127))
    else:
        top = most.max(axis=1)
        row = np.exp2(np.maximum(np.floor(np.log2(np.where(top > 0, top, 2.0 ** -200))) - 10, -100))
        step = _nearest(np.minimum(most / (6.0 * row[:, None]), 448.0), _e4m3_grid()) * row[:, None]
    y = np.divide(b, step[:, :, None], out=np.zeros_like(b), where=step[:, :, None] > 0)
    values = np.sign(y) * _nearest(np.minimum(np.abs(y), 6.0), E2M1) * step[:, :, None]
    return values.reshape(T, -1)[:, :K], row


def _exact_held(r):
    """What 4-bit rows in memory stand for, byte by byte."""
    T, K, n = r["T"], r["K"], BLOCK[r["fmt"]]
    q, s = r["q"].cpu().numpy(), r["scale"].cpu().numpy()
    k = np.arange(K)
    code = (q[:, k // 2] >> (4 * (k % 2)).astype(np.uint8)) & 15
    per = T // r["parts"]
    t = np.arange(T)
    j = np.arange(-(-K // n))
    tile = (t // per) * -(-per // 128) + (t % per) // 128
    u = t % per % 128
    byte = s[tile[:, None], (j // 4)[None, :], ((u % 32) * 16 + u // 32 * 4)[:, None] + (j % 4)[None, :]].astype(np.int64)
    if n == 32:
        scale = np.exp2(byte - 127.0)
    else:
        e, f = byte >> 3 & 15, byte & 7
        scale = np.where(e > 0, (8 + f) * np.exp2(e - 10.0), f * 2.0 ** -9)
    v = np.where(code > 7, -1.0, 1.0) * E2M1[code & 7] * scale[:, k // n]
    return v if r["row"] is None else v * _np(r["row"])[:, None]


def _exact_gelu(v):
    return v * 0.5 * (1.0 + np.tanh(np.sqrt(2.0 / np.pi) * v * (1.0 + 0.044715 * np.square(v))))


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quant":
        values, row = _exact_rows(_np(s["x"]), case["fmt"])
        return {"values": values} if row is None else {"values": values, "row_scale": row}
    if case["op"] == "linear":
        v = np.matmul(_exact_held(s["x"]), _exact_held(s["w"]).T)
        if s["bias"] is not None:
            v += _np(s["bias"])[None, :]
        if case["epi"] == "geglu":
            gate, up = np.split(v, 2, axis=1)
            return _exact_gelu(gate) * up
        if case["epi"] == "silu":
            with np.errstate(over="ignore"):
                return v * np.reciprocal(1.0 + np.exp(-v))
        return _exact_gelu(v) if case["epi"] == "gelu" else v
    B, S, Hq, Hkv, n = (case[k] for k in ("B", "S", "Hq", "Hkv", "shared"))
    G = Hq // Hkv
    held = lambda r: (_np(r["k"]) * _np(r["ks"])[..., None], _np(r["v"]) * _np(r["vs"])[..., None])  # noqa: E731
    sk, sv = held(s["shared"])
    if s["valid"] is not None:
        keep = s["valid"].cpu().numpy() != 0
        sk, sv = sk[:, :, keep], sv[:, :, keep]
    ok, ov = held(s["own"]) if s["own"] is not None else (None, None)
    q, kn, vn = _np(s["q"]), _np(s["k"]), _np(s["v"])
    out = np.zeros((B, S, Hq, D))
    for b in range(B):
        for h in range(Hkv):
            k, v = [sk[0, h]], [sv[0, h]]
            if ok is not None:
                have = int(s["own_len"][b])
                k.append(ok[b, h, :have])
                v.append(ov[b, h, :have])
            seen = np.ones((S, sum(len(x) for x in k)), dtype=bool)
            if kn is not None:
                k.append(kn[b, h])
                v.append(vn[b, h])
                blk = np.zeros(S) if s["block"] is None else s["block"].cpu().numpy()
                seen = np.concatenate([seen, blk[None, :] <= blk[:, None]], axis=1)
            k, v = np.concatenate(k), np.concatenate(v)
            z = np.matmul(q[b, h * G:(h + 1) * G].reshape(G * S, D), k.T) * s["scale"]
            z = np.where(np.tile(seen, (G, 1)), z, -np.inf)
            if z.shape[1] == 0:
                continue
            top = z.max(axis=1, keepdims=True)
            e = np.exp(z - np.where(np.isinf(top), 0.0, top))
            total = e.sum(axis=1, keepdims=True)
            o = np.divide(e @ v, total, out=np.zeros((G * S, D)), where=total > 0)
            out[b, :, h * G:(h + 1) * G] = o.reshape(G, S, D).transpose(1, 0, 2)
    return out.reshape(B * S, Hq * D)
