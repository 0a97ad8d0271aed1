"""The measured cases of the int8 layer operators, with their plain forms.

Four operators that run one after another through a transformer layer whose
weights and activations are held as 8-bit integers:

* ``quant_rows``  rows of a matrix to int8 with one fp32 scale per row
  (activations per token, weights per output channel);
* ``linear_i8``   x_q @ w_q^T over those integers, scaled back by token and
  channel, with bias and activation;
* ``rope``        a QKV row split into q, k and v with the rotary positions
  applied (half or interleaved pairs, part of the head, scaled frequencies);
* ``block_norm``  what lies between two blocks: the norm of the block's output,
  its gate and residual scale, the residual add, and the next block's norm,
  whose output is stored as it is or as int8 rows.

With ``own`` false ``run`` computes them in elementary torch operations; with
``own`` true it calls the library.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases ---
def listed():
    return [
        # one token's MLP activations before its down projection: pure latency
        {"name": "quant_token", "op": "quant_rows", "type": "bf16", "T": 1, "K": 4096},
        # the GeGLU output of a 768-token camera frame (2B-shape prefix layer)
        {"name": "quant_frame", "op": "quant_rows", "type": "bf16", "T": 768, "K": 16384},
        # one token through the prefix layer's fused QKV projection
        {"name": "linear_token_qkv", "op": "linear_i8", "type": "bf16", "T": 1, "K": 2048, "O": 2560, "epi": "store",
         "bias": False},
        # the action expert's gate/up projection for one stream's 50 tokens
        {"name": "linear_expert_geglu", "op": "linear_i8", "type": "bf16", "T": 50, "K": 1024, "O": 8192,
         "epi": "geglu", "bias": False},
        # the vision tower's fc2 over three cameras: K and O no multiple of a tile, fp32 out
        {"name": "linear_vision_fc2", "op": "linear_i8", "type": "fp32", "T": 768, "K": 4304, "O": 1152,
         "epi": "store", "bias": True},
        # the prefix layer's down projection of a frame: a long K over few tiles
        {"name": "linear_frame_down", "op": "linear_i8", "type": "bf16", "T": 768, "K": 16384, "O": 2048,
         "epi": "store", "bias": False},
        # the prefix layer's gate/up projection of a frame: the largest product
        {"name": "linear_frame_geglu", "op": "linear_i8", "type": "bf16", "T": 768, "K": 2048, "O": 32768,
         "epi": "geglu", "bias": False},
        # one stream's 50 tokens: gated residual, then the next norm (scale and shift) as int8 rows
        {"name": "norm_expert_int8", "op": "block_norm", "type": "bf16", "T": 50, "S": 50, "K": 1024, "post": False,
         "gate": True, "mod": True, "int8": True},
        # 64 streams of 50 tokens, with the norm after the block too
        {"name": "norm_streams_int8", "op": "block_norm", "type": "bf16", "T": 3200, "S": 50, "K": 1024, "post": True,
         "gate": True, "mod": True, "int8": True},
        # a frame with its residual stream in fp32, norms before and after, no modulation
        {"name": "norm_frame_fp32", "op": "block_norm", "type": "fp32", "T": 768, "S": 768, "K": 2048, "post": True,
         "gate": False, "mod": False, "int8": False},
        # one stream's 50 action tokens after the 818-token context: 8 query heads, one KV head
        {"name": "rope_expert", "op": "rope", "type": "bf16", "B": 1, "S": 50, "Hq": 8, "Hkv": 1, "D": 256,
         "rot": 256, "pairs": "half", "first": 818, "factor": 1.0},
        # a long context: interleaved pairs over half of the head, frequencies stretched eightfold
        {"name": "rope_long", "op": "rope", "type": "bf16", "B": 1, "S": 6344, "Hq": 8, "Hkv": 1, "D": 256,
         "rot": 128, "pairs": "interleaved", "first": 50000, "factor": 8.0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quant_rows", "linear_i8", "linear_i8", "block_norm", "rope"])
    kind = rng.choice(["bf16", "bf16", "fp32"])
    if op == "quant_rows":
        K = _log_int(rng, 16, 16384)
        T = _log_int(rng, 1, min(4096, (1 << 23) // K))
        return {"op": op, "type": kind, "T": T, "K": K}
    if op == "linear_i8":
        epi = rng.choice(["store", "geglu", "gelu", "silu"])
        K = _log_int(rng, 64, 16384)
        T = _log_int(rng, 1, 3200)
        O = _log_int(rng, 64, min(32768, 50_000_000_000 // (K * T)))
        if epi == "geglu":
            O += O % 2
        return {"op": op, "type": kind, "T": T, "K": K, "O": O, "epi": epi, "bias": epi != "geglu" and rng.random() < 0.5}
    if op == "block_norm":
        K = _log_int(rng, 64, 8192)
        if rng.random() < 0.7:
            K = (K + 7) // 8 * 8
        S = _log_int(rng, 1, 768)
        B = _log_int(rng, 1, max(1, min(64, (1 << 22) // (K * S))))
        return {"op": op, "type": kind, "T": B * S, "S": S, "K": K, "post": rng.random() < 0.5,
                "gate": rng.random() < 0.5, "mod": rng.random() < 0.5, "int8": rng.random() < 0.5}
    D = rng.choice([64, 72, 128, 256])
    Hkv = rng.choice([1, 1, 2, 4])
    Hq = Hkv * rng.choice([1, 2, 4, 8])
    S = _log_int(rng, 1, 6344)
    B = _log_int(rng, 1, max(1, min(64, (1 << 24) // (S * (Hq + 2 * Hkv) * D))))
    rot = D if rng.random() < 0.5 else 2 * rng.randint(4, D // 2)
    return {"op": op, "type": kind, "B": B, "S": S, "Hq": Hq, "Hkv": Hkv, "D": D, "rot": rot,
            "pairs": rng.choice(["half", "interleaved"]), "first": rng.randint(0, 100000),
            "factor": rng.choice([1.0, 4.0, 8.0])}


# ----------------------------------------------------------------- inputs ---
def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _activations(gen, T, K):
    """Token rows as they come out of a block: each row with a size of its own,
    and a few channels far larger than the rest."""
    x = _normal(gen, T, K) * torch.exp(0.5 * _normal(gen, T, 1))
    big = (torch.rand(K, generator=gen, device="cuda") < 0.01).float()
    return x * (1.0 + 7.0 * big)


def _int8_rows(x):
    scale = x.abs().amax(dim=1) / 127.0
    q = torch.round(x / scale.clamp_min(1e-30)[:, None]).clamp_(-127, 127).to(torch.int8)
    return q, scale


def _padded(q):
    """The same rows in memory whose rows begin on 16-byte boundaries."""
    T, K = q.shape
    ld = (K + 15) // 16 * 16
    if ld == K:
        return q.contiguous()
    buf = torch.zeros(T, ld, dtype=q.dtype, device=q.device)
    buf[:, :K] = q
    return buf[:, :K]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[case["type"]]
    s = {"case": case}
    if case["op"] == "quant_rows":
        T, K = case["T"], case["K"]
        s["x"] = _activations(gen, T, K).to(dt)
        s["q"] = torch.empty(T, K, dtype=torch.int8, device="cuda")
        s["scale"] = torch.empty(T, dtype=torch.float32, device="cuda")
        s["values"] = torch.empty(T, K, dtype=dt, device="cuda")
    elif case["op"] == "linear_i8":
        T, K, O = case["T"], case["K"], case["O"]
        xq, s["x_scale"] = _int8_rows(_activations(gen, T, K))
        wq, s["w_scale"] = _int8_rows(_normal(gen, O, K) * K ** -0.5)
        s["x"], s["w"] = _padded(xq), _padded(wq)
        s["bias"] = _normal(gen, O) * 0.5 if case["bias"] else None
        s["y"] = torch.empty(T, O // 2 if case["epi"] == "geglu" else O, dtype=dt, device="cuda")
    elif case["op"] == "block_norm":
        T, S, K = case["T"], case["S"], case["K"]
        s["h"] = _activations(gen, T, K).to(dt)
        s["y"] = _normal(gen, T, K).to(dt)
        vec = lambda on, *shape, mean=0.0: mean + 0.2 * _normal(gen, *shape) if on else None  # noqa: E731
        s["post"] = vec(case["post"], K, mean=1.0)
        s["gate"] = vec(case["gate"], T // S, K, mean=0.5)
        s["a1"] = vec(True, K, mean=1.0)
        s["a2"] = vec(case["mod"], T // S, K, mean=1.0)
        s["b2"] = vec(case["mod"], T // S, K)
        s["rscale"] = 0.75
        s["h_out"] = torch.empty(T, K, dtype=dt, device="cuda")
        s["z"] = torch.empty(T, K, dtype=torch.bfloat16 if case["int8"] else dt, device="cuda")
        s["z_q"] = torch.empty(T, K, dtype=torch.int8, device="cuda")
        s["z_scale"] = torch.empty(T, dtype=torch.float32, device="cuda")
    else:
        B, S, Hq, Hkv, D, rot = (case[k] for k in ("B", "S", "Hq", "Hkv", "D", "rot"))
        T = B * S
        s["x"] = _normal(gen, T, (Hq + 2 * Hkv) * D).to(dt)
        s["positions"] = (case["first"] + torch.arange(S, device="cuda")).repeat(B).to(torch.int32)
        # radians per position of each pair, stretched for contexts longer than the trained one
        pair = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
        s["freq"] = 10000.0 ** (-2.0 * pair / rot) / case["factor"]
        s["mag"] = 1.0 if case["factor"] == 1.0 else 0.1 * math.log(case["factor"]) + 1.0
        s["q_out"] = torch.empty(B, Hq, S, D, dtype=dt, device="cuda")
        s["k_out"] = torch.empty(B, S, Hkv, D, dtype=dt, device="cuda").transpose(1, 2)
        s["v_out"] = torch.empty(B, S, Hkv, D, dtype=dt, device="cuda").transpose(1, 2)
    return s


# ------------------------------------------------------------ plain forms ---
def _plain_int8(z):
    """int8 rows of fp32 values: scale = absmax / 127, q = rne(z / scale).  The
    divisor is a tensor: torch multiplies by the reciprocal of a plain number,
    and a scale that is one rounding off moves values that lie next to a half."""
    absmax = z.abs().amax(dim=1)
    scale = absmax / torch.full_like(absmax, 127.0)
    q = torch.where(scale[:, None] > 0, torch.round(z / scale[:, None]), torch.zeros_like(z)).clamp(-127, 127)
    return q, scale


def _plain_quant(s):
    q, scale = _plain_int8(s["x"].float())
    return {"values": (q * scale[:, None]).to(s["x"].dtype), "scale": scale}


def _gelu(v):
    return 0.5 * v * (1.0 + torch.tanh(0.7978845608028654 * (v + 0.044715 * v * v * v)))


def _plain_linear(s):
    c = s["case"]
    # the integer sum is exact in 64 bits, where 32-bit floats would lose its low end
    acc = (s["x"].double() @ s["w"].double().t()).float()
    v = acc * s["x_scale"][:, None] * s["w_scale"]
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


def _rms(v):
    return v * torch.rsqrt((v * v).mean(dim=1, keepdim=True) + EPS)


def _plain_norm(s):
    c = s["case"]
    per_token = lambda m: m.repeat_interleave(c["S"], dim=0)  # noqa: E731
    u = s["y"].float()
    if s["post"] is not None:
        u = _rms(u) * s["post"]
    if s["gate"] is not None:
        u = per_token(s["gate"]) * u
    h = (s["h"].float() + s["rscale"] * u).to(s["h"].dtype)
    z = _rms(h.float()) * s["a1"]
    if s["a2"] is not None:
        z = z * per_token(s["a2"]) + per_token(s["b2"])
    if not c["int8"]:
        return {"h": h, "z": z.to(s["h"].dtype)}
    q, scale = _plain_int8(z)
    return {"h": h, "z": (q * scale[:, None]).to(torch.bfloat16), "z_scale": scale}


def _plain_rope(s):
    c = s["case"]
    B, S, Hq, Hkv, D, rot = (c[k] for k in ("B", "S", "Hq", "Hkv", "D", "rot"))
    x = s["x"].view(B, S, Hq + 2 * Hkv, D).transpose(1, 2)
    angle = s["positions"].double().view(B, 1, S, 1) * s["freq"]
    cos, sin = (torch.cos(angle) * s["mag"]).float(), (torch.sin(angle) * s["mag"]).float()
    part = x[:, :Hq + Hkv, :, :rot].float()
    if c["pairs"] == "half":
        a, b = part[..., :rot // 2], part[..., rot // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    else:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    out = torch.cat([turned.to(x.dtype), x[:, :Hq + Hkv, :, rot:]], dim=-1)
    return {"q": out[:, :Hq].contiguous(), "k": out[:, Hq:].contiguous(), "v": x[:, Hq + Hkv:].contiguous()}


# -------------------------------------------------------- the library's own ---
def _own(s):
    from reflex_b200 import _lib as L
    from reflex_b200 import kernels as K

    c = s["case"]
    if c["op"] == "quant_rows":
        K.quant_rows(x=s["x"], q=s["q"], scale=s["scale"])
        return {"values": torch.mul(s["q"], s["scale"][:, None], out=s["values"]), "scale": s["scale"]}
    if c["op"] == "linear_i8":
        epi = {"store": L.RFX_EPI_STORE, "silu": L.RFX_EPI_SILU, "gelu": L.RFX_EPI_GELU, "geglu": L.RFX_EPI_GEGLU}
        K.linear_i8(w=s["w"], w_scale=s["w_scale"], x=s["x"], x_scale=s["x_scale"], y=s["y"], epilogue=epi[c["epi"]],
                    bias=s["bias"])
        return s["y"]
    if c["op"] == "block_norm":
        out = {"z_q": s["z_q"], "z_scale": s["z_scale"]} if c["int8"] else {"z": s["z"]}
        K.block_norm(h=s["h"], y=s["y"], S=c["S"], post_w=s["post"], gate=s["gate"], residual_scale=s["rscale"],
                     h_out=s["h_out"], norm_a1=s["a1"], norm_a2=s["a2"], norm_b2=s["b2"], eps=EPS, **out)
        if not c["int8"]:
            return {"h": s["h_out"], "z": s["z"]}
        return {"h": s["h_out"], "z": torch.mul(s["z_q"], s["z_scale"][:, None], out=s["z"]), "z_scale": s["z_scale"]}
    K.rope(x=s["x"], positions=s["positions"], inv_freq=s["freq"], magnitude=s["mag"], q_out=s["q_out"],
           k_out=s["k_out"], v_out=s["v_out"],
           pairs=L.RFX_ROPE_HALF if c["pairs"] == "half" else L.RFX_ROPE_INTERLEAVED)
    return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}


_PLAIN = {"quant_rows": _plain_quant, "linear_i8": _plain_linear, "block_norm": _plain_norm, "rope": _plain_rope}


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["case"]["op"]](state)


# --------------------------------------------------------------- the work ---
def work(case):
    e = 2 if case["type"] == "bf16" else 4
    if case["op"] == "quant_rows":
        n = case["T"] * case["K"]
        return {"bytes": n * e + n + 4 * case["T"], "flops": 4 * n}
    if case["op"] == "linear_i8":
        T, K, O = case["T"], case["K"], case["O"]
        out = T * (O // 2 if case["epi"] == "geglu" else O)
        return {"bytes": T * K + O * K + 4 * T + 4 * O * (2 if case["bias"] else 1) + e * out, "flops": 2 * T * K * O}
    if case["op"] == "block_norm":
        T, S, K = case["T"], case["S"], case["K"]
        n = T * K
        vectors = K * (1 + case["post"]) + (T // S) * K * (case["gate"] + 2 * case["mod"])
        return {"bytes": 3 * n * e + (n + 4 * T if case["int8"] else n * e) + 4 * vectors, "flops": 12 * n}
    T = case["B"] * case["S"]
    n = T * (case["Hq"] + 2 * case["Hkv"]) * case["D"]
    return {"bytes": 2 * n * e + 4 * T + 4 * case["rot"], "flops": 3 * T * (case["Hq"] + case["Hkv"]) * case["rot"]}


# ---------------------------------------------------- 64-bit definitions ---
def _np(t):
    return None if t is None else t.double().cpu().numpy()


def _exact_int8(z):
    """What int8 rows of z stand for, with their scales; a row of zeros stays zero."""
    scale = np.max(np.abs(z), axis=1) / 127.0
    q = np.rint(np.divide(z, scale[:, None], out=np.zeros_like(z), where=scale[:, None] > 0))
    return np.clip(q, -127, 127) * scale[:, None], scale


def _exact_gelu(v):
    return v * 0.5 * (1.0 + np.tanh(np.sqrt(2.0 / np.pi) * v * (1.0 + 0.044715 * np.square(v))))


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quant_rows":
        values, scale = _exact_int8(_np(s["x"]))
        return {"values": values, "scale": scale}
    if case["op"] == "linear_i8":
        v = np.matmul(_np(s["x"]), _np(s["w"]).T)
        v *= np.outer(_np(s["x_scale"]), _np(s["w_scale"]))
        if s["bias"] is not None:
            v += _np(s["bias"])[None, :]
        if case["epi"] == "geglu":
            gate, up = np.split(v, 2, axis=1)
            return _exact_gelu(gate) * up
        if case["epi"] == "silu":
            with np.errstate(over="ignore"):
                return v * np.reciprocal(1.0 + np.exp(-v))
        return _exact_gelu(v) if case["epi"] == "gelu" else v
    if case["op"] == "block_norm":
        T, S, K = case["T"], case["S"], case["K"]
        blocks = lambda t: _np(t).reshape(T // S, 1, K)  # noqa: E731
        u = _np(s["y"]).reshape(T // S, S, K)
        if s["post"] is not None:
            u = u / np.sqrt(np.mean(np.square(u), axis=-1, keepdims=True) + EPS) * _np(s["post"])
        if s["gate"] is not None:
            u = u * blocks(s["gate"])
        h = _np(s["h"]).reshape(T // S, S, K) + s["rscale"] * u
        # the next norm reads the stream as it is held, in its type
        held = torch.from_numpy(h).to(TYPES[case["type"]]).double().numpy()
        z = held / np.sqrt(np.mean(np.square(held), axis=-1, keepdims=True) + EPS) * _np(s["a1"])
        if s["a2"] is not None:
            z = z * blocks(s["a2"]) + blocks(s["b2"])
        h, z = h.reshape(T, K), z.reshape(T, K)
        if not case["int8"]:
            return {"h": h, "z": z}
        values, scale = _exact_int8(z)
        return {"h": h, "z": values, "z_scale": scale}
    B, S, Hq, Hkv, D, rot = (case[k] for k in ("B", "S", "Hq", "Hkv", "D", "rot"))
    x = _np(s["x"]).reshape(B, S, Hq + 2 * Hkv, D).transpose(0, 2, 1, 3).copy()
    turn = s["mag"] * np.exp(1j * np.outer(_np(s["positions"])[:S], _np(s["freq"])))
    first = slice(0, rot // 2) if case["pairs"] == "half" else slice(0, rot, 2)
    second = slice(rot // 2, rot) if case["pairs"] == "half" else slice(1, rot, 2)
    z = (x[:, :Hq + Hkv, :, first] + 1j * x[:, :Hq + Hkv, :, second]) * turn
    x[:, :Hq + Hkv, :, first], x[:, :Hq + Hkv, :, second] = z.real, z.imag
    return {"q": x[:, :Hq], "k": x[:, Hq:Hq + Hkv], "v": x[:, Hq + Hkv:]}
