"""The int8 layer operators without a GPU: struct layouts, the refusals of the
C entry points and of the tensor wrappers, empty calls, and the scaled rotary
frequencies against their formulas."""
import ctypes
import math
import os
import random
import subprocess

import pytest
import torch

from reflex_b200 import _lib
from reflex_b200 import kernels as K

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"rfx_quant_rows_desc": "QuantRowsDesc", "rfx_linear_i8_desc": "LinearI8Desc",
           "rfx_block_norm_desc": "BlockNormDesc", "rfx_rope_desc": "RopeDesc"}
ENTRIES = {"rfx_quant_rows": "quant_rows", "rfx_linear_i8": "linear_i8", "rfx_block_norm": "block_norm",
           "rfx_rope": "rope"}
A = 1 << 20  # an aligned address that is never dereferenced


def test_structs_match_c_layout(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "rfx.h"', "int main(void) {"]
    for c_name, py_name in STRUCTS.items():
        lines.append(f'  printf("{py_name} size %zu\\n", sizeof({c_name}));')
        for field, _ in getattr(_lib, py_name)._fields_:
            lines.append(f'  printf("{py_name} {field} %zu\\n", offsetof({c_name}, {field}));')
    lines.append("  return 0; }")
    c = tmp_path / "layout.c"
    c.write_text("\n".join(lines))
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(c), "-o", str(tmp_path / "layout")],
                   check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split("\n")
    for line in filter(None, out):
        py_name, key, val = line.split()
        cls = getattr(_lib, py_name)
        got = ctypes.sizeof(cls) if key == "size" else getattr(cls, key).offset
        assert got == int(val), f"{py_name}.{key}: ctypes {got}, C {val}"


@pytest.mark.parametrize("name", sorted(ENTRIES))
def test_null_descriptor_is_rejected(name):
    assert getattr(_lib.load(), name)(None, None) == _lib.RFX_E_INVAL


def quant():
    return _lib.QuantRowsDesc(4, 64, _lib.RFX_DTYPE_BF16, A, 64, 2 * A, 64, 3 * A)


def linear():
    return _lib.LinearI8Desc(4, 64, 64, _lib.RFX_EPI_STORE, _lib.RFX_DTYPE_BF16, A, 64, 2 * A, 3 * A, 64, 4 * A, None,
                             5 * A, 64)


def norm():
    d = _lib.BlockNormDesc()
    d.T, d.K, d.tokens_per_batch, d.dtype = 4, 64, 4, _lib.RFX_DTYPE_BF16
    d.h, d.y, d.h_out, d.z = A, 2 * A, 3 * A, 4 * A
    d.ldh = d.ldy = d.ldho = d.ldz = d.ldzq = 64
    d.residual_scale, d.eps = 1.0, 1e-6
    return d


def rope():
    d = _lib.RopeDesc()
    d.B, d.S, d.num_q_heads, d.num_kv_heads, d.head_dim, d.rot_dim = 1, 4, 2, 1, 64, 64
    d.pairs, d.dtype, d.magnitude = _lib.RFX_ROPE_HALF, _lib.RFX_DTYPE_BF16, 1.0
    d.x, d.positions, d.inv_freq, d.q_out, d.k_out, d.v_out = A, 2 * A, 3 * A, 4 * A, 5 * A, 6 * A
    d.ldx = 4 * 64
    return d


BAD = [
    ("rfx_quant_rows", quant, dict(T=-1)), ("rfx_quant_rows", quant, dict(K=0)),
    ("rfx_quant_rows", quant, dict(K=16385, ldx=16385, ldq=16385)), ("rfx_quant_rows", quant, dict(in_dtype=2)),
    ("rfx_quant_rows", quant, dict(x=None)), ("rfx_quant_rows", quant, dict(q=None)),
    ("rfx_quant_rows", quant, dict(scale=None)), ("rfx_quant_rows", quant, dict(ldx=63)),
    ("rfx_quant_rows", quant, dict(ldq=63)), ("rfx_quant_rows", quant, dict(x=A + 1)),
    ("rfx_quant_rows", quant, dict(scale=A + 2)),
    ("rfx_linear_i8", linear, dict(T=-1)), ("rfx_linear_i8", linear, dict(O=0)), ("rfx_linear_i8", linear, dict(K=0)),
    ("rfx_linear_i8", linear, dict(K=65537, ldx=65552, ldw=65552)),
    ("rfx_linear_i8", linear, dict(epilogue=_lib.RFX_EPI_RESIDUAL)),
    ("rfx_linear_i8", linear, dict(epilogue=_lib.RFX_EPI_QKV_ROPE)), ("rfx_linear_i8", linear, dict(epilogue=6)),
    ("rfx_linear_i8", linear, dict(epilogue=_lib.RFX_EPI_GEGLU, O=63)), ("rfx_linear_i8", linear, dict(out_dtype=5)),
    ("rfx_linear_i8", linear, dict(x=A + 8)), ("rfx_linear_i8", linear, dict(w=A + 1)),
    ("rfx_linear_i8", linear, dict(ldx=72)), ("rfx_linear_i8", linear, dict(ldw=48)),
    ("rfx_linear_i8", linear, dict(ldy=63)), ("rfx_linear_i8", linear, dict(y=None)),
    ("rfx_linear_i8", linear, dict(x_scale=None)), ("rfx_linear_i8", linear, dict(w_scale=A + 2)),
    ("rfx_linear_i8", linear, dict(T=2147483647, O=2147483646, ldy=2147483646)),
    ("rfx_linear_i8", linear, dict(T=(1 << 30) + 1)), ("rfx_linear_i8", linear, dict(O=(1 << 30) + 1, ldy=1 << 31)),
    ("rfx_linear_i8", linear, dict(T=1 << 30, O=1 << 20, ldy=1 << 20)),
    ("rfx_block_norm", norm, dict(T=-1)), ("rfx_block_norm", norm, dict(K=16385)),
    ("rfx_block_norm", norm, dict(tokens_per_batch=0)), ("rfx_block_norm", norm, dict(dtype=3)),
    ("rfx_block_norm", norm, dict(h=None)), ("rfx_block_norm", norm, dict(h_out=None)),
    ("rfx_block_norm", norm, dict(y=None)), ("rfx_block_norm", norm, dict(y=None, h_out=None, gate=A)),
    ("rfx_block_norm", norm, dict(y=None, h_out=None, z=None)), ("rfx_block_norm", norm, dict(z_q=A, z_scale=A)),
    ("rfx_block_norm", norm, dict(z=None, z_q=A)), ("rfx_block_norm", norm, dict(z=None, norm_a1=A)),
    ("rfx_block_norm", norm, dict(ldz=63)), ("rfx_block_norm", norm, dict(h_out=A, ldho=128)),
    ("rfx_block_norm", norm, dict(z=3 * A)), ("rfx_block_norm", norm, dict(post_w=A + 2)),
    ("rfx_rope", rope, dict(B=-1)), ("rfx_rope", rope, dict(num_q_heads=0)), ("rfx_rope", rope, dict(head_dim=257)),
    ("rfx_rope", rope, dict(rot_dim=63)), ("rfx_rope", rope, dict(rot_dim=66)), ("rfx_rope", rope, dict(rot_dim=0)),
    ("rfx_rope", rope, dict(pairs=2)), ("rfx_rope", rope, dict(dtype=7)), ("rfx_rope", rope, dict(ldx=255)),
    ("rfx_rope", rope, dict(k_out=None)), ("rfx_rope", rope, dict(num_kv_heads=0)),
    ("rfx_rope", rope, dict(positions=None)), ("rfx_rope", rope, dict(inv_freq=A + 4)),
    ("rfx_rope", rope, dict(B=65536, S=65536)),
]


@pytest.mark.parametrize("entry,make,change", BAD)
def test_bad_descriptors_are_refused(entry, make, change):
    """Refused by the direct call and by the plan add, with a message that
    names the entry point; the plan stays empty."""
    lib = _lib.load()
    d = make()
    for k, v in change.items():
        setattr(d, k, v)
    assert getattr(lib, entry)(ctypes.byref(d), None) == _lib.RFX_E_INVAL
    assert entry.encode() in lib.rfx_last_error()
    plan = ctypes.c_void_p()
    assert lib.rfx_plan_create(ctypes.byref(plan)) == _lib.RFX_OK
    try:
        add = getattr(lib, "rfx_plan_add_" + ENTRIES[entry])
        assert add(plan, ctypes.byref(d)) == _lib.RFX_E_INVAL
        n = ctypes.c_int(-1)
        assert lib.rfx_plan_num_launches(plan, ctypes.byref(n)) == _lib.RFX_OK and n.value == 0
    finally:
        lib.rfx_plan_destroy(plan)


@pytest.mark.parametrize("entry,make,change", [
    ("rfx_quant_rows", quant, dict(T=0, x=None, q=None, scale=None)),
    ("rfx_linear_i8", linear, dict(T=0, x=None, y=None, x_scale=None)),
    ("rfx_block_norm", norm, dict(T=0, h=None, y=None, h_out=None, z=None)),
    ("rfx_rope", rope, dict(S=0, x=None)),
])
def test_no_rows_is_a_no_op(entry, make, change):
    """No rows: accepted without a device, nothing launched."""
    lib = _lib.load()
    d = make()
    for k, v in change.items():
        setattr(d, k, v)
    assert getattr(lib, entry)(ctypes.byref(d), None) == _lib.RFX_OK
    plan = ctypes.c_void_p()
    assert lib.rfx_plan_create(ctypes.byref(plan)) == _lib.RFX_OK
    try:
        assert getattr(lib, "rfx_plan_add_" + ENTRIES[entry])(plan, ctypes.byref(d)) == _lib.RFX_OK
        n = ctypes.c_int(-1)
        assert lib.rfx_plan_num_launches(plan, ctypes.byref(n)) == _lib.RFX_OK and n.value == 0
    finally:
        lib.rfx_plan_destroy(plan)


ROW = 4 * 64 * 2  # bytes of a row of rope()'s x: 2 q heads, one k, one v
OVER_X = dict(q_out=A, qs_b=4 * 256, qs_h=64, qs_s=256, k_out=A + 256, ks_b=4 * 256, ks_h=64, ks_s=256,
              v_out=A + 384, vs_b=4 * 256, vs_h=64, vs_s=256)
PLACES = [  # which memory outputs and inputs may share
    (quant, {}, True),
    (quant, dict(q=A), False),                                        # rows of half the pitch over x
    (quant, dict(q=A + 511), False), (quant, dict(q=A + 512), True),  # its last byte; right behind it
    (quant, dict(q=A - 255), False), (quant, dict(q=A - 256), True),
    (quant, dict(scale=A + 256), False), (quant, dict(scale=2 * A + 252), False),
    (quant, dict(ldx=96, q=A + 128, ldq=192), True),                  # the free columns of x's own rows
    (quant, dict(ldx=95, q=A + 128, ldq=190), False),                 # two bytes too few of them
    (quant, dict(ldx=96, q=A + 127, ldq=192), False), (quant, dict(ldx=96, q=A + 128, ldq=191), False),
    (quant, dict(T=1, q=A + 128), True), (quant, dict(T=1, q=A + 127), False),
    (linear, {}, True),
    (linear, dict(y=A), False), (linear, dict(y=3 * A + 64), False), (linear, dict(y=2 * A), False),
    (linear, dict(y=4 * A + 252), False), (linear, dict(y=4 * A + 256), True), (linear, dict(bias=5 * A), False),
    (linear, dict(bias=5 * A + 512), True), (linear, dict(ldx=192, y=A + 64, ldy=96), True),
    (norm, {}, True),
    (norm, dict(h_out=A), True), (norm, dict(z=A), True), (norm, dict(z=2 * A), True),
    (norm, dict(h_out=A, z=A), False), (norm, dict(h_out=2 * A), False), (norm, dict(h_out=A + 128), False),
    (norm, dict(z=A, ldz=72), False), (norm, dict(z=2 * A + 128), False), (norm, dict(z=3 * A + 2), False),
    (norm, dict(z=None, z_q=5 * A, z_scale=6 * A), True), (norm, dict(z=None, z_q=A, z_scale=6 * A), False),
    (norm, dict(z=None, z_q=2 * A + 511, z_scale=6 * A), False), (norm, dict(z=None, z_q=3 * A, z_scale=6 * A), False),
    (norm, dict(z=None, z_q=5 * A, z_scale=5 * A), False), (norm, dict(z=None, z_q=5 * A, z_scale=3 * A), False),
    (rope, {}, True),
    (rope, OVER_X, True),
    (rope, dict(OVER_X, k_out=A), False),                             # k over the q heads
    (rope, dict(OVER_X, q_out=A + 128), False), (rope, dict(OVER_X, qs_h=128), False),
    (rope, dict(OVER_X, qs_s=128), False), (rope, dict(OVER_X, vs_s=264), False),
    (rope, dict(q_out=A, qs_b=512, qs_h=256, qs_s=64), False),        # head-major over x
    (rope, dict(q_out=A + 4 * ROW, qs_b=512, qs_h=256, qs_s=64), True),
    (rope, dict(q_out=A + 4 * ROW - 2, qs_b=512, qs_h=256, qs_s=64), False),
    (rope, dict(q_out=A - 1024, qs_b=512, qs_h=256, qs_s=64), True),
    (rope, dict(q_out=A - 1022, qs_b=512, qs_h=256, qs_s=64), False),
    (rope, dict(ldx=384, q_out=A + 512, qs_b=4 * 384, qs_h=64, qs_s=384), True),  # the free columns of x's rows
    (rope, dict(ldx=384, q_out=A + 510, qs_b=4 * 384, qs_h=64, qs_s=384), False),
    (rope, dict(q_out=A + 4 * ROW, qs_h=-256, qs_s=64), False),       # strides that lead back into x
]


@pytest.mark.parametrize("make,change,fine", PLACES)
def test_shared_memory_is_in_place_or_refused(make, change, fine):
    """An output lies over an input exactly where the operator may work in
    place, or apart from it; what reads and writes across rows is refused."""
    lib = _lib.load()
    d = make()
    for k, v in change.items():
        setattr(d, k, v)
    name = {"quant": "quant_rows", "linear": "linear_i8", "norm": "block_norm", "rope": "rope"}[make.__name__]
    plan = ctypes.c_void_p()
    assert lib.rfx_plan_create(ctypes.byref(plan)) == _lib.RFX_OK
    try:
        rc = getattr(lib, "rfx_plan_add_" + name)(plan, ctypes.byref(d))
        if name == "linear_i8" and fine:  # without a driver its tensor maps cannot be made
            assert rc != _lib.RFX_E_INVAL or b"shares memory" not in lib.rfx_last_error()
        else:
            assert rc == (_lib.RFX_OK if fine else _lib.RFX_E_INVAL)
        if not fine:
            assert any(w in lib.rfx_last_error() for w in (b"share", b"overlap", b"lies across"))
    finally:
        lib.rfx_plan_destroy(plan)


def test_plan_counts_launches():
    lib = _lib.load()
    plan = ctypes.c_void_p()
    assert lib.rfx_plan_create(ctypes.byref(plan)) == _lib.RFX_OK
    try:
        for name, d in (("quant_rows", quant()), ("block_norm", norm()), ("rope", rope())):
            assert getattr(lib, "rfx_plan_add_" + name)(plan, ctypes.byref(d)) == _lib.RFX_OK
        n = ctypes.c_int(-1)
        assert lib.rfx_plan_num_launches(plan, ctypes.byref(n)) == _lib.RFX_OK and n.value == 3
    finally:
        lib.rfx_plan_destroy(plan)


def test_cpu_tensors_are_refused():
    x, q, s = torch.zeros(2, 16), torch.zeros(2, 16, dtype=torch.int8), torch.zeros(2)
    with pytest.raises(ValueError, match="CUDA"):
        K.quant_rows(x=x, q=q, scale=s)
    with pytest.raises(ValueError, match="CUDA"):
        K.linear_i8(w=q, w_scale=s, x=q, x_scale=s, y=torch.zeros(2, 2))
    with pytest.raises(ValueError, match="CUDA"):
        K.block_norm(h=x, S=2, z=x)
    with pytest.raises(ValueError, match="CUDA"):
        K.rope(x=x, positions=torch.zeros(2, dtype=torch.int32), inv_freq=torch.ones(4, dtype=torch.float64),
               q_out=torch.zeros(1, 1, 2, 16))


def test_rope_frequencies():
    """The published formulas, pair by pair (fp64)."""
    rot, theta, s, L0 = 64, 10000.0, 8.0, 4096
    base = [theta ** (-2 * i / rot) for i in range(rot // 2)]
    f, m = K.rope_frequencies(rot, theta, device="cpu")
    assert f.dtype == torch.float64 and m == 1.0
    assert torch.allclose(f, torch.tensor(base, dtype=torch.float64), rtol=1e-14, atol=0)
    f, m = K.rope_frequencies(rot, theta, scaling="linear", factor=s, device="cpu")
    assert torch.allclose(f, torch.tensor([b / s for b in base], dtype=torch.float64), rtol=1e-14, atol=0) and m == 1.0
    f, m = K.rope_frequencies(rot, theta, scaling="ntk", factor=s, device="cpu")
    # the fastest pair is kept, the slowest divided by the factor
    assert f[0] == 1.0 and math.isclose(f[-1].item(), base[-1] / s, rel_tol=1e-12) and m == 1.0
    f, m = K.rope_frequencies(rot, theta, scaling="yarn", factor=s, trained_len=L0, device="cpu")
    for i, b in enumerate(base):
        turns = L0 * b / (2 * math.pi)
        g = min(max((turns - 1.0) / (32.0 - 1.0), 0.0), 1.0)
        assert math.isclose(f[i].item(), (1 - g) * b / s + g * b, rel_tol=1e-12)
    assert f[0].item() == base[0] and math.isclose(f[-1].item(), base[-1] / s, rel_tol=1e-12)
    assert math.isclose(m, 0.1 * math.log(s) + 1.0)


@pytest.mark.parametrize("kw", [dict(rot_dim=0), dict(rot_dim=7), dict(rot_dim=64, factor=0.5),
                                dict(rot_dim=64, scaling="yarn", factor=4.0), dict(rot_dim=2, scaling="ntk", factor=2.0),
                                dict(rot_dim=64, scaling="other")])
def test_rope_frequencies_refusals(kw):
    with pytest.raises(ValueError):
        K.rope_frequencies(device="cpu", **kw)


def plan_add(name, d):
    """The plan add's return code and, where it refused, its message."""
    lib = _lib.load()
    plan = ctypes.c_void_p()
    assert lib.rfx_plan_create(ctypes.byref(plan)) == _lib.RFX_OK
    try:
        rc = getattr(lib, "rfx_plan_add_" + name)(plan, ctypes.byref(d))
        return rc, lib.rfx_last_error() if rc else b""
    finally:
        lib.rfx_plan_destroy(plan)


def rope_at(**change):
    """rope()'s tensors (x, positions, inv_freq, q, k, v at 1 to 6 A), every output packed head-major."""
    d = rope()
    for k, v in change.items():
        setattr(d, k, v)
    for n, h in (("q", d.num_q_heads), ("k", d.num_kv_heads), ("v", d.num_kv_heads)):
        for s, packed in (("b", h * d.S * d.head_dim), ("h", d.S * d.head_dim), ("s", d.head_dim)):
            if f"{n}s_{s}" not in change:
                setattr(d, f"{n}s_{s}", packed)
    d.ldx = max(d.ldx, (d.num_q_heads + 2 * d.num_kv_heads) * d.head_dim)
    return d


OWN_PLACES = [  # the strides of one rope output: whether its heads and tokens lie apart
    ({}, True), (dict(B=3, num_kv_heads=2), True),
    (dict(qs_h=64, qs_s=64), False),                      # head 1 of a token over head 0 of the next
    (dict(qs_h=63), False), (dict(qs_s=63), False), (dict(B=2, qs_b=511), False), (dict(B=2, qs_b=448), False),
    (dict(qs_h=64, qs_s=128), True), (dict(qs_h=64, qs_s=127), False),
    (dict(qs_h=0), False), (dict(qs_s=0), False), (dict(qs_h=0, qs_s=0), False),
    (dict(qs_h=192, qs_s=128), True),                     # 0, 128, 256, 384 and 192, 320, 448, 576: apart, nested in no order
    (dict(qs_h=191, qs_s=128), False),
    (dict(qs_h=-64, qs_s=128), True), (dict(qs_h=-256, qs_s=-64), True), (dict(qs_h=-64, qs_s=-64), False),
    (dict(qs_b=1), True),                                 # one stream: its stride is not used
    (dict(S=1, qs_s=0), True), (dict(ks_h=0), True), (dict(num_kv_heads=2, ks_h=0), False),
    (dict(num_kv_heads=2, vs_h=64, vs_s=64), False), (dict(num_kv_heads=2, vs_h=64, vs_s=128), True),
    (dict(B=2, qs_b=0, qs_h=0, qs_s=0), True),            # none given: packed, head-major
    (dict(B=2, num_kv_heads=4, vs_b=0, vs_h=0, vs_s=0), True),
]


@pytest.mark.parametrize("change,fine", OWN_PLACES)
def test_rope_outputs_lie_apart_from_themselves(change, fine):
    """Two heads or tokens of an output at one place would be written by two
    threads at once; three strides of 0 stand for a packed output."""
    rc, why = plan_add("rope", rope_at(**change))
    assert rc == (_lib.RFX_OK if fine else _lib.RFX_E_INVAL), why
    assert fine or (b"rfx_rope" in why and b"overlap" in why)


def places(d, n, heads):
    """Every element's offset of output `n`, one per (stream, head, token, dim)."""
    sb, sh, ss = (getattr(d, f"{n}s_{c}") for c in "bhs")
    if not (sb or sh or ss):
        sb, sh, ss = heads * d.S * d.head_dim, d.S * d.head_dim, d.head_dim
    return [b * sb + h * sh + s * ss + e for b in range(d.B) for h in range(heads) for s in range(d.S)
            for e in range(d.head_dim)]


def test_rope_overlap_of_any_strides():
    """Random strides, negative and tangled ones among them, against the
    places written down one by one."""
    rng = random.Random(1)
    seen = [0, 0]
    for _ in range(4000):
        D = rng.choice([2, 4, 6])
        top = rng.choice([8, 30, 100])
        d = rope_at(B=rng.randint(1, 3), S=rng.randint(1, 4), num_q_heads=rng.randint(1, 4), num_kv_heads=0, head_dim=D,
                    rot_dim=2, k_out=None, v_out=None, qs_b=rng.randint(-top, top), qs_h=rng.randint(-top, top),
                    qs_s=rng.randint(-top, top))
        at = places(d, "q", d.num_q_heads)
        fine = len(set(at)) == len(at)
        seen[fine] += 1
        rc, why = plan_add("rope", d)
        assert rc == (_lib.RFX_OK if fine else _lib.RFX_E_INVAL), (why, d.B, d.num_q_heads, d.S, D, d.qs_b, d.qs_h, d.qs_s)
    assert min(seen) > 400, seen


# q 1024 bytes at 4 A, k and v 512 bytes at 5 A and 6 A, positions 16 bytes at 2 A, inv_freq 256 at 3 A
STREAMS = dict(B=2, positions=2 * A, qs_b=1024, qs_h=64, qs_s=128)  # a workspace of 1024 elements per stream
FAR = dict(B=64, S=6344, num_q_heads=8, num_kv_heads=4, x=1 << 40, q_out=2 << 40, k_out=3 << 40, v_out=(3 << 40) + 128)
OTHER_PLACES = [  # rope outputs beside one another and beside the inputs
    ({}, True),
    (dict(k_out=4 * A), False), (dict(k_out=4 * A + 1022), False), (dict(k_out=4 * A + 1024), True),
    (dict(k_out=4 * A - 510), False), (dict(k_out=4 * A - 512), True),
    (dict(v_out=5 * A), False), (dict(v_out=5 * A + 510), False), (dict(v_out=5 * A + 512), True),
    (dict(v_out=4 * A + 512), False),
    (dict(k_out=5 * A, ks_s=128, v_out=5 * A + 128, vs_s=128), True),   # one cache, [S][k | v]
    (dict(k_out=5 * A, ks_s=128, v_out=5 * A + 126, vs_s=128), False),
    (dict(k_out=5 * A, ks_s=127, v_out=5 * A + 128, vs_s=127), False),
    (dict(k_out=5 * A, ks_s=128, v_out=5 * A + 128, vs_s=192), False),  # the third token of each meets
    (dict(num_kv_heads=2, ks_h=128, ks_s=256, v_out=5 * A + 128, vs_h=128, vs_s=256), True),  # [S][heads][k | v]
    (dict(num_kv_heads=2, ks_h=128, ks_s=256, v_out=5 * A + 128, vs_h=64, vs_s=256), False),
    (dict(STREAMS, k_out=4 * A + 1024, ks_b=1024, v_out=4 * A + 1536, vs_b=1024), True),
    (dict(STREAMS, k_out=4 * A + 1024, ks_b=1024, v_out=4 * A + 1408, vs_b=1024), False),
    (dict(STREAMS, k_out=4 * A + 896, ks_b=1024, v_out=4 * A + 1536, vs_b=1024), False),
    (dict(STREAMS, k_out=4 * A + 1024, ks_b=512, v_out=6 * A, vs_b=256), False),  # stream 1's k over its q
    (dict(k_out=5 * A + 384, ks_s=-64, v_out=5 * A + 512), True), (dict(k_out=5 * A + 384, ks_s=-64, v_out=5 * A), False),
    (dict(q_out=2 * A), False), (dict(q_out=2 * A + 14), False), (dict(q_out=2 * A + 16), True),
    (dict(q_out=2 * A - 1022), False), (dict(q_out=2 * A - 1024), True), (dict(v_out=2 * A), False),
    (dict(k_out=3 * A), False), (dict(k_out=3 * A + 254), False), (dict(k_out=3 * A + 256), True),
    (dict(v_out=3 * A + 2), False), (dict(rot_dim=32, v_out=3 * A + 128), True),
    (dict(positions=4 * A + 128, qs_h=64, qs_s=256), False),            # positions in q's rows,
    (dict(positions=4 * A + 256, qs_h=64, qs_s=256), True),             # or in the columns between them
    (dict(q_out=4 * A, k_out=4 * A, v_out=4 * A, positions=4 * A, inv_freq=4 * A), False),
    # caches of 64 streams, [stream][S][heads][k | v] and [stream][heads][S][k | v]
    (dict(FAR, ks_b=6400 * 512, ks_h=128, ks_s=512, vs_b=6400 * 512, vs_h=128, vs_s=512), True),
    (dict(FAR, ks_b=6400 * 512, ks_h=6400 * 128, ks_s=128, vs_b=6400 * 512, vs_h=6400 * 128, vs_s=128), True),
    (dict(FAR, ks_b=6400 * 512, ks_h=6400 * 128, ks_s=128, vs_b=6400 * 512, vs_h=6400 * 128, vs_s=126), False),
    (OVER_X, True), (dict(OVER_X, k_out=5 * A, ks_b=256, ks_s=64), True),
    (dict(OVER_X, positions=A + 512), False), (dict(OVER_X, positions=A + 2048), True),
    (dict(OVER_X, k_out=5 * A, ks_b=256, ks_s=64, v_out=5 * A, vs_b=256, vs_s=64), False),
]


@pytest.mark.parametrize("change,fine", OTHER_PLACES)
def test_rope_outputs_lie_apart_from_the_rest(change, fine):
    """CTAs read positions and inv_freq, and write q, k and v, in no order."""
    rc, why = plan_add("rope", rope_at(**change))
    assert rc == (_lib.RFX_OK if fine else _lib.RFX_E_INVAL), why
    assert fine or (b"rfx_rope" in why and (b"share memory" in why or b"shares memory" in why or b"lies across" in why))


def test_rope_sharing_of_any_strides():
    """Random layouts of q, k and x in one small buffer, against the places
    written down one by one."""
    rng = random.Random(2)
    seen = [0, 0]
    for _ in range(6000):
        D, S, B = rng.choice([2, 4]), rng.randint(1, 4), rng.randint(1, 2)
        Hq, Hk = rng.randint(1, 2), rng.randint(1, 3)
        T, width = B * S, (Hq + Hk) * D
        ldx = width + rng.choice([0, 0, 2, 8, 13])
        st = {}
        for n in "qk":
            st.update({f"{n}s_b": rng.choice([S * ldx, ldx * S + 5, 64, 31]), f"{n}s_h": rng.choice([D, S * D, -D, 9, 17]),
                       f"{n}s_s": rng.choice([ldx, D, 2 * D, 33])})
        at = lambda: A + 2 * rng.randint(-40, 160)  # noqa: E731
        d = rope_at(B=B, S=S, num_q_heads=Hq, num_kv_heads=Hk, head_dim=D, rot_dim=2, v_out=None, **st)
        d.ldx, d.x, d.q_out, d.k_out = ldx, A, rng.choice([A, at()]), rng.choice([A + 2 * Hq * D, at(), at()])
        x = {t * ldx + e for t in range(T) for e in range(width)}
        sets = []
        fine = True
        for n, h, own in (("q", Hq, 0), ("k", Hk, Hq * D)):
            p = places(d, n, h)
            off = (getattr(d, n + "_out") - A) // 2
            p = [off + e for e in p]
            over = p == [own + (b * S + s) * ldx + i * D + e for b in range(B) for i in range(h) for s in range(S)
                         for e in range(D)]
            fine &= len(set(p)) == len(p) and (over or not x & set(p))
            sets.append(set(p))
        fine &= not sets[0] & sets[1]
        seen[fine] += 1
        rc, why = plan_add("rope", d)
        assert rc == (_lib.RFX_OK if fine else _lib.RFX_E_INVAL), (why, st, B, S, Hq, Hk, D, ldx, d.q_out - A, d.k_out - A)
    assert min(seen) > 300, seen


def norm_at(**change):
    """norm() over two streams of two tokens, with all five vectors, gate and a2 / b2 at a batch stride of 64."""
    d = norm()
    d.tokens_per_batch = 2
    d.post_w, d.gate, d.norm_a1, d.norm_a2, d.norm_b2 = (i * A for i in range(7, 12))
    d.gate_stride = d.norm_ab_stride = 64
    for k, v in change.items():
        setattr(d, k, v)
    return d


TO_INT8 = dict(z=None, z_q=5 * A, z_scale=6 * A)
VECTOR_PLACES = [  # block_norm's outputs (512 bytes each of h_out and z, 256 of z_q, 16 of z_scale) and its vectors
    ({}, True), (TO_INT8, True),
    (dict(post_w=3 * A), False), (dict(post_w=3 * A + 508), False), (dict(post_w=3 * A + 512), True),
    (dict(post_w=3 * A - 252), False), (dict(post_w=3 * A - 256), True),
    (dict(norm_a1=4 * A), False), (dict(norm_a1=3 * A), False), (dict(norm_a1=4 * A + 512), True),
    (dict(gate=4 * A), False), (dict(gate=4 * A - 256), False), (dict(gate=4 * A - 512), True),  # its second stream's row
    (dict(gate=4 * A - 256, gate_stride=0), True), (dict(gate=4 * A - 252, gate_stride=0), False),
    (dict(gate=4 * A - 256, tokens_per_batch=4), True),                                          # one stream only
    (dict(norm_a2=3 * A), False), (dict(norm_b2=3 * A), False), (dict(norm_a2=4 * A), False), (dict(norm_b2=4 * A), False),
    (dict(norm_b2=4 * A - 1024, norm_ab_stride=256), False), (dict(norm_b2=4 * A - 1280, norm_ab_stride=256), True),
    (dict(TO_INT8, norm_a1=5 * A), False), (dict(TO_INT8, gate=5 * A + 252), False), (dict(TO_INT8, gate=5 * A + 256), True),
    (dict(TO_INT8, post_w=6 * A), False), (dict(TO_INT8, norm_b2=6 * A + 12), False), (dict(TO_INT8, norm_b2=6 * A + 16), True),
    (dict(T=3, gate=4 * A - 256), False), (dict(T=2, gate=4 * A - 256), True),                   # the last stream cut short
    # vectors in the columns between the outputs' rows
    (dict(ldho=192, post_w=3 * A + 128), True), (dict(ldho=190, post_w=3 * A + 128), False),
    (dict(ldho=192, gate=3 * A + 128, gate_stride=192), True), (dict(ldho=192, gate=3 * A + 128, gate_stride=96), True),
    (dict(ldho=192, gate=3 * A + 128, gate_stride=64), False),
    (dict(h_out=A, post_w=A), False), (dict(h_out=A, z=2 * A, norm_a1=2 * A), False),            # outputs in place
    (dict(gate=7 * A), True), (dict(norm_a1=A), True), (dict(norm_b2=10 * A), True),             # inputs may share
]


@pytest.mark.parametrize("change,fine", VECTOR_PLACES)
def test_block_norm_outputs_lie_apart_from_the_vectors(change, fine):
    """Every CTA reads the vectors while others write their rows."""
    rc, why = plan_add("block_norm", norm_at(**change))
    assert rc == (_lib.RFX_OK if fine else _lib.RFX_E_INVAL), why
    assert fine or (b"rfx_block_norm" in why and b"share" in why)


HUGE = (1 << 32) + 16  # a 32-bit size would hold 16 of it


@pytest.fixture
def meta(monkeypatch):
    """Makes the descriptor builders take meta tensors, which have sizes and no memory."""
    monkeypatch.setattr(K, "_current", lambda dev: dev)
    return lambda *shape, dt=torch.float32: torch.empty(*shape, dtype=dt, device="meta")


@pytest.mark.parametrize("T,Kc", [(1, HUGE), (2, HUGE), (HUGE, 1), (1 << 31, 1), (1, 1 << 31)])
def test_sizes_past_32_bits_are_refused(meta, T, Kc):
    """Descriptors hold sizes in 32 bits: a larger one is refused, not cut."""
    i8 = torch.int8
    with pytest.raises(ValueError, match="2\\^31"):
        K.quant_rows_desc(x=meta(T, Kc), q=meta(T, Kc, dt=i8), scale=meta(T))
    with pytest.raises(ValueError, match="2\\^31"):
        K.block_norm_desc(h=meta(T, Kc), S=1, z=meta(T, Kc))
    with pytest.raises(ValueError, match="2\\^31"):
        K.linear_i8_desc(w=meta(8, Kc, dt=i8), w_scale=meta(8), x=meta(T, Kc, dt=i8), x_scale=meta(T), y=meta(T, 8))
    with pytest.raises(ValueError, match="2\\^31"):
        K.linear_i8_desc(w=meta(T, Kc, dt=i8), w_scale=meta(T), x=meta(1, Kc, dt=i8), x_scale=meta(1), y=meta(1, T))


@pytest.mark.parametrize("B,Hq,S,D,Hkv,pairs", [
    (1, 1, 1, HUGE, 0, 8), (1, HUGE, 1, 16, 0, 8), (1, 1, HUGE, 16, 0, 8), (HUGE, 1, 1, 16, 0, 8), (1 << 16, 1, 1 << 16, 16, 0, 8),
    (1, 1, 1, 16, HUGE, 8), (1, 1, 1, 16, 0, (1 << 31) + 8), (1, 1, 1, 16, 0, 1 << 30),
])
def test_rope_sizes_past_32_bits_are_refused(meta, B, Hq, S, D, Hkv, pairs):
    kv = dict(k_out=meta(B, Hkv, S, D)) if Hkv else {}
    with pytest.raises(ValueError, match="2\\^31"):
        K.rope_desc(x=meta(B * S, (Hq + Hkv) * D), positions=meta(B * S, dt=torch.int32),
                    inv_freq=meta(pairs, dt=torch.float64), q_out=meta(B, Hq, S, D), **kv)


def test_largest_sizes_are_passed_on(meta):
    """Sizes that fit reach the C entry's own limits unchanged."""
    top = (1 << 31) - 1
    d = K.quant_rows_desc(x=meta(1, top), q=meta(1, top, dt=torch.int8), scale=meta(1))
    assert (d.T, d.K) == (1, top)
    d = K.quant_rows_desc(x=meta(top, 1), q=meta(top, 1, dt=torch.int8), scale=meta(top))
    assert (d.T, d.K) == (top, 1)
    d = K.rope_desc(x=meta(top, 2), positions=meta(top, dt=torch.int32), inv_freq=meta(1, dt=torch.float64),
                    q_out=meta(1, 1, top, 2))
    assert (d.B, d.S, d.rot_dim) == (1, top, 2)
