"""The 4-bit layer operators and the attention over a shared context without a
GPU: struct layouts, the refusals of the C entry points and of the tensor
wrappers, empty calls, sizes of scales and workspaces."""
import ctypes
import os
import subprocess

import pytest
import torch

from reflex_b200 import _lib as L
from reflex_b200 import kernels as K

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"rfx_quant_fp4_desc": "QuantFp4Desc", "rfx_dequant_fp4_desc": "DequantFp4Desc",
           "rfx_linear_fp4_desc": "LinearFp4Desc", "rfx_kv_view": "KvView", "rfx_attn_shared_desc": "AttnSharedDesc"}
ENTRIES = {"rfx_quant_fp4": "quant_fp4", "rfx_dequant_fp4": "dequant_fp4", "rfx_linear_fp4": "linear_fp4",
           "rfx_attention_shared": "attention_shared"}
A = 1 << 24  # an aligned address that is never dereferenced
MX, NV, BF, F32 = L.RFX_FP4_MX, L.RFX_FP4_NV, L.RFX_DTYPE_BF16, L.RFX_DTYPE_F32


def test_structs_match_c_layout(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "rfx.h"', "int main(void) {"]
    for c_name, py_name in STRUCTS.items():
        lines.append(f'  printf("{py_name} size %zu\\n", sizeof({c_name}));')
        for field, _ in getattr(L, py_name)._fields_:
            lines.append(f'  printf("{py_name} {field} %zu\\n", offsetof({c_name}, {field}));')
    lines.append("  return 0; }")
    c = tmp_path / "layout.c"
    c.write_text("\n".join(lines))
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(c), "-o", str(tmp_path / "layout")],
                   check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split("\n")
    for line in filter(None, out):
        py_name, key, val = line.split()
        cls = getattr(L, py_name)
        got = ctypes.sizeof(cls) if key == "size" else getattr(cls, key).offset
        assert got == int(val), f"{py_name}.{key}: ctypes {got}, C {val}"


def quant():  # 4 rows of 64, a row scale each
    return L.QuantFp4Desc(4, 64, NV, BF, 0, A, 64, 2 * A, 32, 3 * A, 4 * A)


def dequant():
    return L.DequantFp4Desc(4, 64, MX, F32, 0, 2 * A, 32, 3 * A, None, A, 64)


def linear():
    return L.LinearFp4Desc(4, 64, 64, NV, L.RFX_EPI_STORE, BF, A, 32, 2 * A, 3 * A, 4 * A, 32, 5 * A, 6 * A, None, 7 * A, 64)


def attention():  # 2 streams of 3 tokens, 2 heads over one, 100 shared slots, rings of 40, new keys
    d = L.AttnSharedDesc()
    d.B, d.S, d.num_q_heads, d.num_kv_heads, d.head_dim = 2, 3, 2, 1, 256
    d.quant_mode, d.scale_dtype, d.n_shared, d.own_max = L.RFX_QUANT_I8_SYM, F32, 100, 40
    d.q, d.qs_b, d.qs_h, d.qs_s = A, 3 * 512, 256, 512
    d.shared = L.KvView(2 * A, 3 * A, 4 * A, 5 * A, None, None, 0, 0, 256, 0, 0, 1)
    d.own = L.KvView(6 * A, 7 * A, 8 * A, 9 * A, None, None, 40 * 256, 40 * 256, 256, 40, 40, 1)
    d.k_new, d.ks_b, d.ks_h, d.ks_s = 10 * A, 768, 768, 256
    d.v_new, d.vs_b, d.vs_h, d.vs_s = 11 * A, 768, 768, 256
    d.softmax_scale, d.out, d.ldo = 1 / 16, 12 * A, 512
    d.workspace, d.workspace_bytes = 16 * A, 1 << 30
    return d


def wide():  # 64 streams of 50 tokens: the form that has a workspace
    d = attention()
    d.B, d.S, d.own_max = 64, 50, 0
    d.qs_b, d.qs_s, d.ks_b, d.vs_b = 50 * 512, 512, 50 * 256, 50 * 256
    return d


def changed(make, change):
    d = make()
    for k, v in change.items():
        at, *rest = k.split("__")
        if rest:
            setattr(getattr(d, at), rest[0], v)
        else:
            setattr(d, k, v)
    return d


def plan_add(entry, d):
    """(return code, launches) of adding the descriptor to an empty plan."""
    lib = L.load()
    plan, n = ctypes.c_void_p(), ctypes.c_int(-1)
    assert lib.rfx_plan_create(ctypes.byref(plan)) == L.RFX_OK
    try:
        rc = getattr(lib, "rfx_plan_add_" + ENTRIES[entry])(plan, ctypes.byref(d))
        assert lib.rfx_plan_num_launches(plan, ctypes.byref(n)) == L.RFX_OK
    finally:
        lib.rfx_plan_destroy(plan)
    return rc, n.value


@pytest.mark.parametrize("name", sorted(ENTRIES))
def test_null_descriptor_is_refused(name):
    lib = L.load()
    assert getattr(lib, name)(None, None) == L.RFX_E_INVAL
    n = ctypes.c_size_t(0)
    assert lib.rfx_attention_shared_workspace_size(None, ctypes.byref(n)) == L.RFX_E_INVAL
    assert lib.rfx_attention_shared_workspace_size(ctypes.byref(attention()), None) == L.RFX_E_INVAL


Q, DQ, LI, AT = ("rfx_quant_fp4", quant), ("rfx_dequant_fp4", dequant), ("rfx_linear_fp4", linear), ("rfx_attention_shared", attention)
BAD = [
    *[(*Q, c) for c in (dict(T=-1), dict(T=(1 << 30) + 1), dict(K=0), dict(K=65537, ldx=65537, ldq=32784), dict(format=2),
                        dict(in_dtype=2), dict(rows_per_part=-1), dict(rows_per_part=3), dict(x=None), dict(q=None),
                        dict(scale=None), dict(row_scale=None), dict(format=MX), dict(ldx=63), dict(ldq=16), dict(ldq=40),
                        dict(q=2 * A + 8), dict(scale=3 * A + 8), dict(x=A + 1), dict(row_scale=4 * A + 2),
                        dict(q=A + 512 - 16), dict(scale=A), dict(row_scale=2 * A + 4), dict(row_scale=3 * A + 508))],
    *[(*DQ, c) for c in (dict(T=-1), dict(K=0), dict(K=65537, ldy=65537, ldq=32784), dict(format=-1), dict(out_dtype=7),
                         dict(rows_per_part=5), dict(y=None), dict(q=None), dict(scale=None), dict(row_scale=4 * A),
                         dict(format=NV), dict(ldy=63), dict(ldq=31), dict(q=2 * A + 1), dict(scale=3 * A + 4),
                         dict(y=A + 2), dict(y=2 * A + 124), dict(y=3 * A + 508))],
    *[(*LI, c) for c in (dict(T=-1), dict(T=(1 << 30) + 1), dict(O=0), dict(O=(1 << 30) + 1), dict(K=0),
                         dict(K=65537, ldx=32784, ldw=32784), dict(format=3), dict(epilogue=L.RFX_EPI_RESIDUAL),
                         dict(epilogue=L.RFX_EPI_QKV_ROPE), dict(epilogue=L.RFX_EPI_GEGLU, O=63), dict(out_dtype=4),
                         dict(x=None), dict(w=None), dict(y=None), dict(x_scale=None), dict(w_scale=None),
                         dict(x_row_scale=None), dict(w_row_scale=None), dict(format=MX),
                         dict(format=MX, x_row_scale=None), dict(x=A + 8), dict(w=4 * A + 8), dict(x_scale=2 * A + 4),
                         dict(w_scale=5 * A + 4), dict(ldx=16), dict(ldw=40), dict(ldy=63), dict(y=7 * A + 1),
                         dict(bias=8 * A + 2), dict(x_row_scale=3 * A + 1), dict(w_row_scale=6 * A + 2),
                         dict(y=A), dict(y=4 * A + 2016), dict(y=2 * A), dict(y=5 * A), dict(y=3 * A), dict(y=6 * A),
                         dict(bias=7 * A), dict(T=1 << 30, O=1 << 26, ldy=1 << 26))],
    *[(*AT, c) for c in (dict(B=-1), dict(S=-1), dict(num_q_heads=0), dict(num_kv_heads=0), dict(num_kv_heads=3),
                         dict(head_dim=128), dict(n_shared=-1), dict(own_max=-1), dict(quant_mode=5), dict(scale_dtype=9),
                         dict(scale_dtype=BF), dict(k_new=None), dict(v_new=None), dict(q=None), dict(out=None),
                         dict(shared__k=None), dict(shared__v_scale=None), dict(own__v=None), dict(own__k_scale=None),
                         dict(quant_mode=L.RFX_QUANT_U8_REF), dict(shared__k=2 * A + 8), dict(shared__qs_c=264),
                         dict(own__qs_b=8), dict(own__qs_h=40), dict(own__k_scale=8 * A + 2), dict(q=A + 8),
                         dict(qs_b=1540), dict(qs_h=252), dict(qs_s=513), dict(out=12 * A + 8), dict(ldo=504),
                         dict(ldo=516), dict(k_new=10 * A + 2), dict(ks_s=257), dict(vs_b=772), dict(vs_h=4),
                         dict(own_len=13 * A + 2), dict(new_block=13 * A + 1), dict(out=A), dict(out=2 * A + 1024),
                         dict(out=7 * A), dict(out=4 * A), dict(out=9 * A + 64), dict(out=10 * A + 512), dict(out=11 * A),
                         dict(own_len=12 * A + 16), dict(B=1 << 20, S=1 << 20), dict(B=1 << 25, S=1),
                         dict(n_shared=0x7fffffff, own_max=0x7fffffff))],
    *[("rfx_attention_shared", wide, c) for c in (
        dict(workspace=None), dict(workspace=16 * A + 512), dict(workspace_bytes=1024), dict(workspace=A),
        dict(workspace=2 * A), dict(workspace=11 * A), dict(workspace=12 * A), dict(shared_valid=16 * A),
        dict(new_block=16 * A + 1024))],
]


@pytest.mark.parametrize("entry,make,change", BAD)
def test_bad_descriptors_are_refused(entry, make, change):
    """Refused by the direct call and by the plan add, with a message that
    names the entry point; the plan stays empty."""
    lib = L.load()
    d = changed(make, change)
    assert getattr(lib, entry)(ctypes.byref(d), None) == L.RFX_E_INVAL
    assert entry.encode() in lib.rfx_last_error()
    assert plan_add(entry, d) == (L.RFX_E_INVAL, 0)


@pytest.mark.parametrize("entry,make,change", [
    (*Q, dict(T=0, x=None, q=None, scale=None, row_scale=None)), (*DQ, dict(T=0, y=None, q=None, scale=None)),
    (*LI, dict(T=0, x=None, y=None, x_scale=None)), (*AT, dict(B=0, q=None, out=None)), (*AT, dict(S=0, q=None, workspace=None)),
])
def test_no_rows_is_a_no_op(entry, make, change):
    """No rows: accepted without a device, nothing launched."""
    d = changed(make, change)
    assert getattr(L.load(), entry)(ctypes.byref(d), None) == L.RFX_OK
    assert plan_add(entry, d) == (L.RFX_OK, 0)


@pytest.mark.parametrize("entry,make,change", [
    (*Q, {}), (*Q, dict(format=MX, row_scale=None)), (*Q, dict(ldx=96, q=A + 128, ldq=192)),  # the free columns of x's rows
    (*Q, dict(q=A + 512)), (*DQ, {}), (*DQ, dict(format=NV, row_scale=4 * A)), (*DQ, dict(y=2 * A + 128)),
])
def test_one_launch_each(entry, make, change):
    assert plan_add(entry, changed(make, change)) == (L.RFX_OK, 1)


def test_attention_launches_and_workspace():
    """Few rows: one kernel and, of one tile with few keys, no workspace; many: the keys'
    copy, attention and, where a tile's parts are many, the kernel that joins them."""
    lib = L.load()

    def need(d):
        n = ctypes.c_size_t(12345)
        assert lib.rfx_attention_shared_workspace_size(ctypes.byref(d), ctypes.byref(n)) == L.RFX_OK
        return n.value
    assert need(changed(attention, dict(B=0))) == 0 and need(changed(attention, dict(S=0))) == 0
    few = changed(attention, dict(n_shared=16, own_max=0))
    assert plan_add("rfx_attention_shared", few)[0] == L.RFX_OK
    big = wide()
    n = need(big)
    blocks = 2 + 64  # of 64 keys: the shared ones, and each stream's 50 new
    assert n >= blocks * 64 * (512 + 512 + 16)
    rc, launches = plan_add("rfx_attention_shared", big)
    assert rc == L.RFX_OK and launches in (2, 3)
    big.workspace_bytes = n
    assert plan_add("rfx_attention_shared", big)[0] == L.RFX_OK
    big.workspace_bytes = n - 1
    assert plan_add("rfx_attention_shared", big)[0] == L.RFX_E_INVAL
    # no keys at all: rows of zeros
    assert plan_add("rfx_attention_shared", changed(attention, dict(n_shared=0, own_max=0, k_new=None, v_new=None)))[0] == L.RFX_OK


def test_scale_bytes():
    """128 rows x 4 blocks in 512 bytes, whole tiles, each part by itself."""
    for T, Kc, fmt, parts, tiles in ((1, 1, MX, 1, 1), (128, 128, MX, 1, 1), (129, 128, MX, 1, 2), (128, 129, MX, 1, 2),
                                     (1, 64, NV, 1, 1), (1, 65, NV, 1, 2), (200, 1000, NV, 2, 2 * 16),
                                     (2 * 129, 64, NV, 2, 4), (0, 64, MX, 1, 0)):
        assert K.fp4_scale_bytes(T, Kc, fmt, parts) == 512 * tiles
        r = K.Fp4Rows.allocate(T, Kc, fmt, parts, device="cpu")
        assert r.scale.numel() == 512 * tiles and r.q.shape == (T, (Kc + 1) // 2)
        assert (r.row_scale is None) == (fmt == MX)


def test_rows_are_checked_when_made():
    r = K.Fp4Rows.allocate(6, 100, NV, 2, device="cpu")
    u8 = torch.uint8

    def make(**change):
        return K.Fp4Rows(**{**dict(q=r.q, scale=r.scale, row_scale=r.row_scale, K=100, fmt=NV, parts=2), **change})
    make()
    for change in (dict(q=r.q.float()), dict(scale=r.scale.float()), dict(K=0), dict(K=101), dict(q=r.q[:, :49]),
                   dict(q=r.q[:5]), dict(parts=0), dict(parts=4), dict(scale=r.scale[:-1]),
                   dict(scale=torch.zeros(2 * r.scale.numel(), dtype=u8)[::2]), dict(row_scale=None), dict(fmt=MX),
                   dict(row_scale=r.row_scale[:5]), dict(row_scale=r.row_scale.double()),
                   dict(q=torch.zeros(6, 50, dtype=u8)), dict(q=torch.zeros(50, 6, dtype=u8).t())):
        with pytest.raises(ValueError):
            make(**change)
    for args in ((-1, 4, MX, 1), (4, 0, MX, 1), (5, 4, MX, 2), (4, 4, MX, 0)):
        with pytest.raises(ValueError):
            K.Fp4Rows.allocate(*args, device="cpu")


def test_cpu_tensors_are_refused():
    x, y = torch.zeros(2, 32), torch.zeros(2, 2)
    r = K.Fp4Rows.allocate(2, 32, MX, device="cpu")
    ring = K.KVRing.allocate(1, 1, 16, 256, L.RFX_QUANT_I8_SYM, device="cpu")
    q = torch.zeros(1, 1, 1, 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        K.quant_fp4(x=x, out=r)
    with pytest.raises(ValueError, match="CUDA"):
        K.dequant_fp4(x=r, out=x)
    with pytest.raises(ValueError, match="CUDA"):
        K.linear_fp4(w=r, x=r, y=y)
    with pytest.raises(ValueError, match="CUDA"):
        K.attention_shared(q=q, shared=ring, n_shared=4, out=q.view(1, 256), softmax_scale=1.0)
