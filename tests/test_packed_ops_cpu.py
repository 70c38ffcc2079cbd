"""Refusals and host helpers of the packed-volume operators (rotary positions, attention with modified scores, gated residual): no GPU needed.
What the C entry points refuse is refused before any launch; what the launchers refuse is refused before the C call."""
import ctypes as C

import pytest
import torch

from mirage_amd import _lib as L
from mirage_amd import kernels as K
from mirage_amd import packed

BF16, F32 = torch.bfloat16, torch.float32


def error():
    return L.lib.mrg_last_error_string().decode()


def rotary_desc(**kw):
    d = L.RotaryDesc()
    d.q = d.q_out = d.pos = d.freqs = 4096
    d.q_bs = d.qo_bs = 256
    d.q_rs = d.qo_rs = 64
    d.q_hs = d.qo_hs = 64
    d.B, d.N, d.Hq, d.head_dim, d.axes = 1, 4, 1, 64, 2
    d.sections[0], d.sections[1] = 16, 16
    for k, v in kw.items():
        if k == "sections":
            for i in range(3):
                d.sections[i] = v[i] if i < len(v) else 0
        else:
            setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=7), "dtype"), (dict(pos_dtype=5), "positions"), (dict(pairing=3), "pairing"), (dict(axes=0), "axes"), (dict(axes=4), "axes"), (dict(B=-1), "negative"),
    (dict(head_dim=258), "head_dim"), (dict(head_dim=1), "head_dim"), (dict(sections=(16, 0)), "section"), (dict(sections=(-3, 4)), "section"),
    (dict(sections=(20, 16)), "do not fit"), (dict(freqs=None), "null"), (dict(q=None), "null"), (dict(Hk=2), "null"), (dict(q=4097), "aligned"),
    (dict(B=1 << 20, N=1 << 20), "too many")])
def test_rotary_refuses(kw, text):
    assert L.lib.mrg_rotary_axes(C.byref(rotary_desc(**kw)), None) < 0 and text in error()


def test_empty_calls_launch_nothing():
    assert L.lib.mrg_rotary_axes(C.byref(rotary_desc(B=0)), None) == 0
    assert L.lib.mrg_rotary_axes(C.byref(rotary_desc(Hq=0)), None) == 0
    assert L.lib.mrg_attn_mod_fwd(C.byref(attn_desc(Nq=0)), None) == 0
    assert L.lib.mrg_attn_mod_bwd(C.byref(attn_desc(B=0)), None) == 0
    assert L.lib.mrg_resid_norm_fwd(C.byref(norm_desc(samples=0)), None) == 0
    for f in (L.lib.mrg_rotary_axes, L.lib.mrg_attn_mod_fwd, L.lib.mrg_attn_mod_bwd, L.lib.mrg_resid_norm_fwd, L.lib.mrg_resid_norm_bwd):
        assert f(None, None) < 0 and "null descriptor" in error()


def norm_desc(**kw):
    d = L.ResidNormDesc()
    d.samples, d.rows_per_sample, d.D, d.alpha, d.eps = 2, 3, 64, 1.0, 1e-6
    for f in ("x", "branch", "x_new", "y", "stats", "pre_w", "dx_new", "dy", "dx", "dbranch", "d_pre_w", "ws"):
        setattr(d, f, 4096)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,text", [
    (dict(D=0), "multiple of 4"), (dict(D=66), "multiple of 4"), (dict(D=4100), "4096"), (dict(samples=-1), "row counts"), (dict(samples=1 << 20, rows_per_sample=1 << 20), "row counts"),
    (dict(norm=2), "unknown norm"), (dict(branch_dtype=2), "branch dtype"), (dict(y_dtype=-1), "y dtype"), (dict(gate_rows=3, gate=4096), "gate rows"),
    (dict(gate_rows=1), "disagree"), (dict(gate=4096), "disagree"), (dict(post_b=4096), "without its weight"), (dict(pre_w=None, pre_b=4096), "without its weight"),
    (dict(x=4100), "aligned")])
def test_resid_norm_refuses(kw, text):
    d = norm_desc(**kw)
    for f in (L.lib.mrg_resid_norm_fwd, L.lib.mrg_resid_norm_bwd):
        assert f(C.byref(d), None) < 0 and text in error()
    assert L.lib.mrg_resid_norm_ws_floats(C.byref(d)) == -1


@pytest.mark.parametrize("kw,f", [(dict(x=None), "fwd"), (dict(y=None), "fwd"), (dict(stats=None), "fwd"), (dict(dy=None), "bwd"), (dict(ws=None), "bwd"), (dict(stats=None), "bwd")])
def test_resid_norm_refuses_null(kw, f):
    assert getattr(L.lib, "mrg_resid_norm_" + f)(C.byref(norm_desc(**kw)), None) < 0 and "null" in error()


def test_resid_norm_needs_every_gradient():
    for kw in (dict(d_pre_w=None), dict(post_w=4096), dict(gate=4096, gate_rows=1), dict(pre_b=4096)):
        assert L.lib.mrg_resid_norm_bwd(C.byref(norm_desc(**kw)), None) < 0 and "gradient destination" in error()
    assert L.lib.mrg_resid_norm_bwd(C.byref(norm_desc(d_pre_w=4100)), None) < 0 and "aligned" in error()


def attn_desc(**kw):
    d = L.AttnModDesc()
    for f in ("q", "k", "v", "o", "lse", "d_o", "dq", "dk", "dv", "ws"):
        setattr(d, f, 4096)
    for f, _ in L.AttnModDesc._fields_:
        if f[-3:] in ("_bs", "_rs", "_hs"):
            setattr(d, f, 64)
    d.B, d.H, d.Hk, d.Nq, d.Nk, d.head_dim, d.scale = 1, 4, 2, 5, 5, 64, 0.125
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,text", [
    (dict(head_dim=128), "head_dim"), (dict(H=3), "bad sizes"), (dict(Hk=0), "bad sizes"), (dict(Nk=-1), "bad sizes"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(cap=-1.0), "cap"), (dict(cap=float("nan")), "cap"), (dict(slopes=4096), "distance bias"),
    (dict(pos_q=4096, pos_k=4096), "distance bias"), (dict(slopes=4096, pos_q=4096, pos_k=4096, axes=4), "axes"), (dict(slopes=4096, pos_q=4096, pos_k=4096, axes=0), "axes"),
    (dict(doc_q=4096), "documents"), (dict(prefix=4096), "prefix"), (dict(Nq=1 << 27), "too many rows"), (dict(B=1 << 20, Nq=1 << 20), "too many rows"), (dict(k_rs=1 << 24), "row strides")])
def test_attention_refuses(kw, text):
    d = attn_desc(**kw)
    for f in (L.lib.mrg_attn_mod_fwd, L.lib.mrg_attn_mod_bwd):
        assert f(C.byref(d), None) < 0 and text in error()
    assert L.lib.mrg_attn_mod_ws_bytes(C.byref(d), 0) == -1


@pytest.mark.parametrize("kw,text,f", [
    (dict(q=None), "null", "fwd"), (dict(o=None), "null", "fwd"), (dict(v=None), "null", "fwd"), (dict(lse=None), "null", "bwd"), (dict(dv=None), "null", "bwd"), (dict(ws=None), "null", "bwd"),
    (dict(q=4104), "16 bytes", "fwd"), (dict(k_rs=60), "16 bytes", "fwd"), (dict(o_hs=4), "16 bytes", "fwd"), (dict(dq_bs=12), "16 bytes", "bwd"), (dict(do_rs=1), "16 bytes", "bwd")])
def test_attention_refuses_pointers(kw, text, f):
    assert getattr(L.lib, "mrg_attn_mod_" + f)(C.byref(attn_desc(**kw)), None) < 0 and text in error()


def test_attention_workspace_grows_with_what_it_holds():
    ws = lambda b, **kw: L.lib.mrg_attn_mod_ws_bytes(C.byref(attn_desc(**kw)), b)
    assert ws(0) == 0                                            # no documents, nothing split
    assert ws(1) >= 4 * 4 * 5                                    # sum(do o)
    assert ws(0, Nq=2000, Nk=2000, doc_q=4096, doc_k=4096) >= 2 * 16 * 32 and ws(0, doc_q=4096, doc_k=4096) == 0    # tables of the documents, for long rows
    assert ws(0, Nq=1, Nk=100_000) >= 2 * 4 * 64 * 4             # a single query is cut over many workgroups
    assert ws(1, Nq=1 << 20, Nk=1 << 20) >= 4 * 4 * (1 << 20)    # sizes in 64 bits


def test_launchers_refuse_cpu_tensors():
    t = torch.zeros(1, 4, 2, 64, dtype=BF16)
    f = torch.zeros(32, dtype=torch.float64)
    x = torch.zeros(2, 3, 64)
    for call in (lambda: K.rotary_axes(t, t, torch.zeros(4, 1, dtype=torch.int32), f, (32,)), lambda: K.attn_mod_fwd(t, t, t, 0.125), lambda: K.resid_norm_fwd(x, x),
                 lambda: K.attn_mod_bwd(t, t, t, t, t, t, 0.125), lambda: K.resid_norm_bwd(x, None, x, x, None)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_score_mod_refuses():
    t = torch.zeros(1)
    for kw in (dict(cap=-1.0), dict(cap=float("nan")), dict(cap=float("inf")), dict(slopes=t), dict(pos_q=t, pos_k=t), dict(slopes=t, pos_q=t), dict(doc_q=t), dict(doc_k=t), dict(prefix=t)):
        with pytest.raises(ValueError):
            K.ScoreMod(**kw)
    assert K.ScoreMod(causal=True, prefix=t).causal and K.ScoreMod().cap == 0.0


def test_memory_of_two_tensors():
    row = torch.zeros(2, 5, 6, 8)
    a, b, c = row[:, :, :2], row[:, :, 2:4], row[:, :, 1:3]
    assert K._apart(a, b) and K._apart(b, a) and not K._apart(a, c) and not K._apart(c, b) and not K._apart(a, a)
    assert K._apart(a, torch.zeros_like(row)) and not K._apart(row, b)
    assert K._apart(row[:1], row[1:]) and K._apart(row[:0], row)
    assert not K._apart(row[:, :3, :2], row[:, 2:, :2]) and K._apart(row[:1, :2, :2], row[:1, 2:, :2])
    ok = lambda t: K._out_heads(t, "t", t.shape, t.device, t.dtype)
    assert ok(a) == a.stride() and ok(row.transpose(1, 2)[..., :4])
    for t in (row[:, :1].expand(2, 5, 6, 8), torch.zeros(8).expand(2, 5, 6, 8), torch.as_strided(torch.zeros(500), (2, 5, 6, 8), (200, 20, 4, 1))):
        with pytest.raises(ValueError, match="same place"):
            ok(t)


def test_grid_positions_and_frequencies():
    at = packed.grid_positions((2, 3, 4), lead=1)
    assert at.shape == (25, 3) and at.dtype == torch.int32 and at[0].tolist() == [0, 0, 0]
    assert at[1].tolist() == [0, 0, 0] and at[2].tolist() == [0, 0, 1] and at[5].tolist() == [0, 1, 0] and at[-1].tolist() == [1, 2, 3]
    f = packed.rotary_frequencies((4, 2), 100.0)
    assert f.dtype == torch.float64 and f[0] == 1.0 and f[4] == 1.0
    assert abs(float(f[2]) - 0.1) < 1e-12 and abs(float(f[5]) - 0.1) < 1e-12


def test_modules_refuse():
    with pytest.raises(NotImplementedError, match="head_dim"):
        packed.PackedAttention(256, 2)
    with pytest.raises(NotImplementedError, match="divide"):
        packed.PackedAttention(256, 4, 3)
    with pytest.raises(ValueError, match="rms"):
        packed.Norm(64, "batch")
    with pytest.raises(ValueError, match="depth"):
        packed.PackedEncoder(128, 0, 2)
    att = packed.PackedAttention(128, 2, sections=(16, 16))
    with pytest.raises(ValueError, match="bf16"):
        att(torch.zeros(1, 4, 128))
    with pytest.raises(ValueError, match="positions"):
        att(torch.zeros(1, 4, 128, dtype=BF16))
    enc = packed.PackedEncoder(128, 2, 2, num_kv_heads=1, sections=(4, 12, 16), norm="rms")
    names = set(dict(enc.named_parameters()))
    assert "blocks.0.attn.qkv.weight" in names and "blocks.1.seam2.gate" in names and "norm.weight" in names and not any("_first" in n or "norm1.bias" in n for n in names)
    with pytest.raises(RuntimeError, match="GPU"):
        enc(torch.zeros(1, 4, 128), torch.zeros(4, 3, dtype=torch.int32))


def test_packed_descriptor_equals_the_constructors():
    sizes = [n * 7919 + 1 for n in range(len(L.RotaryDesc._fields_))]
    one = L.RotaryDesc(*sizes[:28], (3, 4, 5), *sizes[29:])
    two = L.rotary_desc(*sizes[:28], 3, 4, 5, *sizes[29:])
    assert bytes(one) == bytes(two) and isinstance(two, L.RotaryDesc)
    assert L.RotaryDesc._fields_[28][0] == "sections"
    with pytest.raises(Exception, match="argument out of range|format requires"):       # the constructor would cut it off
        L.rotary_desc(*sizes[:17], 1 << 31, *sizes[18:28], 3, 4, 5, *sizes[29:])
