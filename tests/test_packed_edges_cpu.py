"""Refusals and host helpers of the packed-volume operators at the edges of what they accept: no GPU needed, nothing is launched."""
import ctypes as C

import pytest
import torch

from mirage_amd import _lib as L
from mirage_amd import kernels as K
from mirage_amd import packed

BF16 = torch.bfloat16


def error():
    return L.lib.mrg_last_error_string().decode()


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


@pytest.mark.parametrize("kw,text", [(dict(scale=1e-38), "scale"), (dict(cap=1e-40), "cap"), (dict(cap=1e-31), "cap"), (dict(cap=1e30), "cap"), (dict(scale=1e10, cap=1e-25), "too small")])
def test_attention_refuses_factors_whose_quotients_leave_fp32(kw, text):
    d = attn_desc(**kw)
    for f in (L.lib.mrg_attn_mod_fwd, L.lib.mrg_attn_mod_bwd):
        assert f(C.byref(d), None) < 0 and text in error()
    assert L.lib.mrg_attn_mod_ws_bytes(C.byref(d), 0) == -1


def test_score_mod_refuses_a_cap_that_fp32_cannot_hold():
    for cap in (1e-46, 1e-40, -0.5, 1e30):                       # the first would arrive as 0: no cap at all
        with pytest.raises(ValueError, match="cap"):
            K.ScoreMod(cap=cap)
    assert K.ScoreMod(cap=1e-30).cap == 1e-30 and K.ScoreMod(cap=-0.0).cap == 0.0
    assert L.lib.mrg_attn_mod_ws_bytes(C.byref(attn_desc(cap=1e-30)), 0) == 0        # the smallest one arrives and is accepted


@pytest.mark.parametrize("name", ["q_rs", "k_rs", "v_rs", "do_rs", "k_bs", "o_hs", "dv_rs"])
def test_attention_refuses_negative_strides(name):
    """rows of a tile lie at unsigned offsets from its first one: a negative stride would be read some GiB behind it"""
    d = attn_desc(Nq=100, Nk=100, **{name: -64})
    for f in (L.lib.mrg_attn_mod_fwd, L.lib.mrg_attn_mod_bwd):
        assert f(C.byref(d), None) < 0 and "negative stride" in error()


def test_rotary_table_made_under_inference_serves_training():
    """the table of a module's first call is kept: made as an inference tensor, no later backward pass could save it"""
    att = packed.PackedAttention(128, 2, sections=(8, 12, 12))
    with torch.inference_mode():
        table = att.freqs(torch.device("cpu"))
        assert att.freqs(torch.device("cpu")) is table
    assert not table.is_inference() and att.freqs(torch.device("cpu")) is table


def test_rotary_table_follows_the_module():
    """theta or sections changed behind the first call: a table of the new ones"""
    att, cpu = packed.PackedAttention(128, 2, sections=(8, 12, 12)), torch.device("cpu")
    first = att.freqs(cpu)
    att.theta = 10_000.0
    assert torch.equal(att.freqs(cpu), packed.rotary_frequencies((8, 12, 12), 10_000.0))
    att.sections = (16, 16)
    assert torch.equal(att.freqs(cpu), packed.rotary_frequencies((16, 16), 10_000.0))
    att.sections, att.theta = (8, 12, 12), 100.0
    assert att.freqs(cpu) is first


def test_attention_module_refuses_a_batch_without_tokens():
    att = packed.PackedAttention(128, 2)
    for shape in ((0, 5, 128), (2, 0, 128)):
        with pytest.raises(ValueError, match="no tokens"):
            att(torch.zeros(shape, dtype=BF16))


def test_padding_that_is_not_finite():
    x = torch.randn(2, 5, 8)
    doc = torch.tensor([[0, 0, 1, -1, -1], [0, -3, 1, 1, -1]], dtype=torch.int32)
    pad = doc < 0
    x[0, 3], x[0, 4, 2], x[1, 1, 0], x[0, 0, 1] = float("nan"), float("inf"), -float("inf"), float("nan")
    x.requires_grad_(True)
    z = packed._finite_padding(x, K.ScoreMod(doc_q=doc, doc_k=doc))
    want = torch.where(pad[..., None] & ~torch.isfinite(x), torch.zeros(()), x)
    assert torch.equal(z.nan_to_num(7.0), want.nan_to_num(7.0)) and bool(torch.isnan(z[0, 0, 1]))
    z.backward(torch.ones_like(z))
    assert torch.equal(x.grad, (~pad[..., None] | torch.isfinite(x)).float())
    asks = torch.where(pad, doc, -1)                              # tokens that ask nothing but are seen
    assert torch.equal(packed._finite_padding(x, K.ScoreMod(doc_q=asks, doc_k=doc)).nan_to_num(7.0), want.nan_to_num(7.0))
    for mod in (None, K.ScoreMod(), K.ScoreMod(doc_q=doc[:, :4], doc_k=doc[:, :4]), K.ScoreMod(doc_q=doc, doc_k=doc[:1])):
        assert packed._finite_padding(x, mod) is x
