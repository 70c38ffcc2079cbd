"""Packed-volume operators at the edges of what they accept, against their formulas in 64 bits: large caps, sizes, gradients and paddings as a caller
may hand them over."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
HALF16, HALF32 = torch.finfo(BF16).eps / 2, torch.finfo(F32).eps / 2


@pytest.fixture(scope="module")
def K():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    from mirage_amd import kernels
    return kernels


def dev():
    return torch.device("cuda:0")


def rnd(*shape, dtype=F32, scale=1.0, seed=0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(dev())


def within(got, ref, bound, what):
    bad = ~((got.double() - ref).abs() <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds, worst {float(((got.double() - ref).abs() / bound)[bad].max()):.3g} x"


def capped_attention(q, k, v, d_o, scale, cap):
    """o, lse, dq, dk, dv with elementwise bounds.  Noise of a score: fp32 accumulation of q.k; the cap's own error, cap 2^-21 for caps up to 256 and
    2^-20 of the score above; factor, running maximum and exponential.  Then the roundings to bf16: p in its products, o, the gradients; ds
    enters its products to 2^-16, o its sum with d_o as well."""
    q, k, v, g = (t.double().transpose(1, 2) for t in (q, k, v, d_o))
    raw = q @ k.transpose(-1, -2) * scale
    th = torch.tanh(raw / cap)
    s, steep = cap * th, 1 - th * th
    noise = (q.abs() @ k.abs().transpose(-1, -2)) * scale * (q.shape[-1] * HALF32) + (s.abs() + 16) * 8 * HALF32
    noise = noise + (cap * 2.0 ** -21 if cap <= 256 else s.abs() * 2.0 ** -20)
    p = torch.softmax(s, -1)
    wob = noise.amax(-1, keepdim=True) * 2                                      # relative error of p in fp32
    o = p @ v
    eo = (p @ v.abs()) * (HALF16 + wob + 64 * HALF32)
    dp = g @ v.transpose(-1, -2)
    ds = p * (dp - (g * o).sum(-1, keepdim=True)) * steep
    eD, fp = (g.abs() * eo).sum(-1, keepdim=True), (wob + 128 * HALF32) * 4
    eds = ds.abs() * 2.0 ** -16 + p * eD + p * ((g.abs() @ v.abs().transpose(-1, -2)) + (g.abs() * o.abs()).sum(-1, keepdim=True)) * fp
    dq, dk, dv = ds @ k * scale, ds.transpose(-1, -2) @ q * scale, p.transpose(-1, -2) @ g
    half = lambda t: t.abs() * HALF16 * 1.01 + 1e-30
    out = {"o": (o, eo + half(o)), "dq": (dq, eds @ k.abs() * scale + half(dq)), "dk": (dk, eds.transpose(-1, -2) @ q.abs() * scale + half(dk)),
           "dv": (dv, (p * (HALF16 + fp)).transpose(-1, -2) @ g.abs() + half(dv))}
    lse = torch.logsumexp(s, -1)
    return {n: (a.transpose(1, 2), e.transpose(1, 2)) for n, (a, e) in out.items()} | {"lse": (lse, wob[..., 0] + 4e-6 * (1 + lse.abs()))}


@pytest.mark.parametrize("Nq,hd,bias", [(150, 64, False), (1, 64, False), (70, 32, False), (150, 64, True)])
@pytest.mark.parametrize("cap,size", [(200.0, 1.5), (256.0, 1.5), (257.0, 1.5), (300.0, 12.0), (1e3, 1.5), (1e3, 20.0), (1e5, 1.5), (1e6, 1.5), (1e8, 1.5), (9e29, 1.5)])
def test_caps_of_any_size(K, cap, size, Nq, hd, bias):
    """a cap far above the scores leaves them as they are; near them (size 12 and 20: scores to some hundreds) it bends them"""
    B, H, Nk = 2, 2, 333
    q, k = rnd(B, Nq, H, hd, dtype=BF16, scale=size, seed=1), rnd(B, Nk, H, hd, dtype=BF16, scale=size, seed=2)
    v, d_o, scale = rnd(B, Nk, H, hd, dtype=BF16, seed=3), rnd(B, Nq, H, hd, dtype=BF16, seed=4), hd ** -0.5
    # a distance of zero everywhere: the kernels with a bias, the same values
    at = dict(slopes=torch.ones(H, device=dev()), pos_q=torch.ones(B, Nq, 1, device=dev()), pos_k=torch.ones(B, Nk, 1, device=dev())) if bias else {}
    mod = K.ScoreMod(cap=cap, **at)
    ref = capped_attention(q, k, v, d_o, scale, cap)
    o, saved = K.attn_mod_fwd(q, k, v, scale, mod)
    within(o, *ref["o"], "o")
    within(saved.lse, *ref["lse"], "lse")
    for got, n in zip(K.attn_mod_bwd(q, k, v, o, saved, d_o, scale, mod), ("dq", "dk", "dv")):
        within(got, *ref[n], n)


@pytest.mark.parametrize("cap", [1e-30, 1e-3, 0.25])
def test_smallest_caps(K, cap):
    """every score at the cap, one of them with nothing to bend (a query of zeros)"""
    q, k, v, d_o = (rnd(1, 100, 2, 64, dtype=BF16, seed=i) for i in range(4))
    q[0, 3] = 0
    ref = capped_attention(q, k, v, d_o, 0.125, cap)
    mod = K.ScoreMod(cap=cap)
    o, saved = K.attn_mod_fwd(q, k, v, 0.125, mod)
    within(o, *ref["o"], "o")
    within(saved.lse, *ref["lse"], "lse")
    for got, n in zip(K.attn_mod_bwd(q, k, v, o, saved, d_o, 0.125, mod), ("dq", "dk", "dv")):
        within(got, *ref[n], n)


def test_attn_mod_of_more_heads_than_workgroups_fit_one_dimension(K):
    """2^24 and some (batch, head) pairs of one token, whose backward pass needs a second dimension of workgroups: o = v, dv = d_o, nothing for q and k"""
    B = (1 << 24) + 5
    g = torch.Generator(device=dev()).manual_seed(1)
    q, k, v, d_o = (torch.randn(B, 1, 1, 32, generator=g, device=dev(), dtype=BF16) for _ in range(4))
    o, saved = K.attn_mod_fwd(q, k, v, 0.125)
    assert torch.equal(o, v)
    dq, dk, dv = K.attn_mod_bwd(q, k, v, o, saved, d_o, 0.125)
    assert torch.equal(dv, d_o)
    # dp - sum(do o) is the difference of two fp32 sums of the same 32 products (sizes below 64 x 8): 64 2^-24 of their sizes, times q or k and the scale
    assert float(dq.abs().amax()) < 1e-2 and float(dk.abs().amax()) < 1e-2


def test_resid_norm_of_more_rows_than_one_dimension_of_workgroups(K):
    """every row as in calls of a part of them, the last ones as well"""
    M, D = (1 << 26) + 5, 4
    x = torch.empty(1, M, D, device=dev())
    b = torch.empty(1, M, D, device=dev(), dtype=BF16)
    tile = 1 << 16
    for at in range(0, M, tile):                                   # rows repeat, but for the first element that counts the tiles
        n = min(tile, M - at)
        if at == 0:
            x[:, :n], b[:, :n] = rnd(1, n, D, seed=1), rnd(1, n, D, dtype=BF16, seed=2)
        else:
            x[:, at:at + n], b[:, at:at + n] = x[:, :n], b[:, :n]
        x[:, at:at + n, 0] = at / tile * 2.0 ** -6
    how = dict(gate=rnd(D, seed=3), alpha=0.5, post=(rnd(D, seed=4), rnd(D, seed=5)), pre=(rnd(D, seed=6), rnd(D, seed=7)))
    x_new, y, stats = K.resid_norm_fwd(x, b, **how)
    for lo, hi in ((0, 1000), (M // 2 - 500, M // 2 + 500), (M - 1000, M)):
        part, py, ps = K.resid_norm_fwd(x[:, lo:hi].clone(), b[:, lo:hi].clone(), **how)   # (clones: rows of 8 bytes)
        assert torch.equal(part, x_new[:, lo:hi]) and torch.equal(py, y[:, lo:hi]) and torch.equal(ps, stats[:, lo:hi])


def test_resid_norm_of_more_gates_than_workgroups(K):
    """2^24 and some samples of one row and a gate each: the gates' gradients are dx' times the branch, element by element"""
    S, D = (1 << 24) + 3, 4
    g = torch.Generator(device=dev()).manual_seed(1)
    x, b, gate, dx_new = (torch.randn(S, 1, D, generator=g, device=dev()) for _ in range(4))
    gate = gate.view(S, D)
    x_new, _, _ = K.resid_norm_fwd(x, b, gate=gate)
    x_, n_ = x.view(S, D), gate * b.view(S, D)
    assert bool(((x_new.view(S, D) - (x_ + n_)).abs() <= 2 * HALF32 * (x_.abs() + 2 * n_.abs())).all())      # a product and a sum, each rounded on either side
    dx, db, grads = K.resid_norm_bwd(dx_new, None, x_new, b, None, gate=gate)
    assert torch.equal(dx, dx_new) and torch.equal(db.view(S, D), dx_new.view(S, D) * gate) and torch.equal(grads["gate"], dx_new.view(S, D) * b.view(S, D))


def test_rotary_of_more_rows_than_one_dimension_of_workgroups(K):
    """2^28 and some rows of two elements (16 rows a workgroup): the last ones as in calls of a part of them"""
    N = (1 << 28) + 37
    q = torch.empty(1, N, 1, 2, device=dev(), dtype=BF16)
    q.view(torch.int16).copy_(torch.arange(2 * N, device=dev(), dtype=torch.int32).view(q.shape) % 16001)      # bits of small numbers, different from row to row
    pos = torch.arange(N, device=dev(), dtype=torch.int32)[:, None]
    freqs = torch.ones(1, dtype=F64, device=dev())
    out, _ = K.rotary_axes(q, None, pos, freqs, (1,))
    for lo, hi in ((0, 1000), (N // 2, N // 2 + 1000), (N - 1000, N)):
        part, _ = K.rotary_axes(q[:, lo:hi].clone(), None, pos[lo:hi].clone(), freqs, (1,))
        assert torch.equal(part, out[:, lo:hi])


# ------------------------------------------------------------------------------------------------------------------ modules
@pytest.fixture(scope="module")
def P():
    from mirage_amd import packed
    return packed


def encoder(P, dim=128, depth=2, heads=2, seed=0, **kw):
    enc = P.PackedEncoder(dim, depth, heads, sections=(8, 12, 12), **kw)
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for p in enc.parameters():
            p.copy_(torch.randn(p.shape, generator=g) * (p.shape[1] ** -0.5 if p.dim() == 2 else 0.3) + (0.0 if p.dim() == 2 else 0.5))
    return enc.to(dev())


def rows(P, K, B=2, pad=9, seed=1, dim=128):
    """two samples in each row and padding behind them"""
    at = torch.cat([P.grid_positions((2, 4, 5), 1), P.grid_positions((3, 3, 7), 1), torch.zeros(pad, 3, dtype=torch.int32)]).to(dev())
    doc = torch.cat([torch.zeros(41), torch.ones(64), torch.full((pad,), -1)]).int().repeat(B, 1).to(dev())
    return rnd(B, len(at), dim, seed=seed), at[None].repeat(B, 1, 1).contiguous(), K.ScoreMod(cap=20.0, doc_q=doc, doc_k=doc)


def step(enc, x, pos, mod, dx, dy, gates=None):
    h, y = enc(x, pos, mod, gates)
    torch.autograd.backward([h, y], [dx, dy])
    return [h.detach(), y.detach()] + [p.grad.clone() for p in enc.parameters() if p.grad is not None]      # (learnt gates behind `gates`: none)


def test_encoder_learns_after_a_first_call_under_inference(K, P):
    x, pos, mod = rows(P, K)
    dx, dy = rnd(*x.shape, seed=2), rnd(*x.shape, dtype=BF16, seed=3)
    want = step(encoder(P), x, pos, mod, dx, dy)
    enc = encoder(P)
    with torch.inference_mode():
        enc(x, pos, mod)
    assert all(torch.equal(a, b) for a, b in zip(step(enc, x, pos, mod, dx, dy), want))


def test_encoder_sees_weights_that_change_behind_the_optimizers_arena(K, P):
    """load_state_dict, or any change through torch, of parameters in an optimizer's arena reaches the next pass, of the encoder and of its parts"""
    from mirage_amd import optim
    x, pos, mod = rows(P, K)
    dx, dy = rnd(*x.shape, seed=2), rnd(*x.shape, dtype=BF16, seed=3)
    enc, other = encoder(P), encoder(P, seed=7)
    opt = optim.FusedAdamW(enc, [1e-3] * 3, [0.0] * 3)
    step(enc, x, pos, mod, dx, dy)
    opt.step()
    enc.load_state_dict(other.state_dict())
    assert all(torch.equal(a, b) for a, b in zip(step(enc, x, pos, mod, dx, dy), step(other, x, pos, mod, dx, dy)))
    opt.step()                                                     # the optimizer's own change too
    other.load_state_dict(enc.state_dict())
    assert all(torch.equal(a, b) for a, b in zip(step(enc, x, pos, mod, dx, dy), step(other, x, pos, mod, dx, dy)))
    with torch.no_grad():                                          # one part by itself
        enc.blocks[1].attn.proj.weight.mul_(-2.0)
        other.blocks[1].attn.proj.weight.mul_(-2.0)
        y16 = rnd(*x.shape, dtype=BF16, seed=4)
        assert torch.equal(enc.blocks[1].attn(y16, pos, mod), other.blocks[1].attn(y16, pos, mod))


def test_gradients_off_alignment(K, P):
    """what torch.cat hands back behind a piece of odd length is dense but starts off the kernels' 16 bytes: the same gradients as from its copy"""
    x, pos, mod = rows(P, K)
    B, N, D = x.shape
    att, seam, pre = P.PackedAttention(D, 2, sections=(8, 12, 12)).to(dev()), P.Seam(D).to(dev()), P.Norm(D).to(dev())
    qkv = rnd(B, N, 6, 64, dtype=BF16, seed=5)

    def grads(of):
        leaves = [t.clone().requires_grad_(True) for t in (qkv[:, :, :2], qkv[:, :, 2:4], qkv[:, :, 4:], x, x.bfloat16())]
        q, k, v, res, y16 = leaves
        outs = [P.attention(q, k, v, 0.125, mod), *P.rotary(q, k, pos, att.freqs(dev()), (8, 12, 12)), att(y16, pos, mod), *seam(res, y16, pre)]
        sum(of(o, i) for i, o in enumerate(outs)).backward()
        return [t.grad for t in leaves] + [p.grad.clone() for m in (att, seam, pre) for p in m.parameters()]

    weights = [rnd(1 + B * N * D, dtype=F32 if i == 4 else BF16, seed=20 + i) for i in range(6)]
    behind = lambda o, i: (torch.cat([torch.ones(1, dtype=o.dtype, device=dev()), o.reshape(-1)]) * weights[i]).float().sum()
    alone = lambda o, i: (o.reshape(-1) * weights[i][1:].clone()).float().sum()
    got, want = grads(behind), grads(alone)
    assert len(got) == 5 + 4 + 3 + 2 and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("junk", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("per_sample", [False, True])
def test_encoder_learns_beside_padding_that_is_not_finite(K, P, junk, per_sample):
    """weight gradients sum over every row of the batch, and zero times NaN is NaN: such padding learns like padding of zeros"""
    x, pos, mod = rows(P, K)
    pad = mod.doc_q < 0
    gates = [tuple(0.5 * rnd(2, 128, seed=10 * i + j) for j in range(2)) for i in range(2)] if per_sample else None
    dx, dy = rnd(*x.shape, seed=2), rnd(*x.shape, dtype=BF16, seed=3)
    dx[pad], dy[pad] = 0, 0                                        # a loss over the samples' tokens

    def learn(fill):
        t = x.clone()
        t[pad] = fill
        t.requires_grad_(True)
        return step(encoder(P), t, pos, mod, dx, dy, gates) + [t.grad]

    got, want = learn(junk), learn(0.0)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(bool(torch.isfinite(t).all()) for t in got)
    finite = learn(3.0)                                            # and finite padding is left alone: its rows differ, nothing that is learnt does
    assert not torch.equal(finite[0][pad], want[0][pad]) and torch.equal(finite[0][~pad], want[0][~pad])
    assert all(torch.equal(a, b) for a, b in zip(finite[2:-1], want[2:-1])) and torch.equal(finite[-1][~pad], want[-1][~pad])


def test_visible_values_that_are_not_finite_still_show(K, P):
    """only padding is replaced: a NaN in a sample's own token reaches that sample, and the gradients"""
    x, pos, mod = rows(P, K)
    x[0, 5, 7] = float("nan")
    asks = mod.doc_q.clone()
    asks[0, 5] = -1                                                # a token that asks nothing, but is seen
    out = step(encoder(P), x, pos, K.ScoreMod(doc_q=asks, doc_k=mod.doc_k), torch.ones_like(x), torch.ones_like(x, dtype=BF16))
    assert bool(torch.isnan(out[0][0, :41]).all()) and bool(torch.isfinite(out[0][0, 41:]).all()) and bool(torch.isnan(out[2]).any())
    out = step(encoder(P), x, pos, mod, torch.ones_like(x), torch.ones_like(x, dtype=BF16))
    assert bool(torch.isnan(out[0][0, :41]).all()) and bool(torch.isfinite(out[0][0, 41:]).all()) and bool(torch.isnan(out[2]).any())


def test_scores_up_to_their_limit(K):
    """scores 2^23 apart up to 99 2^23 (exact in fp32): each row's largest one takes all"""
    N = 100
    q, k = (torch.zeros(1, N, 1, 64, dtype=BF16, device=dev()) for _ in range(2))
    q[..., 0] = 2.0 ** 15
    q[0, 50:, 0, 0] = -(2.0 ** 15)                                 # these rows want the smallest
    order = torch.randperm(N, generator=torch.Generator().manual_seed(1)).to(dev())
    k[0, :, 0, 0] = order.to(BF16)
    v = rnd(1, N, 1, 64, dtype=BF16, seed=2)
    for scale, shift in ((256.0, 0.0), (256.0, 1.0)):              # the second: every score of the first rows is far from zero
        k[0, :, 0, 0] = (order + shift * 28).to(BF16)
        o, saved = K.attn_mod_fwd(q, k, v, scale)
        best = torch.where(torch.arange(N, device=dev()) < 50, order.argmax(), order.argmin())
        want, top = v[:, best].double(), (q[0, :, 0, 0].double() * k[0, best, 0, 0].double() * scale)
        within(o, want, want.abs() * 2 * HALF16, "o")              # p and the result rounded
        within(saved.lse[0, 0], top, top.abs() * 4 * HALF32 + 1e-6, "lse")


def test_encoder_in_training_refuses_documents_that_do_not_fit(K, P):
    x, pos, mod = rows(P, K)
    for doc in (mod.doc_q[:, :-1].contiguous(), mod.doc_q[:1], mod.doc_q.t().contiguous()):
        with pytest.raises(ValueError, match="ScoreMod doc_q must have shape"):
            encoder(P)(x, pos, K.ScoreMod(doc_q=doc, doc_k=doc))
    with pytest.raises(RuntimeError, match="GPU"):
        encoder(P)(x, pos, K.ScoreMod(doc_q=mod.doc_q.cpu(), doc_k=mod.doc_k.cpu()))
