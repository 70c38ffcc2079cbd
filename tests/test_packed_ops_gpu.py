"""Rotary positions with several axes, attention with modified scores and the gated residual with its norms, against their formulas in 64 bits.

Bounds are formed elementwise from the same 64-bit run and count the roundings: an operand or result held in bf16 is off by at most half a step,
2^-8 of its value; fp32 sums of n terms by n 2^-24 of the sum of their sizes."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
HALF16 = torch.finfo(BF16).eps / 2
HALF32 = torch.finfo(F32).eps / 2


@pytest.fixture(scope="module")
def K():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    from mirage_amd import kernels
    return kernels


def dev():
    return torch.device("cuda:0")


def rnd(*shape, dtype=F32, scale=1.0, seed=0):
    g = torch.Generator().manual_seed(seed + 1000 * len(shape))
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(dev())


def within(got, ref, bound, what):
    got = got.double()
    bad = ~((got - ref).abs() <= bound) & ~(torch.isnan(got) & torch.isnan(ref))
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds, worst {float(((got - ref).abs() / bound.clamp_min(1e-300))[bad].max()):.3g} x, "
                           f"first at {bad.nonzero()[0].tolist()}: {float(got[bad][0])} vs {float(ref[bad][0])}")


# ------------------------------------------------------------------------------------------------------------------ rotary
def rotary_ref(t, pos, freqs, sections, pairing, inverse):
    P = sum(sections)
    t = t.double()
    axis = [a for a, s in enumerate(sections) for _ in range(s)]
    first, second = [], []
    for p in range(P):
        start = sum(sections[:axis[p]])
        if pairing == "half":
            f, s = p, p + P
        elif pairing == "interleaved":
            f, s = 2 * p, 2 * p + 1
        else:
            f = start + p
            s = f + sections[axis[p]]
        first.append(f)
        second.append(s)
    pos = pos if pos.dim() == 3 else pos[None]
    th = pos.double()[..., axis] * freqs
    c, s = torch.cos(th)[:, :, None], torch.sin(th)[:, :, None] * (-1 if inverse else 1)
    out, size = t.clone(), t.abs()
    a, b = t[..., first], t[..., second]
    out[..., first], out[..., second] = a * c - b * s, a * s + b * c
    size[..., first] = size[..., second] = a.abs() + b.abs()
    return out, size


def rotary_bound(ref, size, dtype):
    # fp32: products and sum 3 roundings, sine / cosine 2^-22 (angle 2^-26 turns, function 2 ulp); then the rounding to the type
    return size * (3 * HALF32 + 2.0 ** -22) + (HALF16 * ref.abs() if dtype == BF16 else HALF32 * ref.abs()) * (1 + 2.0 ** -10) + 1e-30


ROTARY = [  # B, N, H, Hk, hd, sections
    (1, 1, 1, 1, 32, (16,)), (2, 257, 12, 12, 64, (16, 16)), (3, 65, 4, 2, 64, (8, 12, 12)), (2, 33, 3, 1, 48, (5, 7, 3)), (1, 300, 2, 2, 64, (4, 6, 6)),
    (2, 19, 2, 1, 6, (1, 1)), (1, 2100, 2, 1, 128, (16, 24, 24)), (1, 5, 1, 1, 2, (1,)), (2, 40, 4, 4, 32, (4, 6, 6)), (1, 7, 2, 3, 256, (64, 64)),
    (3, 13337, 2, 1, 16, (3, 2))]                                  # 16 rows a workgroup, the last one short


@pytest.mark.parametrize("pairing", ["half", "interleaved", "axial"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,N,H,Hk,hd,sections", ROTARY)
def test_rotary_matches_the_formula(K, B, N, H, Hk, hd, sections, dtype, pairing):
    row = rnd(B, N, H + 2 * Hk, hd, dtype=dtype, seed=N)
    q, k = row[:, :, :H], row[:, :, H:H + Hk]
    keep = row.clone()
    g = torch.Generator().manual_seed(N)
    for pos in (torch.randint(-50, 1_000_000, (B, N, len(sections)), generator=g).to(dev(), torch.int32),
                (torch.rand(N, len(sections), generator=g) * 40 - 5).to(dev())):
        freqs = (10000.0 ** -torch.rand(sum(sections), generator=g, dtype=F64)).to(dev())
        for inverse in (False, True):
            oq, ok = K.rotary_axes(q, k, pos, freqs, sections, pairing=pairing, inverse=inverse)
            for got, src, what in ((oq, q, "q"), (ok, k, "k")):
                ref, size = rotary_ref(src, pos, freqs, sections, pairing, inverse)
                within(got, ref, rotary_bound(ref, size, dtype), what)
    assert torch.equal(row, keep), "the inputs stay as they are"
    # in place on the fused buffer, v untouched, the same bits
    K.rotary_axes(q, k, pos, freqs, sections, pairing=pairing, inverse=True, out_q=q, out_k=k)
    assert torch.equal(q, oq) and torch.equal(k, ok) and torch.equal(row[:, :, H + Hk:], keep[:, :, H + Hk:])


def test_rotary_odd_strides_one_side_and_empty(K):
    pos = torch.arange(10, device=dev(), dtype=torch.int32).view(5, 2)
    freqs = torch.tensor([1.0, 0.5, 0.25, 0.1], dtype=F64, device=dev())
    for dtype in (BF16, F32):
        base = rnd(2, 5, 3, 11, dtype=dtype, seed=3)
        q = base[..., 1:10]                                  # 9 elements of a head, one element off alignment: 8 turned, 1 copied
        out, none = K.rotary_axes(q, None, pos, freqs, (2, 2), pairing="axial")
        assert none is None
        ref, size = rotary_ref(q, pos, freqs, (2, 2), "axial", False)
        within(out, ref, rotary_bound(ref, size, dtype), "q")
        e, f = K.rotary_axes(q[:0], q[:0], pos, freqs, (2, 2))
        assert e.shape == (0, 5, 3, 9) and f.shape == e.shape
        # heads and rows swapped in memory
        swapped = base.transpose(1, 2).contiguous().transpose(1, 2)[..., :8]
        out, _ = K.rotary_axes(swapped, None, pos, freqs, (2, 2))
        ref, size = rotary_ref(swapped, pos, freqs, (2, 2), "half", False)
        within(out, ref, rotary_bound(ref, size, dtype), "swapped")


def test_rotary_inverse_undoes_and_is_the_gradient(K):
    q = rnd(2, 37, 4, 64, seed=5)
    pos = torch.randint(0, 1000, (2, 37, 3), generator=torch.Generator().manual_seed(1)).to(dev(), torch.int32)
    freqs = (100.0 ** -torch.linspace(0, 1, 32, dtype=F64)).to(dev())
    w = rnd(2, 37, 4, 64, seed=6)
    there, _ = K.rotary_axes(q, None, pos, freqs, (8, 12, 12))
    back, _ = K.rotary_axes(there, None, pos, freqs, (8, 12, 12), inverse=True)
    within(back, q.double(), torch.full_like(q, 2e-6 * float(q.abs().max())).double(), "inverse")
    # <w, R q> = <R^T w, q>
    grad, _ = K.rotary_axes(w, None, pos, freqs, (8, 12, 12), inverse=True)
    a, b = float((w.double() * there.double()).sum()), float((grad.double() * q.double()).sum())
    assert abs(a - b) <= 2e-6 * float((w.double() * there.double()).abs().sum())


# ------------------------------------------------------------------------------------------------------------------ residual norm
def norm_ref(x, b, gate, alpha, post, pre, kind, eps, dx_new=None, dy=None):
    leaf = lambda t: None if t is None else t.double().clone().requires_grad_(True)
    x, b, gate = leaf(x), leaf(b), leaf(gate)
    post, pre = [None if p is None else [leaf(t) for t in p] for p in (post, pre)]

    def norm(v, wb):
        c = v - v.mean(-1, keepdim=True) if kind == "layer" else v
        c = c / torch.sqrt((c * c).mean(-1, keepdim=True) + eps) * wb[0]
        return c if wb[1] is None else c + wb[1]

    n = b if post is None else norm(b, post)
    if gate is not None:
        n = n * (gate if gate.dim() == 1 else gate.view(gate.shape[0], *([1] * (x.dim() - 2)), gate.shape[1]))
    x_new = alpha * x + n
    y = norm(x_new, pre) if pre is not None else None
    out = {"x_new": x_new.detach(), "y": None if y is None else y.detach()}
    if dx_new is not None:
        torch.autograd.backward([x_new] + ([y] if y is not None else []), [dx_new.double()] + ([dy.double()] if y is not None else []))
        out.update(dx=x.grad, dbranch=b.grad, gate=None if gate is None else gate.grad)
        for name, p in (("post", post), ("pre", pre)):
            out[name + "_weight"] = None if p is None else p[0].grad
            out[name + "_bias"] = None if p is None or p[1] is None else p[1].grad
    return out


def rows_bound(ref, dtype, D):
    # row values: sums over D in a tree of depth <= 20 and a dozen further roundings, relative to the row's own size (its largest entry)
    big = ref.abs().amax(-1, keepdim=True) + 1.0
    return 64 * HALF32 * big + (HALF16 * 1.01 * ref.abs() if dtype == BF16 else 0.0)


def sums_bound(ref, terms, rows):
    # column sums of `rows` terms whose sizes stay below `terms` each, the terms themselves a few dozen roundings off
    return (rows ** 0.5 + 64) * HALF32 * terms * rows ** 0.5 * 8 + 1e-6 * ref.abs() + 1e-12


NORM = [  # shape, kind, gate, post bias, pre bias (None: no norm), alpha, branch
    ((1, 1, 4), "layer", "channel", True, True, 1.0, F32), ((2, 129, 768), "layer", "channel", True, True, 1.0, BF16),
    ((3, 50, 1024), "rms", "sample", False, False, 0.75, BF16), ((5, 7, 260), "layer", "sample", False, True, 0.5, F32),
    ((4, 33, 256), "rms", "none", None, False, 1.0, BF16), ((2, 20, 64), "layer", "channel", None, None, -0.5, F32),
    ((1, 70, 1028), "layer", "channel", True, False, 1.0, BF16), ((3, 9, 2052), "rms", "sample", True, True, 1.0, F32),
    ((2, 11, 4096), "layer", "sample", True, True, 0.3, BF16), ((700, 1, 128), "layer", "sample", True, True, 1.0, BF16),
    ((2, 3, 40, 192), "rms", "channel", True, True, 1.0, BF16), ((6, 516), "layer", "sample", False, False, 1.0, F32),
    ((1, 2500, 132), "layer", "none", True, True, 1.0, BF16),
    # more gates than workgroups run at once; parts of a gate's rows that do not divide
    ((2500, 3, 64), "layer", "sample", True, True, 1.0, BF16), ((700, 2, 2052), "rms", "sample", False, False, 1.0, BF16), ((300, 1, 4096), "layer", "sample", True, True, 0.9, F32),
    ((33, 517, 768), "layer", "sample", True, True, 1.0, BF16)]


@pytest.mark.parametrize("shape,kind,gate,post,pre,alpha,branch", NORM)
def test_resid_norm_matches_the_formula(K, shape, kind, gate, post, pre, alpha, branch):
    D, S = shape[-1], shape[0]
    eps = 1e-6
    x, b = rnd(*shape, seed=1), rnd(*shape, dtype=branch, scale=0.7, seed=2)
    vec = lambda i: 1 + 0.2 * rnd(D, seed=i)
    gt = {"none": None, "channel": 0.3 * rnd(D, seed=3), "sample": 0.5 * rnd(S, D, seed=4)}[gate]
    post = None if post is None else (vec(5), vec(6) - 1 if post else None)
    pre = None if pre is None else (vec(7), vec(8) - 1 if pre else None)
    how = dict(gate=gt, alpha=alpha, post=post, pre=pre, kind=kind, eps=eps)
    dxn, dy = rnd(*shape, seed=9), (rnd(*shape, dtype=BF16, seed=10) if pre is not None else None)
    ref = norm_ref(x, b, gt, alpha, post, pre, kind, eps, dxn, dy)
    for out_dtype in (BF16, F32):
        x_new, y, stats = K.resid_norm_fwd(x, b, out_dtype=out_dtype, **how)
        within(x_new, ref["x_new"], rows_bound(ref["x_new"], F32, D), "x_new")
        if pre is None:
            assert y is None
        else:
            assert y.dtype == out_dtype
            within(y, ref["y"], rows_bound(ref["y"], out_dtype, D), "y")
    dx, db, grads = K.resid_norm_bwd(dxn, dy, x_new, b, stats, **how)
    within(dx, ref["dx"], rows_bound(ref["dx"], F32, D), "dx")
    within(db, ref["dbranch"], rows_bound(ref["dbranch"], branch, D), "dbranch")
    assert db.dtype == branch
    want = {n for n in ("gate", "post_weight", "post_bias", "pre_weight", "pre_bias") if ref[n] is not None}
    assert set(grads) == want
    rows = x.numel() // D
    for n in want:
        within(grads[n], ref[n], sums_bound(ref[n], 8.0, rows), n)
    # the same bits again, into given destinations, with the workspace's memory in another state
    torch.full((1 << 20,), float("nan"), device=dev())
    dst = {n: torch.full_like(grads[n], float("nan")) for n in want}
    dx2, db2, g2 = K.resid_norm_bwd(dxn, dy, x_new, b, stats, grads=dst, **how)
    assert torch.equal(dx, dx2) and torch.equal(db, db2) and all(torch.equal(grads[n], dst[n]) and g2[n] is dst[n] for n in want)


def test_resid_norm_no_rows(K):
    w = torch.ones(64, device=dev())
    for shape, gate in (((0, 5, 64), torch.ones(64, device=dev())), ((3, 0, 64), torch.ones(3, 64, device=dev()))):
        x = torch.empty(shape, device=dev())
        how = dict(gate=gate, post=(w, w), pre=(w, w))
        x_new, y, stats = K.resid_norm_fwd(x, x.to(BF16), **how)
        assert x_new.shape == shape and y.shape == shape
        dx, db, g = K.resid_norm_bwd(x, x.to(BF16), x_new, x.to(BF16), stats, **how)
        assert dx.shape == shape and all(bool((t == 0).all()) for t in g.values()) and len(g) == 5


def test_resid_norm_gradient_by_differences(K):
    shape, D = (2, 6, 32), 32
    x, b = rnd(*shape, seed=1), rnd(*shape, seed=2)
    gt, post, pre = 0.5 * rnd(2, D, seed=3), (1 + 0.2 * rnd(D, seed=4), rnd(D, seed=5)), (1 + 0.2 * rnd(D, seed=6), None)
    wx, wy = rnd(*shape, seed=7), rnd(*shape, seed=8)

    def loss(x, b, gt):
        x_new, y, _ = K.resid_norm_fwd(x, b, gate=gt, alpha=0.8, post=post, pre=pre, out_dtype=F32)
        return float((x_new.double() * wx).sum() + (y.double() * wy).sum())

    x_new, y, stats = K.resid_norm_fwd(x, b, gate=gt, alpha=0.8, post=post, pre=pre, out_dtype=F32)
    dx, db, g = K.resid_norm_bwd(wx, wy, x_new, b, stats, gate=gt, alpha=0.8, post=post, pre=pre)
    h = 2.0 ** -7
    for name, t, grad in (("x", x, dx), ("branch", b, db), ("gate", gt, g["gate"])):
        step = rnd(*t.shape, seed=11)
        args = {"x": x, "branch": b, "gate": gt}
        up, down = [loss(*(args[n] + s * h * step if n == name else args[n] for n in ("x", "branch", "gate"))) for s in (1, -1)]
        want = float((grad.double() * step.double()).sum())
        # central difference: h^2 / 6 of the third derivative (sizes of order |step|^3 |w| / row deviation^2) and the values' fp32 rounding over 2 h
        assert abs((up - down) / (2 * h) - want) <= 2e-3 * float((grad.double() * step.double()).abs().sum()) + 1e-3, name


# ------------------------------------------------------------------------------------------------------------------ attention
def attn_ref(q, k, v, scale, cap, slopes, pos_q, pos_k, doc_q, doc_k, causal, prefix, d_o=None):
    """values and elementwise bounds, in 64 bits; masked places never enter a sum"""
    B, Nq, H, hd = q.shape
    Nk, Hk = k.shape[1], k.shape[2]
    G = H // Hk
    qh, kh, vh = q.double().transpose(1, 2), k.double().transpose(1, 2).repeat_interleave(G, 1), v.double().transpose(1, 2).repeat_interleave(G, 1)
    see = torch.ones(B, 1, Nq, Nk, dtype=torch.bool, device=q.device)
    if doc_q is not None:
        see &= ((doc_q[:, :, None] == doc_k[:, None]) & (doc_k >= 0)[:, None])[:, None]
    if causal:
        i, j = torch.arange(Nq, device=q.device)[:, None] + Nk - Nq, torch.arange(Nk, device=q.device)[None]
        see &= (j <= i) | (j < (prefix.view(B, 1, 1, 1) if prefix is not None else 0))
    kh = torch.where(see.any(2)[..., None], kh, torch.zeros_like(kh))          # keys and values that nobody sees: whatever they hold
    vh = torch.where(see.any(2)[..., None], vh, torch.zeros_like(vh))
    qh = torch.where(see.any(3)[..., None], qh, torch.zeros_like(qh))
    raw = qh @ kh.transpose(-1, -2) * scale
    noise = (qh.abs() @ kh.abs().transpose(-1, -2)) * scale * (hd * HALF32)     # fp32 accumulation of q.k
    s, steep = raw, torch.ones_like(raw)
    if cap:
        th = torch.tanh(raw / cap)
        s, steep = cap * th, 1 - th * th
        noise = noise + cap * 2.0 ** -20
    if slopes is not None:
        far = (pos_q[:, :, None].double() - pos_k[:, None].double()).abs().sum(-1)[:, None]
        s = s - slopes.double().view(1, H, 1, 1) * far
        noise = noise + slopes.double().view(1, H, 1, 1).abs() * far * 8 * HALF32
    noise = noise + (s.abs() + 16) * 8 * HALF32                                  # factor, exponential, running maximum
    s = torch.where(see, s, torch.full_like(s, -math.inf))
    some = see.any(-1, keepdim=True)
    p = torch.where(some, torch.softmax(torch.where(some, s, torch.zeros_like(s)), -1), torch.zeros_like(s))
    wob = torch.where(see, noise, torch.zeros_like(noise)).amax(-1, keepdim=True) * 2   # relative error of p in fp32
    o = p @ vh
    eo = (p @ vh.abs()) * (HALF16 + wob + 64 * HALF32) + o.abs() * HALF16 * 1.01
    lse = torch.where(some, torch.logsumexp(torch.where(some, s, torch.zeros_like(s)), -1, keepdim=True), torch.full_like(some, -math.inf, dtype=F64))[..., 0]
    out = {"o": (o, eo + 1e-30), "lse": (lse, wob[..., 0] + 4e-6 * (1 + torch.where(some[..., 0], lse.abs(), torch.zeros_like(lse))))}
    if d_o is not None:
        g = torch.where(see.any(3)[..., None], d_o.double().transpose(1, 2), torch.zeros_like(qh))
        dp = g @ vh.transpose(-1, -2)
        D = (g * o).sum(-1, keepdim=True)
        ds = p * (dp - D) * steep
        # D is formed with o to 2^-16 of its value, whose weights were rounded to bf16; fp32 noise of p, dp, D; ds enters its products to 2^-16
        eD = (g.abs() * (eo - o.abs() * HALF16)).sum(-1, keepdim=True)
        fp = (wob + 128 * HALF32) * 4
        eds = ds.abs() * 2.0 ** -16 + p * eD + p * ((g.abs() @ vh.abs().transpose(-1, -2)) + (g.abs() * o.abs()).sum(-1, keepdim=True)) * fp
        fold = lambda t: t.view(B, Hk, G, Nk, hd).sum(2)
        dq = ds @ kh * scale
        dk, dv = fold(ds.transpose(-1, -2) @ qh * scale), fold(p.transpose(-1, -2) @ g)
        out["dq"] = dq, eds @ kh.abs() * scale + dq.abs() * HALF16 * 1.01 + 1e-30
        out["dk"] = dk, fold(eds.transpose(-1, -2) @ qh.abs() * scale) + dk.abs() * HALF16 * 1.01 + 1e-30
        out["dv"] = dv, fold((p * (HALF16 + fp)).transpose(-1, -2) @ g.abs()) + dv.abs() * HALF16 * 1.01 + 1e-30
    return {n: ((a.transpose(1, 2), e.transpose(1, 2)) if a.dim() == 4 else (a, e)) for n, (a, e) in out.items()}


def documents(B, N, kind, seed=0):
    g = torch.Generator().manual_seed(seed)
    if kind == "packed":                                      # sorted documents, padding behind
        cut = torch.sort(torch.randint(0, N + 1, (B, 4), generator=g), 1)[0]
        d = (torch.arange(N)[None, :, None] >= cut[:, None]).sum(-1)
        d = torch.where(d == 4, torch.full_like(d, -1), d)
    elif kind == "mixed":                                     # any order, some padding in between
        d = torch.randint(-1, 3, (B, N), generator=g)
    elif kind == "one":                                       # one document and its padding, the first row all padding
        d = torch.where(torch.arange(N)[None] < torch.randint(1, N + 1, (B, 1), generator=g), 0, -1)
        d[0] = -7
    else:
        d = torch.full((B, N), 3)
    return d.to(dev(), torch.int32)


ATTN = [  # B, H, Hk, Nq, Nk, hd, cap, axes, docs, causal, prefix
    (1, 1, 1, 1, 1, 64, 0.0, 0, None, False, None), (2, 3, 3, 1, 777, 64, 0.0, 0, None, False, None), (2, 2, 1, 7, 130, 32, 12.0, 2, "packed", False, None),
    (1, 2, 2, 64, 64, 64, 0.0, 0, None, False, None), (2, 2, 2, 129, 129, 64, 0.0, 2, None, False, None), (2, 4, 2, 200, 200, 64, 30.0, 0, "packed", False, None),
    (2, 2, 2, 256, 99, 32, 20.0, 0, None, False, None), (1, 4, 1, 333, 333, 64, 0.0, 0, None, True, None), (2, 2, 2, 150, 150, 32, 0.0, 1, None, True, "some"),
    (2, 2, 2, 90, 260, 64, 0.0, 0, None, True, None), (2, 2, 2, 260, 90, 64, 0.0, 0, None, True, "some"), (3, 2, 2, 140, 140, 64, 5.0, 3, "mixed", True, "some"),
    (3, 2, 1, 190, 190, 32, 0.0, 3, "one", False, None), (2, 2, 2, 128, 128, 64, 0.0, 0, "whole", False, None), (2, 2, 2, 33, 500, 64, 0.0, 1, "mixed", False, None),
    (1, 1, 1, 1, 9000, 64, 0.0, 0, "packed", False, None), (1, 2, 1, 700, 700, 64, 0.0, 2, "packed", False, None), (1, 1, 1, 65, 5000, 32, 0.0, 0, "packed", True, "some"),
    (1, 2, 1, 5000, 65, 32, 8.0, 0, "packed", False, None), (2, 2, 2, 31, 64, 32, 0.0, 0, "mixed", False, None), (5, 3, 3, 257, 257, 64, 0.0, 2, None, False, None),
    # more workgroups than run at once: the row blocks are put in order
    (8, 12, 12, 1100, 1100, 32, 0.0, 0, "packed", False, None), (9, 10, 10, 1200, 1150, 64, 0.0, 0, "mixed", True, "some"), (3, 24, 8, 1500, 1500, 32, 9.0, 0, "packed", True, None),
    # rows split although the blocks cover the chip; as many splits as there may be
    (2, 8, 2, 2083, 2083, 32, 0.0, 1, "packed", True, "some"), (1, 1, 1, 2, 33000, 32, 0.0, 0, "packed", False, None),
    # key blocks in order and split as well
    (4, 16, 8, 2083, 2083, 32, 0.0, 0, "packed", True, "some")]


def attn_case(case, seed=0):
    B, H, Hk, Nq, Nk, hd, cap, axes, docs, causal, prefix = case
    same = Nq == Nk
    if same:
        row = rnd(B, Nk, H + 2 * Hk, hd, dtype=BF16, scale=1.5, seed=seed)
        q, k, v = row[:, :, :H], row[:, :, H:H + Hk], row[:, :, H + Hk:]
    else:
        row = rnd(B, Nk, 2 * Hk, hd, dtype=BF16, scale=1.5, seed=seed)
        q, k, v = rnd(B, Nq, H, hd, dtype=BF16, scale=1.5, seed=seed + 1), row[:, :, :Hk], row[:, :, Hk:]
    m = dict(cap=cap, slopes=None, pos_q=None, pos_k=None, doc_q=None, doc_k=None, causal=causal, prefix=None)
    if axes:
        m["slopes"] = torch.linspace(0.02, 0.4, H, device=dev())
        m["pos_k"] = torch.rand(B, Nk, axes, generator=torch.Generator().manual_seed(1)).to(dev()) * 20
        m["pos_q"] = m["pos_k"] if same else torch.rand(B, Nq, axes, generator=torch.Generator().manual_seed(2)).to(dev()) * 20
    if docs:
        m["doc_k"] = documents(B, Nk, docs, 3)
        m["doc_q"] = m["doc_k"] if same else documents(B, Nq, docs, 4)
    if prefix:
        m["prefix"] = torch.randint(-2, Nk + 3, (B,), generator=torch.Generator().manual_seed(5)).to(dev(), torch.int32)
    return q, k, v, rnd(B, Nq, H, hd, dtype=BF16, seed=seed + 2), hd ** -0.5, m


@pytest.mark.parametrize("case", ATTN)
def test_attn_mod_matches_the_formula(K, case):
    q, k, v, d_o, scale, m = attn_case(case)
    ref = attn_ref(q, k, v, scale, *m.values(), d_o=d_o)
    mod = K.ScoreMod(**m)
    o, saved = K.attn_mod_fwd(q, k, v, scale, mod)
    lse = saved.lse
    within(o, *ref["o"], "o")
    assert bool((saved.o_rest.float().abs() <= HALF16 * o.float().abs()).all())
    empty = torch.isinf(ref["lse"][0])
    assert torch.equal(empty, lse == -math.inf)
    within(torch.where(empty, torch.zeros_like(lse), lse), torch.where(empty, torch.zeros_like(ref["lse"][0]), ref["lse"][0]), ref["lse"][1], "lse")
    assert bool((o.transpose(1, 2)[empty] == 0).all())
    o2, none = K.attn_mod_fwd(q, k, v, scale, mod, need_lse=False)
    assert none is None and torch.equal(o, o2)
    dq, dk, dv = K.attn_mod_bwd(q, k, v, o, saved, d_o, scale, mod)
    for got, n in ((dq, "dq"), (dk, "dk"), (dv, "dv")):
        within(got, *ref[n], n)
    again = K.attn_mod_bwd(q, k, v, o, saved, d_o, scale, mod)
    assert all(torch.equal(a, b) for a, b in zip((dq, dk, dv), again)), "the same bits on every run"


def test_attn_mod_no_keys_no_queries(K):
    for B, Nq, Nk in ((2, 5, 0), (2, 0, 5), (0, 4, 4), (1, 0, 0)):
        q, k, v = (torch.ones(B, n, 2, 64, dtype=BF16, device=dev()) for n in (Nq, Nk, Nk))
        for mod in (None, K.ScoreMod(doc_q=torch.zeros(B, Nq, dtype=torch.int32, device=dev()), doc_k=torch.zeros(B, Nk, dtype=torch.int32, device=dev()), causal=True)):
            o, lse = K.attn_mod_fwd(q, k, v, 0.125, mod)
            assert bool((o == 0).all()) and bool((lse.lse == -math.inf).all()) and o.shape == q.shape
            for g, src in zip(K.attn_mod_bwd(q, k, v, o, lse, torch.ones_like(q), 0.125, mod), (q, k, v)):
                assert g.shape == src.shape and bool((g == 0).all())


@pytest.mark.parametrize("case", [c for c in ATTN if c[8] in ("packed", "mixed", "one") or (c[9] and c[4] < 400)])
def test_attn_mod_what_is_masked_may_be_anything(K, case):
    """NaN and infinities in every row that nobody sees (padding, keys behind the last causal row, queries that see nothing) leave results as they are"""
    q, k, v, d_o, scale, m = attn_case(case)
    q, k, v = q.clone(), k.clone(), v.clone()
    ref = attn_ref(q, k, v, scale, *m.values(), d_o=d_o)
    B, Nq, Nk = q.shape[0], q.shape[1], k.shape[1]
    see = torch.ones(B, Nq, Nk, dtype=torch.bool, device=dev())
    if m["doc_q"] is not None:
        see &= (m["doc_q"][:, :, None] == m["doc_k"][:, None]) & (m["doc_k"] >= 0)[:, None]
    if m["causal"]:
        i, j = torch.arange(Nq, device=dev())[:, None] + Nk - Nq, torch.arange(Nk, device=dev())[None]
        see &= (j <= i) | (j < (m["prefix"].view(B, 1, 1) if m["prefix"] is not None else 0))
    blind, unseen = ~see.any(2), ~see.any(1)
    for junk in (float("nan"), float("inf"), -float("inf"), torch.finfo(BF16).min):
        q[blind], d_o[blind], k[unseen], v[unseen] = junk, junk, junk, junk
        mod = K.ScoreMod(**m)
        o, lse = K.attn_mod_fwd(q, k, v, scale, mod)
        within(o, *ref["o"], "o")
        for got, n in zip(K.attn_mod_bwd(q, k, v, o, lse, d_o, scale, mod), ("dq", "dk", "dv")):
            within(got, *ref[n], n)


def test_attn_mod_not_finite_stays_in_its_document(K):
    """an infinity in one document makes rows of that document NaN and no others, in a tile both share"""
    B, N, H = 1, 100, 1
    q, k, v, d_o = (rnd(B, N, H, 64, dtype=BF16, seed=i) for i in range(4))
    doc = torch.where(torch.arange(N) < 40, 0, 1)[None].to(dev(), torch.int32)
    mod = K.ScoreMod(doc_q=doc, doc_k=doc)
    clean, lse = K.attn_mod_fwd(q, k, v, 0.125, mod)
    grads = K.attn_mod_bwd(q, k, v, clean, lse, d_o, 0.125, mod)
    for t in (q, k, v, d_o):
        keep = t.clone()
        t[0, 10, 0, 5] = float("inf")
        o, l = K.attn_mod_fwd(q, k, v, 0.125, mod)
        dq, dk, dv = K.attn_mod_bwd(q, k, v, o, l, d_o, 0.125, mod)
        assert torch.equal(o[:, 40:], clean[:, 40:])
        for got, want in zip((dq, dk, dv), grads):
            assert torch.equal(got[:, 40:], want[:, 40:])
        if t is v or t is k:
            assert not torch.isfinite(o[:, :40].float()).all()
        assert not torch.isfinite(torch.stack([dq, dk, dv])[:, :, :40].float()).all()
        t.copy_(keep)


def test_attn_mod_gradient_by_differences(K):
    """directional derivatives in 64 bits of the formula agree with the kernels' gradients to the bf16 bounds"""
    case = (1, 2, 1, 70, 70, 32, 6.0, 2, "packed", True, "some")
    q, k, v, d_o, scale, m = attn_case(case)
    mod = K.ScoreMod(**m)
    o, lse = K.attn_mod_fwd(q, k, v, scale, mod)
    grads = K.attn_mod_bwd(q, k, v, o, lse, d_o, scale, mod)
    h = 1e-5
    ref = attn_ref(q, k, v, scale, *m.values(), d_o=d_o)
    for n, (t, got) in enumerate(zip((q, k, v), grads)):
        step = rnd(*t.shape, seed=20 + n).double()
        ends = []
        for sgn in (1, -1):
            args = [x.double() for x in (q, k, v)]
            args[n] = args[n] + sgn * h * step
            ends.append(float((attn_ref(*args, scale, *m.values())["o"][0] * d_o.double()).sum()))
        want = (ends[0] - ends[1]) / (2 * h)
        bound = float((ref[("dq", "dk", "dv")[n]][1] * step.abs()).sum()) + 1e-5
        assert abs(float((got.double() * step).sum()) - want) <= bound


def test_rows_beyond_32_bits(K):
    """q, k and v as columns of rows that lie 2^22 elements apart (the last one behind 2^32): the same bits as from dense copies, gradients in place too"""
    N, rs = 1100, 1 << 22
    far = torch.empty((N - 1) * rs + 512, dtype=BF16, device=dev())
    rows = torch.as_strided(far, (1, N, 8, 64), (N * rs, rs, 64, 1))
    rows.copy_(rnd(1, N, 8, 64, dtype=BF16, seed=1))
    doc = documents(1, N, "packed", 3)
    mod = K.ScoreMod(cap=20.0, doc_q=doc, doc_k=doc)
    pos, freqs = torch.arange(N, device=dev(), dtype=torch.int32)[:, None].contiguous(), torch.linspace(1, 0.01, 32, dtype=torch.float64, device=dev())
    d_o = rnd(1, N, 4, 64, dtype=BF16, seed=2)

    def go(t, grads):
        q, k, v = t[:, :, :4], t[:, :, 4:6], t[:, :, 6:]
        K.rotary_axes(q, k, pos, freqs, (32,), out_q=q, out_k=k)
        o, saved = K.attn_mod_fwd(q, k, v, 0.125, mod)
        one, _ = K.attn_mod_fwd(q[:, -1:], k, v, 0.125, K.ScoreMod(causal=True), need_lse=False)
        outs = [None] * 3 if grads is None else [grads[:, :, :4], grads[:, :, 4:6], grads[:, :, 6:]]
        return [o, one, saved.lse, *K.attn_mod_bwd(q, k, v, o, saved, d_o, 0.125, mod, *outs)]

    dense = go(rows.contiguous(), None)
    into = torch.as_strided(torch.empty_like(far), (1, N, 8, 64), (N * rs, rs, 64, 1))
    assert all(torch.equal(a, b) for a, b in zip(go(rows, into), dense))
