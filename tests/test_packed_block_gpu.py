"""The packed-volume operators together: PackedEncoder against the same network in 64 bits, packed rows against single ones, captured and replayed
calls, other streams, the optimizer's arena.

Tolerances of the network test: a value passes at most R products with operands rounded to bf16 (2^-8 of the value each) between x and the
compared tensor, and the roundings of different elements are independent, so the error relative to the tensor's root mean square stays below
2^-8 sqrt(R) with room for the amplification of the norms (a factor of 2)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


@pytest.fixture(scope="module")
def P():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    from mirage_amd import packed
    return packed


def dev():
    return torch.device("cuda:0")


def rnd(*shape, dtype=F32, scale=1.0, seed=0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(dev())


def rel(a, b):
    a, b = a.detach(), b.detach()
    return float((a.double() - b.double()).pow(2).mean().sqrt() / b.double().pow(2).mean().sqrt())


def fill(model, seed=0):
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for n, p in model.named_parameters():
            if p.dim() == 2:
                p.copy_((torch.randn(p.shape, generator=g) * p.shape[1] ** -0.5).bfloat16().float())     # exact in bf16: the products see these weights
            elif "norm" in n or "post" in n:
                p.copy_((1.0 if n.endswith("weight") else 0.0) + 0.2 * torch.randn(p.shape, generator=g))
            else:
                p.copy_(0.3 * torch.randn(p.shape, generator=g))
    return model


def reference(model, x, pos, mod, gates, dx, dy):
    """the network and its gradients in 64 bits, from its formulas"""
    p = {n: t.detach().double().requires_grad_(True) for n, t in model.named_parameters()}
    x0 = x.double().requires_grad_(True)
    g64 = None if gates is None else [tuple(g.detach().double().requires_grad_(True) for g in pair) for pair in gates]
    kind = model._first.kind

    def norm(v, n):
        c = v - v.mean(-1, keepdim=True) if kind == "layer" else v
        c = c * torch.rsqrt((c * c).mean(-1, keepdim=True) + 1e-6) * p[n + ".weight"]
        return c + p[n + ".bias"] if n + ".bias" in p else c

    lin = lambda v, n: v @ p[n + ".weight"].T + p[n + ".bias"]
    B, N, D = x.shape
    h = x0
    for i, blk in enumerate(model.blocks):
        b, att = f"blocks.{i}.", blk.attn
        qkv = lin(norm(h, b + "norm1"), b + "attn.qkv").view(B, N, -1, att.head_dim)
        q, k, v = att.split(qkv)
        if att.sections:
            th = (pos.double()[..., [a for a, s in enumerate(att.sections) for _ in range(s)]] * att.freqs(x.device))
            th = (th if th.dim() == 3 else th[None])[:, :, None]
            first = [sum(att.sections[:a]) * 2 + j for a, s in enumerate(att.sections) for j in range(s)]
            second = [f + att.sections[a] for a, s in enumerate(att.sections) for f in first[sum(att.sections[:a]):sum(att.sections[:a]) + s]]

            def turn(t):
                o = t.clone()
                o[..., first] = t[..., first] * th.cos() - t[..., second] * th.sin()
                o[..., second] = t[..., first] * th.sin() + t[..., second] * th.cos()
                return o
            q, k = turn(q), turn(k)
        G = att.num_heads // att.num_kv_heads
        s = torch.einsum("bihd,bjhd->bhij", q, k.repeat_interleave(G, 2)) * att.scale
        if mod.cap:
            s = mod.cap * torch.tanh(s / mod.cap)
        if mod.slopes is not None:
            s = s - mod.slopes.double().view(1, -1, 1, 1) * (mod.pos_q[:, :, None].double() - mod.pos_k[:, None].double()).abs().sum(-1)[:, None]
        see = ((mod.doc_q[:, :, None] == mod.doc_k[:, None]) & (mod.doc_k >= 0)[:, None])[:, None]
        w = torch.where(see.any(-1, keepdim=True), torch.softmax(s.masked_fill(~see, -1e30), -1), torch.zeros_like(s))
        a = lin(torch.einsum("bhij,bjhd->bihd", w, v.repeat_interleave(G, 2)).reshape(B, N, D), b + "attn.proj")
        for seam, branch in (("seam1", lambda: a), ("seam2", lambda: lin(torch.nn.functional.gelu(lin(norm(h, b + "norm2"), b + "mlp.fc1")), b + "mlp.fc2"))):
            r = branch()
            if b + seam + ".post.weight" in p:
                r = norm(r, b + seam + ".post")
            j = 0 if seam == "seam1" else 1
            gate = g64[i][j][:, None] if g64 is not None else p.get(b + seam + ".gate")
            h = getattr(blk, seam).alpha * h + (r if gate is None else gate * r)
    y = norm(h, "norm")
    torch.autograd.backward([h, y], [dx.double(), dy.double()])
    return h.detach(), y.detach(), x0.grad, {n: t.grad for n, t in p.items()}, None if g64 is None else [tuple(t.grad for t in pair) for pair in g64]


def volume(P, B=2, lead=1):
    """two samples of different grids and padding in each row: documents, positions"""
    a, b = P.grid_positions((2, 4, 5), lead), P.grid_positions((3, 3, 7), lead)
    pad = 9
    row = torch.cat([a, b, torch.zeros(pad, 3, dtype=torch.int32)])
    doc = torch.cat([torch.zeros(len(a)), torch.ones(len(b)), torch.full((pad,), -1)]).int()
    flip = torch.cat([torch.ones(len(b)), torch.zeros(len(a)), torch.full((pad,), -1)]).int()
    rowf = torch.cat([b, a, torch.zeros(pad, 3, dtype=torch.int32)])
    pos = torch.stack([row if i % 2 == 0 else rowf for i in range(B)]).to(dev())
    docs = torch.stack([doc if i % 2 == 0 else flip for i in range(B)]).to(dev())
    return pos, docs, len(a), len(b)


@pytest.mark.parametrize("norm,post,gate,kv,cap,bias,per_sample", [("layer", True, 1.0, 4, 0.0, False, False), ("rms", True, 0.7, 2, 20.0, True, False),
                                                                  ("rms", False, None, 1, 0.0, True, True)])
def test_encoder_matches_the_network_in_64_bits(P, norm, post, gate, kv, cap, bias, per_sample):
    from mirage_amd import kernels as K
    D, H = 256, 4
    enc = fill(P.PackedEncoder(D, 2, H, num_kv_heads=kv, sections=(8, 12, 12), norm=norm, post_norm=post, gate=gate, alpha=0.9).to(dev()))
    pos, doc, _, _ = volume(P)
    B, N = doc.shape
    extra = dict(slopes=torch.linspace(0.05, 0.4, H, device=dev()), pos_q=pos.float(), pos_k=pos.float()) if bias else {}
    mod = K.ScoreMod(cap=cap, doc_q=doc, doc_k=doc, **extra)
    x = rnd(B, N, D, seed=1).requires_grad_(True)
    gates = [tuple((0.5 * rnd(B, D, seed=10 * i + j)).requires_grad_(True) for j in range(2)) for i in range(2)] if per_sample else None
    dx, dy = rnd(B, N, D, seed=2), rnd(B, N, D, seed=3, dtype=BF16)
    h, y = enc(x, pos, mod, gates)
    torch.autograd.backward([h, y], [dx, dy])
    rh, ry, rx, rp, rg = reference(enc, x.detach(), pos, mod, gates, dx, dy)
    # per block and branch: y, the branch's two (mlp) to five (attention) products and the branch itself
    fwd, bwd = 2 * 2.0 ** -8 * math.sqrt(2 * 9), 2 * 2.0 ** -8 * math.sqrt(2 * 2 * 9)
    assert rel(h, rh) < fwd and rel(y, ry) < fwd
    assert rel(x.grad, rx) < bwd
    for n, p in enc.named_parameters():
        assert rel(p.grad, rp[n]) < bwd, n
    if per_sample:
        for got, want in zip(gates, rg):
            for a, b in zip(got, want):
                assert rel(a.grad, b) < bwd


def test_packed_rows_equal_single_samples(P):
    from mirage_amd import kernels as K
    enc = fill(P.PackedEncoder(128, 2, 2, sections=(8, 12, 12)).to(dev()))
    pos, doc, na, nb = volume(P, B=1)
    x = rnd(1, doc.shape[1], 128, seed=1)
    with torch.no_grad():
        x[:, na + nb:] = float("nan")                              # padding may hold anything
        h, y = enc(x, pos, K.ScoreMod(doc_q=doc, doc_k=doc))
        for lo, hi in ((0, na), (na, na + nb)):
            hs, ys = enc(x[:, lo:hi].contiguous(), pos[:, lo:hi].contiguous())
            # the same roundings, but for the order of sums in tiles that start elsewhere: a few fp32 steps that may turn a bf16 rounding
            assert rel(h[:, lo:hi], hs) < 2.0 ** -8 and rel(y[:, lo:hi], ys) < 2.0 ** -8


def training_pass(K, s):
    """the operators one after the other as a block uses them, forward and backward, on tensors made before"""
    q, k = K.rotary_axes(s["qkv"][:, :, :4], s["qkv"][:, :, 4:6], s["pos"], s["freqs"], (8, 12, 12), pairing="axial")
    o, lse = K.attn_mod_fwd(q, k, s["qkv"][:, :, 6:], 0.125, s["mod"])
    how = dict(gate=s["gate"], alpha=0.9, post=s["post"], pre=s["pre"], kind="layer")
    x_new, y, stats = K.resid_norm_fwd(s["x"], o.view(s["x"].shape), **how)
    dx, db, grads = K.resid_norm_bwd(s["dx"], s["dy"], x_new, o.view(s["x"].shape), stats, **how)
    dq, dk, dv = K.attn_mod_bwd(q, k, s["qkv"][:, :, 6:], o, lse, db.view(o.shape), 0.125, s["mod"])
    dq, dk = K.rotary_axes(dq, dk, s["pos"], s["freqs"], (8, 12, 12), pairing="axial", inverse=True)
    return [x_new, y, dx, dq, dk, dv] + [grads[n] for n in sorted(grads)]


def pass_state(P, B=2, N=None, seed=0, causal=False):
    from mirage_amd import kernels as K
    pos, doc, _, _ = volume(P, B)
    if N is not None:
        pos, doc = pos[:, :1].repeat(1, N, 1).contiguous(), torch.zeros(B, N, dtype=torch.int32, device=dev())
    N = doc.shape[1]
    D = 256
    vec = lambda i: 1 + 0.1 * rnd(D, seed=seed + i)
    return dict(qkv=rnd(B, N, 8, 64, dtype=BF16, seed=seed), pos=pos, freqs=P.rotary_frequencies((8, 12, 12), device=dev()),
                mod=K.ScoreMod(cap=15.0, doc_q=doc, doc_k=doc, causal=causal, prefix=torch.full((B,), 3, dtype=torch.int32, device=dev()) if causal else None),
                x=rnd(B, N, D, seed=seed + 1), gate=0.5 * rnd(B, D, seed=seed + 2), post=(vec(3), vec(4)), pre=(vec(5), vec(6)), dx=rnd(B, N, D, seed=seed + 7),
                dy=rnd(B, N, D, dtype=BF16, seed=seed + 8))


@pytest.mark.parametrize("N,causal", [(None, False), (None, True), (1500, True)])
def test_captured_passes_replay_to_the_eager_result(P, N, causal):
    """two graphs of the same calls on different states: replayed in turn, with eager passes and other allocations between, new inputs in place"""
    from mirage_amd import kernels as K
    states = [pass_state(P, 2, N, seed, causal) for seed in (0, 100)]
    for s in states:
        training_pass(K, s)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(training_pass(K, s))
        graphs.append(g)
    for turn in range(4):
        for s, g, out in zip(states, graphs, outs):
            if turn >= 2:                                          # new values in the captured inputs, other documents too
                s["qkv"].copy_(rnd(*s["qkv"].shape, dtype=BF16, seed=turn))
                s["mod"].doc_k.copy_(torch.where(s["mod"].doc_k >= 0, 1 - s["mod"].doc_k.clamp(0, 1), s["mod"].doc_k))
            g.replay()
            torch.empty(1 << 22, device=dev()).fill_(float("nan"))
            want = training_pass(K, s)
            torch.cuda.synchronize()
            g.replay()
            for a, b in zip(out, want):
                assert torch.equal(a, b)


def test_calls_on_two_streams_at_once(P):
    from mirage_amd import kernels as K
    states = [pass_state(P, 2, 700, seed, True) for seed in (0, 50)]
    want = [training_pass(K, s) for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    for _ in range(3):
        got = []
        for st, s in zip(streams, states):
            with torch.cuda.stream(st):
                got.append(training_pass(K, s))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(g, w))


def test_encoder_with_the_optimizers_arena(P):
    """gradients land in the optimizer's arena and are overwritten by the next pass; one step of AdamW moves every parameter by its formula"""
    from mirage_amd import kernels as K, optim
    enc = fill(P.PackedEncoder(128, 1, 2, sections=(8, 12, 12)).to(dev()))
    opt = optim.FusedAdamW(enc, [1e-3, 1e-3], [0.0, 0.0])
    pos, doc, _, _ = volume(P)
    mod = K.ScoreMod(doc_q=doc, doc_k=doc)
    x, w = rnd(2, doc.shape[1], 128, seed=1), rnd(2, doc.shape[1], 128, seed=2)

    def go():
        opt.zero_grad()
        h, y = enc(x, pos, mod)
        ((h * w).sum() + (y.float() * w).sum()).backward()
        return {n: p.grad.clone() for n, p in enc.named_parameters()}

    first, second = go(), go()
    assert all(torch.equal(first[n], second[n]) for n in first)
    before = {n: p.detach().clone() for n, p in enc.named_parameters()}
    norm = float(opt.step())
    assert abs(norm - math.sqrt(sum(float(g.double().pow(2).sum()) for g in first.values()))) < 1e-4 * norm
    for n, p in enc.named_parameters():
        g = first[n]
        assert p.grad.data_ptr() == p._mrg.grad.data_ptr()
        step = 1e-3 * g / (g.abs() + 1e-8)                         # the first step of AdamW without decay
        assert float((before[n] - p.detach() - step).abs().max()) < 1e-3 * 1e-3 + 2.0 ** -22 * float(before[n].abs().max()), n


def test_functions_have_their_gradients(P):
    """packed.rotary and packed.attention through autograd: the same tensors as the kernels' own backward calls"""
    from mirage_amd import kernels as K
    s = pass_state(P)
    q, k, v = (s["qkv"][:, :, a:b].clone().requires_grad_(True) for a, b in ((0, 4), (4, 6), (6, 8)))
    qr, kr = P.rotary(q, k, s["pos"], s["freqs"], (8, 12, 12))
    o = P.attention(qr, kr, v, 0.125, s["mod"])
    d_o = rnd(*o.shape, dtype=BF16, seed=4)
    o.backward(d_o)
    o2, lse = K.attn_mod_fwd(qr.detach(), kr.detach(), v.detach(), 0.125, s["mod"])
    dq, dk, dv = K.attn_mod_bwd(qr.detach(), kr.detach(), v.detach(), o2, lse, d_o, 0.125, s["mod"])
    dq, dk = K.rotary_axes(dq, dk, s["pos"], s["freqs"], (8, 12, 12), pairing="axial", inverse=True)
    assert torch.equal(o, o2) and torch.equal(q.grad, dq) and torch.equal(k.grad, dk) and torch.equal(v.grad, dv)


def test_launchers_refuse_on_the_gpu(P):
    from mirage_amd import kernels as K
    t = torch.zeros(1, 8, 4, 64, dtype=BF16, device=dev())
    pos, f = torch.zeros(8, 1, dtype=torch.int32, device=dev()), torch.ones(32, dtype=F64, device=dev())
    x, w = torch.zeros(2, 3, 64, device=dev()), torch.ones(64, device=dev())
    q, k, l = t[:, :, :2], t[:, :, 2:], torch.zeros(1, 4, 8, device=dev())
    bad = [
        (ValueError, lambda: K.rotary_axes(t.half(), None, pos, f, (32,))), (ValueError, lambda: K.rotary_axes(t, k.float(), pos, f, (32,))),
        (ValueError, lambda: K.rotary_axes(q, k, pos.long(), f, (32,))), (ValueError, lambda: K.rotary_axes(q, k, pos, f.float(), (32,))),
        (ValueError, lambda: K.rotary_axes(q, k, pos, f, (31,))), (ValueError, lambda: K.rotary_axes(q, k, pos, f, (16, 16))), (ValueError, lambda: K.rotary_axes(q, k, pos, f, (33,))),
        (ValueError, lambda: K.rotary_axes(q, k, pos, f, (32,), pairing="spiral")), (ValueError, lambda: K.rotary_axes(q, k, pos[:7], f, (32,))),
        (ValueError, lambda: K.rotary_axes(q, k[:, :7], pos, f, (32,))), (ValueError, lambda: K.rotary_axes(q, k, pos, f, (32,), out_q=k)),
        (ValueError, lambda: K.rotary_axes(q, k, pos, f, (32,), out_q=t[:, :, 1:3])), (ValueError, lambda: K.rotary_axes(q, k, pos, f, (32,), out_k=q)),
        (ValueError, lambda: K.rotary_axes(q, None, pos, f, (32,), out_k=k)), (ValueError, lambda: K.rotary_axes(q, None, pos, f, (32,), out_q=t[:, :, :1].expand(1, 8, 2, 64))),
        (ValueError, lambda: K.rotary_axes(t.transpose(2, 3), None, pos, f, (1,))), (RuntimeError, lambda: K.rotary_axes(q, k.cpu(), pos, f, (32,))),
        (RuntimeError, lambda: K.rotary_axes(q, k, pos.cpu(), f, (32,))),
        (ValueError, lambda: K.resid_norm_fwd(x.bfloat16(), x)), (ValueError, lambda: K.resid_norm_fwd(x, x.half())), (ValueError, lambda: K.resid_norm_fwd(x, x[:1])),
        (ValueError, lambda: K.resid_norm_fwd(x, x, kind="batch")), (ValueError, lambda: K.resid_norm_fwd(x, x, gate=w[:60])), (ValueError, lambda: K.resid_norm_fwd(x, x, gate=torch.ones(3, 64, device=dev()))),
        (ValueError, lambda: K.resid_norm_fwd(x, x, pre=(None, w))), (ValueError, lambda: K.resid_norm_fwd(x, x, pre=(w, w[:4]))), (ValueError, lambda: K.resid_norm_fwd(x.transpose(0, 1), x.transpose(0, 1))),
        (ValueError, lambda: K.resid_norm_fwd(x[..., :62].contiguous(), x[..., :62].contiguous())), (ValueError, lambda: K.resid_norm_fwd(x, x, out_dtype=torch.float16)),
        (ValueError, lambda: K.resid_norm_bwd(x, x, x, x, None)), (ValueError, lambda: K.resid_norm_bwd(x, None, x, x, None, pre=(w, w))), (ValueError, lambda: K.resid_norm_bwd(x, x, x, x, None, pre=(w, w))),
        (ValueError, lambda: K.resid_norm_bwd(x, None, x, x, None, gate=w, grads={"gate": w[:32]})),
        (ValueError, lambda: K.attn_mod_fwd(t.float(), t, t, 0.1)), (ValueError, lambda: K.attn_mod_fwd(t, t, t[:, :7], 0.1)), (ValueError, lambda: K.attn_mod_fwd(t, t[:, :, :3], t[:, :, :3], 0.1)),
        (NotImplementedError, lambda: K.attn_mod_fwd(t[..., :48], t[..., :48], t[..., :48], 0.1)), (RuntimeError, lambda: K.attn_mod_fwd(t[..., 4:36], t[..., 4:36], t[..., 4:36], 0.1)),
        (RuntimeError, lambda: K.attn_mod_fwd(t, t, t, -0.1)), (ValueError, lambda: K.attn_mod_fwd(t, t, t, 0.1, K.ScoreMod(doc_q=pos[None, :, 0], doc_k=pos[None, :, 0].long()))),
        (ValueError, lambda: K.attn_mod_fwd(t, t, t, 0.1, K.ScoreMod(slopes=w[:3], pos_q=x, pos_k=x))), (ValueError, lambda: K.attn_mod_fwd(t, t, t, 0.1, K.ScoreMod(causal=True, prefix=pos[:2, 0]))),
        (ValueError, lambda: K.attn_mod_bwd(t, t, t, t, None, t, 0.1)), (ValueError, lambda: K.attn_mod_bwd(t, t, t, t, l, t, 0.1)),
        (ValueError, lambda: K.attn_mod_bwd(t, t, t, t, K.AttnSaved(x, t), t, 0.1)), (ValueError, lambda: K.attn_mod_bwd(t, t, t, t, K.AttnSaved(l, q), t, 0.1)),
        (ValueError, lambda: K.attn_mod_bwd(t, t, t, t, K.AttnSaved(l, t), t, 0.1, dq=t)),
    ]
    for i, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            pytest.fail(f"call {i} was not refused")
    torch.cuda.synchronize()


def test_functions_take_any_gradient(P):
    """autograd hands over broadcast gradients (a sum's) and slices on odd strides: the same result as their dense copies'"""
    s = pass_state(P)
    def grads(join):
        q, k, v = (s["qkv"][:, :, a:b].clone().requires_grad_(True) for a, b in ((0, 4), (4, 6), (6, 8)))
        qr, kr = P.rotary(q, k, s["pos"], s["freqs"], (8, 12, 12))
        o = P.attention(qr, kr, v, 0.125, s["mod"])
        join(qr, kr, o)
        return q.grad, k.grad, v.grad

    whole = [torch.ones(*s["qkv"].shape[:2], h, 64, dtype=BF16, device=dev()) for h in (4, 2, 4)]
    dense = grads(lambda *t: torch.autograd.backward(t, whole))
    for join in (lambda *t: sum(x.sum() for x in t).backward(), lambda *t: torch.autograd.backward(t, [torch.ones((), dtype=BF16, device=dev()).expand(x.shape) for x in t]),
                 lambda *t: torch.autograd.backward(t, [torch.ones(*x.shape[:3], 67, dtype=BF16, device=dev())[..., 1:65] for x in t])):
        assert all(torch.equal(a, b) for a, b in zip(grads(join), dense))
    q = s["qkv"][:, :, :4].clone().requires_grad_(True)            # one of the two outputs goes unused, or there is only one
    P.rotary(q, s["qkv"][:, :, 4:6], s["pos"], s["freqs"], (8, 12, 12))[0].sum().backward()
    alone = s["qkv"][:, :, :4].clone().requires_grad_(True)
    P.rotary(alone, None, s["pos"], s["freqs"], (8, 12, 12))[0].sum().backward()
    assert torch.equal(q.grad, alone.grad)


def test_what_the_backward_pass_needs_is_watched(P):
    """masks changed between the passes, and a gradient of the gradient, are errors"""
    s = pass_state(P)
    q = s["qkv"][:, :, :4].clone().requires_grad_(True)
    o = P.attention(q, s["qkv"][:, :, 4:6], s["qkv"][:, :, 6:], 0.125, s["mod"])
    s["mod"].doc_q[0, 0] = 5
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()
    qr, _ = P.rotary(q, None, s["pos"], s["freqs"], (8, 12, 12))
    (g,) = torch.autograd.grad(qr, q, torch.ones_like(qr).requires_grad_(True), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_learnt_gate_gets_no_stale_gradient(P):
    """a pass with gates per sample does not use the learnt one: its gradient is zero, not the one of the pass before"""
    enc = fill(P.PackedEncoder(128, 1, 2).to(dev()))
    x, gates = rnd(2, 20, 128, seed=1), [tuple(0.5 * rnd(2, 128, seed=i) for i in (2, 3))]
    enc(x)[0].sum().backward()
    assert float(enc.blocks[0].seam1.gate.grad.abs().max()) > 0 and float(enc.blocks[0].seam2.gate.grad.abs().max()) > 0
    enc(x, gates=gates)[0].sum().backward()
    assert float(enc.blocks[0].seam1.gate.grad.abs().max()) == 0 and float(enc.blocks[0].seam2.gate.grad.abs().max()) == 0


def test_captured_training_pass_beside_a_living_graph(P):
    """forward and backward of the modules captured while an eager pass of the same parameters waits for its backward: replays equal the eager passes"""
    from mirage_amd import kernels as K
    enc = fill(P.PackedEncoder(128, 2, 2, sections=(8, 12, 12), norm="rms").to(dev()))
    pos, doc, _, _ = volume(P)
    mod = K.ScoreMod(cap=20.0, doc_q=doc, doc_k=doc)
    x, dx, dy = rnd(2, doc.shape[1], 128, seed=1), rnd(2, doc.shape[1], 128, seed=2), rnd(2, doc.shape[1], 128, dtype=BF16, seed=3)

    def go():
        h, y = enc(x, pos, mod)
        torch.autograd.backward([h, y], [dx, dy])
        return [h.detach(), y.detach()] + [p.grad for p in enc.parameters()]

    go()
    waiting = enc(x, pos, mod)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = go()
    for turn in range(3):
        x.copy_(rnd(*x.shape, seed=10 + turn))
        want = [t.clone() for t in go()]
        torch.cuda.synchronize()
        for p in enc.parameters():
            p.grad.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert len(waiting) == 2


def test_modules_refuse_another_device(P, monkeypatch):
    att = P.PackedAttention(128, 2).to(dev())
    y = torch.zeros(1, 4, 128, dtype=BF16, device=dev())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    with pytest.raises(ValueError, match="current device"):
        att(y)


def test_resid_norm_refuses_one_destination_for_two(P):
    from mirage_amd import kernels as K
    x, w, g = torch.zeros(2, 3, 64, device=dev()), torch.ones(64, device=dev()), torch.zeros(64, device=dev())
    x_new, y, stats = K.resid_norm_fwd(x, x, post=(w, None), pre=(w, None))
    with pytest.raises(ValueError, match="destination"):
        K.resid_norm_bwd(x, y, x_new, x, stats, post=(w, None), pre=(w, None), grads={"post_weight": g, "pre_weight": g})
