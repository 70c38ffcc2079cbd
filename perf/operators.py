"""Work lists of the packed-volume block's operators: rotary positions with several axes, attention with a score cap, a distance bias and
document / prefix masks, and the gated residual with the norms around it.  Each case in its plain form (elementary torch operations in 32
bits) and, with `own`, through the entry points of mirage_amd.kernels."""
import math

import torch

own = False

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
# pairs of the rotary dimension given to each axis, for a share of the head dimension: stack, height, width (1 axis: all of it)
SECTIONS = {(32, 1): (16,), (32, 2): (8, 8), (32, 3): (4, 6, 6), (64, 1): (32,), (64, 2): (16, 16), (64, 3): (8, 12, 12)}


# ------------------------------------------------------------------------------------------------------------------ cases
def _rotary(name, B, N, H, Hk, hd, axes, pairing, dtype, train, far=False):
    return dict(name=name, op="rotary", B=B, N=N, H=H, Hk=Hk, hd=hd, axes=axes, pairing=pairing, dtype=dtype, train=train, far=far)


def _norm(name, B, N, D, kind, gate, post, bias, branch, alpha, train):
    return dict(name=name, op="norm", B=B, N=N, D=D, kind=kind, gate=gate, post=post, bias=bias, branch=branch, alpha=alpha, train=train)


def _attn(name, B, H, Hk, Nq, Nk, hd, cap, axes, docs, causal, train):
    return dict(name=name, op="attn", B=B, H=H, Hk=Hk, Nq=Nq, Nk=Nk, hd=hd, cap=cap, axes=axes, docs=docs, causal=causal, train=train)


def listed():
    return [
        # one 512 x 512 image in patches of 32 and its global token, Base heads: inference on a single sample, a launch-bound call
        _rotary("rotary one image", 1, 257, 12, 12, 64, 2, "axial", "bf16", False),
        # a training step on volumes of 16 scans (16 x 256 tokens and the global one), Large heads: rotation and the gradients' rotation
        _rotary("rotary volumes step", 8, 4097, 16, 16, 64, 3, "half", "bf16", True),
        # fp32 features with far positions on a long stack, shared key heads, ragged token count, the adapters' head width
        _rotary("rotary far fp32", 3, 1003, 8, 2, 32, 1, "interleaved", "fp32", True, True),
        # a block's seam on a single sample: LayerScale gate, post- and pre-norm, inference
        _norm("norm one image", 1, 257, 768, "layer", "channel", True, True, "bf16", 1.0, False),
        # the Base training shape: 64 samples of 128 kept tokens and the global one
        _norm("norm base step", 64, 129, 768, "layer", "channel", True, True, "bf16", 1.0, True),
        # gates per sample (conditioned blocks) on Large rows, RMS norms without bias, scaled residual: the widest streaming case
        _norm("norm gated samples step", 256, 257, 1024, "rms", "sample", True, False, "bf16", 0.75, True),
        # attention pooling: one query over a volume's tokens, ragged lengths (padding after the last scan)
        _attn("attn pool one token", 16, 12, 12, 1, 4097, 64, 0.0, 0, 1, False, False),
        # inference on a batch of images, scores falling with the distance on the patch grid
        _attn("attn images distance", 64, 12, 12, 257, 257, 64, 0.0, 2, 0, False, False),
        # training, several samples packed to rows of 1024 tokens, capped scores
        _attn("attn packed capped step", 8, 12, 12, 1024, 1024, 64, 30.0, 0, 5, False, True),
        # the output adapters' cross attention (256 queries on 129 context tokens, 8 heads of 32), capped
        _attn("attn adapter cross step", 32, 8, 8, 256, 129, 32, 20.0, 0, 0, False, True),
        # volumes packed to one long row, three axes of distance: scans of some hundred tokens that only see their own volume
        _attn("attn long packed step", 1, 16, 16, 8192, 8192, 64, 0.0, 3, 12, False, True),
        # autoregressive completion behind a visible prefix, four key heads shared by 16 query heads, odd length
        _attn("attn prefix shared step", 2, 16, 4, 4095, 4095, 64, 0.0, 0, 0, True, True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "norm", "attn", "attn"])
    if op == "rotary":
        hd = rng.choice([32, 64])
        Hk = rng.choice([1, 2, 4, 8])
        H = Hk * rng.choice([1, 2])
        N = _log(rng, 1, 4500)
        B = _log(rng, 1, max(1, 30000 // N))
        c = _rotary("", min(B, 64), N, H, Hk, hd, rng.choice([1, 2, 3]), rng.choice(["half", "interleaved", "axial"]), rng.choice(["bf16", "fp32"]),
                    rng.random() < 0.5, rng.random() < 0.3)
    elif op == "norm":
        D = rng.choice([4 * _log(rng, 16, 512), 64 * _log(rng, 1, 24), 256, 768, 1024])
        N = _log(rng, 1, 2000)
        B = _log(rng, 1, max(1, min(40000, 60_000_000 // D) // N))
        c = _norm("", min(B, 256), N, D, rng.choice(["layer", "rms"]), rng.choice(["none", "channel", "sample"]), rng.random() < 0.7, rng.random() < 0.5,
                  rng.choice(["bf16", "fp32"]), rng.choice([1.0, 0.5, 0.75]), rng.random() < 0.6)
    else:
        hd = rng.choice([32, 64])
        Hk = rng.choice([1, 2, 4, 8])
        H = Hk * rng.choice([1, 1, 2, 3])
        train = rng.random() < 0.6
        Nk = _log(rng, 64 if train else 1, 4500)       # (a query with a single key has no gradient: nothing but rounding to compare)
        Nq = min(rng.choice([Nk, Nk, 1, _log(rng, 1, Nk)]), 250_000_000 // (H * Nk))
        B = _log(rng, 1, max(1, min(64, 80_000_000 // (H * Nk * max(Nq, 1)))))
        causal = rng.random() < 0.3
        docs = 0 if Nk < 8 else rng.choice([0, 0, 1, rng.randint(2, 9)])
        c = _attn("", B, H, Hk, Nq, Nk, hd, rng.choice([0.0, 0.0, 15.0, 50.0]), rng.choice([0, 0, 1, 2, 3]), docs, causal, train)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------------------------ inputs
def _grid(N, axes):
    """Token positions: the global token first (at the origin), then a raster over stack, height and width."""
    n = torch.arange(N) - 1
    side = 16
    cols = [n % side, (n // side) % side, n // (side * side)]
    at = torch.stack(([n] if axes == 1 else [cols[1], cols[0]] if axes == 2 else [cols[2], cols[1], cols[0]]), dim=1)
    at[0] = 0
    return at


def _doc_lengths(N, docs):
    """Lengths of the documents of one row, from the case alone; what they leave of the row (about a sixteenth) is padding."""
    if docs == 0:
        return []
    total = N - N // 16
    share = [1.0 + (i % 4) for i in range(docs)]
    cut = [int(total * x / sum(share)) for x in share]
    return [max(1, x) for x in cut]


def _documents(B, N, docs, rng):
    ids = torch.full((B, N), -1, dtype=torch.int32)
    for b in range(B):
        lengths = _doc_lengths(N, docs)
        order = torch.randperm(len(lengths), generator=rng).tolist()
        at = 0
        for d, i in enumerate(order):
            ids[b, at:at + lengths[i]] = d
            at += lengths[i]
    return ids


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rng = torch.Generator().manual_seed(seed)
    rand = lambda *shape, dtype=torch.float32, scale=1.0: (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)  # noqa: E731
    s = dict(case)
    if case["op"] == "rotary":
        B, N, H, Hk, hd, dt = case["B"], case["N"], case["H"], case["Hk"], case["hd"], DT[case["dtype"]]
        # q and k as the fused projection leaves them: side by side in one row
        row = rand(B, N, H + 2 * Hk, hd, dtype=dt)
        s["q"], s["k"] = row[:, :, :H], row[:, :, H:H + Hk]
        pos = _grid(N, case["axes"])[None].repeat(B, 1, 1)
        pos = pos + torch.randint(0, 1_000_000 if case["far"] else 8, (B, 1, case["axes"]), generator=rng)
        s["pos"] = pos.to(DEV, torch.int32)
        s["sections"] = SECTIONS[(hd, case["axes"])]
        base = 10000.0 if case["axes"] == 1 else 100.0
        s["freqs"] = torch.cat([base ** (-torch.arange(n, dtype=torch.float64) / n) for n in s["sections"]]).to(DEV)
        if case["train"]:
            s["dq"], s["dk"] = rand(B, N, H, hd, dtype=dt), rand(B, N, Hk, hd, dtype=dt)
    elif case["op"] == "norm":
        B, N, D = case["B"], case["N"], case["D"]
        s["x"], s["branch"] = rand(B, N, D), rand(B, N, D, dtype=DT[case["branch"]], scale=0.7)
        weight = lambda: (1.0 + 0.2 * rand(D), 0.2 * rand(D) if case["bias"] else None)  # noqa: E731
        s["pre"] = weight()
        s["post"] = weight() if case["post"] else None
        s["gate"] = {"none": None, "channel": 0.3 * rand(D), "sample": 0.5 * rand(B, D)}[case["gate"]]
        if case["train"]:
            s["dx_new"], s["dy"] = rand(B, N, D), rand(B, N, D, dtype=torch.bfloat16)
    else:
        B, H, Hk, Nq, Nk, hd = (case[n] for n in ("B", "H", "Hk", "Nq", "Nk", "hd"))
        bf = torch.bfloat16
        if Nq == Nk:
            row = rand(B, Nk, H + 2 * Hk, hd, dtype=bf, scale=1.5)
            s["q"], s["k"], s["v"] = row[:, :, :H], row[:, :, H:H + Hk], row[:, :, H + Hk:]
        else:
            row = rand(B, Nk, 2 * Hk, hd, dtype=bf, scale=1.5)
            s["q"], s["k"], s["v"] = rand(B, Nq, H, hd, dtype=bf, scale=1.5), row[:, :, :Hk], row[:, :, Hk:]
        s["scale"] = hd ** -0.5
        s["doc_q"] = s["doc_k"] = s["slopes"] = s["pos_q"] = s["pos_k"] = s["prefix"] = None
        if case["docs"]:
            s["doc_k"] = _documents(B, Nk, case["docs"], rng).to(DEV)
            # as many queries as keys: the same tokens; fewer: the queries are spread over the row's documents
            s["doc_q"] = s["doc_k"] if Nq == Nk else s["doc_k"][:, :: max(1, Nk // Nq)][:, :Nq].contiguous()
        if case["axes"]:
            s["pos_k"] = (_grid(Nk, case["axes"]).float() + 0.25 * torch.rand(1, case["axes"], generator=rng))[None].repeat(B, 1, 1).to(DEV)
            s["pos_q"] = s["pos_k"] if Nq == Nk else s["pos_k"][:, :Nq].contiguous()
            s["slopes"] = (2.0 ** (-4.0 * torch.arange(1, H + 1) / H)).to(DEV)
        if case["causal"]:
            s["prefix"] = torch.randint(0, max(1, Nk // 4) + 1, (B,), generator=rng).to(DEV, torch.int32)
        if case["train"]:
            s["d_o"] = rand(B, Nq, H, hd, dtype=bf)
    return s


# ------------------------------------------------------------------------------------------------------------------ plain forms
def _pairs(sections, pairing):
    """Elements (first, second) of every pair, and the axis that turns it."""
    P = sum(sections)
    p = torch.arange(P)
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections))
    if pairing == "half":
        return p, p + P, axis
    if pairing == "interleaved":
        return 2 * p, 2 * p + 1, axis
    width = torch.tensor(sections)[axis]
    start = (torch.cumsum(torch.tensor(sections), 0) - torch.tensor(sections))[axis]
    return p + start, p + start + width, axis


def _plain_turn(t, cos, sin, first, second):
    a, b = t[..., first].float(), t[..., second].float()
    out = t.float()
    out[..., first] = a * cos - b * sin
    out[..., second] = a * sin + b * cos
    return out.to(t.dtype)


def _plain_rotary(s):
    first, second, axis = (i.to(DEV) for i in _pairs(s["sections"], s["pairing"]))
    angle = s["pos"][..., axis].double() * s["freqs"]                   # in 64 bits: a far position times a frequency
    cos, sin = torch.cos(angle).float().unsqueeze(2), torch.sin(angle).float().unsqueeze(2)
    out = {"q": _plain_turn(s["q"], cos, sin, first, second), "k": _plain_turn(s["k"], cos, sin, first, second)}
    if s["train"]:
        out["dq"], out["dk"] = _plain_turn(s["dq"], cos, -sin, first, second), _plain_turn(s["dk"], cos, -sin, first, second)
    return out


EPS = 1e-6


def _plain_stats(v, kind):
    mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    rstd = 1.0 / torch.sqrt((v - mean).square().mean(-1, keepdim=True) + EPS)
    return (v - mean) * rstd, rstd


def _plain_norm_grad(dn, w, hat, rstd, kind):
    t = dn * w
    m1 = t.mean(-1, keepdim=True) if kind == "layer" else 0.0
    return rstd * (t - m1 - hat * (t * hat).mean(-1, keepdim=True))


def _plain_norm(s):
    kind, x, b = s["kind"], s["x"], s["branch"].float()
    gate = s["gate"] if s["gate"] is None or s["gate"].dim() == 1 else s["gate"].unsqueeze(1)
    n = b
    if s["post"] is not None:
        bhat, brstd = _plain_stats(b, kind)
        n = bhat * s["post"][0]
        if s["post"][1] is not None:
            n = n + s["post"][1]
    x_new = s["alpha"] * x + (n if gate is None else gate * n)
    xhat, xrstd = _plain_stats(x_new, kind)
    y = xhat * s["pre"][0]
    if s["pre"][1] is not None:
        y = y + s["pre"][1]
    out = {"x_new": x_new, "y": y.to(torch.bfloat16)}
    if not s["train"]:
        return out
    dy = s["dy"].float()
    t = s["dx_new"] + _plain_norm_grad(dy, s["pre"][0], xhat, xrstd, kind)
    out["pre_weight"] = (dy * xhat).sum((0, 1))
    if s["pre"][1] is not None:
        out["pre_bias"] = dy.sum((0, 1))
    out["dx"] = s["alpha"] * t
    if gate is not None:
        out["gate"] = (t * n).sum((0, 1)) if s["gate"].dim() == 1 else (t * n).sum(1)
        t = gate * t
    if s["post"] is not None:
        out["post_weight"] = (t * bhat).sum((0, 1))
        if s["post"][1] is not None:
            out["post_bias"] = t.sum((0, 1))
        t = _plain_norm_grad(t, s["post"][0], bhat, brstd, kind)
    out["dbranch"] = t.to(s["branch"].dtype)
    return out


def _plain_attn(s):
    B, H, Hk, Nq, Nk, hd = (s[n] for n in ("B", "H", "Hk", "Nq", "Nk", "hd"))
    heads = lambda t: t.float().transpose(1, 2).repeat_interleave(H // t.shape[2], dim=1)  # noqa: E731
    q, k, v = heads(s["q"]), heads(s["k"]), heads(s["v"])
    z = torch.matmul(q, k.transpose(-1, -2)) * s["scale"]
    slope = None
    if s["cap"]:
        tanh = torch.tanh(z / s["cap"])
        z = s["cap"] * tanh
        slope = 1.0 - tanh * tanh
    if s["slopes"] is not None:
        far = (s["pos_q"].unsqueeze(2) - s["pos_k"].unsqueeze(1)).abs().sum(-1)
        z = z - s["slopes"][None, :, None, None] * far.unsqueeze(1)
    hidden = None
    if s["doc_q"] is not None:
        hidden = ((s["doc_q"].unsqueeze(2) != s["doc_k"].unsqueeze(1)) | (s["doc_q"].unsqueeze(2) < 0)).unsqueeze(1)
    if s["causal"]:
        i, j = torch.arange(Nq, device=DEV).unsqueeze(1) + (Nk - Nq), torch.arange(Nk, device=DEV).unsqueeze(0)
        late = (j > i) & (j >= s["prefix"][:, None, None, None])
        hidden = late if hidden is None else hidden | late
    if hidden is not None:
        z = z.masked_fill(hidden, -math.inf)
    top = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)      # a row that may see nothing gives zeros
    o = torch.matmul(p, v)
    out = {"o": o.transpose(1, 2).to(torch.bfloat16)}
    if s["train"]:
        d_o = heads(s["d_o"])
        dz = torch.matmul(d_o, v.transpose(-1, -2))
        dz = p * (dz - (d_o * o).sum(-1, keepdim=True))
        if slope is not None:
            dz = dz * slope
        shared = lambda t: t.view(B, Hk, H // Hk, Nk, hd).sum(2).transpose(1, 2).to(torch.bfloat16)  # noqa: E731
        out["dq"] = (torch.matmul(dz, k) * s["scale"]).transpose(1, 2).to(torch.bfloat16)
        out["dk"] = shared(torch.matmul(dz.transpose(-1, -2), q) * s["scale"])
        out["dv"] = shared(torch.matmul(p.transpose(-1, -2), d_o))
    return out


# ------------------------------------------------------------------------------------------------------------------ the framework's calls
def _own_rotary(s):
    from mirage_amd import kernels as K
    # fp32 tensors are turned where they lie, as the plain form turns them; bf16 ones into new tensors
    at = (lambda q, k: dict(out_q=s[q], out_k=s[k])) if s["dtype"] == "fp32" else (lambda q, k: {})  # noqa: E731
    q, k = K.rotary_axes(s["q"], s["k"], s["pos"], s["freqs"], s["sections"], pairing=s["pairing"], **at("q", "k"))
    out = {"q": q, "k": k}
    if s["train"]:
        out["dq"], out["dk"] = K.rotary_axes(s["dq"], s["dk"], s["pos"], s["freqs"], s["sections"], pairing=s["pairing"], inverse=True, **at("dq", "dk"))
    return out


def _own_norm(s):
    from mirage_amd import kernels as K
    how = dict(gate=s["gate"], alpha=s["alpha"], post=s["post"], pre=s["pre"], kind=s["kind"], eps=EPS)
    x_new, y, stats = K.resid_norm_fwd(s["x"], s["branch"], **how)
    out = {"x_new": x_new, "y": y}
    if s["train"]:
        out["dx"], out["dbranch"], grads = K.resid_norm_bwd(s["dx_new"], s["dy"], x_new, s["branch"], stats, **how)
        out.update(grads)
    return out


def _own_attn(s):
    from mirage_amd import kernels as K
    mod = K.ScoreMod(cap=s["cap"], slopes=s["slopes"], pos_q=s["pos_q"], pos_k=s["pos_k"], doc_q=s["doc_q"], doc_k=s["doc_k"],
                     causal=s["causal"], prefix=s["prefix"])
    o, lse = K.attn_mod_fwd(s["q"], s["k"], s["v"], s["scale"], mod, need_lse=s["train"])
    out = {"o": o}
    if s["train"]:
        out["dq"], out["dk"], out["dv"] = K.attn_mod_bwd(s["q"], s["k"], s["v"], o, lse, s["d_o"], s["scale"], mod)
    return out


def run(state):
    if own:
        return {"rotary": _own_rotary, "norm": _own_norm, "attn": _own_attn}[state["op"]](state)
    return {"rotary": _plain_rotary, "norm": _plain_norm, "attn": _plain_attn}[state["op"]](state)


# ------------------------------------------------------------------------------------------------------------------ work
def _visible(case):
    """Score pairs of one (batch row, head) that the masks leave; with a prefix, its mean length."""
    Nq, Nk = case["Nq"], case["Nk"]
    pairs = float(Nq) * Nk
    if case["docs"]:
        pairs = sum(float(n) * n for n in _doc_lengths(Nk, case["docs"])) * Nq / Nk
    if case["causal"]:
        seen = sum(max(min(Nk, i + Nk - Nq + 1), Nk / 8) for i in range(Nq))
        pairs *= seen / (float(Nq) * Nk)
    return pairs


def work(case):
    passes = 2 if case["train"] else 1
    if case["op"] == "rotary":
        elems = case["B"] * case["N"] * (case["H"] + case["Hk"]) * case["hd"]
        size = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": passes * 2 * elems * size + 4 * case["B"] * case["N"] * case["axes"], "flops": passes * 3 * elems}
    if case["op"] == "norm":
        elems = case["B"] * case["N"] * case["D"]
        size = 2 if case["branch"] == "bf16" else 4
        fwd = elems * (4 + size + 4 + 2)
        bwd = elems * (4 + 2 + 4 + size)       # dx', dy in, dx, dbranch out; x' and the branch are in hand from the forward pass's side
        return {"bytes": fwd + (bwd if case["train"] else 0), "flops": elems * (16 + (30 if case["train"] else 0))}
    B, H, Hk, Nq, Nk, hd = (case[n] for n in ("B", "H", "Hk", "Nq", "Nk", "hd"))
    rows = B * hd * 2 * (2 * Nq * H + 2 * Nk * Hk)
    more = B * hd * 2 * (2 * Nq * H + 2 * Nk * Hk) if case["train"] else 0
    return {"bytes": rows + more, "flops": _visible(case) * B * H * hd * (14 if case["train"] else 4)}


# ------------------------------------------------------------------------------------------------------------------ 64 bits
def _exact_rotary(s):
    first, second, axis = (i.to(DEV) for i in _pairs(s["sections"], s["pairing"]))
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), s["pos"].double()[..., axis] * s["freqs"])[:, :, None]

    def turned(t, by):
        t = t.double()
        z = torch.complex(t[..., first], t[..., second]) * by
        out = t.clone()
        out[..., first], out[..., second] = z.real, z.imag
        return out

    out = {"q": turned(s["q"], turn), "k": turned(s["k"], turn)}
    if s["train"]:
        out["dq"], out["dk"] = turned(s["dq"], turn.conj()), turned(s["dk"], turn.conj())
    return out


def _exact_norm(s):
    leaf = lambda t: None if t is None else t.double().requires_grad_(s["train"])  # noqa: E731
    x, b, gate = leaf(s["x"]), leaf(s["branch"]), leaf(s["gate"])
    pre = [leaf(t) for t in s["pre"]]
    post = [leaf(t) for t in s["post"]] if s["post"] is not None else None

    def norm(v, wb):
        if s["kind"] == "layer":
            v = v - v.mean(-1, keepdim=True)
        v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS) * wb[0]
        return v if wb[1] is None else v + wb[1]

    n = b if post is None else norm(b, post)
    if gate is not None:
        n = n * (gate if gate.dim() == 1 else gate[:, None])
    x_new = s["alpha"] * x + n
    y = norm(x_new, pre)
    out = {"x_new": x_new.detach(), "y": y.detach()}
    if s["train"]:
        torch.autograd.backward([x_new, y], [s["dx_new"].double(), s["dy"].double()])
        out["dx"], out["dbranch"] = x.grad, b.grad
        for name, t in [("gate", gate), ("pre_weight", pre[0]), ("pre_bias", pre[1])] + ([("post_weight", post[0]), ("post_bias", post[1])] if post else []):
            if t is not None:
                out[name] = t.grad
    return out


def _exact_attn(s):
    B, H, Hk, Nq, Nk, hd = (s[n] for n in ("B", "H", "Hk", "Nq", "Nk", "hd"))
    if float(B) * H * Nq * Nk > 2.2e9:
        return None
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    o, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b in range(B):
        see = torch.ones(Nq, Nk, dtype=torch.bool, device=DEV)
        if s["doc_q"] is not None:
            see &= (s["doc_q"][b][:, None] == s["doc_k"][b][None]) & (s["doc_k"][b] >= 0)
        if s["causal"]:
            j = torch.arange(Nk, device=DEV)
            see &= (j < s["prefix"][b]) | (j <= torch.arange(Nk - Nq, Nk, device=DEV)[:, None])
        some = see.any(1)
        for h in range(H):
            c = h // (H // Hk)
            z = q[b, :, h] @ k[b, :, c].T * s["scale"]
            if s["cap"]:
                z = torch.tanh(z / s["cap"]) * s["cap"]
            steep = 1 - (z / s["cap"]) ** 2 if s["cap"] else None
            if s["slopes"] is not None:
                for a in range(s["axes"]):
                    z = z - s["slopes"][h].double() * torch.abs(s["pos_q"][b, :, a].double()[:, None] - s["pos_k"][b, :, a].double())
            p = torch.softmax(torch.where(see, z, torch.full_like(z, -1e300)), -1) * some[:, None]
            o[b, :, h] = p @ v[b, :, c]
            if s["train"]:
                g = s["d_o"][b, :, h].double()
                dp = g @ v[b, :, c].T
                dz = p * (dp - (p * dp).sum(-1, keepdim=True))
                if steep is not None:
                    dz = dz * steep
                dq[b, :, h] = dz @ k[b, :, c] * s["scale"]
                dk[b, :, c] += dz.T @ q[b, :, h] * s["scale"]
                dv[b, :, c] += p.T @ g
    return {"o": o, "dq": dq, "dk": dk, "dv": dv} if s["train"] else {"o": o}


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "norm": _exact_norm, "attn": _exact_attn}[s["op"]](s)
