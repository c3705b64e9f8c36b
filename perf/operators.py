"""Cases of three operator families of this library, for timing and for comparing their outputs: rotary
positions (``ops.rotary``), a block's norms with its gate and residual scale (``ops.block_norm``) and
distillation from a teacher's top logits (``ops.distill``).

``own`` False runs each operator in its plain form (elementary torch operations in 32 bits), True runs
this library's kernels.  A case is a dict of plain values; ``prepare`` makes its inputs from the seed.
"""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one new token of each of 32 sequences, far into a scaled context (latency)
        _rot("rotary_one_token", 32, 1, 32, 8, 128, 128, "bf16", False, "llama3", "far", False, False),
        # the attention of a Llama-3-8B micro-batch, forward and backward
        _rot("rotary_llama_block", 2, 4096, 32, 8, 128, 128, "bf16", False, "llama3", "none", False, True),
        # half of each 64-wide head rotated, neighbouring pairs, q and k as slices of a packed projection
        _rot("rotary_packed_part", 3, 1023, 20, 20, 64, 32, "fp16", True, "ntk", "none", True, True),
        # one long fp32 sequence whose positions go on from a prefix
        _rot("rotary_long_fp32", 1, 32768, 16, 4, 128, 128, "fp32", True, "yarn", "far", False, True),
        # a few rows, forward only (latency)
        _norm("norm_few_rows", 16, 1, 4096, "bf16", "rms", "channel", False),
        # both norms around the attention of a Llama-3-8B micro-batch, forward and backward
        _norm("norm_llama_block", 2, 4096, 4096, "bf16", "rms", "channel", True),
        # LayerNorm at GPT-2 large's width, odd lengths, one gate for each sequence
        _norm("norm_sequence_gate", 7, 577, 1280, "fp16", "layer", "sequence", True),
        # wide rows with a gate of their own for each token
        _norm("norm_token_gate_wide", 4, 2048, 8192, "bf16", "rms", "token", True),
        # the loss of a few tokens, forward only (latency)
        _distill("distill_few_rows", 8, 128256, 32, "bf16", 1.0, 1.0, "none", False),
        # a Llama-3-8B micro-batch, loss and gradient of the logits
        _distill("distill_llama_head", 4096, 128256, 64, "bf16", 2.0, 0.5, "mean", True),
        # GPT-2's odd vocabulary (rows that start at any 2-byte boundary) in fp16, with a loss scale
        _distill("distill_gpt_head", 2047, 50257, 16, "fp16", 1.0, 0.9, "mean", True),
        # fp32 logits, a loss for each token
        _distill("distill_fp32_rows", 1023, 32001, 8, "fp32", 1.5, 1.0, "none", True),
    ]


def _rot(name, batch, seq, hq, hkv, dim, rdim, dtype, interleaved, scaling, positions, packed, grad):
    return {"name": name, "op": "rotary", "batch": batch, "seq": seq, "hq": hq, "hkv": hkv, "dim": dim, "rdim": rdim,
            "dtype": dtype, "interleaved": interleaved, "scaling": scaling, "positions": positions, "packed": packed,
            "grad": grad}


def _norm(name, batch, seq, dim, dtype, norm, gate, grad):
    return {"name": name, "op": "norm", "batch": batch, "seq": seq, "dim": dim, "dtype": dtype, "norm": norm,
            "gate": gate, "grad": grad}


def _distill(name, rows, vocab, top, dtype, tau, alpha, reduction, grad):
    return {"name": name, "op": "distill", "rows": rows, "vocab": vocab, "top": top, "dtype": dtype, "tau": tau,
            "alpha": alpha, "reduction": reduction, "grad": grad}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    grad = rng.random() < 0.75
    op = rng.choice(["rotary", "norm", "distill"])
    if op == "rotary":
        dim = rng.choice([32, 64, 80, 96, 128, 192, 256])
        rdim = rng.choice([dim, dim, dim // 2, dim // 4])
        hkv = rng.choice([1, 2, 4, 8])
        hq = hkv * rng.choice([1, 2, 4])
        batch = rng.randint(1, 8)
        most = (1 << 30) // (batch * (hq + hkv) * dim * BYTES[dtype] * 4)
        seq = _log(rng, 1, max(1, min(32768, most)))
        c = _rot("", batch, seq, hq, hkv, dim, rdim, dtype, rng.random() < 0.5,
                 rng.choice(["none", "linear", "ntk", "llama3", "yarn"]), rng.choice(["none", "far"]), rng.random() < 0.4, grad)
    elif op == "norm":
        dim = _log(rng, 64, 8192)
        if rng.random() < 0.7:
            dim = dim // 8 * 8
        batch = rng.randint(1, 8)
        most = (1 << 30) // (batch * dim * BYTES[dtype] * 13)
        seq = _log(rng, 1, max(1, min(8192, most)))
        c = _norm("", batch, seq, dim, dtype, rng.choice(["rms", "layer"]), rng.choice(["none", "channel", "sequence", "token"]), grad)
    else:
        vocab = _log(rng, 1000, 131072)
        if rng.random() < 0.6:
            vocab = vocab // 8 * 8
        most = (1 << 30) // (vocab * BYTES[dtype] * 2)
        c = _distill("", _log(rng, 1, max(1, min(8192, most))), vocab, _log(rng, 1, 256), dtype, rng.choice([1.0, 2.0, 1.5, 0.7]),
                     rng.choice([1.0, 0.5, 0.9]), rng.choice(["mean", "mean", "none"]), grad)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------- state
THETA = 500000.0
FACTOR, TRAINED = 8.0, 8192  # the context is stretched eightfold over this trained length
RHO, SCALE, EPS = 0.9, 0.5, 1e-5


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DT[case["dtype"]]

    def rand(*shape, scale=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + mean).to(dt)

    s = {"case": dict(case)}
    if case["op"] == "rotary":
        B, T, hq, hkv, D = (case[k] for k in ("batch", "seq", "hq", "hkv", "dim"))
        if case["packed"]:
            qkv = rand(B, T, (hq + 2 * hkv) * D)
            s["q"] = qkv[..., :hq * D].view(B, T, hq, D)
            s["k"] = qkv[..., hq * D:(hq + hkv) * D].view(B, T, hkv, D)
        else:
            s["q"], s["k"] = rand(B, T, hq, D), rand(B, T, hkv, D)
        if case["positions"] == "far":
            start = torch.randint(0, 8 * TRAINED - (T if T > 1 else 0), (B, 1), generator=g, device="cuda")
            s["positions"] = start + torch.arange(T, device="cuda")
        else:
            s["positions"] = None
        if case["grad"]:
            s["dq"], s["dk"] = rand(B, T, hq, D), rand(B, T, hkv, D)
        s["freq"], s["magnitude"] = _frequencies(case)
        s["freq"] = torch.tensor(s["freq"], dtype=torch.float64, device="cuda")
        if own:
            from my_muon_fsdp2_b200.ops.rotary import RopeScaling, RotaryEmbedding

            scaling = None if case["scaling"] == "none" else \
                RopeScaling(case["scaling"], factor=FACTOR, original_max_position=TRAINED)
            s["rotary"] = RotaryEmbedding(D, THETA, rotary_dim=case["rdim"], interleaved=case["interleaved"], scaling=scaling)
    elif case["op"] == "norm":
        B, T, D = case["batch"], case["seq"], case["dim"]
        s["x"], s["y"] = rand(B, T, D, scale=2.0), rand(B, T, D, scale=0.7, mean=0.1)
        s["wp"], s["wn"] = rand(D, scale=0.1, mean=1.0), rand(D, scale=0.1, mean=1.0)
        s["bp"], s["bn"] = (rand(D, scale=0.1), rand(D, scale=0.1)) if case["norm"] == "layer" else (None, None)
        shape = {"none": None, "channel": (D,), "sequence": (B, 1, D), "token": (B, T, D)}[case["gate"]]
        s["gate"] = None if shape is None else rand(*shape, scale=0.5, mean=0.5)
        if case["grad"]:
            s["dh"], s["dn"] = rand(B, T, D, scale=0.1), rand(B, T, D, scale=0.1)
    else:
        N, V, K = case["rows"], case["vocab"], case["top"]
        z = torch.randn(N, V, generator=g, device="cuda") * 2.0
        # a teacher's ids: K different ones spread over the vocabulary, where the student has mass too
        ids = (torch.randint(0, V, (N, 1), generator=g, device="cuda")
               + torch.arange(K, device="cuda") * torch.randint(1, max(2, V // K), (N, 1), generator=g, device="cuda")) % V
        a = torch.sort(torch.randn(N, K, generator=g, device="cuda") * 2.0 + 6.0, dim=1, descending=True).values
        z.scatter_add_(1, ids, a)
        s["logits"] = z.to(dt)
        del z
        a = a + torch.randn(N, K, generator=g, device="cuda")
        u = torch.rand(N, 1, generator=g, device="cuda")
        kept = torch.where(u < 0.05, 0, torch.where(u < 0.2, (K + 1) // 2, K))  # some rows keep fewer, some none
        ids = torch.where(torch.arange(K, device="cuda") < kept, ids, -1)
        s["ids"], s["teacher"] = ids, a
        if case["alpha"] < 1.0:
            y = torch.randint(0, V, (N,), generator=g, device="cuda")
            s["targets"] = torch.where(torch.rand(N, generator=g, device="cuda") < 0.05, -100, y)
        else:
            s["targets"] = None
        # fp16 gradients come with a loss scale, without which most of a mean's would underflow
        up = 65536.0 if case["dtype"] == "fp16" else 1.0
        s["dloss"] = torch.full((), up, device="cuda") if case["reduction"] == "mean" else \
            (torch.rand(N, generator=g, device="cuda") + 0.5) * min(up, 1024.0)
    if case["grad"]:
        for k in ("q", "k", "x", "y", "wp", "wn", "bp", "bn", "gate", "logits"):
            if s.get(k) is not None:
                s[k].requires_grad_(True)
    return s


def _frequencies(case):
    """([radians a position for each pair], factor on cos and sin) of a case, in 64 bits."""
    R, kind = case["rdim"], case["scaling"]
    theta = THETA * FACTOR ** (R / (R - 2)) if kind == "ntk" else THETA
    f = [theta ** (-2.0 * i / R) for i in range(R // 2)]
    magnitude = 1.0
    if kind == "linear":
        f = [v / FACTOR for v in f]
    elif kind == "llama3":  # long waves are stretched, short ones kept, a ramp of 1 to 4 turns between
        t = [min(1.0, max(0.0, (TRAINED * v / (2 * math.pi) - 1.0) / 3.0)) for v in f]
        f = [(1 - w) * v / FACTOR + w * v for v, w in zip(f, t)]
    elif kind == "yarn":  # a ramp over the pair's index, from 32 turns in the trained length to 1
        at = [R * math.log(TRAINED / (b * 2 * math.pi)) / (2 * math.log(THETA)) for b in (32.0, 1.0)]
        lo, hi = max(0, math.floor(at[0])), min(R - 1, math.ceil(at[1]))
        w = [min(1.0, max(0.0, (i - lo) / max(hi - lo, 1e-3))) for i in range(R // 2)]
        f = [v / FACTOR * t + v * (1 - t) for v, t in zip(f, w)]
        magnitude = 0.1 * math.log(FACTOR) + 1.0
    return f, magnitude


# --------------------------------------------------------------------------------------- run
def run(s):
    f = {"rotary": _run_rotary, "norm": _run_norm, "distill": _run_distill}[s["case"]["op"]]
    if own:
        return f(s)
    with torch.no_grad():  # the plain forms write their gradients out
        return f(s)


def _rotate(x, cos, sin, case):
    R = case["rdim"]
    r = x[..., :R].float()
    if case["interleaved"]:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = r[..., :R // 2], r[..., R // 2:]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return r.to(x.dtype) if R == x.shape[-1] else torch.cat([r.to(x.dtype), x[..., R:]], dim=-1)


def _run_rotary(s):
    c = s["case"]
    if own:
        from my_muon_fsdp2_b200.ops.rotary import apply_rotary

        q, k = apply_rotary(s["q"], s["k"], s["rotary"], positions=s["positions"])
        if not c["grad"]:
            return q, k
        return (q, k) + torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
    pos = s["positions"] if s["positions"] is not None else torch.arange(c["seq"], device="cuda")[None]
    angle = pos[..., None].double() * s["freq"]
    cos = (angle.cos() * s["magnitude"]).float()[:, :, None]
    sin = (angle.sin() * s["magnitude"]).float()[:, :, None]
    out = [_rotate(s[n], cos, sin, c) for n in ("q", "k")]
    if c["grad"]:
        out += [_rotate(s[n], cos, -sin, c) for n in ("dq", "dk")]
    return tuple(out)


def _run_norm(s):
    c = s["case"]
    if own:
        from my_muon_fsdp2_b200.ops.block_norm import gated_residual_norm

        h, n = gated_residual_norm(s["x"], s["y"], post_weight=s["wp"], post_bias=s["bp"], gate=s["gate"],
                                   pre_weight=s["wn"], pre_bias=s["bn"], norm=c["norm"], eps=EPS,
                                   residual_scale=RHO, branch_scale=SCALE)
        if not c["grad"]:
            return {"h": h, "n": n}
        names = [k for k in ("x", "y", "wp", "bp", "gate", "wn", "bn") if s[k] is not None]
        grads = torch.autograd.grad((h, n), [s[k] for k in names], (s["dh"], s["dn"]))
        return {"h": h, "n": n, **{"d" + k: v for k, v in zip(names, grads)}}
    layer, dt = c["norm"] == "layer", DT[c["dtype"]]
    f = {k: s[k].float() for k in ("x", "y", "wp", "bp", "wn", "bn", "gate") if s[k] is not None}

    def norm(v, w, b):
        d = v - v.mean(-1, keepdim=True) if layer else v
        r = torch.rsqrt(d.square().mean(-1, keepdim=True) + EPS)
        u = d * r
        return (u * w if b is None else u * w + b), u, r

    p, uy, ry = norm(f["y"], f["wp"], f.get("bp"))
    gate = f.get("gate")
    h = RHO * f["x"] + SCALE * (p if gate is None else p * gate)
    n, uh, rh = norm(h, f["wn"], f.get("bn"))
    out = {"h": h.to(dt), "n": n.to(dt)}
    if not c["grad"]:
        return out

    def back(dout, u, r, w):
        du = dout * w
        d = du - u * (du * u).mean(-1, keepdim=True)
        return r * (d - du.mean(-1, keepdim=True) if layer else d)

    dn = s["dn"].float()
    dh = s["dh"].float() + back(dn, uh, rh, f["wn"])
    out["dx"] = RHO * dh
    dp = SCALE * (dh if gate is None else dh * gate)
    out["dy"] = back(dp, uy, ry, f["wp"])
    out["dwp"], out["dwn"] = (dp * uy).sum((0, 1)), (dn * uh).sum((0, 1))
    if layer:
        out["dbp"], out["dbn"] = dp.sum((0, 1)), dn.sum((0, 1))
    if gate is not None:
        dg = SCALE * dh * p
        out["dgate"] = {"channel": lambda: dg.sum((0, 1)), "sequence": lambda: dg.sum(1, keepdim=True), "token": lambda: dg}[c["gate"]]()
    return {k: v.to(dt) for k, v in out.items()}


def _run_distill(s):
    c = s["case"]
    tau, alpha = c["tau"], c["alpha"]
    if own:
        from my_muon_fsdp2_b200.ops.distill import distillation_loss

        loss = distillation_loss(s["logits"], s["ids"], s["teacher"], s["targets"], temperature=tau, alpha=alpha,
                                 reduction=c["reduction"])
        if not c["grad"]:
            return loss
        return (loss,) + torch.autograd.grad(loss, (s["logits"],), (s["dloss"],))
    ids, y = s["ids"], s["targets"]
    z = s["logits"].float()

    def lse(v):
        m = v.max(dim=1, keepdim=True).values
        return m + (v - m).exp().sum(1, keepdim=True).log()

    mean = c["reduction"] == "mean"
    slot = ids >= 0
    at = ids.clamp_min(0)
    a = torch.where(slot, s["teacher"].float() / tau, -math.inf)
    row = slot.any(1, keepdim=True)
    logp = torch.where(slot, a - torch.where(row, lse(a), 0.0), 0.0)
    p = torch.where(slot, logp.exp(), 0.0)
    zt = z if tau == 1.0 else z / tau
    lt = lse(zt)
    kd = tau * tau * (p * (logp - (zt.gather(1, at) - lt))).sum(1)
    ckd = alpha / row.sum().clamp_min(1) if mean else torch.full((), alpha, device="cuda")
    loss = ckd * kd
    if y is not None:
        l1 = lt if tau == 1.0 else lse(z)
        hard = (y >= 0)[:, None]
        yt = y.clamp_min(0)[:, None]
        cce = (1 - alpha) / hard.sum().clamp_min(1) if mean else torch.full((), 1 - alpha, device="cuda")
        loss = loss + cce * torch.where(hard, l1 - z.gather(1, yt), 0.0)[:, 0]
    if mean:
        loss = loss.sum()
    if not c["grad"]:
        return loss
    up = s["dloss"] if mean else s["dloss"][:, None]
    k = up * ckd * tau
    grad = (zt - lt).exp() * torch.where(row, k, 0.0)
    grad.scatter_add_(1, at, -k * p)
    if y is not None:
        k = up * cce
        grad += (z - l1).exp() * torch.where(hard, k, 0.0)
        grad.scatter_add_(1, yt, torch.where(hard, -k, 0.0))
    return loss, grad.to(DT[c["dtype"]])


# -------------------------------------------------------------------------------------- work
def work(case):
    b, grad = BYTES[case["dtype"]], case["grad"]
    if case["op"] == "rotary":
        tokens = case["batch"] * case["seq"]
        n = tokens * (case["hq"] + case["hkv"]) * case["dim"]
        pos = 8 * tokens if case["positions"] == "far" else 0
        return {"bytes": (4 if grad else 2) * n * b + pos, "flops": (6 if grad else 3) * n * case["rdim"] // case["dim"]}
    if case["op"] == "norm":
        rows, D = case["batch"] * case["seq"], case["dim"]
        gates = {"none": 0, "channel": D, "sequence": case["batch"] * D, "token": rows * D}[case["gate"]]
        vectors = (4 if case["norm"] == "layer" else 2) * D + gates
        # x, y, h, n and with gradients dh, dn, dx, dy (that the backward pass reads y and h again is left out)
        return {"bytes": b * (8 if grad else 4) * rows * D + b * (2 if grad else 1) * vectors,
                "flops": (32 if grad else 10) * rows * D}
    N, V, K = case["rows"], case["vocab"], case["top"]
    return {"bytes": N * ((2 if grad else 1) * V * b + K * 12 + (8 if case["alpha"] < 1.0 else 0)),
            "flops": (10 if grad else 4) * N * V}


# ------------------------------------------------------------------------------------- exact
def exact(case, seed):
    """The operators' definitions in 64 bits; gradients by automatic differentiation."""
    global own
    was, own = own, False
    s = prepare(case, seed)
    own = was
    leaves = {k: s[k].detach().double().requires_grad_(case["grad"])
              for k in ("q", "k", "x", "y", "wp", "bp", "gate", "wn", "bn", "logits") if s.get(k) is not None}
    if case["op"] == "rotary":
        B, T, R = case["batch"], case["seq"], case["rdim"]
        pos = s["positions"] if s["positions"] is not None else torch.arange(T, device="cuda").expand(B, T)
        turn = torch.polar(torch.full((), s["magnitude"], dtype=torch.float64, device="cuda"),
                           pos.double()[:, :, None, None] * s["freq"])
        outs = []
        for n in ("q", "k"):
            x = leaves[n]
            r = x[..., :R]
            # the pairs as complex numbers, turned by the angle
            pairs = r.unflatten(-1, (R // 2, 2)) if case["interleaved"] else r.unflatten(-1, (2, R // 2)).transpose(-1, -2)
            r = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            r = r if case["interleaved"] else r.transpose(-1, -2)
            outs.append(torch.cat([r.flatten(-2), x[..., R:]], dim=-1))
        if case["grad"]:
            outs += torch.autograd.grad(outs, (leaves["q"], leaves["k"]), (s["dq"].double(), s["dk"].double()))
        return tuple(t.detach() for t in outs)
    if case["op"] == "norm":
        def norm(v, w, b):
            if case["norm"] == "layer":
                return torch.nn.functional.layer_norm(v, (v.shape[-1],), w, b, EPS)
            return v / torch.sqrt((v * v).sum(-1, keepdim=True) / v.shape[-1] + EPS) * w

        branch = norm(leaves["y"], leaves["wp"], leaves.get("bp"))
        h = RHO * leaves["x"] + SCALE * leaves.get("gate", 1.0) * branch
        n = norm(h, leaves["wn"], leaves.get("bn"))
        out = {"h": h, "n": n}
        if case["grad"]:
            grads = torch.autograd.grad((h, n), list(leaves.values()), (s["dh"].double(), s["dn"].double()))
            out |= {"d" + k: v for k, v in zip(leaves, grads)}
        return {k: v.detach() for k, v in out.items()}
    tau, alpha, ids, y = case["tau"], case["alpha"], s["ids"], s["targets"]
    a = s["teacher"].double().masked_fill(ids < 0, -math.inf)
    row = (ids >= 0).any(1)
    p = torch.softmax(a[row] / tau, dim=1)
    logq = torch.log_softmax(leaves["logits"] / tau, dim=1)[row].gather(1, ids[row].clamp_min(0))
    kd = torch.zeros(case["rows"], dtype=torch.float64, device="cuda")
    kd = kd.index_put((row.nonzero()[:, 0],), tau ** 2 * (torch.xlogy(p, p) - p * logq).sum(1))
    ce = torch.zeros_like(kd)
    if y is not None:
        ce = torch.nn.functional.cross_entropy(leaves["logits"], y, ignore_index=-100, reduction="none")
    if case["reduction"] == "mean":
        loss = alpha * kd.sum() / max(1, int(row.sum()))
        if y is not None:
            loss = loss + (1 - alpha) * ce.sum() / max(1, int((y >= 0).sum()))
    else:
        loss = alpha * kd + (1 - alpha) * ce
    if not case["grad"]:
        return loss.detach()
    return loss.detach(), torch.autograd.grad(loss, leaves["logits"], s["dloss"].double())[0]
