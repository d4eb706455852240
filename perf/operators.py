"""The training operators' cases: what is timed, the plain forms they are compared with, and 64-bit results.

Operators (warchest_b200.train_ops): policy_loss; block_norm and
block_norm_backward; act8_pack / act8_unpack; gelu8 / gelu8_backward;
act8_wgrad. `own` chooses between the plain form (elementary torch operations
in 32 bits) and the framework's calls.
"""
import math
import sys

import torch

own = False

HEXES = 37  # cells of the board: a position is 37 rows of the trunk
F = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
CLIP_LOW, CLIP_HIGH, KL_COEF, ENTROPY_COEF = 0.2, 0.28, 0.05, 0.01
EPS = 1e-5
BLOCK = 32  # values that share a scale in the 8-bit form


def _ops():
    if "war-chest-bot-9000-_b200" not in sys.path:
        sys.path.insert(1, "war-chest-bot-9000-_b200")
    from warchest_b200 import train_ops

    return train_ops


# ------------------------------------------------------------------ cases

def listed():
    return [
        # the decisions of one game under way: 512 is the longest list of legal actions the engine hands out
        {"name": "policy one game", "op": "policy", "rows": 64, "width": 512, "type": "f32", "legal": True, "kl": True,
         "entropy": True},
        # a replay batch of decisions, the legal actions marked
        {"name": "policy replay batch", "op": "policy", "rows": 131072, "width": 512, "type": "bf16", "legal": True,
         "kl": True, "entropy": True},
        # a generic language-sized vocabulary, one batch of tokens
        {"name": "policy vocabulary", "op": "policy", "rows": 2048, "width": 131072, "type": "bf16", "legal": False,
         "kl": True, "entropy": False},
        # the trunk of one search's few positions: latency
        {"name": "norm forward few", "op": "norm", "rows": 4 * HEXES, "width": 96, "type": "f32", "kind": "layer",
         "post": True, "pre": True, "per_gate": HEXES},
        # a wide transformer block's two norms and channel gate
        {"name": "norm forward wide", "op": "norm", "rows": 16384, "width": 4096, "type": "bf16", "kind": "rms",
         "post": True, "pre": True, "per_gate": 0},
        # the trunk's training batch of 16384 positions, one gate row to a position
        {"name": "norm backward trunk", "op": "norm_backward", "rows": 16384 * HEXES, "width": 96, "type": "f16",
         "kind": "layer", "post": True, "pre": True, "per_gate": HEXES},
        # one token of an odd width kept and read back
        {"name": "pack one token", "op": "pack", "rows": 1, "width": 4099, "type": "bf16"},
        # the net's 897 public features over a long batch
        {"name": "pack features", "op": "pack", "rows": 131071, "width": 897, "type": "f32"},
        # the trunk's activation in a training batch of 8192 positions, forward and backward
        {"name": "gelu trunk", "op": "gelu", "rows": 8192 * HEXES, "width": 96, "type": "bf16"},
        # a wide block's activation over one sequence of odd length
        {"name": "gelu wide", "op": "gelu", "rows": 4095, "width": 16384, "type": "bf16"},
        # the weight gradient of the trunk's pooled mix, 192 to 96, over 16384 positions: a long sum, a small result
        {"name": "wgrad trunk", "op": "wgrad", "rows": 16384 * HEXES, "k": 192, "n": 96, "type": "bf16", "out": "f32"},
        # the weight gradient of a wide square projection
        {"name": "wgrad wide", "op": "wgrad", "rows": 8192, "k": 4096, "n": 4096, "type": "bf16", "out": "bf16"},
    ]


def draw(rng):
    def log(low, high):
        return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))

    op = rng.choice(["policy", "policy", "norm", "norm_backward", "pack", "gelu", "wgrad", "wgrad"])
    kind = rng.choice(["f32", "bf16", "bf16", "f16"])
    if op == "wgrad":
        case = {"op": op, "k": log(8, 4096), "n": log(8, 4096), "type": kind, "out": rng.choice(["f32", kind])}
        cost = 2.0 * case["k"] * case["n"]
        most = min(2e11 / cost, 2.5e8 / (case["k"] + 4 * case["n"]), 606208)
        case["rows"] = log(1, max(1, int(most)))
        return case
    if op == "policy":
        width = log(8, 131072)
        most = int(min(131072, 1.2e8 / width))
        return {"op": op, "rows": log(1, max(1, most)), "width": width, "type": kind, "legal": rng.random() < 0.5,
                "kl": rng.random() < 0.7, "entropy": rng.random() < 0.5}
    width = log(8, 16384)
    rows = log(1, max(1, int(min(606208, 6e7 / width))))
    if op in ("norm", "norm_backward"):
        post, pre = rng.choice([(True, True), (True, False), (False, True)])
        return {"op": op, "rows": rows, "width": width, "type": kind, "kind": rng.choice(["layer", "rms"]), "post": post,
                "pre": pre, "per_gate": rng.choice([-1, 0, 1, HEXES, 512])}
    return {"op": op, "rows": rows, "width": width, "type": kind}


# ----------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, dtype, T = case["op"], F[case["type"]], case["rows"]

    def normal(*shape, scale=1.0, kind=dtype):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(kind)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    s = {"case": case}
    if op == "policy":
        V = case["width"]
        s["logits"] = normal(T, V, scale=2.0)
        s["legal"] = (uniform(T, V) < 0.2) if case["legal"] else None
        s["actions"] = torch.randint(0, V, (T,), generator=g, device="cuda")
        if case["legal"]:  # the action taken was legal, except in a few rows that have none left
            some = uniform(T) < 0.98
            s["legal"][torch.arange(T, device="cuda"), s["actions"]] = True
            s["legal"] &= some[:, None]
        # sampled under a policy a little off the present one; off the clip's edges, where the gradient jumps
        z = s["logits"].float()
        if s["legal"] is not None:
            z = z.masked_fill(~s["legal"], -1e30)
        now = torch.log_softmax(z, 1).gather(1, s["actions"][:, None])[:, 0].clamp(min=-60.0)
        del z
        step = normal(T, scale=0.2, kind=torch.float32)
        for edge in (math.log(1 - CLIP_LOW), math.log(1 + CLIP_HIGH)):
            step = torch.where((step - edge).abs() < 1e-3, step + 4e-3, step)
        s["old"] = now - step
        s["ref"] = now + normal(T, scale=0.2, kind=torch.float32) if case["kl"] else None
        s["advantages"] = normal(T, kind=torch.float32)
        # a mean over the rows that count: padding has weight 0
        s["weights"] = (uniform(T) < 0.9).float() / T
        return s
    if op in ("norm", "norm_backward"):
        D, R = case["width"], case["per_gate"]
        s["x"], s["h"] = normal(T, D, scale=1.5), normal(T, D, scale=0.7) + torch.tensor(0.1, dtype=dtype, device="cuda")
        s["per_gate"] = T if R == 0 else R
        s["gate"] = None if R < 0 else normal(-(-T // s["per_gate"]), D, scale=0.5)
        for name in ("post", "pre"):
            s[name] = None
            if case[name]:
                w = 1 + normal(D, scale=0.1, kind=torch.float32)
                s[name] = (w, normal(D, scale=0.1, kind=torch.float32)) if case["kind"] == "layer" else w
        if op == "norm_backward":
            s["dy"] = normal(T, D, scale=0.01 if case["type"] != "f16" else 0.25)
            s["dn"] = normal(T, D, scale=0.01 if case["type"] != "f16" else 0.25) if case["pre"] else None
            s["stats"] = _norm_stats(s)
        return s
    if op == "pack":
        D = case["width"]
        # rows of different loudness, as activations are
        s["x"] = (normal(T, D, kind=torch.float32) * torch.exp(normal(T, 1, kind=torch.float32))).to(dtype)
        return s
    if op == "gelu":
        D = case["width"]
        s["z"], s["bias"] = normal(T, D, scale=1.2), normal(D, scale=0.2, kind=torch.float32)
        s["da"] = normal(T, D, scale=0.5)
        return s
    K, N = case["k"], case["n"]
    s["q"], s["scale"] = _pack(normal(T, K, kind=torch.float32))
    s["dy"] = normal(T, N, scale=1.0 / math.sqrt(T))
    return s


# -------------------------------------------------------------- plain form

def _pack(v):
    """32-bit rows in blocks of 32: whole numbers of at most 127 and the exponent (plus 127) of their unit, the
    smallest power of two that the block's largest value allows. Rows are padded to whole blocks."""
    T, D = v.shape
    b = torch.nn.functional.pad(v, (0, -D % BLOCK)).view(T, -1, BLOCK)
    m, e = torch.frexp(b.abs().amax(2))
    code = (torch.where(m * 128 <= 127, e - 7, e - 6) + 127).clamp(min=1)
    q = torch.round(b * ((254 - code) << 23).to(torch.int32).view(torch.float32)[:, :, None])
    return q.to(torch.int8).view(T, -1), code.to(torch.uint8)


def _unpack(q, code, D):
    T = q.shape[0]
    unit = (code.to(torch.int32) << 23).view(torch.float32)
    return (q.view(T, -1, BLOCK).float() * unit[:, :, None]).view(T, -1)[:, :D]


def _moments(v, kind):
    mean = v.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(v[:, :1])
    return mean, torch.rsqrt((v - mean).square().mean(1, keepdim=True) + EPS)


def _affine(v, w):
    return v * w[0] + w[1] if isinstance(w, tuple) else v * w


def _gate_rows(s):
    T = s["x"].shape[0]
    return s["gate"].float()[torch.arange(T, device="cuda") // s["per_gate"]]


def _norm_parts(s):
    c = s["case"]
    x, h = s["x"].float(), s["h"].float()
    hm, hr = _moments(h, c["kind"]) if s["post"] is not None else (torch.zeros_like(h[:, :1]), torch.ones_like(h[:, :1]))
    hh = (h - hm) * hr
    u = _affine(hh, s["post"]) if s["post"] is not None else h
    y = RESIDUAL * x + (u if s["gate"] is None else _gate_rows(s) * u)
    ym, yr = _moments(y, c["kind"]) if s["pre"] is not None else (torch.zeros_like(h[:, :1]), torch.ones_like(h[:, :1]))
    return hh, hm, hr, u, y, ym, yr


RESIDUAL = 0.9


def _norm_stats(s):
    """The row statistics that the forward pass leaves for the backward: means and reciprocal deviations, 32 bits."""
    _, hm, hr, _, _, ym, yr = _norm_parts(s)
    return torch.cat([hm, hr, ym, yr], 1)


def _plain_policy(s):
    c = s["case"]
    z = s["logits"].float()
    T, V = z.shape
    a = s["actions"]
    legal = s["legal"] if s["legal"] is not None else torch.ones_like(z, dtype=torch.bool)
    w = s["weights"]
    live = (w != 0) & legal.gather(1, a[:, None])[:, 0]
    z = torch.where(legal & live[:, None], z, -math.inf)
    top = torch.where(live, z.amax(1), 0.0)
    e = torch.exp(z - top[:, None])
    total = torch.where(live, e.sum(1), 1.0)
    p = e / total[:, None]
    lnp = z - top[:, None] - torch.log(total)[:, None]
    pl = torch.where(p > 0, p * lnp, 0.0)
    logp = torch.where(live, lnp.gather(1, a[:, None])[:, 0], 0.0)
    entropy = -pl.sum(1)
    ratio = torch.exp(logp - s["old"])
    A = s["advantages"]
    inside = ~((A > 0) & (ratio > 1 + CLIP_HIGH) | (A < 0) & (ratio < 1 - CLIP_LOW))
    gain = torch.minimum(ratio * A, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * A)
    d = s["ref"] - logp if c["kl"] else torch.zeros_like(logp)
    kl = torch.expm1(d) - d
    ce = ENTROPY_COEF if c["entropy"] else 0.0
    row = torch.where(live, -gain + KL_COEF * kl - ce * entropy, 0.0)
    pull = torch.where(live, w * (-ratio * A * inside - KL_COEF * torch.expm1(d)), 0.0)
    grad = -pull[:, None] * p
    grad += (w * ce)[:, None] * (pl + p * entropy[:, None])
    grad[torch.arange(T, device="cuda"), a] += pull
    zero = torch.zeros_like(logp)
    return {"loss": (w * row).sum(), "row_loss": row, "logp": logp, "entropy": torch.where(live, entropy, zero),
            "kl": torch.where(live, kl, zero), "dlogits": grad.to(s["logits"].dtype)}


def _plain_norm(s):
    _, _, _, _, y, ym, yr = _norm_parts(s)
    out = {"y": y.to(s["x"].dtype)}
    if s["pre"] is not None:
        out["n"] = _affine((y - ym) * yr, s["pre"]).to(s["x"].dtype)
    return out


def _norm_grad(d, hat, r, w, kind):
    """The gradient at a norm's input, and at its weight and bias, from the gradient `d` at its output."""
    wd = d * (w[0] if isinstance(w, tuple) else w)
    inner = wd - hat * (wd * hat).mean(1, keepdim=True)
    if kind == "layer":
        inner = inner - wd.mean(1, keepdim=True)
    return inner * r, (d * hat).sum(0), d.sum(0)


def _plain_norm_backward(s):
    kind, dtype = s["case"]["kind"], s["x"].dtype
    hh, _, hr, u, y, _, _ = _norm_parts(s)
    ym, yr = s["stats"][:, 2:3], s["stats"][:, 3:4]
    out, dy = {}, s["dy"].float()
    if s["pre"] is not None:
        d, out["dpre"], bias = _norm_grad(s["dn"].float(), (y - ym) * yr, yr, s["pre"], kind)
        dy = dy + d
        if kind == "layer":
            out["dpre_bias"] = bias
    out["dx"] = (RESIDUAL * dy).to(dtype)
    du = dy
    if s["gate"] is not None:
        T, D = dy.shape
        R, G = s["per_gate"], s["gate"].shape[0]
        rows = torch.nn.functional.pad(dy * u, (0, 0, 0, G * R - T))
        out["dgate"] = rows.view(G, R, D).sum(1).to(dtype)
        du = dy * _gate_rows(s)
    if s["post"] is not None:
        du, out["dpost"], bias = _norm_grad(du, hh, hr, s["post"], kind)
        if kind == "layer":
            out["dpost_bias"] = bias
    out["dh"] = du.to(dtype)
    return out


GELU_A, GELU_B = math.sqrt(2.0 / math.pi), 0.044715


def _plain_gelu(s):
    z = s["z"].float() + s["bias"]
    a = 0.5 * z * (1 + torch.tanh(GELU_A * (z + GELU_B * z * z * z)))
    k = _unpack(*_pack(z), z.shape[1])
    t = torch.tanh(GELU_A * (k + GELU_B * k * k * k))
    slope = 0.5 * (1 + t) + 0.5 * k * (1 - t * t) * GELU_A * (1 + 3 * GELU_B * k * k)
    dz = s["da"].float() * slope
    return {"a": a.to(s["z"].dtype), "dz": dz.to(s["z"].dtype), "dbias": dz.sum(0)}


def _plain_wgrad(s):
    x = _unpack(s["q"], s["scale"], s["case"]["k"])
    dy = s["dy"].float()
    return {"dw": (x.t() @ dy).to(F[s["case"]["out"]]), "db": dy.sum(0)}


# -------------------------------------------------------------------- run

def run(s):
    c = s["case"]
    op = c["op"]
    if not own:
        if op == "policy":
            return _plain_policy(s)
        if op == "norm":
            return _plain_norm(s)
        if op == "norm_backward":
            return _plain_norm_backward(s)
        if op == "pack":
            return {"values": _unpack(*_pack(s["x"].float()), c["width"]).to(s["x"].dtype)}
        if op == "gelu":
            return _plain_gelu(s)
        return _plain_wgrad(s)
    t = _ops()
    if op == "policy":
        r = t.policy_loss(s["logits"], s["actions"], s["old"], s["advantages"], weights=s["weights"], ref_logp=s["ref"],
                          legal=s["legal"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_coef=KL_COEF if c["kl"] else 0.0,
                          entropy_coef=ENTROPY_COEF if c["entropy"] else 0.0)
        return {"loss": r.loss, "row_loss": r.row_loss, "logp": r.logp, "entropy": r.entropy, "kl": r.kl,
                "dlogits": r.dlogits}
    if op in ("norm", "norm_backward"):
        more = {"gate": s["gate"], "rows_per_gate": s["per_gate"], "residual_scale": RESIDUAL, "post": s["post"],
                "pre": s["pre"], "kind": c["kind"], "eps": EPS}
        if op == "norm":
            r = t.block_norm(s["x"], s["h"], **more)
            return {"y": r.y, "n": r.n} if s["pre"] is not None else {"y": r.y}
        r = t.block_norm_backward(s["dy"], s["dn"], s["x"], s["h"], s["stats"], **more)
        return {k: v for k, v in r._asdict().items() if v is not None}
    if op == "pack":
        return {"values": t.act8_unpack(t.act8_pack(s["x"]), s["x"].dtype)}
    if op == "gelu":
        a, z8 = t.gelu8(s["z"], s["bias"])
        dz, dbias = t.gelu8_backward(s["da"], z8)
        return {"a": a, "dz": dz, "dbias": dbias}
    dw, db = t.act8_wgrad(t.Act8(s["q"], s["scale"], c["k"]), s["dy"], dtype=F[c["out"]])
    return {"dw": dw, "db": db}


# ------------------------------------------------------------------- work

def work(case):
    op, e, T = case["op"], SIZE[case["type"]], case["rows"]
    if op == "wgrad":
        K, N = case["k"], case["n"]
        blocks = -(-K // BLOCK)
        return {"bytes": T * (blocks * (BLOCK + 1) + N * e) + K * N * SIZE[case["out"]] + 4 * N, "flops": 2.0 * T * K * N}
    D = case["width"]
    if op == "policy":
        # the logits and their gradient, the mask; per row the action, the weight, the log-probabilities and the results
        return {"bytes": T * D * (2 * e + (1 if case["legal"] else 0)) + T * (8 + 4 * 4 + 16), "flops": 10.0 * T * D}
    blocks = -(-D // BLOCK)
    if op == "pack":
        return {"bytes": T * (D * 2 * e + 2 * blocks * (BLOCK + 1)), "flops": 4.0 * T * D}
    if op == "gelu":
        return {"bytes": T * (4 * D * e + 2 * blocks * (BLOCK + 1)) + 8 * D, "flops": 30.0 * T * D}
    groups = 0 if case["per_gate"] < 0 else 1 if case["per_gate"] == 0 else -(-T // case["per_gate"])
    norms = int(case["post"]) + int(case["pre"])
    affine = 4 * D * (2 if case["kind"] == "layer" else 1)
    if op == "norm":
        return {"bytes": (T * (3 + int(case["pre"])) + groups) * D * e + norms * affine, "flops": (2.0 + 6.0 * norms) * T * D}
    return {"bytes": (T * (5 + int(case["pre"])) + 2 * groups) * D * e + 2 * norms * affine + 16 * T,
            "flops": (4.0 + 14.0 * norms) * T * D}


# ------------------------------------------------------------------ exact

def exact(case, seed):
    """Results from the definitions in 64 bits; gradients by differentiating the definition."""
    s = prepare(case, seed)
    op, T = case["op"], case["rows"]
    d = lambda v: None if v is None else tuple(x.double() for x in v) if isinstance(v, tuple) else v.double()  # noqa: E731
    if op == "policy":
        return _exact_policy(s)
    if op in ("norm", "norm_backward"):
        leaf = {k: d(s[k]) for k in ("x", "h", "gate", "post", "pre")}
        if op == "norm_backward":
            for v in leaf.values():
                for x in v if isinstance(v, tuple) else (v,):
                    if x is not None:
                        x.requires_grad_(True)

        def norm(v, w):
            if case["kind"] == "layer":
                v = v - v.mean(-1, keepdim=True)
            v = v / (v.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
            return v * w[0] + w[1] if isinstance(w, tuple) else v * w

        u = leaf["h"] if leaf["post"] is None else norm(leaf["h"], leaf["post"])
        if leaf["gate"] is not None:
            u = u * leaf["gate"].repeat_interleave(s["per_gate"], 0)[:T]
        y = leaf["x"] * RESIDUAL + u
        n = None if leaf["pre"] is None else norm(y, leaf["pre"])
        if op == "norm":
            return {"y": y} if n is None else {"y": y, "n": n}
        total = (y * d(s["dy"])).sum()
        if n is not None:
            total = total + (n * d(s["dn"])).sum()
        total.backward()
        out = {"dx": leaf["x"].grad, "dh": leaf["h"].grad}
        if leaf["gate"] is not None:
            out["dgate"] = leaf["gate"].grad
        for k in ("post", "pre"):
            if isinstance(leaf[k], tuple):
                out["d" + k], out["d" + k + "_bias"] = leaf[k][0].grad, leaf[k][1].grad
            elif leaf[k] is not None:
                out["d" + k] = leaf[k].grad
        return out

    # every power of two that can be a unit, exact in 64 bits
    units = ((torch.arange(-126, 123, device="cuda") + 1023) << 52).view(torch.float64)

    def kept(v):
        rows, width = v.shape
        b = torch.zeros(rows, -(-width // BLOCK) * BLOCK, dtype=torch.float64, device=v.device)
        b[:, :width] = v
        b = b.view(rows, -1, BLOCK)
        unit = units[torch.searchsorted(127 * units, b.abs().max(2).values)][:, :, None]  # the first one that suffices
        return (torch.round(b / unit) * unit).view(rows, -1)[:, :width]

    if op == "pack":
        return {"values": kept(d(s["x"]))}
    if op == "gelu":
        z = s["z"].float() + s["bias"]  # the definition keeps the 32-bit sum

        def gelu(v):
            return v / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v.pow(3))))

        v = kept(d(z)).requires_grad_(True)
        gelu(v).backward(d(s["da"]))
        return {"a": gelu(d(z)), "dz": v.grad, "dbias": v.grad.sum(0)}
    K = case["k"]
    unit = units[s["scale"].long() - 1]
    x = s["q"].double()[:, :K] * unit.repeat_interleave(BLOCK, 1)[:, :K]
    return {"dw": torch.einsum("tk,tn->kn", x, d(s["dy"])), "db": d(s["dy"]).sum(0)}


def _exact_policy(s):
    c = s["case"]
    z = s["logits"].double().requires_grad_(True)
    T, V = z.shape
    at = torch.arange(T, device="cuda")
    a, w, A, old = s["actions"], s["weights"].double(), s["advantages"].double(), s["old"].double()
    hold = torch.zeros(T, V, dtype=torch.float64, device="cuda")
    if s["legal"] is not None:
        hold.masked_fill_(~s["legal"], -math.inf)
    live = (w != 0) & (hold[at, a] == 0)
    hold[~live] = 0  # rows that do not count: any finite logits, then left out
    lnp = torch.log_softmax(z + hold, 1)
    logp = lnp[at, a]
    entropy = -(lnp.exp() * lnp.clamp(min=-1e4)).sum(1)
    ratio = (logp - old).exp()
    gain = torch.min(ratio * A, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * A)
    kl = torch.zeros_like(logp)
    if c["kl"]:
        diff = s["ref"].double() - logp
        kl = diff.exp() - diff - 1
    row = torch.where(live, KL_COEF * kl - gain - (ENTROPY_COEF if c["entropy"] else 0.0) * entropy, 0.0)
    loss = (w * row).sum()
    loss.backward()
    none = torch.zeros_like(logp)
    keep = lambda v: torch.where(live, v, none).detach()  # noqa: E731
    return {"loss": loss.detach(), "row_loss": row.detach(), "logp": keep(logp), "entropy": keep(entropy), "kl": keep(kl),
            "dlogits": z.grad}
