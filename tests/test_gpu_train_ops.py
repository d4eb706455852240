"""The training operators on the device against the same definitions in 64 bits.

Tolerances follow from the arithmetic, not from runs. u = 2^-24 is the relative
rounding of 32 bits; an output in 16 bits is rounded once more, by at most
EPS of its type. Sums of n terms in 32 bits, added pairwise or in runs, are
held to 32 u times the sum of the magnitudes.
"""
import math

import pytest

torch = pytest.importorskip("torch")

from warchest_b200 import SolveError  # noqa: E402
from warchest_b200 import train_layers as layers  # noqa: E402
from warchest_b200 import train_ops as ops  # noqa: E402

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
EPS = {F32: U, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F32: 1e-37, F16: 2.0 ** -24, BF16: 1e-37}  # what underflows


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def near(got, want, slack, what=""):
    """|got - want| within the output's rounding and `slack` (an absolute bound, element by element)."""
    assert got.shape == want.shape, what
    bound = EPS[got.dtype] * want.abs() + slack + TINY[got.dtype]
    off = (got.double() - want).abs()
    bad = ~(off <= bound) & ~(got.isnan() & want.isnan()) & ~(got.double() == want)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / bound)[bad].max())} bounds"


# ------------------------------------------------------------------ policy loss

def policy_case(T, V, dtype, seed=0, legal=None, scale=2.0):
    g = gen(seed)
    c = {"logits": randn(g, T, V, dtype=dtype, scale=scale), "actions": torch.randint(0, V, (T,), generator=g, device="cuda"),
         "advantages": randn(g, T), "weights": torch.rand(T, generator=g, device="cuda"), "legal": None}
    if legal is not None:
        c["legal"] = torch.rand(T, V, generator=g, device="cuda") < legal
        c["legal"][torch.arange(T, device="cuda"), c["actions"]] = True
    l = policy_plain(c, {})["logp"]
    # ratios off the clip's edges, where the gradient jumps
    step = randn(g, T, scale=0.3)
    for edge in (math.log(0.8), math.log(1.3)):
        step = torch.where((step - edge).abs() < 1e-3, step + 4e-3, step)
    c["old_logp"] = (l - step).float()
    c["ref_logp"] = (l + randn(g, T, scale=0.3)).float()
    return c


OPTIONS = {"clip_low": 0.2, "clip_high": 0.3, "kl_coef": 0.1, "entropy_coef": 0.05}


def policy_plain(c, options, upstream=1.0):
    o = {"clip_low": 0.2, "clip_high": 0.2, "kl_coef": 0.0, "entropy_coef": 0.0} | options
    z = c["logits"].double()
    T, V = z.shape
    at = torch.arange(T, device="cuda")
    a = c["actions"].long()
    legal = torch.ones_like(z, dtype=torch.bool) if c.get("legal") is None else c["legal"].bool()
    legal = legal & (z != -math.inf)
    w = c["weights"].double() if c.get("weights") is not None else torch.ones(T, dtype=torch.float64, device="cuda")
    there = (a >= 0) & (a < V)
    live = there & (w != 0) & legal[at, a.clamp(0, V - 1)]
    a = a.clamp(0, V - 1)
    z = torch.where(live[:, None], z, 0.0)
    lnp = torch.log_softmax(torch.where(legal | ~live[:, None], z, -math.inf), 1)
    p = lnp.exp()
    pl = torch.where(p > 0, p * lnp, torch.where(p.isnan(), p, 0.0))
    logp, H = lnp[at, a], -pl.sum(1)
    out = {"logp": torch.where(live, logp, 0.0), "entropy": torch.where(live, H, 0.0), "live": live}
    if "old_logp" not in c:
        return out
    A = c["advantages"].double()
    ratio = (logp - c["old_logp"].double()).exp()
    lo, hi = 1 - o["clip_low"], 1 + o["clip_high"]
    held = ((A > 0) & (ratio > hi)) | ((A < 0) & (ratio < lo))
    d = c["ref_logp"].double() - logp if c.get("ref_logp") is not None else torch.zeros_like(logp)
    kl = torch.expm1(d) - d
    row = -torch.minimum(ratio * A, ratio.clamp(lo, hi) * A) + o["kl_coef"] * kl - o["entropy_coef"] * H
    pull = torch.where(held, 0.0, -ratio * A) - o["kl_coef"] * torch.expm1(d)
    hit = torch.zeros_like(p)
    hit[at, a] = 1.0
    s = (upstream * w)[:, None]
    grad = s * (pull[:, None] * (hit - p) + o["entropy_coef"] * (pl + p * H[:, None]))
    # what an error of 1 in l, in ln p and in H does to each result
    size = s.abs() * ((ratio * A).abs() + o["kl_coef"] * torch.exp(d) + pull.abs() + o["entropy_coef"] * (1 + H.abs()))[:, None] * (hit + p * (2 + lnp.clamp(min=-1e3).abs()))
    keep = lambda v: torch.where(live, v, 0.0)  # noqa: E731
    return out | {"kl": keep(kl), "row_loss": keep(row), "loss": (w * keep(row)).sum(), "dlogits": torch.where(live[:, None] & legal, grad, 0.0),
                  "size": torch.where(live[:, None] & legal, size, 0.0), "slope": keep(((ratio * A).abs() + o["kl_coef"] * torch.expm1(d).abs() + o["entropy_coef"])),
                  "dkl": keep(torch.expm1(d).abs())}


# l: the result's rounding and 3e-7 for the sum of powers (a power is good to 2^-22, entries that weigh little have
# exponents rounded at more) and the subtraction; H likewise, from |H| + 1
def check_policy(c, options, r, upstream=1.0):
    w = policy_plain(c, options, upstream)
    l_off = 3e-7
    near(r.logp, w["logp"], l_off, "logp")
    near(r.entropy, w["entropy"], 4 * U * w["entropy"].abs() + 8e-7 * w["live"], "entropy")
    near(r.kl, w["kl"], l_off * w["dkl"] + 4 * U * w["kl"], "kl")
    slack = l_off * w["slope"] + 8 * U * (w["row_loss"].abs() + 10 * w["live"])
    near(r.row_loss, w["row_loss"], slack, "row_loss")
    weights = c["weights"].double() if c.get("weights") is not None else torch.ones_like(slack)
    near(r.loss, w["loss"], (weights.abs() * slack).sum() + 4 * U * (weights * w["row_loss"]).abs().sum(), "loss")
    # p: 2^-22 and the exponent's rounding, 3e-7 and u |ln p|; the rest of the product 4 u
    near(r.dlogits, w["dlogits"], 1.5e-6 * w["size"], "dlogits")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V", [(1, 1), (3, 2), (5, 8), (37, 33), (64, 512), (9, 513), (20, 1000), (7, 1024), (5, 1025), (6, 4096),
                                 (3, 16385), (2, 32768), (2, 70001), (3, 131072), (2, 140000)])
def test_policy_loss(T, V, dtype):
    for legal in (None, 0.3):
        c = policy_case(T, V, dtype, seed=T + V, legal=legal)
        check_policy(c, OPTIONS, ops.policy_loss(**c, **OPTIONS))
        plain = {k: v for k, v in c.items() if k != "ref_logp"}
        check_policy(plain | {"weights": None}, {}, ops.policy_loss(**plain | {"weights": None}))


@pytest.mark.parametrize("V", [16, 513, 3000, 40000])
def test_policy_rows_that_count_for_nothing(V):
    c = policy_case(9, V, BF16, seed=4, legal=0.5)
    c["legal"][0] = False  # nothing left
    c["legal"][1, c["actions"][1]] = False  # the action masked
    c["actions"][2], c["actions"][3] = -100, V  # outside
    c["weights"][4] = 0.0
    c["logits"][4] = math.nan  # and not even numbers
    c["logits"][5, c["actions"][5]] = -math.inf
    c["logits"][6] = torch.where(torch.arange(V, device="cuda") == c["actions"][6], c["logits"][6], -math.inf)  # the action alone
    r = ops.policy_loss(**c, **OPTIONS)
    check_policy(c, OPTIONS, r)
    for name in ("row_loss", "logp", "entropy", "kl"):
        assert (getattr(r, name)[:6] == 0).all()
    assert (r.dlogits[:6] == 0).all() and r.logp[6] == 0 and r.loss.isfinite()
    assert (r.dlogits[~c["legal"]] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [24, 2000, 33000])
def test_policy_masks_of_the_lowest_value(V, dtype):
    c = policy_case(6, V, dtype, seed=5)
    low = torch.finfo(dtype).min
    c["logits"][0, 1:] = low
    c["actions"][0], c["old_logp"][0], c["ref_logp"][0] = 0, -0.1, -0.2  # one entry left by a finite mask
    c["logits"][1] = low  # all equal, at the lowest value
    c["old_logp"][1] = c["ref_logp"][1] = -math.log(V)
    c["logits"][2, ::2] = -math.inf
    c["actions"][2] = 1
    c["old_logp"][2] = c["ref_logp"][2] = policy_plain(c, {})["logp"][2].float() - 0.05
    r = ops.policy_loss(**c, **OPTIONS)
    check_policy(c, OPTIONS, r)
    assert abs(float(r.entropy[1]) - math.log(V)) < 2e-6 * math.log(V)


@pytest.mark.parametrize("V", [24, 2000, 33000, 140000])
def test_policy_nan_and_infinity_stay_in_their_row(V):
    c = policy_case(5, V, F32, seed=6)
    c["logits"][1, V // 2] = math.nan
    c["logits"][3, V - 1] = math.inf
    r = ops.policy_loss(**c, **OPTIONS)
    assert r.loss.isnan() and r.row_loss[[1, 3]].isnan().all() and r.logp[[1, 3]].isnan().all()
    keep = [0, 2, 4]
    part = {k: (v[keep].contiguous() if v is not None else None) for k, v in c.items()}
    near(r.row_loss[keep], policy_plain(part, OPTIONS)["row_loss"], 1e-5, "row_loss")
    assert r.dlogits[keep].isfinite().all() and r.dlogits[1].isnan().any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,ld,skip", [(40, 48, 8), (40, 41, 0), (33, 64, 5), (1500, 1503, 1), (20000, 20016, 16), (20001, 20002, 1)])
def test_policy_strides_and_addresses(V, ld, skip, dtype):
    c = policy_case(11, V, dtype, seed=7, legal=0.4)
    wide = torch.full((11, ld + skip), math.nan, dtype=dtype, device="cuda")
    wide[:, skip:skip + V] = c["logits"]
    mask = torch.zeros(11, ld + skip + 3, dtype=torch.uint8, device="cuda")
    mask[:, skip:skip + V] = c["legal"].to(torch.uint8) * 2  # any nonzero byte marks
    v = c | {"logits": wide[:, skip:skip + V], "legal": mask[:, skip:skip + V], "actions": c["actions"].to(torch.int32)}
    check_policy(c, OPTIONS, ops.policy_loss(**v, **OPTIONS))


def test_policy_without_gradient_and_with_upstream():
    c = policy_case(30, 200, F32, seed=8)
    r = ops.policy_loss(**c, **OPTIONS, want_grad=False)
    assert r.dlogits is None
    full = ops.policy_loss(**c, **OPTIONS)
    assert torch.equal(r.row_loss, full.row_loss) and torch.equal(r.loss, full.loss)
    up = torch.tensor(-3.0, device="cuda")
    check_policy(c, OPTIONS, ops.policy_loss(**c, **OPTIONS, upstream=up), upstream=-3.0)


def test_policy_gradient_against_differences():
    c = policy_case(4, 9, F32, seed=9)
    r = ops.policy_loss(**c, **OPTIONS)
    h = 1e-4  # of the definition in 64 bits: an error of h^2
    for t in range(4):
        for j in range(9):
            sides = []
            for sign in (1, -1):
                z = c["logits"].double()
                z[t, j] += sign * h
                sides.append(float(policy_plain(c | {"logits": z}, OPTIONS)["loss"]))
            assert abs((sides[0] - sides[1]) / (2 * h) - float(r.dlogits[t, j])) < 1e-6


def test_policy_no_rows():
    e = torch.empty(0, device="cuda")
    r = ops.policy_loss(torch.empty(0, 7, device="cuda"), e.long(), e, e)
    assert r.loss == 0 and r.dlogits.shape == (0, 7)
    r = ops.policy_loss(torch.empty(3, 0, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda"), *[torch.zeros(3, device="cuda")] * 2)
    assert r.loss == 0 and (r.row_loss == 0).all()


# ------------------------------------------------------------------- block norms

def norm_case(T, D, dtype, kind, post=True, pre=True, per=None, seed=0):
    g = gen(seed)
    w = lambda: (1 + randn(g, D, scale=0.2), randn(g, D, scale=0.2)) if kind == "layer" else 1 + randn(g, D, scale=0.2)  # noqa: E731
    per = max(1, T) if per == 0 else per
    return {"x": randn(g, T, D, dtype=dtype), "h": randn(g, T, D, dtype=dtype, scale=0.7) + 0.25, "kind": kind,
            "post": w() if post else None, "pre": w() if pre else None, "residual_scale": 0.8, "rows_per_gate": per,
            "gate": None if per is None else randn(g, -(-T // per), D, dtype=dtype)}


def norm_plain(c, x, h, gate, post, pre):
    def norm(v, w):
        if c["kind"] == "layer":
            v = v - v.mean(1, keepdim=True)
        v = v * torch.rsqrt(v.square().mean(1, keepdim=True) + 1e-5)
        return v * w[0] + w[1] if isinstance(w, tuple) else v * w

    u = h if post is None else norm(h, post)
    if gate is not None:
        u = gate.repeat_interleave(c["rows_per_gate"], 0)[: len(u)] * u
    y = c["residual_scale"] * x + u
    return y, None if pre is None else norm(y, pre)


def double(v):
    return None if v is None else tuple(t.double().requires_grad_() for t in v) if isinstance(v, tuple) else v.double().requires_grad_()


def check_norm(c):
    r = ops.block_norm(**c)
    leaves = {k: double(c[k]) for k in ("x", "h", "gate", "post", "pre")}
    y, n = norm_plain(c, **leaves)
    # a normalised value is good to 32 u times the largest of its row: means of up to 16384 values, a root, two products
    at = lambda v: 64 * U * (1 + v.detach().abs().amax(1, keepdim=True))  # noqa: E731
    near(r.y, y.detach(), at(y), "y")
    if n is not None:
        near(r.n, n.detach(), at(n), "n")
    g = gen(3)
    dy, dn = randn(g, *y.shape, dtype=c["x"].dtype), randn(g, *y.shape, dtype=c["x"].dtype) if n is not None else None
    for dy_, dn_ in ((dy, dn),) + (((None, dn), (dy, None)) if n is not None else ()):
        back = ops.block_norm_backward(dy_, dn_, c["x"], c["h"], r.stats, **{k: v for k, v in c.items() if k not in ("x", "h")})
        total = (0 if dy_ is None else (y * dy_.double()).sum()) + (0 if dn_ is None else (n * dn_.double()).sum())
        total.backward(retain_graph=True)
        for name, leaf in (("dx", "x"), ("dh", "h"), ("dgate", "gate"), ("dpost", "post"), ("dpre", "pre")):
            v = leaves[leaf]
            for key, t in (((name, v[0]), (name + "_bias", v[1])) if isinstance(v, tuple) else ((name, v),)):
                got = getattr(back, key)
                if t is None:
                    assert got is None
                    continue
                want = torch.zeros_like(t) if t.grad is None else t.grad
                # products of normalised values: 64 u of the row's largest; sums over rows: of the sum of magnitudes,
                # which for gradients like these is at most sqrt(rows) times a few of the result's root mean square
                if want.dim() == 2:
                    slack = 128 * U * (1 + want.abs().amax(1, keepdim=True)) * (math.sqrt(c["rows_per_gate"]) if key == "dgate" else 1)
                else:
                    slack = 128 * U * math.sqrt(len(y)) * 4 * (1 + want.abs())
                near(got, want, slack, key)
                t.grad = None
    return r


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("T,D", [(1, 8), (3, 5), (37, 96), (75, 97), (20, 256), (33, 257), (10, 1000), (9, 1001), (5, 4096), (4, 4097),
                                 (3, 8200), (2, 16384), (3, 16383)])
def test_block_norm(T, D, kind, dtype):
    for i, (post, pre, per) in enumerate(((True, True, 0), (True, False, 1), (False, True, 37), (True, True, None))):
        check_norm(norm_case(T, D, dtype, kind, post, pre, per, seed=T + D + i))


@pytest.mark.parametrize("T,per", [(1000, 0), (1000, 37), (999, 512), (4000, 3)])
@pytest.mark.parametrize("D", [40, 300, 5000])
def test_block_norm_gates_of_many_rows(T, per, D):
    check_norm(norm_case(T, D, F32, "layer", per=per, seed=T + per))


def test_block_norm_neither():
    c = norm_case(6, 64, F32, "rms", post=False, pre=False, per=2)
    check_norm(c)


@pytest.mark.parametrize("D,ld,skip", [(96, 104, 8), (96, 97, 0), (300, 333, 3), (5000, 5001, 1)])
def test_block_norm_strides_and_addresses(D, ld, skip):
    c = norm_case(12, D, BF16, "layer", per=5, seed=1)
    wide = {}
    for k in ("x", "h"):
        wide[k] = torch.full((12, ld + skip), math.nan, dtype=BF16, device="cuda")
        wide[k][:, skip:skip + D] = c[k]
        wide[k] = wide[k][:, skip:skip + D]
    a, b = ops.block_norm(**c), ops.block_norm(**(c | wide))
    near(b.n, a.n.double(), 2.0 ** -7 * a.n.double().abs() + 1e-4, "n")
    rest = {k: v for k, v in c.items() if k not in ("x", "h")}
    dy, dn = randn(gen(2), 12, D, dtype=BF16), randn(gen(3), 12, D, dtype=BF16)
    ga = ops.block_norm_backward(dy, dn, c["x"], c["h"], a.stats, **rest)
    gb = ops.block_norm_backward(dy, dn, wide["x"], wide["h"], a.stats, **rest)
    for u, v in zip(ga, gb):
        near(v, u.double(), 2.0 ** -7 * u.double().abs() + 1e-3, "gradient")


@pytest.mark.parametrize("D", [8, 40, 96, 97, 1024, 1111])
def test_block_norm_packs_its_output(D):
    c = norm_case(7, D, F32, "layer")
    r = ops.block_norm(**c, pack=True)
    _, n = norm_plain(c, **{k: double(c[k]) for k in ("x", "h", "gate", "post", "pre")})
    kept = ops.act8_unpack(r.n8, F32).double()
    unit = (r.n8.scale.double() - 127).exp2().repeat_interleave(32, 1)[:, :D]
    assert ((kept - n.detach()).abs() <= unit * 0.5001 + 1e-5).all()
    assert torch.equal(r.n8.scale, ops.act8_pack(r.n).scale)


def test_block_norm_nan_stays_in_its_row():
    c = norm_case(5, 96, F32, "layer", per=1)
    c["h"][2, 7] = math.nan
    r = ops.block_norm(**c)
    keep = [0, 1, 3, 4]
    assert r.n[2].isnan().all() and r.n[keep].isfinite().all()


def test_block_norm_no_rows():
    c = norm_case(0, 16, F32, "layer")
    r = ops.block_norm(**c)
    assert r.y.shape == (0, 16)
    g = ops.block_norm_backward(r.y, r.n, c["x"], c["h"], r.stats, **{k: v for k, v in c.items() if k not in ("x", "h")})
    assert (g.dpost == 0).all() and (g.dpre_bias == 0).all()


# -------------------------------------------------------- activations in 8 bits

def packed(v):
    """The definition, in 64 bits: whole numbers and the units' exponents (plus 127)."""
    T, D = v.shape
    b = torch.nn.functional.pad(v.double(), (0, -D % 32)).view(T, -1, 32)
    units = ((torch.arange(-126, 123, device="cuda") + 1023) << 52).view(torch.float64)
    top = b.abs().amax(2)
    i = torch.searchsorted(127 * units, torch.nan_to_num(top, nan=0.0, posinf=0.0))
    q = torch.round(b / units[i][:, :, None])
    q = torch.where((i == 248)[:, :, None], q.clamp(-63, 63), q)  # the largest unit: 64 of it are no number of 32 bits
    broken = ~top.isfinite()
    return torch.where(broken[:, :, None], 0.0, q).view(T, -1), torch.where(broken, 255, i + 1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,D", [(1, 1), (1, 32), (3, 31), (5, 33), (7, 96), (100, 897), (4, 4099), (50, 2048)])
def test_act8_pack_and_back(T, D, dtype):
    x = (randn(gen(T), T, D) * torch.exp(3 * randn(gen(D), T, 1))).to(dtype)
    x[0, 0] = 0.0
    p = ops.act8_pack(x)
    q, scale = packed(x)
    assert torch.equal(p.q.double(), q) and torch.equal(p.scale.long(), scale)
    for out in TYPES:
        want = (q * (scale.double() - 127).exp2().repeat_interleave(32, 1))[:, :D]
        got = ops.act8_unpack(p, out)
        assert torch.equal(got.double(), want.to(out).double())
    again = ops.act8_unpack(p, F32)
    unit = (scale.double() - 127).exp2().repeat_interleave(32, 1)[:, :D]
    assert ((again.double() - x.double()).abs() <= 0.5 * unit).all()


@pytest.mark.parametrize("D", [64, 63])
def test_act8_extremes(D):
    x = torch.zeros(9, D, device="cuda")
    x[1], x[2] = 1e-44, torch.finfo(F32).tiny  # below what a unit can hold, and the smallest normal number
    x[3], x[4] = torch.finfo(F32).max, -torch.finfo(F32).max
    x[5, 40], x[6, 3], x[7, 50] = math.inf, math.nan, -math.inf
    x[8] = 127.0
    x[8, 0] = 127.00001  # one step past a unit's reach
    p = ops.act8_pack(x)
    q, scale = packed(x)
    assert torch.equal(p.q.double(), q) and torch.equal(p.scale.long(), scale)
    back = ops.act8_unpack(p, F32)
    assert (back[0] == 0).all() and back[3].isfinite().all()
    assert back[5, 32:].isnan().all() and back[5, :32].isfinite().all() and back[6, :32].isnan().all() and back[7, 32:].isnan().all()


def gelu_plain(z):
    u = math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    return z / (1 + torch.exp(-2 * u))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,D", [(1, 1), (3, 40), (37, 96), (50, 97), (9, 2048), (300, 264), (5, 2500)])
@pytest.mark.parametrize("bias", [True, False])
def test_gelu8(T, D, dtype, bias):
    g = gen(T + D)
    z, b, da = randn(g, T, D, dtype=dtype, scale=2.0), randn(g, D) if bias else None, randn(g, T, D, dtype=dtype)
    a, z8 = ops.gelu8(z, b)
    s = z.float() + b if bias else z.float()
    # a gate of 2^-22 and a product; the exponent's rounding weighs u |2 u(x)|, at most 60 u where GELU is not 0
    near(a, gelu_plain(s.double()), 96 * U * s.double().abs() * torch.sigmoid(1.6 * s.double()), "a")
    q, scale = packed(s)
    assert torch.equal(z8.q.double(), q) and torch.equal(z8.scale.long(), scale)
    v = ops.act8_unpack(z8, F32).double().requires_grad_()
    gelu_plain(v).backward(da.double())
    dz, db = ops.gelu8_backward(da, z8)
    near(dz, v.grad, 128 * U * da.double().abs(), "dz")
    near(db, v.grad.sum(0), 128 * U * da.double().abs().sum(0), "dbias")
    assert ops.gelu8_backward(da, z8, want_bias=False)[1] is None


def test_gelu8_slope_against_differences():
    z = torch.linspace(-8, 8, 512, device="cuda").view(4, 128)
    a, z8 = ops.gelu8(z)
    v, h = ops.act8_unpack(z8, F32).double(), 1e-5
    dz, _ = ops.gelu8_backward(torch.ones_like(z), z8)
    assert ((gelu_plain(v + h) - gelu_plain(v - h)) / (2 * h) - dz.double()).abs().max() < 1e-6


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,K,N", [(1, 1, 1), (1, 40, 33), (63, 33, 7), (64, 128, 32), (65, 129, 128), (200, 192, 96), (1000, 300, 520),
                                   (4097, 257, 130), (3000, 96, 96), (300, 1100, 700), (50, 31, 1025)])
def test_act8_wgrad(T, K, N, dtype):
    g = gen(T + K + N)
    x8, dy = ops.act8_pack(randn(g, T, K, dtype=BF16)), randn(g, T, N, dtype=dtype)
    x = ops.act8_unpack(x8, F32).double()
    want, size = x.t() @ dy.double(), x.abs().t() @ dy.double().abs()
    for out in {F32, dtype}:
        dw, db = ops.act8_wgrad(x8, dy, dtype=out)
        # a run of the tensor core sums at most 160 products of 16 rows, each good to a last place (2 u) of the sum
        near(dw, want, 160 * 2 * U * size, "dw")
        near(db, dy.double().sum(0), 32 * U * dy.double().abs().sum(0), "db")
    assert ops.act8_wgrad(x8, dy, want_bias=False)[1] is None


def test_act8_wgrad_long_sums_in_32_bits():
    g = gen(1)
    x8, dy = ops.act8_pack(randn(g, 20000, 300, dtype=BF16)), randn(g, 20000, 260, dtype=BF16)
    x = ops.act8_unpack(x8, F32).double()
    dw, _ = ops.act8_wgrad(x8, dy)
    want = x.t() @ dy.double()
    # relative to the whole: 160 steps of 2 u / sqrt(3) of a sum that grows like a root, and the runs' own sums
    assert float((dw.double() - want).norm() / want.norm()) < 2e-6


@pytest.mark.parametrize("T,K,N,dtype", [(100000, 512, 336, F32), (150000, 192, 96, BF16), (100000, 320, 200, F16), (60000, 128, 384, F32)])
def test_act8_wgrad_long_walks(T, K, N, dtype):
    """Many stages a CTA, in rings of different lengths: every call's bits alike, and right."""
    g = gen(T + K)
    x8, dy = ops.act8_pack(randn(g, T, K, dtype=BF16)), randn(g, T, N, dtype=dtype)
    x = ops.act8_unpack(x8, F32)
    want = sum(a.double().t() @ b.double() for a, b in zip(x.split(20000), dy.split(20000)))
    first, db = ops.act8_wgrad(x8, dy)
    # as above relative to the whole: a run's bias, and the runs' own sums
    assert float((first.double() - want).norm() / want.norm()) < 2e-6
    near(db, dy.double().sum(0), 32 * U * dy.double().abs().sum(0), "db")
    for i in range(30):
        dw, other = ops.act8_wgrad(x8, dy, want_bias=i % 2 == 0)
        assert torch.equal(dw, first) and (other is None or torch.equal(other, db))


@pytest.mark.parametrize("ld,skip", [(104, 8), (97, 0), (99, 3)])
def test_act8_wgrad_strides_and_addresses(ld, skip):
    g = gen(2)
    x8, dy = ops.act8_pack(randn(g, 500, 200, dtype=BF16)), randn(g, 500, 96, dtype=BF16)
    wide = torch.full((500, ld + skip), math.nan, dtype=BF16, device="cuda")
    wide[:, skip:skip + 96] = dy
    for a, b in zip(ops.act8_wgrad(x8, dy), ops.act8_wgrad(x8, wide[:, skip:skip + 96])):
        assert torch.equal(a, b)


def test_act8_wgrad_units_at_any_address():
    """Blocks a row that are no multiple of 4, and a scale matrix that starts on an odd byte."""
    g = gen(3)
    x8, dy = ops.act8_pack(randn(g, 300, 33 * 32, dtype=BF16)), randn(g, 300, 64, dtype=BF16)
    room = torch.full((300 * 33 + 1,), 255, dtype=torch.uint8, device="cuda")
    room[1:] = x8.scale.view(-1)
    moved = ops.Act8(x8.q, room[1:].view(300, 33), x8.width)
    for a, b in zip(ops.act8_wgrad(x8, dy), ops.act8_wgrad(moved, dy)):
        assert torch.equal(a, b)


def test_act8_wgrad_broken_blocks_and_infinities():
    g = gen(4)
    x, dy = randn(g, 100, 64), randn(g, 100, 40, dtype=F16)
    x[10, 5] = math.nan  # its block: channels 0 to 31
    dy[20, 7] = math.inf
    x8 = ops.act8_pack(x)
    dw, db = ops.act8_wgrad(x8, dy)
    assert dw[:32].isnan().all() and db[7] == math.inf
    rest = [j for j in range(40) if j != 7]
    assert dw[32:, rest].isfinite().all()
    column = dw[32:, 7]
    sign = ops.act8_unpack(x8, F32)[20, 32:].sign()
    assert ((column == sign * math.inf) | (sign == 0)).all()


def test_act8_wgrad_nothing_to_sum():
    x8 = ops.act8_pack(torch.empty(0, 40, device="cuda"))
    dw, db = ops.act8_wgrad(x8, torch.empty(0, 24, device="cuda"))
    assert (dw == 0).all() and (db == 0).all() and dw.shape == (40, 24)


# ----------------------------------------------------------------- all of them

def every_result(seed=0):
    """Each operator once, on inputs of the seed."""
    c = policy_case(300, 1000, BF16, seed=seed, legal=0.5)
    long = policy_case(40, 50001, F16, seed=seed)
    n = norm_case(2000, 96, BF16, "layer", per=37, seed=seed)
    wide = norm_case(300, 2048, F32, "rms", per=0, seed=seed)
    out = [*ops.policy_loss(**c, **OPTIONS), *ops.policy_loss(**long, **OPTIONS)]
    for v in (n, wide):
        r = ops.block_norm(**v, pack=True)
        out += [r.y, r.n, r.n8.q, r.n8.scale, r.stats]
        out += ops.block_norm_backward(r.y, r.n, v["x"], v["h"], r.stats, **{k: w for k, w in v.items() if k not in ("x", "h")})
    z = randn(gen(seed), 3000, 200, dtype=F16)
    a, z8 = ops.gelu8(z, randn(gen(seed + 1), 200))
    out += [a, z8.q, *ops.gelu8_backward(a, z8)]
    out += ops.act8_wgrad(ops.act8_pack(a), z)
    return [t for t in out if t is not None]


def test_equal_calls_give_equal_bits():
    first = every_result()
    for _ in range(3):
        for a, b in zip(first, every_result()):
            assert torch.equal(a, b) or (a.isnan() == b.isnan()).all()


def test_another_stream():
    want = every_result(5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = every_result(5)
    side.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_inside_a_cuda_graph():
    x, h = randn(gen(1), 100, 96), randn(gen(2), 100, 96)
    w = (torch.ones(96, device="cuda"), torch.zeros(96, device="cuda"))
    dy = randn(gen(3), 100, 64, dtype=BF16)
    step = lambda: (ops.block_norm(x, h, pre=w).n, ops.act8_wgrad(ops.act8_pack(x), dy)[0])  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    x.copy_(randn(gen(9), 100, 96))
    graph.replay()
    for a, b in zip(got, step()):
        assert torch.equal(a, b)


def test_offsets_past_32_bits():
    """Matrices of more than 2^31 elements: the last rows are as they are by themselves."""
    T, D = 70000, 32768
    x = torch.zeros(T, D, dtype=BF16, device="cuda")
    x[-3:] = randn(gen(1), 3, D, dtype=BF16)
    tail = x[-3:].clone()
    p, q = ops.act8_pack(x), ops.act8_pack(tail)
    assert torch.equal(p.q[-3:], q.q) and torch.equal(p.scale[-3:], q.scale)
    assert torch.equal(ops.act8_unpack(p)[-3:], ops.act8_unpack(q))
    dy = torch.zeros(T, 32, dtype=BF16, device="cuda")
    dy[-3:] = randn(gen(2), 3, 32, dtype=BF16)
    near(ops.act8_wgrad(p, dy)[0], ops.act8_wgrad(q, dy[-3:].contiguous())[0].double(), 1e-5, "dw")
    del p
    a = torch.zeros(T, dtype=torch.int64, device="cuda")
    o = torch.full((T,), -10.0, device="cuda")
    w = torch.zeros(T, device="cuda")
    w[-3:] = 1.0
    r = ops.policy_loss(x, a, o, o, weights=w)
    s = ops.policy_loss(tail, a[:3], o[:3], o[:3])
    assert torch.equal(r.dlogits[-3:], s.dlogits) and torch.equal(r.row_loss[-3:], s.row_loss) and not r.dlogits[:-3].any()
    del r
    v = torch.empty(T * 2, 16384, dtype=BF16, device="cuda").copy_(x.view(T * 2, 16384))
    w = torch.ones(16384, device="cuda")
    n = ops.block_norm(v, v, pre=w, kind="rms")
    assert torch.equal(n.n[-6:], ops.block_norm(v[-6:].clone(), v[-6:].clone(), pre=w, kind="rms").n)


def test_wrong_tensors_are_refused():
    x = torch.zeros(8, 16, device="cuda")
    v = torch.zeros(8, device="cuda")
    for call in (lambda: ops.act8_pack(x.t()[::2]), lambda: ops.act8_pack(x.double()), lambda: ops.act8_pack(x[0]),
                 lambda: ops.policy_loss(x, v, v, v), lambda: ops.policy_loss(x, v.long()[:7], v, v),
                 lambda: ops.policy_loss(x, v.long(), v.double(), v), lambda: ops.policy_loss(x, v.long(), v, v, legal=x),
                 lambda: ops.policy_loss(x, v.long(), v, v, clip_low=-1.0), lambda: ops.policy_loss(x, v.long(), None, v),
                 lambda: ops.block_norm(x, x.half()), lambda: ops.block_norm(x, x, post=v), lambda: ops.block_norm(x, x, kind="batch"),
                 lambda: ops.block_norm(x, x, gate=x, rows_per_gate=2), lambda: ops.block_norm(x, x, pack=True),
                 lambda: ops.block_norm_backward(None, None, x, x, torch.zeros(8, 4, device="cuda")),
                 lambda: ops.gelu8_backward(x, ops.act8_pack(x[:4])), lambda: ops.act8_wgrad(ops.act8_pack(x), x[:4]),
                 lambda: ops.act8_wgrad(ops.act8_pack(x), x, dtype=torch.int32),
                 lambda: ops.act8_unpack(ops.Act8(torch.zeros(8, 16, dtype=torch.int8, device="cuda"), v.byte(), 16))):
        with pytest.raises(SolveError) as e:
            call()
        assert e.value.code == 1


# ------------------------------------------------------------------ as layers

def test_layers_differentiate():
    """A block of layers, its loss and all gradients against the same in torch with 64 bits (activations that the
    layers keep in 8 bits move only the gradients at weights that read them, by about half a unit of 1/64)."""
    g = gen(11)
    T, D, H, V = 74, 96, 192, 50
    x, h = randn(g, T, D), randn(g, T, D)
    w1, b1, w2 = randn(g, D, H, scale=0.1), randn(g, H, scale=0.1), randn(g, H, V, scale=0.1)
    post, pre = (1 + randn(g, D, scale=0.1), randn(g, D, scale=0.1)), (1 + randn(g, D, scale=0.1), randn(g, D, scale=0.1))
    gate = randn(g, 2, D)
    c = policy_case(T, V, F32, seed=12)
    names = ("x", "h", "w1", "b1", "w2", "post", "post_bias", "pre", "pre_bias", "gate")
    values = (x, h, w1, b1, w2, *post, *pre, gate)
    p = {k: v.clone().requires_grad_() for k, v in zip(names, values)}
    y, n, n8 = layers.block_norm(p["x"], p["h"], gate=p["gate"], rows_per_gate=37, residual_scale=0.9,
                                 post=(p["post"], p["post_bias"]), pre=(p["pre"], p["pre_bias"]), kind="layer", pack=True)
    z = layers.linear8(layers.gelu8(layers.linear8(n, p["w1"], x8=n8), p["b1"]), p["w2"]) + y[:, :V]
    r = layers.policy_loss(z, c["actions"], c["old_logp"], c["advantages"], weights=c["weights"], ref_logp=c["ref_logp"], **OPTIONS)
    r.loss.backward()

    q = {k: v.double().requires_grad_() for k, v in zip(names, values)}
    yq, nq = norm_plain({"kind": "layer", "residual_scale": 0.9, "rows_per_gate": 37}, q["x"], q["h"], q["gate"],
                        (q["post"], q["post_bias"]), (q["pre"], q["pre_bias"]))
    zq = gelu_plain(nq @ q["w1"] + q["b1"]) @ q["w2"] + yq[:, :V]
    d = policy_plain(c | {"logits": zq.detach()}, OPTIONS)["dlogits"]
    zq.backward(d)
    for k in names:
        rel = float((p[k].grad.double() - q[k].grad).norm() / q[k].grad.norm())
        assert rel < 2e-2, (k, rel)  # half a unit of 1/64 is 8e-3 of a block's largest value
    want = policy_plain(c | {"logits": zq.detach()}, OPTIONS)["loss"]
    assert abs(float(r.loss) - float(want)) < 1e-3 * (1 + abs(float(want)))


def test_layers_notice_what_changed_before_the_backward_pass():
    c = policy_case(20, 30, F32, seed=13)
    z = c["logits"].clone().requires_grad_()
    r = layers.policy_loss(z, c["actions"], c["old_logp"], c["advantages"], weights=c["weights"])
    c["weights"].mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        r.loss.backward()


def test_the_example_learns():
    import os
    import sys

    sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples"))
    import policy_step

    gains = policy_step.train(32, 12)
    assert gains[-1] > gains[0] + 0.2, gains


# ------------------------------------------------------------- sums of any length

def act8_product(x8, dy):
    want = torch.zeros(x8.width, dy.shape[1], dtype=torch.float64, device="cuda")
    for t in range(0, len(dy), 16384):
        part = ops.Act8(x8.q[t:t + 16384], x8.scale[t:t + 16384], x8.width)
        want += ops.act8_unpack(part, F32).double().t() @ dy[t:t + 16384].double()
    return want


# Values of one sign, so that whatever a long sum loses shows in the mean; enough tiles that CTAs sum whole ones. Rounding
# to the nearest is unbiased: the mean of K N of them, each at most EPS, lies within six deviations.

def test_act8_wgrad_long_sums_in_f16():
    g = gen(21)
    T, K, N = 131072, 4096, 1280
    positive = lambda n, scale: (0.5 + torch.rand(T, n, generator=g, device="cuda")) * scale  # noqa: E731
    x8, dy = ops.act8_pack(positive(K, 1.0)), positive(N, 1.5 * 2.0 ** -7).to(F16)
    dw, _ = ops.act8_wgrad(x8, dy, dtype=F16)  # about 1536, where places are 1 and values spread over 10
    off = dw.double() / act8_product(x8, dy) - 1
    # and a run's bias: at most 3.84e-6, a 64th of the least that the rounding can move a value by
    assert abs(float(off.mean())) < 6 * EPS[F16] / math.sqrt(3 * K * N) + 3.84e-6
    assert float(off.abs().max()) < EPS[F16] + 1e-5
    # what is rounded is the 32-bit result
    assert torch.equal(dw, ops.act8_wgrad(x8, dy)[0].to(F16))


def test_act8_wgrad_long_sums_in_bf16():
    g = gen(22)
    T, K, N = 131072, 4096, 2560
    positive = lambda n: 0.5 + torch.rand(T, n, generator=g, device="cuda")  # noqa: E731
    octave = torch.linspace(0, 1, K, device="cuda").exp2()  # results over all places of a power of two
    x8, dy = ops.act8_pack(positive(K) * octave), positive(N).to(BF16)
    dw, _ = ops.act8_wgrad(x8, dy, dtype=BF16)
    off = dw.double() / act8_product(x8, dy) - 1
    # a run's bias: 1024 products, each half a last place of a sum that grows to the result (u of the result)
    assert abs(float(off.mean())) < 6 * EPS[BF16] / math.sqrt(3 * K * N) + 1024 * U
    assert float(off.abs().max()) < EPS[BF16] + 1e-4


# --------------------------------------------------------------------- long gates

@pytest.mark.parametrize("T", [1, 2, 3, 100])
@pytest.mark.parametrize("D", [40, 300, 5000])
def test_block_norm_one_gate_for_any_number_of_rows(T, D):
    c = norm_case(T, D, F32, "layer", per=0, seed=T)
    r, rest = ops.block_norm(**c), {k: v for k, v in c.items() if k not in ("x", "h")}
    dy, dn = randn(gen(1), T, D), randn(gen(2), T, D)
    want = [r.y, r.n, *ops.block_norm_backward(dy, dn, c["x"], c["h"], r.stats, **rest)]
    for per in (2 ** 63 - 1, 2 ** 63 - T, T + 1):
        s = ops.block_norm(**(c | {"rows_per_gate": per}))
        got = [s.y, s.n, *ops.block_norm_backward(dy, dn, c["x"], c["h"], s.stats, **(rest | {"rows_per_gate": per}))]
        for a, b in zip(want, got):
            assert torch.equal(a, b)


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_block_norm_one_gate_for_no_rows(kind):
    c = norm_case(4, 16, F32, kind, per=0) | {"rows_per_gate": None}
    c["x"], c["h"] = c["x"][:0], c["h"][:0]
    r = ops.block_norm(**c)
    assert r.y.shape == r.n.shape == (0, 16)
    g = ops.block_norm_backward(r.y, r.n, c["x"], c["h"], r.stats, **{k: v for k, v in c.items() if k not in ("x", "h")})
    assert g.dgate.shape == (1, 16) and not g.dgate.any()
    with pytest.raises(SolveError, match="0 x 16"):
        ops.block_norm(**(c | {"rows_per_gate": 4}))


# ------------------------------------------------------------------ waits that run out

@pytest.fixture
def wait_limit():
    """Sets the limit of the kernels' waits for their own copies and products, which complete all the same."""
    from warchest_b200 import _check, lib

    yield lambda ns: _check(lib().wc_debug_set_train_wait_limit(ns))
    torch.cuda.synchronize()
    _check(lib().wc_debug_set_train_wait_limit(0))


LIMITS = [1, 300, 1000, 3000, 10000]


def gives_up(wait_limit, call, sure=True):
    """call's results under short limits: each element NaN or, to the bit, what it is without; at the shortest there is NaN
    (`sure`: where not all that is waited for may have come before the first look). Then as before."""
    want = call()
    for ns in LIMITS:
        wait_limit(ns)
        got = call()
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert (b.isnan() | (a == b) | a.isnan()).all(), ns
        assert ns > LIMITS[0] or not sure or any(b.isnan().any() for b in got)
    wait_limit(0)
    for a, b in zip(want, call()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("T,K,N,dtype,out", [
    (40, 96, 64, BF16, F32), (150, 192, 96, BF16, F32), (150, 192, 96, F16, F16), (250, 300, 500, BF16, BF16), (1000, 64, 2000, F32, F32),
    (2500, 1000, 1000, BF16, BF16), (60000, 192, 96, BF16, F32), (30000, 320, 200, F16, F16), (20000, 512, 336, F32, F32)])
def test_act8_wgrad_waits_that_run_out(wait_limit, T, K, N, dtype, out):
    g = gen(31)
    x8, dy = ops.act8_pack(randn(g, T, K, dtype=BF16)), randn(g, T, N, dtype=dtype)
    gives_up(wait_limit, lambda: ops.act8_wgrad(x8, dy, dtype=out))


@pytest.mark.parametrize("T,D,dtype,per,post,pre", [
    (3, 300, F32, 0, True, True), (500, 1000, BF16, 0, True, True), (2000, 2048, F16, 37, True, True), (1500, 1001, BF16, None, False, True),
    (3000, 4096, BF16, 0, True, False), (700, 4095, F32, 1, False, False),
    # (more than the caches hold: copies take longer than a row)
    (40000, 4096, BF16, 0, True, True), (40000, 2047, F32, None, False, False)])
def test_block_norm_backward_waits_that_run_out(wait_limit, T, D, dtype, per, post, pre):
    c = norm_case(T, D, dtype, "layer", post, pre, per)
    r, rest = ops.block_norm(**c), {k: v for k, v in c.items() if k not in ("x", "h")}
    dy, dn = randn(gen(1), T, D, dtype=dtype), randn(gen(2), T, D, dtype=dtype) if pre else None
    gives_up(wait_limit, lambda: [g for g in ops.block_norm_backward(dy, dn, c["x"], c["h"], r.stats, **rest) if g is not None],
             sure=T * D > 1 << 26)


@pytest.mark.parametrize("T,V,dtype,legal", [
    (5, 1025, F32, None), (700, 2001, F16, 0.4), (600, 9000, BF16, None), (2000, 16384, BF16, None), (300, 40000, F32, 0.5), (500, 50001, BF16, None),
    (300, 131072, BF16, None)])
def test_policy_waits_that_run_out(wait_limit, T, V, dtype, legal):
    c = policy_case(T, V, dtype, seed=41, legal=legal)
    c["weights"][::7] = 0.0
    gives_up(wait_limit, lambda: ops.policy_loss(**c, **OPTIONS), sure=T * V > 1 << 24)


# ----------------------------------------------------------------- equal bits, layers

def test_equal_calls_give_the_same_bits():
    first = every_result(3)
    for _ in range(3):
        for a, b in zip(first, every_result(3)):
            assert torch.equal(a, b) and not (a.is_floating_point() and a.isnan().any())


def test_layers_refuse_second_derivatives():
    g = gen(14)
    x, w = randn(g, 20, 40).requires_grad_(), randn(g, 40, 30).requires_grad_()
    y = layers.gelu8(layers.linear8(layers.block_norm(x, x.detach(), pre=torch.ones(40, device="cuda"))[1], w))
    want = torch.autograd.grad(y.sum(), (x, w), retain_graph=True)
    got = torch.autograd.grad(y.sum(), (x, w), create_graph=True)
    for a, b in zip(want, got):
        assert torch.equal(a, b)
        with pytest.raises(SolveError, match="second derivative"):
            torch.autograd.grad(b.square().sum() + w.sum(), w, retain_graph=True)


@pytest.mark.parametrize("V", [16, 600, 3000, 40000])
def test_policy_kl_that_is_only_watched(V):
    """With kl_coef 0 the loss and the gradient are those without a reference, however far off it is."""
    c = policy_case(6, V, F32, seed=15)
    c["ref_logp"] = c["ref_logp"] + torch.tensor([0.0, 50.0, 87.0, 95.0, 200.0, 1e6], device="cuda")
    options = OPTIONS | {"kl_coef": 0.0}
    r, s = ops.policy_loss(**c, **options), ops.policy_loss(**(c | {"ref_logp": None}), **options)
    assert r.loss.isfinite() and torch.equal(r.loss, s.loss) and torch.equal(r.row_loss, s.row_loss) and torch.equal(r.dlogits, s.dlogits)
    assert (r.kl[3:] == math.inf).all() and r.kl[:2].isfinite().all()


def test_policy_results_are_the_users_own():
    """They can be changed in place, and hold no more memory than they are."""
    c = policy_case(40, 60, F32, seed=16)
    z = c["logits"].clone().requires_grad_()
    r = layers.policy_loss(z, c["actions"], c["old_logp"], c["advantages"], weights=c["weights"])
    s = ops.policy_loss(c["logits"], c["actions"], c["old_logp"], c["advantages"], weights=c["weights"])
    want, row = s.loss.clone(), s.row_loss.clone()
    r.loss.div_(4)
    r.row_loss.mul_(2)
    s.loss.div_(4)
    s.row_loss.mul_(2)
    assert torch.equal(r.loss, want / 4) and torch.equal(s.loss, want / 4) and torch.equal(r.row_loss, 2 * row) and torch.equal(s.row_loss, 2 * row)
    r.loss.backward()
    near(z.grad, s.dlogits.double() / 4, 1e-7, "dlogits")
    assert s.loss.untyped_storage().nbytes() == 4 and s.logp.untyped_storage().nbytes() == 4 * 4 * 40


@pytest.mark.parametrize("T,D", [(40, 96), (40, 97), (50, 1000), (30, 5000)])
def test_block_norm_gradients_one_at_a_time(T, D):
    c = norm_case(T, D, BF16, "layer", per=7)
    r, rest = ops.block_norm(**c), {k: v for k, v in c.items() if k not in ("x", "h")}
    dy, dn = randn(gen(1), T, D, dtype=BF16), randn(gen(2), T, D, dtype=BF16)
    full = ops.block_norm_backward(dy, dn, c["x"], c["h"], r.stats, **rest)
    for i in range(7):
        some = ops.block_norm_backward(dy, dn, c["x"], c["h"], r.stats, **rest, want=[j == i for j in range(7)])
        assert torch.equal(some[i], full[i]) and all(some[j] is None for j in range(7) if j != i)
    with pytest.raises(SolveError, match="seven"):
        ops.block_norm_backward(dy, dn, c["x"], c["h"], r.stats, **rest, want=(True,))


# ---------------------------------------------- widths, strides and lengths between the others

def strided(v, ld, skip, fill=math.nan):
    """v's values in rows that are `ld` apart and start `skip` entries into theirs."""
    room = torch.full((len(v), ld + skip), fill, dtype=v.dtype, device="cuda")
    room[:, skip:skip + v.shape[1]] = v
    return room[:, skip:skip + v.shape[1]]


# rows that no cluster of CTAs can hold: from 213,000 entries of 32 bits on (170,400 with legal bytes), twice that of 16
@pytest.mark.parametrize("T,V,dtype,legal", [(3, 220000, F32, None), (2, 180001, F32, 0.3), (2, 430001, BF16, None), (3, 350003, F16, 0.4)])
def test_policy_loss_of_the_longest_rows(T, V, dtype, legal):
    c = policy_case(T, V, dtype, seed=17, legal=legal)
    check_policy(c, OPTIONS, ops.policy_loss(**c, **OPTIONS))
    wide = c | {"logits": strided(c["logits"], V + 3, 1), "actions": c["actions"].to(torch.int32)}
    if legal is not None:
        wide["legal"] = strided(c["legal"].to(torch.uint8) * 4, V + 5, 2, fill=1)
    check_policy(wide, OPTIONS | {"entropy_coef": 0.0}, ops.policy_loss(**wide, **(OPTIONS | {"entropy_coef": 0.0})))


def test_policy_longest_rows_that_count_for_nothing():
    V = 180000
    c = policy_case(7, V, F32, seed=18, legal=0.5)
    c["legal"][0] = False
    c["legal"][1, c["actions"][1]] = False
    c["actions"][2], c["weights"][3] = V, 0.0
    c["logits"][3] = math.nan
    c["logits"][4] = torch.where(torch.arange(V, device="cuda") == c["actions"][4], c["logits"][4], -math.inf)
    c["logits"][5] = torch.finfo(F32).min
    c["logits"][5, c["actions"][5]] = 0.5
    c["old_logp"][5], c["ref_logp"][5] = -0.1, -0.2
    r = ops.policy_loss(**c, **OPTIONS)
    check_policy(c, OPTIONS, r)
    assert (r.row_loss[:4] == 0).all() and (r.dlogits[:4] == 0).all() and (r.logp[4:6] == 0).all() and r.loss.isfinite()
    c["logits"][6, 5], c["legal"][6, 5] = math.nan, True
    r = ops.policy_loss(**c, **OPTIONS)
    assert r.row_loss[6].isnan() and r.row_loss[:6].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("D", [9, 16, 20, 24, 37, 60, 130, 201, 255, 500])
def test_block_norm_widths_between(D, kind, dtype):
    for i, (post, pre, per) in enumerate(((True, True, 0), (True, False, 37), (False, True, None))):
        check_norm(norm_case(75, D, dtype, kind, post, pre, per, seed=D + i))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [24, 33, 96, 97, 520, 1111, 4099])
def test_block_norm_packs_16_bit_outputs(D, dtype):
    """The 8 bits are those of n before it is rounded."""
    c = norm_case(20, D, dtype, "layer", per=7)
    r = ops.block_norm(**c, pack=True)
    _, n = norm_plain(c, **{k: double(c[k]) for k in ("x", "h", "gate", "post", "pre")})
    kept = ops.act8_unpack(r.n8, F32).double()
    unit = (r.n8.scale.double() - 127).exp2().repeat_interleave(32, 1)[:, :D]
    # half a unit and what a normalised value is off
    assert ((kept - n.detach()).abs() <= unit * 0.5 + 64 * U * (1 + n.detach().abs().amax(1, keepdim=True))).all()
    near(r.n, n.detach(), 64 * U * (1 + n.detach().abs().amax(1, keepdim=True)), "n")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,ld,skip", [(24, 25, 1), (96, 97, 0), (96, 104, 8), (200, 203, 3), (333, 336, 3), (1000, 1003, 1), (4097, 4100, 1)])
def test_block_norm_strides_of_every_matrix(D, ld, skip, dtype):
    c = norm_case(40, D, dtype, "layer", per=9, seed=4)
    v = c | {k: strided(c[k], ld, skip) for k in ("x", "h")}
    leaves = {k: double(c[k]) for k in ("x", "h", "gate", "post", "pre")}
    y, n = norm_plain(c, **leaves)
    r = ops.block_norm(**v)
    at = lambda w: 64 * U * (1 + w.detach().abs().amax(1, keepdim=True))  # noqa: E731
    near(r.y, y.detach(), at(y), "y")
    near(r.n, n.detach(), at(n), "n")
    dy, dn = randn(gen(5), 40, D, dtype=dtype), randn(gen(6), 40, D, dtype=dtype)
    g = ops.block_norm_backward(strided(dy, ld, skip), strided(dn, ld + 1, skip), v["x"], v["h"], r.stats,
                                **{k: w for k, w in c.items() if k not in ("x", "h")})
    ((y * dy.double()).sum() + (n * dn.double()).sum()).backward()
    # as check_norm has them
    for name, t in zip(("dx", "dh", "dgate"), ("x", "h", "gate")):
        want = leaves[t].grad
        near(getattr(g, name), want, 128 * U * (1 + want.abs().amax(1, keepdim=True)) * (3 if name == "dgate" else 1), name)
    for name, t in zip(("dpost", "dpost_bias", "dpre", "dpre_bias"), (*leaves["post"], *leaves["pre"])):
        near(getattr(g, name), t.grad, 128 * U * math.sqrt(40) * 4 * (1 + t.grad.abs()), name)


def check_gelu8(z, b, da):
    a, z8 = ops.gelu8(z, b)
    s = z.float() + b if b is not None else z.float()
    near(a, gelu_plain(s.double()), 96 * U * s.double().abs() * torch.sigmoid(1.6 * s.double()), "a")
    q, scale = packed(s)
    assert torch.equal(z8.q.double(), q) and torch.equal(z8.scale.long(), scale)
    v = ops.act8_unpack(z8, F32).double().requires_grad_()
    gelu_plain(v).backward(da.double())
    dz, db = ops.gelu8_backward(da, z8)
    near(dz, v.grad, 128 * U * da.double().abs(), "dz")
    near(db, v.grad.sum(0), 128 * U * da.double().abs().sum(0), "dbias")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,D", [(40, 33), (300, 63), (7, 161), (50, 31), (3, 8), (1, 4099)])
def test_gelu8_widths_between(T, D, dtype):
    g = gen(T + D)
    check_gelu8(randn(g, T, D, dtype=dtype, scale=2.0), randn(g, D), randn(g, T, D, dtype=dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,ld,skip", [(8, 9, 0), (40, 43, 3), (64, 65, 1), (96, 104, 8), (96, 97, 0), (161, 168, 5), (256, 257, 1), (2048, 2051, 3)])
def test_act8_and_gelu8_strides_and_addresses(D, ld, skip, dtype):
    g = gen(D + ld)
    x, da = randn(g, 30, D, dtype=dtype, scale=2.0), randn(g, 30, D, dtype=dtype)
    p = ops.act8_pack(strided(x, ld, skip))
    q, scale = packed(x)
    assert torch.equal(p.q.double(), q) and torch.equal(p.scale.long(), scale)
    for bias in (None, randn(g, D), randn(g, D + 1)[1:]):
        check_gelu8(strided(x, ld, skip), bias, strided(da, ld + 2, skip))


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("ld,skip", [(104, 8), (97, 0), (99, 3)])
def test_act8_wgrad_strides_of_every_type(ld, skip, dtype):
    g = gen(7)
    x8, dy = ops.act8_pack(randn(g, 500, 200, dtype=BF16)), randn(g, 500, 96, dtype=dtype)
    for a, b in zip(ops.act8_wgrad(x8, dy), ops.act8_wgrad(x8, strided(dy, ld, skip))):
        assert torch.equal(a, b)


def test_backward_passes_past_32_bits():
    """Matrices of more than 2^31 elements: the last rows' results are as they are by themselves."""
    T, D = 140000, 16384
    x = torch.zeros(T, D, dtype=BF16, device="cuda")
    x[-3:] = randn(gen(1), 3, D, dtype=BF16)
    tail, one = x[-3:].clone(), torch.ones(D, device="cuda")
    a, z8 = ops.gelu8(x)
    b, y8 = ops.gelu8(tail)
    assert torch.equal(a[-3:], b) and torch.equal(z8.q[-3:], y8.q) and torch.equal(z8.scale[-3:], y8.scale)
    del a
    dz, db = ops.gelu8_backward(x, z8)
    dw, dc = ops.gelu8_backward(tail, y8)
    assert torch.equal(dz[-3:], dw)
    near(db, dc.double(), 4 * U * dw.double().abs().sum(0), "dbias")  # (the other rows add zeros)
    del dz, z8
    for width in (D, 4096, 96):
        rows = T * D // width
        v, w = x.view(-1)[:rows * width].view(rows, width), tail.view(-1)[-3 * width:].view(3, width)
        v[-3:] = w
        s, t = (ops.block_norm(u, u, post=one[:width], kind="rms") for u in (v, w))
        assert torch.equal(s.y[-3:], t.y) and torch.equal(s.stats[-3:], t.stats)
        big = ops.block_norm_backward(v, None, v, v, s.stats, post=one[:width], kind="rms")
        small = ops.block_norm_backward(w, None, w, w, t.stats, post=one[:width], kind="rms")
        assert torch.equal(big.dx[-3:], small.dx) and torch.equal(big.dh[-3:], small.dh)
        v[:-3] = 0
        del s, big


@pytest.mark.parametrize("T,V,dtype", [(300, 70001, BF16), (2000, 30000, F32), (33000, 18000, F16)])
def test_policy_loss_sums_clusters_rows_in_an_order_of_the_sizes_alone(T, V, dtype):
    """Runs of 32768 rows, 1024 chains each, joined by halves: to the bit, where the terms cancel to their last places."""
    g = gen(19)
    l = lambda: -math.log(V) + randn(g, T, scale=0.3)  # noqa: E731
    c = {"logits": randn(g, T, V, dtype=dtype, scale=0.1), "actions": torch.randint(0, V, (T,), generator=g, device="cuda"),
         "advantages": randn(g, T), "old_logp": l(), "ref_logp": l()}
    row = ops.policy_loss(**c, **OPTIONS, want_grad=False).row_loss.cpu()
    w = torch.rand(T, generator=g, device="cuda").cpu()

    def total(sum_of):
        return sum_of((w * row).double())

    w[T - 2:] = 0.0
    for t in (T - 1, T - 2):  # two weights that cancel the rest: some 2^-48 of it is left
        w[t] = -float(total(torch.sum)) / float(row[t])

    def ordered(p):
        runs = torch.zeros(-(-T // 32768) * 32768, dtype=torch.float64)
        runs[:T] = p
        chains = torch.zeros(len(runs) // 32768, 1024, dtype=torch.float64)
        for part in runs.view(-1, 32, 1024).unbind(1):
            chains = chains + part
        tree = lambda v: v if v.shape[-1] == 1 else tree(v[..., :v.shape[-1] // 2] + v[..., v.shape[-1] // 2:])  # noqa: E731
        runs = tree(tree(chains.view(-1, 32, 32))[..., 0].view(-1, 32))[:, 0]
        return tree(torch.nn.functional.pad(runs, (0, 32 - len(runs))))[0] if len(runs) > 1 else runs[0]

    got = ops.policy_loss(**c, weights=w.cuda(), **OPTIONS).loss
    assert abs(float(got)) < 1e-11 * float((w * row).double().abs().sum())
    assert float(got) == float(total(ordered).float())


def test_every_operator_inside_a_cuda_graph():
    """Every kernel family's launch, captured once and replayed on other inputs."""
    short, long = policy_case(64, 512, F32, seed=51, legal=0.5), policy_case(20, 40000, BF16, seed=52)
    longest = policy_case(2, 220000, F32, seed=53)
    narrow, wide, widest = (norm_case(40, D, BF16, "layer", per=0, seed=D) for D in (96, 1000, 5000))
    z, da = randn(gen(1), 500, 192, dtype=BF16), randn(gen(2), 500, 96, dtype=F16)
    inputs = [short["logits"], long["logits"], longest["logits"], narrow["x"], wide["x"], widest["x"], z, da]

    def step():
        out = []
        for c in (short, long, longest):
            out += ops.policy_loss(**c, **OPTIONS)
        for c in (narrow, wide, widest):
            r = ops.block_norm(**c, pack=True)
            out += [r.y, r.n, r.n8.q, *ops.block_norm_backward(r.y, r.n, c["x"], c["h"], r.stats, **{k: v for k, v in c.items() if k not in ("x", "h")})]
        a, z8 = ops.gelu8(z)
        return out + [a, z8.q, *ops.gelu8_backward(a, z8), *ops.act8_wgrad(ops.act8_pack(z), da), ops.act8_unpack(z8)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for t in inputs:
        t.copy_(t.flip(0))
    graph.replay()
    for a, b in zip(got, step()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("T,V,dtype,legal", [(20, 290000, F32, None), (12, 430001, F16, None), (12, 430001, BF16, 0.9)])
def test_policy_longest_rows_of_few_large_entries(T, V, dtype, legal):
    """Most entries are small beside the sum, and many."""
    c = policy_case(T, V, dtype, seed=20, legal=legal, scale=4.0)
    check_policy(c, OPTIONS, ops.policy_loss(**c, **OPTIONS))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [16, 513, 1000, 3000, 40000, 350003])
def test_policy_what_lies_under_the_mask_does_not_count(V, dtype):
    c = policy_case(5, V, dtype, seed=23, legal=0.5)
    want = ops.policy_loss(**c, **OPTIONS)
    under = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dtype).max], device="cuda").to(dtype)
    hidden = torch.where(c["legal"], c["logits"], under[torch.arange(V, device="cuda") % 4])
    for a, b in zip(want, ops.policy_loss(**(c | {"logits": hidden}), **OPTIONS)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("T,K,N,dtype", [(5000, 37 * 256, 4 * 128, F16), (20000, 37 * 256, 4 * 256, BF16), (17000, 37 * 256, 8 * 256, BF16)])
def test_act8_wgrad_whole_tiles_of_several_runs(T, K, N, dtype):
    """As many tiles as CTAs, or twice that: none is shared, and each is summed up in the workspace."""
    from warchest_b200 import lib

    g = gen(24)
    x8, dy = ops.act8_pack(randn(g, T, K, dtype=BF16)), randn(g, T, N, dtype=dtype)
    kind, sizes = ops._TYPES[dtype], [T, K, N, N]
    need = lib().wc_act8_wgrad_workspace(ops._ACT8_WGRAD.pack(0, 0, 0, 0, 0, 0, *sizes, kind, kind))
    space = torch.full((need + 64,), 99, dtype=torch.uint8, device="cuda")
    dw = torch.empty(K, N, dtype=dtype, device="cuda")
    ops._call(lib().wc_act8_wgrad, 0, ops._ACT8_WGRAD.pack(x8.q.data_ptr(), x8.scale.data_ptr(), dy.data_ptr(), dw.data_ptr(), 0,
                                                           space.data_ptr(), *sizes, kind, kind))
    assert (space[need:] == 99).all()
    # relative to the whole: the result's rounding, and as for 32-bit results a run's bias and the runs' own sums
    want = act8_product(x8, dy)
    assert float((dw.double() - want).norm() / want.norm()) < EPS[dtype] / math.sqrt(3) + 1e-5
    if dtype == F16:
        assert torch.equal(dw, ops.act8_wgrad(x8, dy)[0].to(F16))
