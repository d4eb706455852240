"""The training operators over torch tensors (include/wc_b200.h, "training
operators"): a clipped policy loss with a KL term and its gradient, a residual
block's norms with its gate and residual scale, and activations kept in 8 bits
between the forward and the backward pass.

Tensors live on one CUDA device; matrices are [rows, width] with unit column
stride (any row stride) in float32, float16 or bfloat16, per-row and
per-channel vectors are contiguous float32 unless said otherwise. torch
supplies memory and the stream: a call enqueues its work on the device's
current stream and returns. Wrong arguments raise SolveError. train_layers
has the same operators as differentiable functions.
"""
from __future__ import annotations

import ctypes as C
from functools import lru_cache
from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import SolveError, _check, lib

BLOCK = 32  # values that share a unit in the 8-bit form
NORM_KINDS = {"layer": 0, "rms": 1}
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}

_VP, _I64, _F, _I = C.c_void_p, C.c_int64, C.c_float, C.c_int32


class _PolicyLossArgs(C.Structure):
    _fields_ = [(n, _VP) for n in ("logits", "legal", "actions", "old_logp", "advantages", "weights", "ref_logp",
                                   "upstream", "loss", "row_out", "dlogits", "workspace")] + \
               [(n, _I64) for n in ("rows", "width", "ld_logits", "ld_legal", "ld_dlogits")] + \
               [(n, _F) for n in ("clip_low", "clip_high", "kl_coef", "entropy_coef")] + \
               [("type", _I), ("action_bytes", _I)]


class _BlockNormArgs(C.Structure):
    _fields_ = [(n, _VP) for n in ("x", "h", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias", "y", "n",
                                   "n_q", "n_scale", "stats")] + \
               [(n, _I64) for n in ("rows", "width", "rows_per_gate", "ld_x", "ld_h", "ld_y", "ld_n")] + \
               [("residual_scale", _F), ("eps", _F), ("type", _I), ("kind", _I)]


class _BlockNormGrads(C.Structure):
    _fields_ = [(n, _VP) for n in ("dy", "dn", "dx", "dh", "dgate", "dpost_weight", "dpost_bias", "dpre_weight",
                                   "dpre_bias", "workspace")] + \
               [(n, _I64) for n in ("ld_dy", "ld_dn", "ld_dx", "ld_dh")]


class _Act8Args(C.Structure):
    _fields_ = [(n, _VP) for n in ("x", "bias", "q", "scale", "out", "dbias", "workspace")] + \
               [(n, _I64) for n in ("rows", "width", "ld_x", "ld_out")] + [("type", _I)]


class _Act8WgradArgs(C.Structure):
    _fields_ = [(n, _VP) for n in ("q", "scale", "dy", "dw", "db", "workspace")] + \
               [(n, _I64) for n in ("rows", "k", "n", "ld_dy")] + [("type", _I), ("out_type", _I)]


class PolicyLoss(NamedTuple):
    """loss: scalar; row_loss, logp, entropy, kl: [rows] float32; dlogits: like the logits, or None."""
    loss: torch.Tensor
    row_loss: torch.Tensor
    logp: torch.Tensor
    entropy: torch.Tensor
    kl: torch.Tensor
    dlogits: Optional[torch.Tensor]


class Act8(NamedTuple):
    """A matrix kept in 8 bits: q int8 [rows, 32 blocks], scale uint8 [rows, blocks], its width."""
    q: torch.Tensor
    scale: torch.Tensor
    width: int


class BlockNorm(NamedTuple):
    """y; n or None; n in 8 bits or None; stats [rows, 4] for the backward pass."""
    y: torch.Tensor
    n: Optional[torch.Tensor]
    n8: Optional[Act8]
    stats: torch.Tensor


class BlockNormGrads(NamedTuple):
    dx: torch.Tensor
    dh: torch.Tensor
    dgate: Optional[torch.Tensor]
    dpost: Optional[torch.Tensor]
    dpost_bias: Optional[torch.Tensor]
    dpre: Optional[torch.Tensor]
    dpre_bias: Optional[torch.Tensor]


Weight = Union[None, torch.Tensor, Tuple[torch.Tensor, Optional[torch.Tensor]]]


def _fail(what: str, why: str):
    raise SolveError(1, f"{what}: {why}")


def _matrix(what: str, name: str, t: torch.Tensor, like: Optional[torch.Tensor] = None) -> None:
    """A [rows, width] CUDA matrix with unit column stride; `like`'s shape, type and device if given."""
    if t.dtype not in _TYPES or t.dim() != 2 or not t.is_cuda:
        _fail(what, f"{name} must be a 2-d float32, float16 or bfloat16 CUDA tensor")
    if like is not None and (t.shape != like.shape or t.dtype != like.dtype or t.device != like.device):
        _fail(what, f"{name} must have the first matrix's shape, type and device")
    rows, width = t.shape
    if rows and width and ((t.stride(1) != 1 and width > 1) or (rows > 1 and t.stride(0) < width)):
        _fail(what, f"{name} must have unit column stride and rows that do not overlap")


def _vector(what: str, name: str, t: Optional[torch.Tensor], n: int, like: torch.Tensor) -> Optional[int]:
    if t is None:
        return None
    if t.dtype != torch.float32 or t.dim() != 1 or t.shape[0] != n or t.device != like.device or not t.is_contiguous():
        _fail(what, f"{name} must be {n} contiguous float32 values on {like.device}")
    return t.data_ptr()


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else max(1, t.shape[1])


def _call(fn, device: torch.device, *args) -> None:
    """The entry on the tensors' device and its current stream."""
    stream = torch.cuda.current_stream(device).cuda_stream
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            _check(fn(*args, stream))
    else:
        _check(fn(*args, stream))


# --------------------------------------------------------------- policy loss

@lru_cache(maxsize=256)
def _policy_workspace(rows: int, width: int) -> int:
    return lib().wc_policy_loss_workspace(rows, width)


def policy_loss(logits, actions, old_logp, advantages, *, weights=None, ref_logp=None, legal=None, clip_low=0.2,
                clip_high=0.2, kl_coef=0.0, entropy_coef=0.0, upstream=None, want_grad=True) -> PolicyLoss:
    """The clipped policy loss of [rows, width] logits, and its gradient.

    Per row: -min(ratio A, clip(ratio, 1 - clip_low, 1 + clip_high) A) +
    kl_coef (exp(r - l) - (r - l) - 1) - entropy_coef H, with l the
    log-probability of actions[row] (int64 or int32) among the entries that
    `legal` ([rows, width] bool or uint8) marks, ratio = exp(l - old_logp), r =
    ref_logp and H the entropy. The loss is their sum under `weights` (1 where
    None); the gradient is scaled by `upstream` (one float32 on the device).
    Rows of weight 0, with an action outside the width, or whose action is not
    a legal entry count for nothing, whatever their logits hold."""
    me = "policy_loss"
    _matrix(me, "logits", logits)
    rows, width = logits.shape
    if actions.dtype not in (torch.int64, torch.int32) or actions.dim() != 1 or actions.shape[0] != rows or \
            actions.device != logits.device or not actions.is_contiguous():
        _fail(me, f"actions must be {rows} contiguous int64 or int32 values on {logits.device}")
    old = _vector(me, "old_logp", old_logp, rows, logits)
    adv = _vector(me, "advantages", advantages, rows, logits)
    wts = _vector(me, "weights", weights, rows, logits)
    ref = _vector(me, "ref_logp", ref_logp, rows, logits)
    if old is None or adv is None:
        _fail(me, "old_logp and advantages are needed")
    if upstream is not None and (upstream.dtype != torch.float32 or upstream.numel() != 1 or
                                 upstream.device != logits.device):
        _fail(me, "upstream must be one float32 value on the logits' device")
    ld_legal = 0
    if legal is not None:
        if legal.dtype not in (torch.bool, torch.uint8) or legal.shape != logits.shape or legal.device != logits.device:
            _fail(me, "legal must be a bool or uint8 matrix of the logits' shape and device")
        if rows and width and ((legal.stride(1) != 1 and width > 1) or (rows > 1 and legal.stride(0) < width)):
            _fail(me, "legal must have unit column stride and rows that do not overlap")
        ld_legal = _ld(legal)
    device = logits.device
    space = (_policy_workspace(rows, width) + 15) // 16 * 4
    flat = torch.empty(space + 4 * rows + 1, dtype=torch.float32, device=device)
    scratch, out, loss = flat.split((space, 4 * rows, 1))  # the workspace first: it has to be aligned
    grad = torch.empty((rows, width), dtype=logits.dtype, device=device) if want_grad else None
    args = _PolicyLossArgs(
        logits.data_ptr(), legal.data_ptr() if legal is not None else None, actions.data_ptr(), old, adv, wts, ref,
        upstream.data_ptr() if upstream is not None else None, loss.data_ptr(), out.data_ptr(),
        grad.data_ptr() if want_grad else None, scratch.data_ptr(), rows, width, _ld(logits), ld_legal, max(1, width),
        clip_low, clip_high, kl_coef, entropy_coef, _TYPES[logits.dtype], actions.element_size())
    _call(lib().wc_policy_loss, device, C.byref(args))
    row_loss, logp, entropy, kl = out.view(4, rows).unbind(0)
    return PolicyLoss(loss[0], row_loss, logp, entropy, kl, grad)


# --------------------------------------------------------------- block norms

def _weight(what: str, name: str, w: Weight, like: torch.Tensor):
    bias = None
    if isinstance(w, tuple):
        w, bias = w
    n = like.shape[1]
    return _vector(what, name, w, n, like), _vector(what, name + " bias", bias, n, like)


def _norm_args(me, x, h, gate, rows_per_gate, residual_scale, post, pre, kind, eps):
    _matrix(me, "x", x)
    _matrix(me, "h", h, x)
    rows, width = x.shape
    if kind not in NORM_KINDS:
        _fail(me, "kind must be 'layer' or 'rms'")
    a = _BlockNormArgs(x=x.data_ptr(), h=h.data_ptr(), rows=rows, width=width, ld_x=_ld(x), ld_h=_ld(h),
                       residual_scale=residual_scale, eps=eps, type=_TYPES[x.dtype], kind=NORM_KINDS[kind])
    if gate is not None:
        per = rows_per_gate if rows_per_gate is not None else max(1, rows)
        if per < 1:
            _fail(me, "rows_per_gate below 1")
        if gate.dim() != 2 or tuple(gate.shape) != (-(-rows // per), width) or gate.dtype != x.dtype or \
                gate.device != x.device or not gate.is_contiguous():
            _fail(me, f"gate must be a contiguous {-(-rows // per)} x {width} matrix of x's type and device")
        a.gate, a.rows_per_gate = gate.data_ptr(), per
    a.post_weight, a.post_bias = _weight(me, "post", post, x)
    a.pre_weight, a.pre_bias = _weight(me, "pre", pre, x)
    return a


def block_norm(x, h, *, gate=None, rows_per_gate=None, residual_scale=1.0, post=None, pre=None, kind="layer", eps=1e-5,
               pack=False) -> BlockNorm:
    """y = residual_scale x + gate post(h) and n = pre(y) of a residual block.

    post and pre: a float32 weight or (weight, bias) of a LayerNorm (kind
    "layer") or the weight of an RMSNorm ("rms"); None leaves that norm out.
    gate: [ceil(rows / rows_per_gate), width] in x's type; rows_per_gate None
    means one gate row for all. pack also returns n in 8 bits."""
    me = "block_norm"
    a = _norm_args(me, x, h, gate, rows_per_gate, residual_scale, post, pre, kind, eps)
    rows, width = x.shape
    y = torch.empty((rows, width), dtype=x.dtype, device=x.device)
    stats = torch.empty((rows, 4), dtype=torch.float32, device=x.device)
    a.y, a.stats, a.ld_y, a.ld_n = y.data_ptr(), stats.data_ptr(), max(1, width), max(1, width)
    n = n8 = None
    if a.pre_weight is not None:
        n = torch.empty_like(y)
        a.n = n.data_ptr()
        if pack:
            n8 = _new_act8(x)
            a.n_q, a.n_scale = n8.q.data_ptr(), n8.scale.data_ptr()
    elif pack:
        _fail(me, "pack needs a pre norm")
    _call(lib().wc_block_norm, x.device, C.byref(a))
    return BlockNorm(y, n, n8, stats)


def block_norm_backward(dy, dn, x, h, stats, *, gate=None, rows_per_gate=None, residual_scale=1.0, post=None, pre=None,
                        kind="layer", eps=1e-5) -> BlockNormGrads:
    """Gradients of block_norm at its inputs and parameters from those at y and n (either may be None) and the
    stats that the forward pass returned."""
    me = "block_norm_backward"
    a = _norm_args(me, x, h, gate, rows_per_gate, residual_scale, post, pre, kind, eps)
    rows, width = x.shape
    if stats.dtype != torch.float32 or tuple(stats.shape) != (rows, 4) or stats.device != x.device or \
            not stats.is_contiguous():
        _fail(me, f"stats must be the forward's contiguous float32 {rows} x 4 matrix")
    a.stats = stats.data_ptr()
    g = _BlockNormGrads()
    for name, d in (("dy", dy), ("dn", dn)):
        if d is not None:
            _matrix(me, name, d, x)
            setattr(g, name, d.data_ptr())
            setattr(g, "ld_" + name, _ld(d))
    dx, dh = torch.empty((rows, width), dtype=x.dtype, device=x.device), torch.empty((rows, width), dtype=x.dtype, device=x.device)
    g.dx, g.dh, g.ld_dx, g.ld_dh = dx.data_ptr(), dh.data_ptr(), max(1, width), max(1, width)
    dgate = None
    if gate is not None:
        dgate = torch.empty_like(gate)
        g.dgate = dgate.data_ptr()
    flat = torch.empty((4, width), dtype=torch.float32, device=x.device)
    grads = [None] * 4
    for i, (name, there) in enumerate((("dpost_weight", a.post_weight), ("dpost_bias", a.post_bias),
                                       ("dpre_weight", a.pre_weight), ("dpre_bias", a.pre_bias))):
        if there is not None:
            grads[i] = flat[i]
            setattr(g, name, grads[i].data_ptr())
    scratch = torch.empty(max(16, lib().wc_block_norm_workspace(C.byref(a))), dtype=torch.uint8, device=x.device)
    g.workspace = scratch.data_ptr()
    _call(lib().wc_block_norm_backward, x.device, C.byref(a), C.byref(g))
    return BlockNormGrads(dx, dh, dgate, *grads)


# ------------------------------------------------------- activations in 8 bits

def _new_act8(like: torch.Tensor) -> Act8:
    rows, width = like.shape
    blocks = -(-width // BLOCK)
    return Act8(torch.empty((rows, blocks * BLOCK), dtype=torch.int8, device=like.device),
                torch.empty((rows, blocks), dtype=torch.uint8, device=like.device), width)


def _check_act8(what: str, a: Act8) -> None:
    blocks = -(-a.width // BLOCK)
    if a.q.dtype != torch.int8 or a.scale.dtype != torch.uint8 or not a.q.is_cuda or a.q.device != a.scale.device or \
            a.q.dim() != 2 or tuple(a.q.shape) != (a.scale.shape[0], blocks * BLOCK) or a.scale.dim() != 2 or \
            a.scale.shape[1] != blocks or not a.q.is_contiguous() or not a.scale.is_contiguous():
        _fail(what, "not an 8-bit matrix: q int8 [rows, 32 blocks] and scale uint8 [rows, blocks], contiguous")


def act8_pack(x) -> Act8:
    """x in 8 bits: whole numbers of at most 127 in a power-of-two unit per block of 32 values of a row."""
    _matrix("act8_pack", "x", x)
    p = _new_act8(x)
    a = _Act8Args(x=x.data_ptr(), q=p.q.data_ptr(), scale=p.scale.data_ptr(), rows=x.shape[0], width=x.shape[1],
                  ld_x=_ld(x), type=_TYPES[x.dtype])
    _call(lib().wc_act8_pack, x.device, C.byref(a))
    return p


def act8_unpack(p: Act8, dtype=torch.bfloat16) -> torch.Tensor:
    """The values an 8-bit matrix stands for (exact in bfloat16 and float32)."""
    _check_act8("act8_unpack", p)
    if dtype not in _TYPES:
        _fail("act8_unpack", "dtype must be float32, float16 or bfloat16")
    rows = p.q.shape[0]
    out = torch.empty((rows, p.width), dtype=dtype, device=p.q.device)
    a = _Act8Args(q=p.q.data_ptr(), scale=p.scale.data_ptr(), out=out.data_ptr(), rows=rows, width=p.width,
                  ld_out=max(1, p.width), type=_TYPES[dtype])
    _call(lib().wc_act8_unpack, p.q.device, C.byref(a))
    return out


def gelu8(z, bias=None) -> Tuple[torch.Tensor, Act8]:
    """GELU (tanh form) of z + bias, and z + bias in 8 bits for gelu8_backward."""
    _matrix("gelu8", "z", z)
    p = _new_act8(z)
    out = torch.empty(z.shape, dtype=z.dtype, device=z.device)
    a = _Act8Args(x=z.data_ptr(), bias=_vector("gelu8", "bias", bias, z.shape[1], z), q=p.q.data_ptr(),
                  scale=p.scale.data_ptr(), out=out.data_ptr(), rows=z.shape[0], width=z.shape[1], ld_x=_ld(z),
                  ld_out=max(1, z.shape[1]), type=_TYPES[z.dtype])
    _call(lib().wc_gelu8, z.device, C.byref(a))
    return out, p


@lru_cache(maxsize=256)
def _gelu8_workspace(rows: int, width: int) -> int:
    return lib().wc_gelu8_workspace(rows, width)


def gelu8_backward(da, z8: Act8, want_bias=True):
    """(dz, dbias): the gradients at gelu8's input and bias (float32, or None) from the one at its output."""
    me = "gelu8_backward"
    _matrix(me, "da", da)
    _check_act8(me, z8)
    rows, width = da.shape
    if z8.width != width or z8.q.shape[0] != rows or z8.q.device != da.device:
        _fail(me, "da and the 8-bit activations differ in shape or device")
    dz = torch.empty((rows, width), dtype=da.dtype, device=da.device)
    a = _Act8Args(x=da.data_ptr(), q=z8.q.data_ptr(), scale=z8.scale.data_ptr(), out=dz.data_ptr(), rows=rows,
                  width=width, ld_x=_ld(da), ld_out=max(1, width), type=_TYPES[da.dtype])
    dbias = None
    if want_bias:
        dbias = torch.empty(width, dtype=torch.float32, device=da.device)
        scratch = torch.empty(max(16, _gelu8_workspace(rows, width)), dtype=torch.uint8, device=da.device)
        a.dbias, a.workspace = dbias.data_ptr(), scratch.data_ptr()
    _call(lib().wc_gelu8_backward, da.device, C.byref(a))
    return dz, dbias


def act8_wgrad(x8: Act8, dy, *, dtype=torch.float32, want_bias=True):
    """(dw, db): x8^T dy as [width of x8, width of dy] in `dtype`, and dy's column sums (float32, or None): the
    gradients of a linear layer's weight [in, out] and bias from its input as kept in 8 bits."""
    me = "act8_wgrad"
    _matrix(me, "dy", dy)
    _check_act8(me, x8)
    rows, n = dy.shape
    if x8.q.shape[0] != rows or x8.q.device != dy.device:
        _fail(me, "dy and the 8-bit activations differ in rows or device")
    if dtype not in _TYPES:
        _fail(me, "dtype must be float32, float16 or bfloat16")
    dw = torch.empty((x8.width, n), dtype=dtype, device=dy.device)
    db = torch.empty(n, dtype=torch.float32, device=dy.device) if want_bias else None
    a = _Act8WgradArgs(x8.q.data_ptr(), x8.scale.data_ptr(), dy.data_ptr(), dw.data_ptr(),
                       db.data_ptr() if want_bias else None, None, rows, x8.width, n, _ld(dy), _TYPES[dy.dtype],
                       _TYPES[dtype])
    scratch = torch.empty(max(16, lib().wc_act8_wgrad_workspace(C.byref(a))), dtype=torch.uint8, device=dy.device)
    a.workspace = scratch.data_ptr()
    _call(lib().wc_act8_wgrad, dy.device, C.byref(a))
    return dw, db
