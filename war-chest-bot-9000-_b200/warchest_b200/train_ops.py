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

import struct
from functools import lru_cache
from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import SolveError, _check, lib

BLOCK = 32  # values that share a unit in the 8-bit form
NORM_KINDS = {"layer": 0, "rms": 1}
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}

# The argument structures of include/wc_b200.h, field by field: pointers, 64-bit sizes, floats, 32-bit numbers. (Packed
# bytes: building a ctypes structure takes longer than the smallest kernels.)
_POLICY_LOSS = struct.Struct("@12Q5q4f2i")
_BLOCK_NORM = struct.Struct("@12Q7q2f2i")
_BLOCK_NORM_GRADS = struct.Struct("@10Q4q")
_ACT8 = struct.Struct("@7Q4qi4x")
_ACT8_WGRAD = struct.Struct("@6Q4q2i")


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
    dx: Optional[torch.Tensor]
    dh: Optional[torch.Tensor]
    dgate: Optional[torch.Tensor]
    dpost: Optional[torch.Tensor]
    dpost_bias: Optional[torch.Tensor]
    dpre: Optional[torch.Tensor]
    dpre_bias: Optional[torch.Tensor]


Weight = Union[None, torch.Tensor, Tuple[torch.Tensor, Optional[torch.Tensor]]]


def _fail(what: str, why: str):
    raise SolveError(1, f"{what}: {why}")


def _matrix(what: str, name: str, t: torch.Tensor, like: Optional[torch.Tensor] = None) -> int:
    """The row stride of a [rows, width] CUDA matrix with unit column stride, of `like`'s shape, type and device if
    given."""
    if t.dtype not in _TYPES or t.dim() != 2 or not t.is_cuda:
        _fail(what, f"{name} must be a 2-d float32, float16 or bfloat16 CUDA tensor")
    if like is not None and (t.shape != like.shape or t.dtype != like.dtype or t.device != like.device):
        _fail(what, f"{name} must have the first matrix's shape, type and device")
    return _row_stride(what, name, t)


def _row_stride(what: str, name: str, t: torch.Tensor) -> int:
    rows, width = t.shape
    if rows > 1:
        ld, step = t.stride()
        if width and (ld < width or (step != 1 and width > 1)):
            _fail(what, f"{name} must have unit column stride and rows that do not overlap")
        return ld if width else 1
    if width > 1 and t.stride(1) != 1 and rows:
        _fail(what, f"{name} must have unit column stride and rows that do not overlap")
    return max(1, width)


def _vector(what: str, name: str, t: Optional[torch.Tensor], n: int, like: torch.Tensor) -> int:
    if t is None:
        return 0
    if t.dtype != torch.float32 or t.dim() != 1 or t.numel() != n or t.get_device() != like.get_device() or not t.is_contiguous():
        _fail(what, f"{name} must be {n} contiguous float32 values on {like.device}")
    return t.data_ptr()


# (Tensor.new_empty takes half as long as torch.empty, which is given a type and a device to look up.)
def _scratch(n: int, like: torch.Tensor) -> torch.Tensor:
    return like.new_empty(max(16, n), dtype=torch.uint8)


def _call(fn, index: int, *args) -> None:
    """The entry on the current stream of the tensors' device."""
    stream = torch._C._cuda_getCurrentRawStream(index)
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(index):
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
    ld = _matrix(me, "logits", logits)
    rows, width = logits.shape
    index = logits.get_device()
    if actions.dtype not in (torch.int64, torch.int32) or actions.dim() != 1 or actions.numel() != rows or \
            actions.get_device() != index or not actions.is_contiguous():
        _fail(me, f"actions must be {rows} contiguous int64 or int32 values on {logits.device}")
    if old_logp is None or advantages is None:
        _fail(me, "old_logp and advantages are needed")
    old = _vector(me, "old_logp", old_logp, rows, logits)
    adv = _vector(me, "advantages", advantages, rows, logits)
    wts = _vector(me, "weights", weights, rows, logits)
    ref = _vector(me, "ref_logp", ref_logp, rows, logits)
    up = on = ld_legal = 0
    if upstream is not None:
        if upstream.dtype != torch.float32 or upstream.numel() != 1 or upstream.get_device() != index:
            _fail(me, "upstream must be one float32 value on the logits' device")
        up = upstream.data_ptr()
    if legal is not None:
        if legal.dtype not in (torch.bool, torch.uint8) or legal.shape != logits.shape or legal.get_device() != index:
            _fail(me, "legal must be a bool or uint8 matrix of the logits' shape and device")
        on, ld_legal = legal.data_ptr(), _row_stride(me, "legal", legal)
    scratch = _scratch(_policy_workspace(rows, width), logits)
    loss, per_row = old_logp.new_empty(()), old_logp.new_empty((4, rows))
    grad = logits.new_empty(rows, width) if want_grad else None
    _call(lib().wc_policy_loss, index, _POLICY_LOSS.pack(
        logits.data_ptr(), on, actions.data_ptr(), old, adv, wts, ref, up, loss.data_ptr(), per_row.data_ptr(),
        grad.data_ptr() if want_grad else 0, scratch.data_ptr(), rows, width, ld, ld_legal, max(1, width), clip_low, clip_high,
        kl_coef, entropy_coef, _TYPES[logits.dtype], actions.element_size()))
    return PolicyLoss(loss, *per_row.unbind(), grad)


# --------------------------------------------------------------- block norms

def _weight(what: str, name: str, w: Weight, like: torch.Tensor):
    bias = None
    if isinstance(w, tuple):
        w, bias = w
    n = like.shape[1]
    return _vector(what, name, w, n, like), _vector(what, name + " bias", bias, n, like)


def _norm_args(me, x, h, gate, rows_per_gate, residual_scale, post, pre, kind, eps):
    """The packed arguments, given y, n, n_q, n_scale, stats and n's and y's row stride; and whether there is a post
    weight and bias, a pre weight and bias."""
    ld_x, ld_h = _matrix(me, "x", x), _matrix(me, "h", h, x)
    rows, width = x.shape
    if kind not in NORM_KINDS:
        _fail(me, "kind must be 'layer' or 'rms'")
    per = gp = 0
    if gate is not None:
        per = rows_per_gate if rows_per_gate is not None else max(1, rows)
        if per < 1:
            _fail(me, "rows_per_gate below 1")
        groups = -(-rows // per) if rows_per_gate is not None else 1
        if gate.shape != (groups, width) or gate.dtype != x.dtype or gate.get_device() != x.get_device() or \
                not gate.is_contiguous():
            _fail(me, f"gate must be a contiguous {groups} x {width} matrix of x's type and device")
        gp = gate.data_ptr()
    there = _weight(me, "post", post, x) + _weight(me, "pre", pre, x)

    def pack(y, n, n_q, n_scale, stats):
        ld = max(1, width)
        return _BLOCK_NORM.pack(x.data_ptr(), h.data_ptr(), gp, *there, y, n, n_q, n_scale, stats, rows, width, per, ld_x, ld_h,
                                ld, ld, residual_scale, eps, _TYPES[x.dtype], NORM_KINDS[kind])

    return pack, there


def block_norm(x, h, *, gate=None, rows_per_gate=None, residual_scale=1.0, post=None, pre=None, kind="layer", eps=1e-5,
               pack=False) -> BlockNorm:
    """y = residual_scale x + gate post(h) and n = pre(y) of a residual block.

    post and pre: a float32 weight or (weight, bias) of a LayerNorm (kind
    "layer") or the weight of an RMSNorm ("rms"); None leaves that norm out.
    gate: [ceil(rows / rows_per_gate), width] in x's type; rows_per_gate None
    means one gate row for all. pack also returns n in 8 bits."""
    me = "block_norm"
    args, there = _norm_args(me, x, h, gate, rows_per_gate, residual_scale, post, pre, kind, eps)
    rows, width = x.shape
    y = x.new_empty(rows, width)
    stats = x.new_empty((rows, 4), dtype=torch.float32)
    n = n8 = None
    if there[2]:
        n = x.new_empty(rows, width)
        if pack:
            n8 = _new_act8(x)
    elif pack:
        _fail(me, "pack needs a pre norm")
    _call(lib().wc_block_norm, x.get_device(), args(y.data_ptr(), n.data_ptr() if n is not None else 0,
                                                    n8.q.data_ptr() if n8 else 0, n8.scale.data_ptr() if n8 else 0,
                                                    stats.data_ptr()))
    return BlockNorm(y, n, n8, stats)


def block_norm_backward(dy, dn, x, h, stats, *, gate=None, rows_per_gate=None, residual_scale=1.0, post=None, pre=None,
                        kind="layer", eps=1e-5, want=(True,) * 7) -> BlockNormGrads:
    """Gradients of block_norm at its inputs and parameters from those at y and n (either may be None) and the
    stats that the forward pass returned. `want` says which of the seven are: the others are None and not formed."""
    me = "block_norm_backward"
    args, there = _norm_args(me, x, h, gate, rows_per_gate, residual_scale, post, pre, kind, eps)
    rows, width = x.shape
    if stats.dtype != torch.float32 or stats.shape != (rows, 4) or stats.get_device() != x.get_device() or \
            not stats.is_contiguous():
        _fail(me, f"stats must be the forward's contiguous float32 {rows} x 4 matrix")
    packed = args(0, 0, 0, 0, stats.data_ptr())
    ld_dy = _matrix(me, "dy", dy, x) if dy is not None else 0
    ld_dn = _matrix(me, "dn", dn, x) if dn is not None else 0
    if len(want) != 7:
        _fail(me, "want is seven truth values, one for each gradient")
    dx = x.new_empty(rows, width) if want[0] else None
    dh = x.new_empty(rows, width) if want[1] else None
    dgate = None if gate is None or not want[2] else torch.empty_like(gate) if rows else torch.zeros_like(gate)
    grads = [x.new_empty(width, dtype=torch.float32) if w and there_is else None for there_is, w in zip(there, want[3:])]
    scratch = _scratch(lib().wc_block_norm_workspace(packed), x)
    _call(lib().wc_block_norm_backward, x.get_device(), packed, _BLOCK_NORM_GRADS.pack(
        dy.data_ptr() if dy is not None else 0, dn.data_ptr() if dn is not None else 0,
        dx.data_ptr() if dx is not None else 0, dh.data_ptr() if dh is not None else 0,
        dgate.data_ptr() if dgate is not None else 0, *[g.data_ptr() if g is not None else 0 for g in grads],
        scratch.data_ptr(), ld_dy, ld_dn, max(1, width), max(1, width)))
    return BlockNormGrads(dx, dh, dgate, *grads)


# ------------------------------------------------------- activations in 8 bits

def _new_act8(like: torch.Tensor) -> Act8:
    rows, width = like.shape
    blocks = -(-width // BLOCK)
    return Act8(like.new_empty((rows, blocks * BLOCK), dtype=torch.int8), like.new_empty((rows, blocks), dtype=torch.uint8), width)


def _check_act8(what: str, a: Act8) -> None:
    q, scale, width = a
    blocks = -(-width // BLOCK)
    if q.dtype != torch.int8 or scale.dtype != torch.uint8 or not q.is_cuda or q.get_device() != scale.get_device() or \
            scale.dim() != 2 or q.shape != (scale.shape[0], blocks * BLOCK) or scale.shape[1] != blocks or \
            not q.is_contiguous() or not scale.is_contiguous():
        _fail(what, "not an 8-bit matrix: q int8 [rows, 32 blocks] and scale uint8 [rows, blocks], contiguous")


def act8_pack(x) -> Act8:
    """x in 8 bits: whole numbers of at most 127 in a power-of-two unit per block of 32 values of a row."""
    ld = _matrix("act8_pack", "x", x)
    rows, width = x.shape
    p = _new_act8(x)
    _call(lib().wc_act8_pack, x.get_device(), _ACT8.pack(
        x.data_ptr(), 0, p.q.data_ptr(), p.scale.data_ptr(), 0, 0, 0, rows, width, ld, 0, _TYPES[x.dtype]))
    return p


def act8_unpack(p: Act8, dtype=torch.bfloat16) -> torch.Tensor:
    """The values an 8-bit matrix stands for (exact in bfloat16 and float32)."""
    _check_act8("act8_unpack", p)
    if dtype not in _TYPES:
        _fail("act8_unpack", "dtype must be float32, float16 or bfloat16")
    rows, width = p.q.shape[0], p.width
    out = p.q.new_empty((rows, width), dtype=dtype)
    _call(lib().wc_act8_unpack, p.q.get_device(), _ACT8.pack(
        0, 0, p.q.data_ptr(), p.scale.data_ptr(), out.data_ptr(), 0, 0, rows, width, 0, max(1, width), _TYPES[dtype]))
    return out


def gelu8(z, bias=None) -> Tuple[torch.Tensor, Act8]:
    """GELU (tanh form) of z + bias, and z + bias in 8 bits for gelu8_backward."""
    ld = _matrix("gelu8", "z", z)
    rows, width = z.shape
    b = _vector("gelu8", "bias", bias, width, z)
    p = _new_act8(z)
    out = z.new_empty(rows, width)
    _call(lib().wc_gelu8, z.get_device(), _ACT8.pack(
        z.data_ptr(), b, p.q.data_ptr(), p.scale.data_ptr(), out.data_ptr(), 0, 0, rows, width, ld, max(1, width),
        _TYPES[z.dtype]))
    return out, p


@lru_cache(maxsize=256)
def _gelu8_workspace(rows: int, width: int) -> int:
    return lib().wc_gelu8_workspace(rows, width)


def gelu8_backward(da, z8: Act8, want_bias=True):
    """(dz, dbias): the gradients at gelu8's input and bias (float32, or None) from the one at its output."""
    me = "gelu8_backward"
    ld = _matrix(me, "da", da)
    _check_act8(me, z8)
    rows, width = da.shape
    if z8.width != width or z8.q.shape[0] != rows or z8.q.get_device() != da.get_device():
        _fail(me, "da and the 8-bit activations differ in shape or device")
    dz = da.new_empty(rows, width)
    dbias = scratch = None
    if want_bias:
        dbias = da.new_empty(width, dtype=torch.float32)
        scratch = _scratch(_gelu8_workspace(rows, width), da)
    _call(lib().wc_gelu8_backward, da.get_device(), _ACT8.pack(
        da.data_ptr(), 0, z8.q.data_ptr(), z8.scale.data_ptr(), dz.data_ptr(), dbias.data_ptr() if want_bias else 0,
        scratch.data_ptr() if want_bias else 0, rows, width, ld, max(1, width), _TYPES[da.dtype]))
    return dz, dbias


@lru_cache(maxsize=256)
def _wgrad_workspace(rows: int, k: int, n: int, ld: int, dy_offset: int, kind: int, out: int) -> int:
    return lib().wc_act8_wgrad_workspace(_ACT8_WGRAD.pack(0, 0, dy_offset, 0, 0, 0, rows, k, n, ld, kind, out))


def act8_wgrad(x8: Act8, dy, *, dtype=torch.float32, want_bias=True):
    """(dw, db): x8^T dy as [width of x8, width of dy] in `dtype`, and dy's column sums (float32, or None): the
    gradients of a linear layer's weight [in, out] and bias from its input as kept in 8 bits. A wait of the kernel
    that runs out (which only a fault of the device would cause) leaves NaN in them."""
    me = "act8_wgrad"
    ld = _matrix(me, "dy", dy)
    _check_act8(me, x8)
    rows, n = dy.shape
    if x8.q.shape[0] != rows or x8.q.get_device() != dy.get_device():
        _fail(me, "dy and the 8-bit activations differ in rows or device")
    if dtype not in _TYPES:
        _fail(me, "dtype must be float32, float16 or bfloat16")
    dw = dy.new_empty((x8.width, n), dtype=dtype)
    db = dy.new_empty(n, dtype=torch.float32) if want_bias else None
    scratch = _scratch(_wgrad_workspace(rows, x8.width, n, ld, dy.data_ptr() & 15, _TYPES[dy.dtype], _TYPES[dtype]), dy)
    _call(lib().wc_act8_wgrad, dy.get_device(), _ACT8_WGRAD.pack(
        x8.q.data_ptr(), x8.scale.data_ptr(), dy.data_ptr(), dw.data_ptr(), db.data_ptr() if want_bias else 0,
        scratch.data_ptr(), rows, x8.width, n, ld, _TYPES[dy.dtype], _TYPES[dtype]))
    return dw, db
