"""The training operators (train_ops) as differentiable functions: torch's
autograd calls their backward entries. What a backward pass needs of an
activation is kept in 8 bits where the operator has that form.

First derivatives only: under create_graph the gradients are the same, and
whatever asks for a derivative of them raises SolveError."""
from __future__ import annotations

import functools
from typing import Optional

import torch

from . import SolveError
from . import train_ops as ops
from .train_ops import Act8, PolicyLoss


class _NoDerivative(torch.autograd.Function):
    @staticmethod
    def forward(ctx, grad, *depends_on):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, unused):
        raise SolveError(1, "train_layers: the gradients have no derivatives (a second derivative was asked for)")


def _handle(ctx, like, *saved):
    """Saves what the backward pass reads and, last, an empty tensor that forward has to return first: a result of the
    function that is cheap to keep, through which the graph of a gradient leads back to all inputs."""
    handle = like.new_empty(0)
    ctx.save_for_backward(*saved, handle)
    ctx.set_materialize_grads(False)
    return handle


def _first_order(backward):
    """A backward pass whose results autograd would take for constants. (torch's once_differentiable does not tie them to
    the inputs, so that a derivative at some of those alone comes out without them, and not as an error.)"""

    @functools.wraps(backward)
    def run(ctx, unused, *grads):
        *saved, handle = ctx.saved_tensors
        with torch.no_grad():
            out = backward(ctx, saved, *grads)
        if not torch.is_grad_enabled():
            return out
        return tuple(g if g is None else _NoDerivative.apply(g, handle, *grads) for g in out)

    return run


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, actions, old_logp, advantages, weights, ref_logp, legal, options):
        r = ops.policy_loss(logits, actions, old_logp, advantages, weights=weights, ref_logp=ref_logp, legal=legal,
                            want_grad=False, **options)
        ctx.options = options
        ctx.mark_non_differentiable(r.row_loss, r.logp, r.entropy, r.kl)
        return _handle(ctx, logits, logits, actions, old_logp, advantages, weights, ref_logp, legal), r.loss, r.row_loss, r.logp, r.entropy, r.kl

    @staticmethod
    @_first_order
    def backward(ctx, saved, g, *unused):
        logits, actions, old_logp, advantages, weights, ref_logp, legal = saved
        r = ops.policy_loss(logits, actions, old_logp, advantages, weights=weights, ref_logp=ref_logp, legal=legal,
                            upstream=g.to(torch.float32), **ctx.options)
        return (r.dlogits,) + (None,) * 7


def policy_loss(logits, actions, old_logp, advantages, *, weights=None, ref_logp=None, legal=None, **options) -> PolicyLoss:
    """train_ops.policy_loss with a loss that is differentiable at the logits (the other results are not, and dlogits is
    None): the logits are read again in the backward pass, which keeps no gradient between the two."""
    return PolicyLoss(*_PolicyLoss.apply(logits, actions, old_logp, advantages, weights, ref_logp, legal, options)[1:], None)


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, h, gate, post, post_bias, pre, pre_bias, options, pack):
        pair = lambda w, b: None if w is None else (w, b)  # noqa: E731
        weights = {"post": pair(post, post_bias), "pre": pair(pre, pre_bias)}
        r = ops.block_norm(x, h, gate=gate, pack=pack, **weights, **options)
        ctx.options = options
        out = (_handle(ctx, x, x, h, gate, post, post_bias, pre, pre_bias, r.stats), r.y) + ((r.n,) if r.n is not None else ())
        if pack:
            ctx.mark_non_differentiable(r.n8.q, r.n8.scale)
            out += (r.n8.q, r.n8.scale)
        return out

    @staticmethod
    @_first_order
    def backward(ctx, saved, dy, dn=None, *unused):
        x, h, gate, post, post_bias, pre, pre_bias, stats = saved
        if dy is None and dn is None:
            return (None,) * 9
        flat = lambda d: None if d is None else d.contiguous()  # noqa: E731
        g = ops.block_norm_backward(flat(dy), flat(dn), x, h, stats, gate=gate,
                                    post=None if post is None else (post, post_bias),
                                    pre=None if pre is None else (pre, pre_bias), want=ctx.needs_input_grad[:7], **ctx.options)
        return *g, None, None


def block_norm(x, h, *, gate=None, post=None, pre=None, pack=False, **options):
    """train_ops.block_norm with gradients at x, h, gate and the norms' weights and biases: y, then n where there is a
    pre norm, then n in 8 bits where `pack` asks for it."""
    split = lambda w: w if isinstance(w, tuple) else (w, None)  # noqa: E731
    out = _BlockNorm.apply(x, h, gate, *split(post), *split(pre), options, pack)[1:]
    if pack:
        return out[0], out[1], Act8(out[2], out[3], x.shape[1])
    return out if len(out) > 1 else out[0]


class _Gelu8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, bias):
        a, z8 = ops.gelu8(z, bias)
        return _handle(ctx, z, z8.q, z8.scale), a

    @staticmethod
    @_first_order
    def backward(ctx, saved, da):
        q, scale = saved
        dz, dbias = ops.gelu8_backward(da.contiguous(), Act8(q, scale, da.shape[1]), want_bias=ctx.needs_input_grad[1])
        return dz, dbias


def gelu8(z, bias=None) -> torch.Tensor:
    """GELU (tanh form) of z + bias; what its backward pass needs is kept in 8 bits."""
    return _Gelu8.apply(z, bias)[1]


class _Linear8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, q, scale, keep):
        if keep and q is None:
            q, scale, _ = ops.act8_pack(x)
        out = x @ w.to(x.dtype)
        return _handle(ctx, x, w, *((q, scale) if keep else (None, None))), out if bias is None else out + bias.to(x.dtype)

    @staticmethod
    @_first_order
    def backward(ctx, saved, dy):
        w, q, scale = saved
        dy = dy.contiguous()
        need_x, need_w, need_bias = ctx.needs_input_grad[:3]
        dx = dy @ w.to(dy.dtype).t() if need_x else None
        dw = db = None
        if need_w:
            dw, db = ops.act8_wgrad(Act8(q, scale, w.shape[0]), dy, dtype=w.dtype, want_bias=need_bias)
        elif need_bias:
            db = dy.sum(0, dtype=torch.float32)
        return dx, dw, db, None, None, None


def linear8(x, w, bias=None, x8: Optional[Act8] = None) -> torch.Tensor:
    """x w + bias with w [in, out]. The input is kept in 8 bits for w's gradient, where that is wanted: as `x8` has it
    (block_norm's pack, say), or packed here. The product is the library's; the weight gradient is act8_wgrad's, in w's
    type."""
    q = scale = None
    if x8 is not None:
        q, scale, width = x8
        if x.dim() != 2 or (q.shape[0], width) != x.shape:
            raise SolveError(1, "linear8: x and the 8-bit activations differ in shape")
    return _Linear8.apply(x, w, bias, q, scale, torch.is_grad_enabled() and w.requires_grad)[1]


__all__ = ["policy_loss", "block_norm", "gelu8", "linear8"]
