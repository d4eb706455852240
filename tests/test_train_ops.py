"""The training operators' entries refuse wrong arguments before anything runs
(no GPU needed: the pointers are never followed)."""
import struct

import pytest

from warchest_b200 import SolveError, _check, lib
from warchest_b200 import train_ops as ops

P = 0x1000  # a 16-byte aligned address that nothing reads


def refused(fn, *args, match):
    with pytest.raises(SolveError, match=match) as e:
        _check(fn(*args))
    assert e.value.code == 1


def policy(**change):
    names = ("logits legal actions old_logp advantages weights ref_logp upstream loss row_out dlogits workspace rows width "
             "ld_logits ld_legal ld_dlogits clip_low clip_high kl_coef entropy_coef type action_bytes").split()
    v = dict.fromkeys(names, 0) | dict(logits=P, actions=P, old_logp=P, advantages=P, loss=P, row_out=P, dlogits=P,
                                       workspace=P, rows=4, width=10, ld_logits=10, ld_dlogits=10, clip_low=0.2,
                                       clip_high=0.2, action_bytes=8)
    assert set(change) <= set(names)
    return ops._POLICY_LOSS.pack(*(v | change).values())


@pytest.mark.parametrize("change,match", [
    (dict(type=3), "unknown element type"), (dict(action_bytes=2), "action_bytes"), (dict(rows=-1), "sizes out of range"),
    (dict(width=1 << 40), "sizes out of range"), (dict(loss=0), "null device pointer"), (dict(workspace=0), "workspace"),
    (dict(workspace=P + 8), "workspace"), (dict(actions=0), "null device pointer"), (dict(logits=0), "null device pointer"),
    (dict(ld_logits=9), "row stride"), (dict(legal=P, ld_legal=9), "row stride"), (dict(ld_dlogits=9), "row stride"),
    (dict(clip_low=-0.1), "clip"), (dict(clip_high=float("nan")), "clip"), (dict(kl_coef=float("inf")), "coefficient"),
    (dict(entropy_coef=float("nan")), "coefficient")])
def test_policy_loss_refuses(change, match):
    refused(lib().wc_policy_loss, policy(**change), None, match=match)


def norm(**change):
    names = ("x h gate post_weight post_bias pre_weight pre_bias y n n_q n_scale stats rows width rows_per_gate ld_x ld_h ld_y "
             "ld_n residual_scale eps type kind").split()
    v = dict.fromkeys(names, 0) | dict(x=P, h=P, post_weight=P, pre_weight=P, y=P, n=P, stats=P, rows=4, width=10, ld_x=10,
                                       ld_h=10, ld_y=10, ld_n=10, residual_scale=1.0, eps=1e-5)
    assert set(change) <= set(names)
    return ops._BLOCK_NORM.pack(*(v | change).values())


@pytest.mark.parametrize("change,match", [
    (dict(type=-1), "unknown element type"), (dict(kind=2), "unknown kind"), (dict(width=16385), "up to 16384"),
    (dict(gate=P), "rows_per_gate"), (dict(kind=1, post_bias=P), "RMSNorm has no bias"),
    (dict(pre_weight=0, n=0, pre_bias=P), "bias without"), (dict(eps=-1.0), "eps"), (dict(residual_scale=float("inf")), "residual_scale"),
    (dict(x=0), "null device pointer"), (dict(ld_h=9), "row stride"), (dict(stats=P + 4), "aligned"),
    (dict(pre_weight=0), "pre norm"), (dict(n_q=P), "together"), (dict(y=0), "null device pointer"), (dict(ld_n=9), "row stride")])
def test_block_norm_refuses(change, match):
    refused(lib().wc_block_norm, norm(**change), None, match=match)


def grads(**change):
    names = ("dy dn dx dh dgate dpost_weight dpost_bias dpre_weight dpre_bias workspace ld_dy ld_dn ld_dx ld_dh").split()
    v = dict.fromkeys(names, 0) | dict(dy=P, dn=P, dx=P, dh=P, workspace=P, ld_dy=10, ld_dn=10, ld_dx=10, ld_dh=10)
    assert set(change) <= set(names)
    return ops._BLOCK_NORM_GRADS.pack(*(v | change).values())


@pytest.mark.parametrize("a,g,match", [
    (dict(pre_weight=0), {}, "dn needs"), ({}, dict(dy=0, dn=0), "neither"), ({}, dict(dgate=P), "without a gate"),
    ({}, dict(dpost_bias=P), "not there"), ({}, dict(workspace=0), "workspace"), ({}, dict(ld_dx=9), "row stride")])
def test_block_norm_backward_refuses(a, g, match):
    refused(lib().wc_block_norm_backward, norm(**a), grads(**g), None, match=match)


def act8(**change):
    names = "x bias q scale out dbias workspace rows width ld_x ld_out type".split()
    v = dict.fromkeys(names, 0) | dict(x=P, q=P, scale=P, out=P, rows=4, width=10, ld_x=10, ld_out=10)
    assert set(change) <= set(names)
    return ops._ACT8.pack(*(v | change).values())


@pytest.mark.parametrize("entry,change,match", [
    ("pack", dict(type=7), "unknown element type"), ("pack", dict(x=0), "null device pointer"), ("pack", dict(ld_x=9), "row stride"),
    ("pack", dict(q=P + 8), "aligned"), ("unpack", dict(out=0), "null device pointer"), ("unpack", dict(ld_out=9), "row stride")])
def test_act8_refuses(entry, change, match):
    refused(getattr(lib(), "wc_act8_" + entry), act8(**change), None, match=match)


def test_gelu8_refuses():
    refused(lib().wc_gelu8, act8(out=0), None, match="null device pointer")
    refused(lib().wc_gelu8_backward, act8(dbias=P), None, match="workspace")


def wgrad(**change):
    names = "q scale dy dw db workspace rows k n ld_dy type out_type".split()
    v = dict.fromkeys(names, 0) | dict(q=P, scale=P, dy=P, dw=P, db=P, workspace=P, rows=4, k=10, n=12, ld_dy=12)
    assert set(change) <= set(names)
    return ops._ACT8_WGRAD.pack(*(v | change).values())


@pytest.mark.parametrize("change,match", [
    (dict(type=5), "unknown element type"), (dict(out_type=5), "unknown element type"), (dict(k=0), "k below 1"),
    (dict(n=1 << 21), "sizes out of range"), (dict(dw=0), "null device pointer"), (dict(workspace=P + 4), "workspace"),
    (dict(dy=0), "null device pointer"), (dict(ld_dy=11), "row stride"), (dict(q=P + 8), "aligned"),
    (dict(rows=1 << 31, k=1 << 20, n=1 << 20, ld_dy=1 << 20), "sizes out of range")])
def test_act8_wgrad_refuses(change, match):
    refused(lib().wc_act8_wgrad, wgrad(**change), None, match=match)


@pytest.mark.parametrize("entry,args", [
    ("wc_policy_loss", [policy(logits=P + 2)]), ("wc_policy_loss", [policy(type=1, dlogits=P + 1)]),
    ("wc_policy_loss", [policy(actions=P + 4)]), ("wc_policy_loss", [policy(old_logp=P + 2)]), ("wc_policy_loss", [policy(loss=P + 1)]),
    ("wc_block_norm", [norm(type=2, x=P + 1)]), ("wc_block_norm", [norm(post_weight=P + 2)]),
    ("wc_block_norm_backward", [norm(), grads(dx=P + 2)]), ("wc_block_norm_backward", [norm(), grads(dpost_weight=P + 1)]),
    ("wc_act8_pack", [act8(x=P + 2)]), ("wc_act8_unpack", [act8(type=1, out=P + 1)]), ("wc_gelu8", [act8(bias=P + 2)]),
    ("wc_act8_wgrad", [wgrad(dy=P + 2)]), ("wc_act8_wgrad", [wgrad(out_type=2, dw=P + 1)]), ("wc_act8_wgrad", [wgrad(db=P + 2)])])
def test_addresses_between_elements_are_refused(entry, args):
    refused(getattr(lib(), entry), *args, None, match="not aligned to its elements")


def test_null_arguments_are_refused():
    for name in ("policy_loss", "block_norm", "act8_pack", "act8_unpack", "gelu8", "gelu8_backward", "act8_wgrad"):
        refused(getattr(lib(), "wc_" + name), None, None, match="null arguments")


def test_argument_bytes_are_the_structures_sizes():
    # pointers and 64-bit numbers first, then pairs of 32-bit ones: no padding but act8's last four bytes
    sizes = {s.size for s in (ops._POLICY_LOSS, ops._BLOCK_NORM, ops._BLOCK_NORM_GRADS, ops._ACT8, ops._ACT8_WGRAD)}
    assert sizes == {160, 168, 112, 96, 88}
    assert struct.calcsize("P") == 8


def test_workspaces_of_nothing():
    assert lib().wc_gelu8_workspace(0, 0) == 0
    assert lib().wc_act8_wgrad_workspace(wgrad(rows=0)) == 0
    assert lib().wc_block_norm_workspace(norm(width=0)) == 0


def test_cpu_tensors_are_refused():
    import torch

    x = torch.zeros(4, 8)
    for call in (lambda: ops.act8_pack(x), lambda: ops.gelu8(x), lambda: ops.block_norm(x, x),
                 lambda: ops.policy_loss(x, torch.zeros(4, dtype=torch.int64), x[:, 0], x[:, 0])):
        with pytest.raises(SolveError, match="CUDA tensor"):
            call()


@pytest.mark.parametrize("rows", [1, 2, 3, 100])
def test_a_gate_for_more_rows_than_there_are_is_one_for_all(rows):
    space = lambda per: lib().wc_block_norm_workspace(norm(rows=rows, gate=P, rows_per_gate=per))  # noqa: E731
    assert space((1 << 63) - 1) == space((1 << 63) - rows) == space(rows)
