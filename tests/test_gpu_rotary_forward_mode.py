"""Derivatives of the rotary embedding beside plain reverse mode, on the GPU: tangents, tangents of gradients, and the
transforms that are refused."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from avqa_b200 import RotaryEmbedding
from paged_reference import DTYPES, assert_within, rotate64

pytestmark = pytest.mark.gpu


def _heads(H, dt="f32", seed=0, B=2, T=9, D=64):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(B, H, T, D, generator=g, device="cuda").to(DTYPES[dt])


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("who", ["q", "k", "both"])
@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("reverse_too", [False, True])
def test_tangents_rotate_with_their_inputs(dt, who, given, reverse_too) -> None:
    rot = RotaryEmbedding(64, sections=(8, 24) if given else None)
    pos = torch.randint(0, 500, (2, 2, 9), device="cuda") if given else None
    axes = pos[:, :, None] if given else torch.arange(7, 16, device="cuda")[None]
    q, k, tq, tk = _heads(4, dt), _heads(2, dt, 1), _heads(4, dt, 2), _heads(2, dt, 3)
    if reverse_too:
        q.requires_grad_()
    with forward_ad.dual_level():
        qd = forward_ad.make_dual(q, tq) if who != "k" else q
        kd = forward_ad.make_dual(k, tk) if who != "q" else k
        outs = rot(qd, kd, positions=pos, offset=7)
        for out, x, t, dual in zip(outs, (q, k), (tq, tk), (who != "k", who != "q")):
            value, tangent = forward_ad.unpack_dual(out)
            assert_within(value.detach(), *rotate64(x.detach(), axes, rot), "value")
            if dual:
                assert_within(tangent.detach(), *rotate64(t, axes, rot), "tangent")
            else:
                assert not tangent.any()
        if who != "k":
            alone = forward_ad.unpack_dual(rot(qd, positions=pos, offset=7))
            assert torch.equal(alone.tangent, forward_ad.unpack_dual(outs[0]).tangent)
            with torch.no_grad():
                assert torch.equal(forward_ad.unpack_dual(rot(qd, positions=pos, offset=7)).tangent, alone.tangent)
    assert forward_ad.unpack_dual(rot(q, positions=pos, offset=7)).tangent is None


def test_tangent_of_a_gradient_and_gradient_of_a_tangent() -> None:
    rot = RotaryEmbedding(64)
    at = torch.arange(9, device="cuda")[None]
    q, g, t = _heads(3), _heads(3, seed=1), _heads(3, seed=2)
    q.requires_grad_()
    with forward_ad.dual_level():
        (grad,) = torch.autograd.grad(rot(q), q, forward_ad.make_dual(g, t))
        value, tangent = forward_ad.unpack_dual(grad)
        assert_within(value, *rotate64(g, at, rot, reverse=True), "gradient")
        assert_within(tangent, *rotate64(t, at, rot, reverse=True), "its tangent")
    t = t.clone().requires_grad_()
    with forward_ad.dual_level():
        tangent = forward_ad.unpack_dual(rot(forward_ad.make_dual(q.detach(), t))).tangent
        (grad,) = torch.autograd.grad(tangent, t, g)
    assert_within(grad, *rotate64(g, at, rot, reverse=True), "a tangent's gradient")


def test_function_transforms_are_refused() -> None:
    rot = RotaryEmbedding(64)
    q = _heads(3)
    calls = [lambda: torch.func.grad(lambda x: rot(x).sum())(q), lambda: torch.func.jvp(rot, (q,), (q,)),
             lambda: torch.func.vmap(rot)(q[None]), lambda: torch.func.vjp(rot, q)]
    for call in calls:
        with pytest.raises(RuntimeError):
            call()
    assert_within(rot(q), *rotate64(q, torch.arange(9, device="cuda")[None], rot), "and nothing is left behind")
