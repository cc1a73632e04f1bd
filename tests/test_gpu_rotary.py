"""The rotary embedding on the GPU against its fp64 formula
(``paged_reference.rotate64``, whose bounds count the roundings): every type,
pairing, partial widths, odd head widths, several axes, far and negative
positions, strided and expanded operands, and the gradient against the formula
and against differences.
"""
from __future__ import annotations

import pytest
import torch

from avqa_b200 import DtypeError, RotaryEmbedding, ShapeError, ops
from paged_reference import DTYPES, assert_within, rotate64

pytestmark = pytest.mark.gpu


def _heads(B, H, T, D, dt, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(B, T, H, D, generator=g, device="cuda") * scale).to(DTYPES[dt]).transpose(1, 2)


CASES = [
    # dtype, B, H, Hk, T, head_dim, embedding, offset
    ("f32", 2, 8, 8, 64, 64, {}, 0),
    ("bf16", 1, 4, 2, 33, 128, {}, 100000),
    ("f16", 3, 2, 1, 7, 64, dict(interleaved=True), 5),
    ("bf16", 1, 3, 3, 1, 128, dict(rotary_dim=32), 2 ** 24 + 3),
    ("f16", 2, 5, 1, 19, 72, dict(rotary_dim=20, interleaved=True), -40),
    ("f32", 1, 1, 1, 5, 5, dict(rotary_dim=4), 3),
    ("bf16", 2, 7, 1, 300, 40, {}, 0),
    ("f32", 1, 2, 2, 11, 256, dict(base=500000.0), 77),
    ("bf16", 1, 2, 2, 2, 2, {}, 1),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}_T{c[4]}_D{c[5]}_{len(c[6])}")
def test_rotary_matches_formula(case) -> None:
    dt, B, H, Hk, T, D, kw, offset = case
    rot = RotaryEmbedding(D, **kw)
    q, k = _heads(B, H, T, D, dt, 1), _heads(B, Hk, T, D, dt, 2)
    qr, kr = rot(q, k, offset=offset)
    pos = (offset + torch.arange(T, device="cuda"))[None]
    for x, y in ((q, qr), (k, kr)):
        assert y.dtype == x.dtype and y.stride() == x.stride()
        assert_within(y, *rotate64(x, pos, rot), f"{case}")
    assert torch.equal(rot(q, offset=offset), qr)
    assert torch.equal(rot(q, positions=pos[0].to(torch.int64), offset=9), qr)  # given positions replace the offset


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("pos_dtype", [torch.int32, torch.int64])
def test_rotary_axes_and_position_shapes(interleaved, pos_dtype) -> None:
    B, H, T, D = 2, 3, 50, 64
    rot = RotaryEmbedding(D, sections=(8, 12, 12), interleaved=interleaved)
    q = _heads(B, H, T, D, "bf16", 3)
    g = torch.Generator(device="cuda").manual_seed(4)
    grid = torch.randint(-5, 5000, (3, B, T), generator=g, device="cuda").to(pos_dtype)
    want = rotate64(q, grid[:, :, None], rot)
    assert_within(rot(q, positions=grid), *want, "axes, batch, tokens")
    assert_within(rot(q, positions=grid[:, :1]), *rotate64(q, grid[:, :1, None], rot), "axes, 1, tokens")
    assert_within(rot(q, positions=grid[:, 0]), *rotate64(q, grid[:, :1, None], rot), "axes, tokens")
    line = grid[1, 1]
    assert_within(rot(q, positions=line), *rotate64(q, line.expand(3, T), rot), "tokens on all axes")
    # a view with strides of its own
    wide = torch.zeros(3, B, T, 2, device="cuda", dtype=pos_dtype)
    wide[..., 0] = grid
    assert torch.equal(rot(q, positions=wide[..., 0]), rot(q, positions=grid))
    one = RotaryEmbedding(D, interleaved=interleaved)
    assert_within(one(q, positions=grid[0]), *rotate64(q, grid[:1, :, None], one), "batch, tokens")


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_rotary_strides_and_alignment(dt) -> None:
    rot = RotaryEmbedding(64)
    fused = _heads(2, 9, 40, 64, dt, 5).transpose(1, 2)  # [B, T, 9, 64]: q, k and v side by side
    q, k = fused[:, :, :6].transpose(1, 2), fused[:, :, 6:8].transpose(1, 2)
    pos = torch.arange(40, device="cuda")[None]
    qr, kr = rot(q, k)
    assert_within(qr, *rotate64(q, pos, rot), "q of a fused projection")
    assert_within(kr, *rotate64(k, pos, rot), "k of a fused projection")
    flat = torch.randn(2 * 3 * 40 * 65 + 1, device="cuda").to(DTYPES[dt])
    odd = flat[1:].view(2, 3, 40, 65)[..., :64]  # rows at odd addresses
    assert_within(rot(odd), *rotate64(odd, pos, rot), "odd addresses")
    shared = _heads(1, 1, 40, 64, dt, 6).expand(2, 4, 40, 64)
    assert_within(rot(shared), *rotate64(shared, pos, rot), "expanded")
    for empty in (odd[:0], odd[:, :, :0]):
        assert rot(empty).shape == empty.shape
    # in place through the C ABI's aliasing rule
    x = q.contiguous()
    want = ops.rotary(rot, x)[0]
    import ctypes
    from avqa_b200 import _lib
    s = _lib.strides3(x)
    _lib.check(_lib.load().avq_rotary(_lib.dtype_code(x.dtype), x.data_ptr(), s, 6, None, None, 0, 2, 40, 64, 64, 0,
                                      rot.c_frequencies, None, 1, None, 0, None, 0, 0, x.data_ptr(), s, None, None,
                                      ctypes.c_void_p(_lib.stream_of(x.device))), "avq_rotary")
    assert torch.equal(x, want)


def test_rotary_keeps_infinities_and_nan_in_their_pairs() -> None:
    rot = RotaryEmbedding(8)
    x = torch.ones(1, 1, 3, 8, device="cuda")
    x[0, 0, 1, 2], x[0, 0, 2, 5] = float("inf"), float("nan")
    y = rot(x, offset=1)
    bad = ~torch.isfinite(y)
    want = torch.zeros_like(bad)
    want[0, 0, 1, [2, 6]] = True
    want[0, 0, 2, [1, 5]] = True
    assert torch.equal(bad, want)


GRADS = [("f32", 128, {}), ("bf16", 64, dict(interleaved=True)), ("f16", 72, dict(rotary_dim=36, sections=(4, 7, 7)))]


@pytest.mark.parametrize("case", GRADS, ids=lambda c: f"{c[0]}_D{c[1]}")
def test_rotary_gradient_matches_formula(case) -> None:
    dt, D, kw = case
    B, H, Hk, T = 2, 4, 2, 29
    rot = RotaryEmbedding(D, **kw)
    q, k = (_heads(B, h, T, D, dt, 7 + h).requires_grad_() for h in (H, Hk))
    gq, gk = _heads(B, H, T, D, dt, 11), _heads(B, Hk, T, D, dt, 12)
    pos = torch.randint(0, 9000, (rot.num_axes, B, T), device="cuda")
    qr, kr = rot(q, k, positions=pos)
    dq, dk = torch.autograd.grad((qr, kr), (q, k), (gq, gk), retain_graph=True)
    assert_within(dq, *rotate64(gq, pos[:, :, None], rot, reverse=True), "dq")
    assert_within(dk, *rotate64(gk, pos[:, :, None], rot, reverse=True), "dk")
    # one output's gradient alone, and a gradient that is expanded along D
    assert torch.equal(torch.autograd.grad(kr, k, gk, retain_graph=True)[0], dk)
    (ds,) = torch.autograd.grad(qr.sum(), q)
    assert_within(ds, *rotate64(torch.ones_like(q), pos[:, :, None], rot, reverse=True), "a sum's gradient")


def test_rotary_gradient_of_shared_and_of_frozen_inputs() -> None:
    rot = RotaryEmbedding(64)
    base = torch.randn(1, 1, 9, 64, device="cuda", requires_grad=True)  # one key head shared by four
    q = torch.randn(2, 4, 9, 64, device="cuda")  # takes no gradient
    qr, kr = rot(q, base.expand(2, 4, 9, 64))
    w = torch.randn_like(kr)
    (kr * w).sum().backward()
    y, bound = rotate64(w, torch.arange(9, device="cuda")[None], rot, reverse=True)
    # 8 rounded terms and their fp32 sum
    assert_within(base.grad, y.sum((0, 1), keepdim=True), bound.sum((0, 1), keepdim=True)
                  + y.abs().sum((0, 1), keepdim=True) * 8 * 2.0 ** -24, "shared head")
    assert q.grad is None


def test_rotary_gradient_matches_differences() -> None:
    """Along a direction v, <g, R(x + v) - R(x)> = <R^T g, v>: the operator is linear, so the step may be 1;
    both sides are sums of 4096 products in fp64 of values with fp32 roundings."""
    rot = RotaryEmbedding(64, sections=(10, 11, 11))
    x = torch.randn(2, 4, 8, 64, device="cuda", requires_grad=True)
    v, g = torch.randn_like(x), torch.randn_like(x)
    pos = torch.randint(0, 100, (3, 8), device="cuda")
    y = rot(x, positions=pos)
    (dx,) = torch.autograd.grad(y, x, g, create_graph=True)
    with torch.no_grad():
        step = rot(x + v, positions=pos).double() - rot(x, positions=pos).double()
    left, right = (g.double() * step).sum(), (dx.double() * v.double()).sum()
    size = (g.double().abs() * (x.abs() + v.abs() + y.abs()).double()).sum()
    assert abs(left - right) <= size * 2.0 ** -20
    # the gradient of the gradient: the rotation again
    h = torch.randn_like(x)
    g2 = g.clone().requires_grad_()
    (dx2,) = torch.autograd.grad(rot(x, positions=pos), x, g2, create_graph=True)
    (dg,) = torch.autograd.grad(dx2, g2, h)
    assert_within(dg, *rotate64(h, pos[:, None], rot), "double backward")


def test_rotary_refuses_on_the_device() -> None:
    rot = RotaryEmbedding(64)
    q = torch.randn(2, 3, 5, 64, device="cuda")
    with pytest.raises(ShapeError):
        rot(q, q[:, :, :4])
    with pytest.raises(ShapeError):
        rot(q[..., :32])
    with pytest.raises(ShapeError):
        rot(q, positions=torch.arange(6, device="cuda"))
    with pytest.raises(ShapeError):
        rot(q, positions=torch.zeros(3, 5, dtype=torch.long, device="cuda"))
    with pytest.raises(DtypeError):
        rot(q, positions=torch.arange(5, device="cuda").float())
    with pytest.raises(DtypeError):
        rot(q, q.bfloat16())


def test_rotary_graph_replays_with_new_positions() -> None:
    rot = RotaryEmbedding(128)
    q, k = _heads(3, 8, 1, 128, "bf16", 21), _heads(3, 2, 1, 128, "bf16", 22)
    pos = torch.zeros(3, 1, dtype=torch.int32, device="cuda")
    rot(q, k, positions=pos)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qr, kr = rot(q, k, positions=pos)
    for step in (0, 5, 70001):
        pos.fill_(step)
        graph.replay()
        assert_within(qr, *rotate64(q, pos[None, :, None], rot), f"step {step}")
        assert_within(kr, *rotate64(k, pos[None, :, None], rot), f"step {step}")
