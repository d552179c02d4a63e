"""Rotary positions with several axes (``rope_axes``) against the formula in 64 bits."""

import pytest
import torch

from _operators_ref import rope_reference

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def inputs(B, T, H, D, axes, dtype, seed=0, far=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, T, H, D, generator=g).to(dtype)
    pos = torch.randint(0, 4000, (B, T, axes), generator=g) + far
    return x, pos


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("shared", [True, False])
@pytest.mark.parametrize("B,T,H,D,sections", [
    (2, 37, 3, 64, (64,)),
    (1, 1, 1, 128, (32, 48, 48)),
    (3, 65, 5, 80, (20, 20)),        # half of the vector stays
    (2, 9, 2, 62, (14, 0, 22)),      # nothing is a whole 16 bytes; an axis that rotates nothing
    (1, 700, 1, 6, (2, 2, 2)),
    (2, 5, 4, 256, (256,)),
    (1, 3, 2, 600, (256, 256)),      # the most pairs
    (2, 4, 2, 32, (0,)),
])
def test_forward_and_gradient(dtype, interleaved, shared, B, T, H, D, sections):
    import probjax_b200 as pj

    x, pos = inputs(B, T, H, D, len(sections), dtype, seed=D)
    xd = x.to(DEV).requires_grad_(True)
    y = pj.rope_axes(xd, pos.to(DEV), sections, shared=shared, interleaved=interleaved)
    want, tol = rope_reference(x, pos, sections, shared=shared, interleaved=interleaved)
    assert bool(((y.detach().cpu().double() - want).abs() <= tol).all())
    dy = torch.randn(B, T, H, D, generator=torch.Generator().manual_seed(1)).to(dtype)
    (dx,) = torch.autograd.grad(y, xd, dy.to(DEV))
    want, tol = rope_reference(dy, pos, sections, shared=shared, interleaved=interleaved, sign=-1)
    assert bool(((dx.cpu().double() - want).abs() <= tol).all())


@pytest.mark.parametrize("far", [0, 131071, 10 ** 6, 2 ** 31 - 5000])
def test_far_positions_keep_their_angles(far):
    import probjax_b200 as pj

    x, pos = inputs(1, 50, 2, 128, 2, torch.float32, far=far)
    y = pj.rope_axes(x.to(DEV), pos.to(DEV), (64, 64))
    want, tol = rope_reference(x, pos, (64, 64))
    assert bool(((y.cpu().double() - want).abs() <= tol + 2.0 ** -20 * (far > 10 ** 7)).all())  # (2^31 radians carry 2^-22 in float64 too)


@pytest.mark.parametrize("dtype", [torch.float32, torch.int32, torch.int64, torch.float64, torch.int16])
def test_position_types_shapes_and_strides(dtype):
    import probjax_b200 as pj

    x, pos = inputs(2, 21, 4, 64, 2, torch.bfloat16)
    want = pj.rope_axes(x.to(DEV), pos.to(DEV), (32, 32))
    assert torch.equal(pj.rope_axes(x.to(DEV), pos.to(DEV, dtype), (32, 32)), want)
    # shared positions, missing and further leading dimensions
    one = pj.rope_axes(x.to(DEV), pos[0].to(DEV, dtype), (32, 32))
    assert torch.equal(one[0], want[0])
    assert torch.equal(pj.rope_axes(x[0].to(DEV), pos[0].to(DEV, dtype), (32, 32)), want[0])
    five = pj.rope_axes(x.to(DEV)[:, None].expand(2, 3, 21, 4, 64), pos.to(DEV, dtype)[:, None].expand(2, 3, 21, 2), (32, 32))
    assert torch.equal(five[:, 1], want)
    # slices of a fused projection, heads in another order, an odd address, the result in place
    fused = torch.cat([x, x + 1], 2).to(DEV)
    assert torch.equal(pj.rope_axes(fused[:, :, :4], pos.to(DEV, dtype), (32, 32)), want)
    assert torch.equal(pj.rope_axes(x.to(DEV).transpose(1, 2).contiguous().transpose(1, 2), pos.to(DEV, dtype), (32, 32)), want)
    odd = torch.empty(x.numel() + 1, dtype=x.dtype, device=DEV)[1:].view(x.shape).copy_(x)
    assert torch.equal(pj.rope_axes(odd, pos.to(DEV, dtype), (32, 32)), want)
    buf = x.to(DEV)
    assert pj.rope_axes(buf, pos.to(DEV, dtype), (32, 32), out=buf).data_ptr() == buf.data_ptr() and torch.equal(buf, want)


def test_one_axis_is_the_layer_with_shared_positions():
    import probjax_b200 as pj

    x = torch.randn(2, 40, 4, 64, generator=torch.Generator().manual_seed(3)).to(DEV)
    a = pj.rope_axes(x, torch.arange(40, device=DEV)[:, None] + 7, (64,))
    b = pj.rope_interleaved(x, torch.arange(40, device=DEV) + 7)
    # the older kernel forms its angles in 32 bits: 47 radians times 2^-23, on values below 6
    assert float((a - b).abs().max()) <= 47 * 2.0 ** -22 * 12


def test_gradient_against_differences_and_twice():
    import probjax_b200 as pj

    x, pos = inputs(1, 3, 2, 16, 2, torch.float32, seed=4)
    xd = x.to(DEV).requires_grad_(True)
    w = torch.randn(1, 3, 2, 16, generator=torch.Generator().manual_seed(5)).to(DEV)
    f = lambda t: (pj.rope_axes(t, pos.to(DEV), (8, 8)) * w).sum()
    (g,) = torch.autograd.grad(f(xd), xd)
    for i in (0, 5, 17, 40, 95):  # the map is linear: a difference of any size is the gradient
        e = torch.zeros(96, device=DEV)
        e[i] = 1.0
        with torch.no_grad():
            d = f(e.view_as(xd))
        assert abs(float(d) - float(g.flatten()[i])) <= 2.0 ** -19
    # a gradient of a gradient, an expanded gradient and a tangent
    xd2 = x.to(DEV).requires_grad_(True)
    dy = w.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(pj.rope_axes(xd2, pos.to(DEV), (8, 8)), xd2, dy, create_graph=True)
    (ddy,) = torch.autograd.grad(dx, dy, x.to(DEV))
    assert torch.equal(ddy, pj.rope_axes(x.to(DEV), pos.to(DEV), (8, 8)))
    (s,) = torch.autograd.grad(pj.rope_axes(xd2, pos.to(DEV), (8, 8)).sum(), xd2)
    want, tol = rope_reference(torch.ones_like(x), pos, (8, 8), sign=-1)
    assert bool(((s.cpu().double() - want).abs() <= tol).all())
    import torch.autograd.forward_ad as fwd_ad

    with fwd_ad.dual_level():
        tangent = fwd_ad.unpack_dual(pj.rope_axes(fwd_ad.make_dual(x.to(DEV), w), pos.to(DEV), (8, 8))).tangent
    assert torch.equal(tangent, pj.rope_axes(w, pos.to(DEV), (8, 8)))


def test_drafts_are_rotated_to_their_own_positions():
    """The use beside drafted trees: every draft sits at its sequence's length plus its depth."""
    import probjax_b200 as pj

    lengths, depth = torch.tensor([100, 7]), torch.tensor([0, 1, 1, 2])
    x, _ = inputs(2, 4, 2, 64, 1, torch.bfloat16, seed=6)
    pos = (lengths[:, None] + depth)[..., None]
    y = pj.rope_axes(x.to(DEV), pos.to(DEV), (64,))
    want, tol = rope_reference(x, pos, (64,))
    assert bool(((y.cpu().double() - want).abs() <= tol).all())


def test_gradient_refuses_positions_that_changed():
    """The gradient turns by the angles of the forward pass: positions that moved on meanwhile are refused, a copy is not."""
    import probjax_b200 as pj

    x = torch.randn(2, 5, 3, 16, device="cuda", requires_grad=True)
    pos = torch.arange(5, device="cuda", dtype=torch.int32)[:, None].contiguous()
    w = torch.randn(2, 5, 3, 16, device="cuda")
    want = torch.autograd.grad((pj.rope_axes(x, pos, (16,)) * w).sum(), x)[0]
    y = pj.rope_axes(x, pos.clone(), (16,))
    z = pj.rope_axes(x, pos, (16,))
    pos += 1
    assert torch.equal(torch.autograd.grad((y * w).sum(), x)[0], want)
    with pytest.raises(RuntimeError, match="changed in place"):
        (z * w).sum().backward()


@pytest.mark.parametrize("shape", [(2, 3, 0, 4, 8), (0, 3, 5, 4, 8), (2, 0, 4, 8), (0, 4, 8)])
def test_empty_tensors(shape):
    import probjax_b200 as pj

    x = torch.zeros(shape, device=DEV, requires_grad=True)
    for pos in (torch.zeros(shape[-3], 1, device=DEV), torch.zeros(shape[:-2] + (1,), device=DEV)):
        y = pj.rope_axes(x, pos, (8,))
        assert y.shape == x.shape
        assert torch.autograd.grad(y.sum(), x)[0].shape == x.shape
