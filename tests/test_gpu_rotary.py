"""Rotary positions with several axes against complex rotations in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
DTYPES = list(HALF)


def _reference(x, pos, widths, frequency, sign=1):
    """x [..., H, D], pos [..., axes]: (value, bound).  Each result is two products of values that are exact in fp32 with a cosine
    or sine rounded to fp32, added in fp32: 4 roundings of 2^-24 of |a| + |b|, then one of the type."""
    y, mag, at = x.double().clone(), torch.zeros_like(x, dtype=torch.float64), 0
    for a, w in enumerate(widths):
        h = w // 2
        ang = sign * pos[..., a].double()[..., None, None] * frequency ** (-torch.arange(h, device=x.device).double() * 2 / w)
        z = torch.complex(x[..., at:at + h].double(), x[..., at + h:at + w].double())
        m = z.real.abs() + z.imag.abs()
        z = z * torch.polar(torch.ones_like(ang), ang)
        y[..., at:at + h], y[..., at + h:at + w] = z.real, z.imag
        mag[..., at:at + h] = mag[..., at + h:at + w] = m
        at += w
    u = HALF[x.dtype]
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    return y, u * y.abs() + (1 + u) * 4 * 2.0 ** -24 * mag + tiny


def _close(got, ref):
    assert ((got.double() - ref[0]).abs() <= ref[1]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,H,Hk,D,widths", [
    (1, 1, 1, 64, (32, 32)), (37, 16, 16, 64, (16, 24, 24)), (129, 16, 4, 128, (32, 48, 40)), (65, 3, 1, 128, (16, 56, 56)),
    (50, 2, 5, 64, (64,)), (33, 4, 2, 32, (8, 12, 12)), (19, 2, 2, 10, (2, 6)), (19, 2, 2, 9, (2, 4, 2)), (7, 33, 40, 256, (64, 64, 64, 64)),
    (11, 2, 1, 256, (2,)), (1041, 16, 0, 64, (32, 32)), (5, 70, 70, 2, (2,)),
])
def test_values_and_gradients(N, H, Hk, D, widths, dtype):
    from geoweave_b200 import check_status
    from geoweave_b200.rotary import apply_rotary_axes, rotary_axes
    from tests.gpu_util import dev

    g = torch.Generator().manual_seed(N + D)
    mk = lambda h: torch.randn(N, h, D, generator=g).to(dtype).to(dev())
    q, k, dq, dk = mk(H), mk(Hk) if Hk else None, mk(H), mk(Hk) if Hk else None
    pos = torch.randint(0, 900, (N, len(widths)), generator=g).to(dev())
    axes = rotary_axes(widths, 900, dev(), 10000.0)
    leaves = [x.requires_grad_() for x in (q, k) if x is not None]
    out = apply_rotary_axes(q, k, pos, axes)
    grads = torch.autograd.grad([x for x in out if x is not None], leaves, [x for x in (dq, dk) if x is not None])
    check_status()
    for x, y in zip((q, k), out):
        if x is not None:
            assert y.dtype == dtype and y.is_contiguous()
            _close(y, _reference(x.detach(), pos, widths, 10000.0))
    for x, y in zip((dq, dk), grads):
        _close(y, _reference(x, pos, widths, 10000.0, -1))
    with torch.no_grad():  # int32 positions and the plain call give the same
        again = apply_rotary_axes(q, k, pos.int(), axes)
    for a, b in zip(out, again):
        assert (a is None and b is None) or torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_batched_strided_and_misaligned_inputs(dtype):
    from geoweave_b200.rotary import apply_rotary_axes, rotary_axes
    from tests.gpu_util import dev

    g = torch.Generator().manual_seed(1)
    B, N, H, D, widths = 3, 41, 4, 64, (16, 24, 24)
    axes = rotary_axes(widths, 50, dev())
    pos = torch.randint(0, 50, (B, N, 3), generator=g).to(dev())
    fused = torch.randn(B, N, 3, H, D, generator=g).to(dtype).to(dev())
    head_major = torch.randn(B, H, N, D, generator=g).to(dtype).to(dev()).transpose(1, 2)
    odd = torch.randn(B * N * H * D + 1, generator=g).to(dtype).to(dev())[1:].view(B, N, H, D)
    every_other = torch.randn(B, N, H, 2 * D, generator=g).to(dtype).to(dev())[..., ::2]
    shared = torch.randn(B, N, 1, D, generator=g).to(dtype).to(dev()).expand(B, N, H, D)
    for q, k in ((fused[:, :, 0], fused[:, :, 1]), (head_major, odd), (every_other, shared)):
        got = apply_rotary_axes(q, k, pos, axes)
        for x, y in zip((q, k), got):
            _close(y, _reference(x, pos, widths, 100.0))
        flat = apply_rotary_axes(q.reshape(B * N, H, D), k.reshape(B * N, H, D), pos.reshape(B * N, 3), axes)
        for a, b in zip(got, flat):
            assert torch.equal(a.reshape(B * N, H, D), b)
    leaf = shared[:, :, :1].clone().requires_grad_()  # the gradient of a broadcast input is the sum over the copies
    up = torch.randn(B, N, H, D, generator=g).to(dtype).to(dev())
    out, _ = apply_rotary_axes(leaf.expand(B, N, H, D), None, pos, axes)
    (grad,) = torch.autograd.grad(out, leaf, up)
    each, _ = apply_rotary_axes(leaf.detach().expand(B, N, H, D).clone().requires_grad_(), None, pos, axes)
    assert grad.shape == leaf.shape
    value, bound = _reference(up, pos, widths, 100.0, -1)
    u = HALF[dtype]
    assert ((grad.double() - value.sum(2, keepdim=True)).abs() <= bound.sum(2, keepdim=True) + H * u * (value.abs() + bound).sum(2, keepdim=True)).all()
    assert torch.equal(each[:, :, 0], out.detach()[:, :, 0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_two_equal_axes_are_the_front_ends_embedding(dtype):
    """Widths (32, 32) with the projection front-end's own tables: the same numbers as its kernel, bit for bit up to the order of
    one fused multiply-add."""
    from geoweave_b200.front_end import FrontEndParams, project_epilogue, rope_tables
    from geoweave_b200.rotary import RotaryAxes, apply_rotary_axes
    from tests.gpu_util import dev

    g = torch.Generator().manual_seed(2)
    N, H, Hi = 77, 4, 2
    cos, sin = rope_tables(40, dev(), dtype)
    fused = torch.randn(1, N, 3 * H * 64 + 2 * Hi * 64 + Hi, generator=g).to(dtype).to(dev())
    pos = torch.randint(0, 40, (1, N, 2), generator=g).to(dev())
    prm = FrontEndParams(torch.empty(0), None, H, Hi, cos=cos, sin=sin)
    q, k = project_epilogue(fused, pos, prm)[:2]
    both = RotaryAxes((32, 32), cos[:, :16].repeat(1, 2), sin[:, :16].repeat(1, 2))
    qr, kr = apply_rotary_axes(fused[..., :H * 64].unflatten(-1, (H, 64)), fused[..., H * 64:2 * H * 64].unflatten(-1, (H, 64)), pos, both)
    # both round the same two products and their sum once (a fused step more or less: 2^-23 of the pair), then to the type
    for a, b, x in ((q, qr, fused[..., :H * 64]), (k, kr, fused[..., H * 64:2 * H * 64])):
        top = 2 * x.double().abs().max()
        assert ((a.double() - b.double()).abs() <= 2 * HALF[dtype] * a.double().abs() + 2.0 ** -22 * top).all()


def test_far_positions_bad_positions_and_empty_calls():
    import geoweave_b200
    from geoweave_b200.rotary import apply_rotary_axes, rotary_axes
    from tests.gpu_util import dev

    q = torch.randn(4, 2, 64, device=dev())
    axes = rotary_axes((32, 32), 1 << 20, dev(), (10000.0, 100.0))
    pos = torch.tensor([[0, 0], [(1 << 20) - 1, 7], [1000003, 99999], [5, (1 << 20) - 1]], device=dev())
    out, none = apply_rotary_axes(q, None, pos, axes)
    assert none is None
    geoweave_b200.check_status()
    # frequencies differ by axis: check them one at a time
    _close(out[..., :32].contiguous(), _reference(q[..., :32], pos[:, :1], (32,), 10000.0))
    _close(out[..., 32:].contiguous(), _reference(q[..., 32:], pos[:, 1:], (32,), 100.0))
    for bad in (-1, 1 << 20, 1 << 40):
        pos2 = pos.clone()
        pos2[2, 1] = bad
        got, _ = apply_rotary_axes(q, None, pos2, axes)
        with pytest.raises(geoweave_b200.GeoWeaveError):
            geoweave_b200.check_status()
        assert torch.equal(got[[0, 1, 3]], out[[0, 1, 3]])
        assert torch.equal(got[2, :, 32:], q[2, :, 32:])  # counts as position 0
    empty, _ = apply_rotary_axes(q[:0], None, pos[:0], axes)
    assert empty.shape == (0, 2, 64)


def test_refusals():
    from geoweave_b200.rotary import RotaryAxes, apply_rotary_axes as f, rotary_axes
    from tests.gpu_util import dev

    q = torch.randn(4, 2, 64, device=dev())
    pos = torch.zeros(4, 2, dtype=torch.int64, device=dev())
    axes = rotary_axes((32, 32), 10, dev())
    for call, error in [
        (lambda: f(q[0], None, pos, axes), ValueError), (lambda: f(q, q[:3], pos, axes), ValueError), (lambda: f(q, q.half(), pos, axes), TypeError),
        (lambda: f(q, q[..., :32], pos, axes), ValueError), (lambda: f(q[..., :32], None, pos, axes), ValueError),
        (lambda: f(q, None, pos[:, :1], axes), ValueError), (lambda: f(q, None, pos.float(), axes), TypeError),
        (lambda: f(q.double(), None, pos, axes), TypeError), (lambda: f(q.cpu(), None, pos.cpu(), axes), ValueError),
        (lambda: f(q, None, pos, RotaryAxes((32, 32), axes.cos[:, :8], axes.sin[:, :8])), ValueError),
        (lambda: f(q, None, pos, RotaryAxes((32, 32), axes.cos.half(), axes.sin.half())), ValueError),
        (lambda: f(q, None, pos, RotaryAxes((31, 33), axes.cos, axes.sin)), ValueError),
        (lambda: f(q[:, :0], None, pos, axes), ValueError),
    ]:
        with pytest.raises(error):
            call()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", [1, 2, 4, 8, 12])
def test_tables_inside_a_larger_buffer(offset, dtype):
    """Tables that start 4 to 48 bytes behind a 256-byte boundary: the widest pieces need 32-byte ones, narrower ones serve as well."""
    from geoweave_b200.rotary import RotaryAxes, apply_rotary_axes, rotary_axes
    from tests.gpu_util import dev

    g = torch.Generator().manual_seed(offset)
    widths, n = (32, 32), 60
    own = rotary_axes(widths, n, dev())
    room = torch.empty(2, n * 32 + 16, device=dev())
    tables = [x[offset:offset + n * 32].view(n, 32).copy_(t) for x, t in zip(room, (own.cos, own.sin))]
    axes = RotaryAxes(widths, *tables)
    assert axes.cos.data_ptr() == tables[0].data_ptr() and axes.cos.data_ptr() % 256 == 4 * offset
    q, k = [torch.randn(77, h, 64, generator=g).to(dtype).to(dev()) for h in (4, 2)]
    pos = torch.randint(0, n, (77, 2), generator=g).to(dev())
    for a, b in zip(apply_rotary_axes(q, k, pos, axes), apply_rotary_axes(q, k, pos, own)):
        assert torch.equal(a, b)
