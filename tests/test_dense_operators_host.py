"""Host side of the rotary and packed-attention operators: tables, and refusals before any launch (no GPU needed)."""
import ctypes
import math

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from geoweave_b200 import _lib, build as gw_build

    gw_build.build()
    return _lib.load()


def test_tables_hold_angles_of_far_positions():
    from geoweave_b200.rotary import rotary_axes

    axes = rotary_axes((16, 24, 24), 5000, "cpu", (100.0, 100.0, 10000.0))
    assert axes.cos.shape == axes.sin.shape == (5000, 32) and axes.cos.dtype == torch.float32
    for p in (0, 1, 4999):
        for at, w, f in ((0, 16, 100.0), (8, 24, 100.0), (20, 24, 10000.0)):
            for j in range(w // 2):
                a = p * f ** (-2.0 * j / w)
                # rounded once from 64 bits; the angle itself is good to 5000 * 2^-51
                assert abs(axes.cos[p, at + j].item() - math.cos(a)) <= 2.0 ** -24
                assert abs(axes.sin[p, at + j].item() - math.sin(a)) <= 2.0 ** -24


def test_rotary_axes_refuses_what_makes_no_sense():
    from geoweave_b200.rotary import rotary_axes

    for widths in ((), (3,), (0, 4), (-2,), (2, 2, 2, 2, 2)):
        with pytest.raises(ValueError):
            rotary_axes(widths, 4, "cpu")
    for kw in ({"max_position": 0}, {"max_position": 4, "frequency": -1.0}, {"max_position": 4, "frequency": (1.0, 2.0)}):
        with pytest.raises(ValueError):
            rotary_axes((4,), device="cpu", **kw)


def test_operators_take_cuda_tensors_only():
    from geoweave_b200.custom_flash_attn import packed_flash_attn_func, packed_flash_attn_inference_func
    from geoweave_b200.rotary import apply_rotary_axes, rotary_axes

    q = torch.zeros(4, 2, 64)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    for f in (packed_flash_attn_func, packed_flash_attn_inference_func):
        with pytest.raises(ValueError):
            f(q, q, q, cu)
    with pytest.raises(ValueError):
        apply_rotary_axes(q, None, torch.zeros(4, 1, dtype=torch.int64), rotary_axes((64,), 4, "cpu"))


def test_entry_points_refuse_bad_arguments_before_any_launch(lib):
    from geoweave_b200 import _lib

    p, two, three = 4096, _lib.i64x2([64, 64]), _lib.i64x3([64, 64, 64])  # an aligned address that is never followed
    wide = (ctypes.c_int * 2)(32, 32)
    fwd = lambda q=p, dt=_lib.GW_BF16, nseq=1, tq=8, tk=8, H=1, Hk=1, D=64, st=two, scale=1.0, o=p: lib.gw_packed_attn_fwd(
        q, p, p, dt, p, p, nseq, tq, tk, H, Hk, D, st, two, two, scale, 0, 0, o, None, None, None, 0, None, None)
    assert fwd(q=None) == fwd(o=None) == fwd(nseq=-1) == fwd(tq=-1) == fwd(H=3, Hk=2) == fwd(H=0) == -1
    assert fwd(q=4097) == fwd(st=_lib.i64x2([60, 64])) == fwd(st=_lib.i64x2([0, 64])) == -1
    assert fwd(scale=0.0) == fwd(scale=-1.0) == fwd(scale=float("nan")) == fwd(scale=float("inf")) == -1
    assert fwd(dt=7) == fwd(D=136) == fwd(D=60) == fwd(H=70000, Hk=70000) == fwd(tq=1 << 31) == -2
    bwd = lambda q=p, lse=p, ws=p, n=1 << 20, st=two, dq=p: lib.gw_packed_attn_bwd(
        q, p, p, p, None, lse, p, _lib.GW_F16, p, p, 1, 8, 8, 1, 1, 64, two, two, two, st, 1.0, 0, dq, p, p, ws, n, None, None)
    assert bwd(q=None) == bwd(lse=None) == bwd(dq=None) == -1
    rot = lambda q=p, pos=p, widths=wide, axes=2, D=64, rows=4, H=1, dt=_lib.GW_F32: lib.gw_rotary_axes(
        q, None, dt, 1, 4, H, 0, D, three, None, pos, 1, axes, widths, p, p, rows, 0, p, None, None, None)
    assert rot(q=None) == rot(pos=None) == rot(D=62) == rot(rows=0) == rot(H=0) == rot(axes=0) == rot(q=4098) == -1
    assert rot(widths=(ctypes.c_int * 2)(31, 33)) == rot(widths=(ctypes.c_int * 2)(0, 32)) == -1
    assert rot(axes=5) == rot(D=512) == rot(dt=9) == -2
    assert lib.gw_packed_attn_bwd_workspace_bytes(1000, 16) == 64000
    assert lib.gw_packed_attn_bwd_workspace_bytes(0, 16) == 0


def test_warps_of_the_packed_kernels_wait_as_one():
    """A wait that runs out must not split a warp: outside blocks that a single lane runs, every wait goes through warp_wait, and so does
    every look at the abort flag, or through warp_sees.  (In a split warp the next warp-wide instruction would wait without a limit.)"""
    import os
    import re

    import geoweave_b200

    csrc = os.path.join(os.path.dirname(geoweave_b200.__file__), "csrc")
    for name in ("gw_packed_fwd.cu", "gw_packed_bwd.cu", "gw_packed_split.cu"):
        blocks, waits = [], 0  # the lines that opened the blocks around the present one
        for number, line in enumerate(open(os.path.join(csrc, name)), 1):
            code = line.split("//")[0]
            one_lane = any("lane == 0" in b for b in blocks) or "if (lane == 0)" in code
            waits += code.count("warp_wait(")
            if re.search(r"mbar_wait_\w+\(", code):
                assert one_lane, f"{name}:{number}: {line.strip()}"
            if re.search(r"abort_flag(?! = )", re.sub(r"int abort_flag;|&sh->abort_flag|warp_sees\(sh->abort_flag\)", "", code)):
                assert one_lane, f"{name}:{number}: {line.strip()}"
            for c in code:
                if c == "{":
                    blocks.append(code)
                elif c == "}":
                    blocks.pop()
        assert waits > 0 and not blocks


def test_one_of_the_key_sides_gradients_alone_is_refused(lib):
    from geoweave_b200 import _lib

    p, two = 4096, _lib.i64x2([64, 64])
    bwd = lambda dk, dv: lib.gw_packed_attn_bwd(p, p, p, p, None, p, p, _lib.GW_F16, p, p, 1, 8, 8, 1, 1, 64, two, two, two, two, 1.0, 0, p, dk, dv,
                                                p, 1 << 20, None, None)
    assert bwd(None, p) == bwd(p, None) == -1


def test_scales_that_fp32_cannot_hold_are_refused(lib):
    """Times log2 e the largest fp32 numbers are infinite, and infinity times a score of zero is not a number."""
    from geoweave_b200 import _lib
    from geoweave_b200.custom_flash_attn.packed_flash_attn import _scale

    p, two = 4096, _lib.i64x2([64, 64])
    fwd = lambda scale: lib.gw_packed_attn_fwd(p, p, p, _lib.GW_BF16, p, p, 1, 8, 8, 1, 1, 64, two, two, two, scale, 0, 0, p, None, None, None, 0,
                                               None, None)
    assert fwd(2.9e38) == fwd(2.4e38) == fwd(float("inf")) == -1
    for scale in (1e-50, 2.4e38, 1e300, float("inf"), float("nan"), 0.0, -1.0):
        with pytest.raises(ValueError):
            _scale(scale, 64)
    assert _scale(2.0 ** 127, 64) == 2.0 ** 127 and _scale(None, 64) == 0.125


def test_pointers_between_the_words_that_they_point_to_are_refused(lib):
    from geoweave_b200 import _lib

    p, odd, two = 4096, 4098, _lib.i64x2([64, 64])
    fwd = lambda cu_q=p, cu_k=p, lse=p, status=p: lib.gw_packed_attn_fwd(p, p, p, _lib.GW_BF16, cu_q, cu_k, 1, 8, 8, 1, 1, 64, two, two, two, 1.0, 0,
                                                                         0, p, None, lse, None, 0, status, None)
    bwd = lambda cu_q=p, cu_k=p, lse=p, status=p, ws=p: lib.gw_packed_attn_bwd(p, p, p, p, None, lse, p, _lib.GW_F16, cu_q, cu_k, 1, 8, 8, 1, 1, 64, two,
                                                                               two, two, two, 1.0, 0, p, p, p, ws, 1 << 20, status, None)
    for call, names in ((fwd, ("cu_q", "cu_k", "lse", "status")), (bwd, ("cu_q", "cu_k", "lse", "status", "ws"))):
        for name in names:
            assert call(**{name: odd}) == -1, name


def test_tables_made_during_inference_serve_training():
    from geoweave_b200.rotary import rotary_axes

    with torch.inference_mode():
        axes = rotary_axes((16, 24, 24), 50, "cpu")
    assert not axes.cos.is_inference() and not axes.sin.is_inference()  # an inference tensor cannot be kept for a backward pass
    (torch.ones(50, 32, requires_grad=True) * axes.cos).sum().backward()
