"""Packed attention over thousands of sequences: windows, single tokens, empty ones among them."""
import math

import pytest
import torch

from tests.packed_reference import HALF, TINY, assert_within, borders, packed_reference

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [31, 32, 33, 64, 65, 66, 1023, 1024, 1025, 1056, 1057, 1089, 40000])
def test_sequences_of_one_token_or_none(n, dtype):
    """One key: o is its value and lse its score to the last bit or two, dv the sum of the incoming gradients over the group's heads, and
    dq = dk = 0 up to the rounding of dP and D (the two are equal; o is exact): (D + 8) 2^-23 sum|d_o||v| for dS."""
    from geoweave_b200 import check_status
    from geoweave_b200.custom_flash_attn import packed_flash_attn_func, packed_flash_attn_inference_func

    g = torch.Generator().manual_seed(n)
    there = (torch.rand(n, generator=g) < 0.6).int()
    T, D = int(there.sum()), 64
    cu = borders(there.tolist(), torch.device("cuda"))
    mk = lambda h, tail=0: torch.randn(T + tail, h, D, generator=g).to(dtype).cuda()
    q, k, v, up = [x.requires_grad_() for x in (mk(2, 70), mk(1, 70), mk(1, 70))] + [mk(2, 70)]
    o = packed_flash_attn_func(q, k, v, cu, None, True)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), up)
    check_status()
    u = HALF[dtype]
    score = (q.double() * k.double()).sum(-1) / 8
    size = (q.double() * k.double()).abs().sum(-1) / 8
    for most in (None, 1):
        again, lse = packed_flash_attn_inference_func(q, k, v, cu, None, True, None, most, True)
        assert torch.equal(again[:T], v.detach()[:T].expand(-1, 2, -1)) and (again[T:] == 0).all()
        assert ((lse[:, :T].T.double() - score[:T]).abs() <= ((D + 8) * size[:T] + 4 * score[:T].abs() + 16) * 2.0 ** -24).all()
        assert (lse[:, T:] == -math.inf).all()
    assert torch.equal(o[:T], again[:T]) and (o[T:] == 0).all()
    # P = 2^(S - lse): a common error of both cancels but for the lse's own
    want = up.double()[:T].sum(1, keepdim=True)
    p_err = ((2 * (D + 8) * size[:T] + 8 * score[:T].abs() + 32) * 2.0 ** -24)[..., None]
    limit = ((u + p_err) * up.double()[:T].abs()).sum(1, keepdim=True) + u * want.abs() + 4 * TINY[dtype]
    assert ((dv[:T].double() - want).abs() <= limit).all()
    s_err = (D + 8) * 2.0 ** -23 * (up.double() * v.double()).abs().sum(-1, keepdim=True)[:T] * (1 + 2 * u)
    assert (dq[:T].double().abs() <= s_err / 8 * k.double()[:T].abs() + TINY[dtype]).all()
    assert (dk[:T].double().abs() <= (s_err / 8 * q.double()[:T].abs()).sum(1, keepdim=True) + TINY[dtype]).all()
    for x in (dq, dk, dv):
        assert (x[T:] == 0).all()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_short_and_long_sequences_among_a_thousand(dtype, causal):
    from geoweave_b200 import check_status
    from geoweave_b200.custom_flash_attn import packed_flash_attn_func, packed_flash_attn_inference_func

    g = torch.Generator().manual_seed(7)
    n = 1100
    lens_q, lens_k = [torch.randint(0, 9, (n,), generator=g).tolist() for _ in range(2)]
    for at, (a, b) in {0: (300, 0), 32: (0, 300), 33: (257, 130), 500: (5, 1500), 1023: (520, 64), 1024: (128, 256), 1099: (200, 129)}.items():
        lens_q[at], lens_k[at] = a, b
    mk = lambda rows, h: torch.randn(rows, h, 64, generator=g).to(dtype).cuda()
    q, k, v, up = mk(sum(lens_q) + 9, 2), mk(sum(lens_k) + 9, 1), mk(sum(lens_k) + 9, 1), mk(sum(lens_q) + 9, 2)
    ref = packed_reference(q, k, v, lens_q, lens_k, causal, 0.125, up)
    cu = borders(lens_q, q.device), borders(lens_k, q.device)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    o = packed_flash_attn_func(*leaves, *cu, causal)
    for name, x in zip(("o", "dq", "dk", "dv"), (o, *torch.autograd.grad(o, leaves, up))):
        assert_within(name, x, ref[name])
    # single tokens against the same keys
    ones = (torch.rand(n, generator=g) < 0.7).int().tolist()
    q = mk(sum(ones) + 5, 2)
    ref = packed_reference(q, k.detach(), v.detach(), ones, lens_k, causal, 0.125)
    o, lse = packed_flash_attn_inference_func(q, k, v, borders(ones, q.device), cu[1], causal, None, 1, True)
    check_status()
    assert_within("o", o, ref["o"])
    assert_within("lse", lse, ref["lse"])


@pytest.mark.parametrize("n", [66, 70, 74])
def test_divided_keys_of_many_sequences(n):
    """One head and just over 64 sequences of long keys: slots that stay empty, and each row's keys in two parts."""
    from geoweave_b200 import check_status
    from geoweave_b200.custom_flash_attn import packed_flash_attn_inference_func

    g = torch.Generator().manual_seed(n)
    lens_q, lens_k = [3 + i % 5 if i % 11 else 0 for i in range(n)], [2100 + 17 * i if i % 13 else 0 for i in range(n)]
    mk = lambda rows: torch.randn(rows, 1, 64, generator=g).bfloat16().cuda()
    q, k, v = mk(sum(lens_q)), mk(sum(lens_k)), mk(sum(lens_k))
    for causal in (False, True):
        ref = packed_reference(q, k, v, lens_q, lens_k, causal, 0.125)
        o, lse = packed_flash_attn_inference_func(q, k, v, borders(lens_q, q.device), borders(lens_k, q.device), causal, return_lse=True)
        check_status()
        assert_within("o", o, ref["o"])
        assert_within("lse", lse, ref["lse"])


def test_finding_a_tile_does_not_cost_a_look_at_every_sequence():
    """300 000 sequences: with work for each tile that grows with their number this took minutes; it is some tens of milliseconds."""
    from geoweave_b200.custom_flash_attn import packed_flash_attn_func, packed_flash_attn_inference_func

    n = 300000
    cu = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    q, k, v, up = [torch.randn(n, 1, 64, device="cuda", dtype=torch.bfloat16) for _ in range(4)]
    leaves = [x.requires_grad_() for x in (q, k, v)]

    def step():
        o = packed_flash_attn_func(*leaves, cu)
        token, _ = packed_flash_attn_inference_func(*leaves, cu, max_seqlen_q=1)
        return o, token, *torch.autograd.grad(o, leaves, up)

    step()
    start, end = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
    start.record()
    o, token, _, _, dv = step()
    end.record()
    torch.cuda.synchronize()
    assert torch.equal(o, v) and torch.equal(token, v)
    assert ((dv - up).abs() <= 2.0 ** -7 * up.abs()).all()
    assert start.elapsed_time(end) < 2000
