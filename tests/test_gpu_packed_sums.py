"""The packed attention on inputs whose results are counts and sums of whole numbers: a row that is left out or taken twice at
a border of tiles, parts, chunks or sequences shows in full, at lengths where bounds on random inputs are wide.

With q = 0 (or k = 0) every score is 0, so each weight is 1 before the division, which every type holds; sums of small whole numbers are
exact in fp32.  What is left is the division and the last rounding: (u^2 + 2^-22) of the value for o with what its rounding took off,
u + 2^-20 for a 16-bit result whose P or dS is a power of two, twice that otherwise (P = 1 / n is rounded too).
"""
import math

import pytest
import torch

from tests.packed_reference import HALF, TINY, borders, packed_reference

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]

# name: query lengths, key lengths, heads, key heads, max_seqlen_q -- each way the forward divides its work
FORMS = {
    "two tiles a block": ([2500, 33], [2999, 1500], 16, 16, None),
    "one tile a block": ([700, 1], [1111, 129], 8, 2, None),
    "keys in parts": ([130], [5003], 4, 2, None),
    "keys in parts, ragged": ([300, 17], [4100, 9], 2, 1, None),
    "single tokens": ([1, 0, 1, 1], [3001, 64, 77, 1], 8, 2, 1),
    "a few queries": ([3, 4], [2600, 513], 8, 2, 4),
}


def _zeros(n, heads, D, dtype):
    return torch.zeros(n, heads, D, dtype=dtype, device="cuda")


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float16, 64), (torch.float16, 80), (torch.float32, 64),
                                     (torch.float32, 128)])
@pytest.mark.parametrize("form", list(FORMS))
def test_every_key_counts_once(form, dtype, D, causal):
    """o = mean of the visible values, whole numbers of up to 8, with what rounding it took off."""
    from geoweave_b200 import check_status
    from geoweave_b200.custom_flash_attn.packed_flash_attn import packed_attention_forward

    lens_q, lens_k, H, Hk, most = FORMS[form]
    g = torch.Generator().manual_seed(D)
    v = torch.randint(-8, 9, (sum(lens_k), Hk, D), generator=g).to(dtype).cuda()
    k = torch.randn(sum(lens_k), Hk, D, generator=g).to(dtype).cuda()
    q = _zeros(sum(lens_q), H, D, dtype)
    low = None if dtype is torch.float32 else torch.full_like(q, float("nan"))
    o, lse = packed_attention_forward(q, k, v, borders(lens_q, q.device), borders(lens_k, q.device), causal, None, most, True, low)
    check_status()
    u = HALF[dtype]
    a = c = 0
    for lq, lk in zip(lens_q, lens_k):
        if lq:
            seen = torch.full((lq,), lk) if not causal else (torch.arange(lq) + lk - lq + 1).clamp(0, lk)
            seen = seen.cuda()
            sums = torch.cat((torch.zeros_like(v[:1]).double(), v[c:c + lk].double().cumsum(0)))[seen]
            want = (sums / seen.clamp(min=1)[:, None, None]).repeat_interleave(H // Hk, 1)
            got = o[a:a + lq].double() + (0 if low is None else low[a:a + lq].double())
            err = u * u + 2.0 ** -22 if low is not None else 2.0 ** -22
            assert ((got - want).abs() <= err * want.abs() + TINY[dtype]).all()
            assert ((o[a:a + lq].double() - want).abs() <= (u + 2.0 ** -22) * want.abs() + TINY[dtype]).all()
            assert ((lse[:, a:a + lq].double() - seen.double().log()).nan_to_num(0.0).abs() <= 2.0 ** -20 * (1 + seen.double().log().abs().nan_to_num(0.0, 0.0, 0.0))).all()
            assert (lse[:, a:a + lq][:, seen == 0] == -math.inf).all()
        a, c = a + lq, c + lk


def _codes(n, D, dtype, heads):
    """[n, heads, D]: row i has a one in column i % 64."""
    x = torch.zeros(n, heads, D)
    x[torch.arange(n), :, torch.arange(n) % 64] = 1
    return x.to(dtype).cuda()


def _sides(lens):
    """[n, 1]: +1 or -1 for each row of each sequence by (row within the batch) % 64, half of them each."""
    n = sum(lens)
    return torch.where(torch.arange(n) % 64 < 32, 1.0, -1.0)[:, None]


def _counts(lens, D):
    """For each sequence: how many of its rows (numbered over the batch) have their one in each column."""
    out, at = [], 0
    for n in lens:
        out.append(torch.bincount(torch.arange(at, at + n) % 64, minlength=D)[:D].double().cuda())
        at += n
    return out


# lengths of keys: powers of two, so that P = 1 / n is exact; multiples of 64 otherwise (borders inside tiles of 128)
GRADS = [([4099, 70], [4096, 64], 2, 2), ([1500], [1024], 4, 2), ([1000, 129], [2048, 512], 1, 1), ([777], [3008], 2, 1), ([2900, 65], [192, 704], 4, 2)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens_q,lens_k,H,Hk", GRADS)
def test_every_pair_counts_once_in_the_gradients(lens_q, lens_k, H, Hk, D, dtype):
    from geoweave_b200 import check_status
    from geoweave_b200.custom_flash_attn import packed_flash_attn_func

    T, S, group, scale, u = sum(lens_q), sum(lens_k), H // Hk, 1 / 8, HALF[dtype]
    cu = borders(lens_q, torch.device("cuda")), borders(lens_k, torch.device("cuda"))
    first = lambda x, heads: torch.cat((x, torch.zeros(x.shape[0], D - 1)), 1)[:, None].expand(-1, heads, -1).to(dtype).cuda()
    v = first(_sides(lens_k), Hk)       # +-1 in column 0
    up = first(torch.ones(T, 1), H)     # dP = +-1, its mean 0 over each sequence of 64 n keys
    sides = _sides(lens_k)[:, 0].double().cuda()
    for n in lens_k:
        assert n % 64 == 0

    # q = 0: dq = scale sum_j dS_j k_j counts the keys with a one in each column; dv = sum_i P d_o the queries
    q, k, v_, g = [x.clone().requires_grad_() for x in (_zeros(T, H, D, dtype), _codes(S, D, dtype, Hk), v)] + [up]
    dq, dk, _ = torch.autograd.grad(packed_flash_attn_func(q, k, v_, *cu, False, scale), (q, k, v_), g)
    g = _codes(T, D, dtype, H)
    _, _, dv = torch.autograd.grad(packed_flash_attn_func(q, k, v_, *cu, False, scale), (q, k, v_), g)
    # k = 0: dk = scale sum_i dS_i q_i counts the queries
    q2, k2 = _codes(T, D, dtype, H).requires_grad_(), _zeros(S, Hk, D, dtype).requires_grad_()
    dq2, dk2, _ = torch.autograd.grad(packed_flash_attn_func(q2, k2, v_, *cu, False, scale), (q2, k2, v_), up)
    check_status()
    assert (dk == 0).all() and (dq2 == 0).all()

    a = c = 0
    column = torch.where(torch.arange(D) % 64 < 32, 1.0, -1.0).double().cuda()
    for lq, lk, rows, keys in zip(lens_q, lens_k, _counts(lens_q, D), _counts(lens_k, D)):
        err = (u if lk & (lk - 1) == 0 else 2 * u) + 2.0 ** -20
        want = scale / lk * keys * column
        assert ((dq[a:a + lq].double() - want).abs() <= err * want.abs() + TINY[dtype]).all(), "dq"
        want = group / lk * rows
        assert ((dv[c:c + lk].double() - want).abs() <= err * want.abs() + TINY[dtype]).all(), "dv"
        want = scale / lk * group * rows * sides[c:c + lk, None, None]
        assert ((dk2[c:c + lk].double() - want).abs() <= err * want.abs() + TINY[dtype]).all(), "dk"
        a, c = a + lq, c + lk


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("form", list(FORMS))
def test_row_sums_come_from_the_output_before_its_rounding(form, D, dtype):
    """Values that hardly differ between the keys, and keys close to 2: dP hardly differs either, so an error of D = sum d_o o, which all keys
    share, is not lost among others.  With o as rounded, dq is off by up to 8 to 21 times (bf16) and 3 to 7 times (fp16) these limits.

    Limits (e = 2^-24, n keys, P = 1 / n): D is off by sum|d_o| ((u^2 + 2^-22)|o| + 2^-25 for fp16) + (D + 8) e sum|d_o||o|; dP by
    (D + 8) e sum|d_o||v|; dS by 1 / n of both and (u + 2^-18) of itself; dq by scale sum |dS error||k| + n e scale sum|dS||k| + u |dq|."""
    from geoweave_b200 import check_status
    from geoweave_b200.custom_flash_attn import packed_flash_attn_func

    lens_q, lens_k, H, Hk, most = FORMS[form]
    g = torch.Generator().manual_seed(D + 1)
    mk = lambda n, h, mean, size: (mean + size * torch.randn(n, h, D, generator=g)).to(dtype).cuda()
    q = _zeros(sum(lens_q), H, D, dtype).requires_grad_()
    k, v, up = mk(sum(lens_k), Hk, 2.0, 0.25), mk(sum(lens_k), Hk, 1 + torch.rand(D, generator=g), 1 / 64), mk(sum(lens_q), H, 0.0, 1.0)
    o = packed_flash_attn_func(q, k, v, borders(lens_q, q.device), borders(lens_k, q.device), False, None, most)
    (dq,) = torch.autograd.grad(o, q, up)
    check_status()
    u, e, scale = HALF[dtype], 2.0 ** -24, D ** -0.5
    a = c = 0
    for lq, lk in zip(lens_q, lens_k):
        for h in range(H if lq else 0):
            K, V, G = k[c:c + lk, h * Hk // H].double(), v[c:c + lk, h * Hk // H].double(), up[a:a + lq, h].double()
            mean = V.mean(0)
            dS = (G @ (V - mean).T) / lk
            want = scale * dS @ K
            size = G.abs() @ mean.abs()
            d_err = (u * u + 2.0 ** -22) * size + TINY[dtype] * G.abs().sum(1) + (D + 8) * e * size
            s_err = (d_err[:, None] + (D + 8) * e * (G.abs() @ V.abs().T)) / lk + (u + 2.0 ** -18) * dS.abs()
            limit = scale * (s_err @ K.abs() + lk * e * (dS.abs() @ K.abs())) + u * want.abs() + TINY[dtype]
            assert ((dq[a:a + lq, h].double() - want).abs() <= limit).all(), (form, h)
        a, c = a + lq, c + lk


def test_a_bound_on_the_queries_may_be_any_number():
    """Through C, where nothing clips it to the number of queries: a bound beyond 2^31, or whose product with the heads of a group passes 64
    bits, says no more than none at all."""
    from geoweave_b200 import _lib, check_status
    from tests.gpu_util import dev

    lib = _lib.load()
    T, S, H, Hk, D = 40, 700, 8, 2, 64
    g = torch.Generator().manual_seed(0)
    q, k, v = [torch.randn(n, h, D, generator=g).bfloat16().to(dev()) for n, h in ((T, H), (S, Hk), (S, Hk))]
    cu_q, cu_k = borders([T], dev()), borders([S], dev())
    outs = []
    for most in (0, T, 1 << 31, (1 << 32) + 1, 1 << 40, 1 << 62, (1 << 62) + 1, (1 << 63) - 1):
        n = lib.gw_packed_attn_fwd_workspace_bytes(_lib.GW_BF16, 1, T, S, H, Hk, D, most)
        ws = torch.empty(max(n, 16), dtype=torch.uint8, device=dev())
        outs.append(torch.empty_like(q))
        strides = [_lib.i64x2((h * D, D)) for h in (H, Hk, Hk)]
        rc = lib.gw_packed_attn_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), _lib.GW_BF16, cu_q.data_ptr(), cu_k.data_ptr(), 1, T, S, H, Hk, D,
                                    *strides, 0.125, 0, most, outs[-1].data_ptr(), None, None, ws.data_ptr(), n, _lib.status_word(dev()).data_ptr(),
                                    _lib.stream_ptr(dev()))
        _lib.check(rc, "gw_packed_attn_fwd")
        assert n == lib.gw_packed_attn_fwd_workspace_bytes(_lib.GW_BF16, 1, T, S, H, Hk, D, 0)
    check_status()
    for o in outs[1:]:
        assert torch.equal(o, outs[0])


@pytest.mark.parametrize("lens_q,lens_k,H,Hk,D,causal", [
    ([1348, 33], [1348, 33], 16, 2, 64, True), ([447] * 4, [447] * 4, 16, 2, 32, True), ([2, 2], [6982, 2327], 8, 1, 80, False), ([900], [900], 8, 1, 128, True),
    ([1, 1], [40000, 9000], 4, 4, 64, False),
])
def test_fp32_sums_over_thousands_of_rows_stay_exact(lens_q, lens_k, H, Hk, D, causal):
    """The error's norm against 64 bits, in half steps u = 2^-24 of the result's, as a root of these squares, times 1.6, since weights of different
    sizes make a sum's steps uneven:
      * a sum of n products of either sign in one go: n / 6, for its k-th partial sum is sqrt(k / n) of the whole and rounded once, by
        u / sqrt(3) of itself on average (16 to 82 u here); in two levels, 64 products and then n / 64 sums: 64 / 6 + n / 384;
      * a score, a sum of D products and 1.5 in size, moves its P by 1.5 sqrt(D / 6) u; dP, for dq and dk, is off by sqrt(D / 6) u of itself;
      * the gradients' P = 2^(S log2 e - lse log2 e): with X = log2 e (ln n + 1.2) for the size of lse and h u the half step of numbers of
        that size (h = 8 from 8 to 16), lse, its product with log2 e and the difference are rounded once each, which moves P by
        h, h ln 2 and h ln 2 over sqrt(3) at most: 0.65 h^2;
      * exp and the last rounding: 2 u.
    (First written as 14 u for every case, then without dP's and the exponents' own roundings: errors of 14.1, 12.8 and 12.6 u, of dq, dq and dk,
    showed that terms were missing, not digits.)"""
    from geoweave_b200 import check_status
    from geoweave_b200.custom_flash_attn import packed_flash_attn_func

    g = torch.Generator().manual_seed(H + D)
    mk = lambda n, h, size=1.0: (torch.randn(n, h, D, generator=g) * size).cuda()
    q, k, v, up = mk(sum(lens_q), H, 1.5), mk(sum(lens_k), Hk), mk(sum(lens_k), Hk), mk(sum(lens_q), H)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    most = 1 if max(lens_q) == 1 else None
    o = packed_flash_attn_func(*leaves, borders(lens_q, q.device), borders(lens_k, q.device), causal, None, most)
    got = (o, *torch.autograd.grad(o, leaves, up))
    check_status()
    ref = packed_reference(q.detach(), k.detach(), v.detach(), lens_q, lens_k, causal, D ** -0.5, up)
    for name, x in zip(("o", "dq", "dk", "dv"), got):
        value = ref[name][0]
        off = (x.double() - value).norm() / value.norm()
        n = max(lens_k) if name in ("o", "dq") else max(lens_q) * (H // Hk)
        h = 2.0 ** math.floor(math.log2((math.log(max(lens_k)) + 1.2) / math.log(2)))
        squares = 64 / 6 + n / 384 + 1.5 ** 2 * D / 6 + 4 + (D / 6 if name in ("dq", "dk") else 0) + (0 if name == "o" else 0.65 * h * h)
        limit = 1.6 * math.sqrt(squares)
        assert off <= limit * 2.0 ** -24, f"{name}: {off * 2 ** 24:.1f} half steps, at most {limit:.1f}"
