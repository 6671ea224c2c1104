"""Attention over packed sequences against a plain implementation in 64 bits, with bounds that follow from the arithmetic."""
import math

import pytest
import torch

from tests.packed_reference import assert_within, borders, packed_reference

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _inputs(lens_q, lens_k, H, Hk, D, dtype, seed, tail_q=0, tail_k=0):
    from tests.gpu_util import dev

    g = torch.Generator().manual_seed(seed)
    T, S = sum(lens_q) + tail_q, sum(lens_k) + tail_k
    mk = lambda *s: torch.randn(s, generator=g).to(dtype).to(dev())
    return mk(T, H, D), mk(S, Hk, D), mk(S, Hk, D), mk(T, H, D)


def _forward(q, k, v, lens_q, lens_k, causal, scale=None, max_q=None):
    from geoweave_b200 import check_status
    from geoweave_b200.custom_flash_attn import packed_flash_attn_inference_func

    o, lse = packed_flash_attn_inference_func(q, k, v, borders(lens_q, q.device), borders(lens_k, q.device), causal, scale, max_q, True)
    check_status()
    return o, lse


def _check(lens_q, lens_k, H, Hk, D, dtype, causal, seed=0, train=True, scale=None, tail_q=0, tail_k=0, max_q=None):
    from geoweave_b200 import check_status
    from geoweave_b200.custom_flash_attn import packed_flash_attn_func

    q, k, v, g = _inputs(lens_q, lens_k, H, Hk, D, dtype, seed, tail_q, tail_k)
    ref = packed_reference(q, k, v, lens_q, lens_k, causal, scale or 1 / math.sqrt(D), g if train else None)
    o, lse = _forward(q, k, v, lens_q, lens_k, causal, scale, max_q)
    assert o.dtype == dtype and lse.dtype == torch.float32
    assert_within("o", o, ref["o"])
    assert_within("lse", lse, ref["lse"])
    if train:
        q, k, v = [x.requires_grad_() for x in (q, k, v)]
        o2 = packed_flash_attn_func(q, k, v, borders(lens_q, q.device), borders(lens_k, q.device), causal, scale, max_q)
        assert torch.equal(o2, o)
        grads = torch.autograd.grad(o2, (q, k, v), g)
        check_status()
        for name, x in zip(("dq", "dk", "dv"), grads):
            assert x.dtype == dtype
            assert_within(name, x, ref[name])


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 127, 128, 129, 255, 256, 257, 400])
def test_one_sequence_of_every_awkward_length(n, dtype, D, causal):
    _check([n], [n], 2, 2, D, dtype, causal, seed=n)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,Hk,D", [(4, 4, 64), (4, 1, 64), (6, 2, 128), (3, 3, 8), (2, 1, 24), (4, 2, 72), (2, 2, 96), (2, 2, 80), (2, 2, 120)])
def test_ragged_sequences_head_groups_and_head_dims(H, Hk, D, dtype, causal):
    _check([5, 0, 130, 1, 300, 64], [5, 0, 130, 1, 300, 64], H, Hk, D, dtype, causal, seed=H + D)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_query_and_key_lengths_differ_empty_sides_and_rows_without_a_key(dtype, causal):
    # causal with more queries than keys leaves the first queries without a key; a side may be empty
    lens_q, lens_k = [7, 300, 40, 0, 129, 128, 3], [19, 20, 0, 33, 500, 128, 257]
    _check(lens_q, lens_k, 4, 2, 64, dtype, causal, seed=3)
    _check(lens_q, lens_k, 2, 2, 128, dtype, causal, seed=4)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_many_short_sequences(dtype, D):
    lens = [(7 * i) % 23 for i in range(150)]  # several rounds of the 32-wide border scan, zero lengths among them
    _check(lens, lens, 2, 1, D, dtype, True, seed=5)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float16, 128), (torch.bfloat16, 40)])
def test_more_work_than_blocks(dtype, D, causal):
    """Several hundred items of every kind (full, half, and empty second tiles, no keys, more than eight key tiles), so that each
    block takes several in a row."""
    lens_q = [270, 17, 256, 129, 700, 0, 128, 1, 385, 513, 90, 260] * 3
    lens_k = [270, 17, 300, 129, 1200, 5, 0, 640, 100, 513, 128, 260] * 3
    _check(lens_q, lens_k, 16, 4, D, dtype, causal, seed=30)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
def test_rows_behind_the_last_sequence_are_zeros(dtype, causal):
    _check([100, 33], [70, 200], 2, 1, 64, dtype, causal, seed=6, tail_q=700, tail_k=450)
    _check([], [], 2, 1, 64, dtype, causal, seed=6, tail_q=70, tail_k=45)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_non_finite_values_stay_in_their_sequence_and_behind_it(dtype, D, causal):
    from geoweave_b200.custom_flash_attn import packed_flash_attn_func

    lens = [77, 130, 140]
    q, k, v, g = _inputs(lens, lens, 2, 2, D, dtype, 7, 90, 90)
    clean = packed_reference(q, k, v, lens, lens, causal, 1 / math.sqrt(D), g)
    for x, bad in ((q, float("nan")), (k, float("inf")), (v, float("nan")), (g, float("inf"))):
        x[77:77 + 130] = bad          # the middle sequence
        x[sum(lens):] = float("nan")  # behind the last one
    q, k, v = [x.requires_grad_() for x in (q, k, v)]
    cu = borders(lens, q.device)
    o = packed_flash_attn_func(q, k, v, cu, None, causal)
    grads = torch.autograd.grad(o, (q, k, v), g)
    for name, x in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        for rows in (slice(0, 77), slice(207, 347)):
            assert_within(name, x[rows], tuple(y[rows] for y in clean[name]))
        assert (x[sum(lens):] == 0).all(), name


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_large_scores_and_a_running_maximum_that_keeps_rising(dtype, D):
    from geoweave_b200 import check_status

    n = 700
    q, k, v, g = _inputs([n], [n], 2, 2, D, dtype, 8)
    k = (k.float() * torch.linspace(0.01, 6.0, n, device=k.device)[:, None, None]).to(dtype)  # later keys score far higher
    for scale in (0.125, 1.0, 1e-4):
        ref = packed_reference(q, k, v, [n], [n], False, scale, None)
        o, lse = _forward(q, k, v, [n], [n], False, scale)
        assert_within("o", o, ref["o"])
        assert_within("lse", lse, ref["lse"])


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_views_equal_contiguous_tensors(dtype):
    from geoweave_b200.custom_flash_attn import packed_flash_attn_func
    from tests.gpu_util import dev

    lens = [150, 61]
    g = torch.Generator().manual_seed(9)
    fused = torch.randn(sum(lens), 4 + 2 + 2, 64, generator=g).to(dtype).to(dev())
    views = [fused[:, :4], fused[:, 4:6], fused[:, 6:]]
    up = torch.randn(4, sum(lens), 64, generator=g).to(dtype).to(dev()).transpose(0, 1)  # a gradient of head-major strides
    odd = torch.randn(sum(lens) * 4 * 64 + 1, generator=g).to(dtype).to(dev())[1:].view(sum(lens), 4, 64)  # off 16-byte alignment
    cu = borders(lens, dev())
    for q in (views[0], odd, fused[:, :1].expand(-1, 4, -1)):
        for grad in (up, torch.ones((), dtype=dtype, device=dev()).expand(sum(lens), 4, 64)):
            results = []
            for a, b, c, d in ((q, views[1], views[2], grad), tuple(x.contiguous().clone() for x in (q, views[1], views[2], grad))):
                a, b, c = [x.detach().requires_grad_() for x in (a, b, c)]
                o = packed_flash_attn_func(a, b, c, cu, None, True)
                results.append((o, *torch.autograd.grad(o, (a, b, c), d)))
            for x, y in zip(*results):
                assert torch.equal(x, y)


def test_gradients_against_differences():
    """fp32: a directional derivative of <o, g> by central differences.  Curvature and rounding: the step h = 1e-2 leaves
    h^2/6 times a third derivative of order one along a unit direction, and 2^-20 / h from rounding: 2e-3 relative."""
    from geoweave_b200.custom_flash_attn import packed_flash_attn_func

    lens = [70, 33]
    q, k, v, g = _inputs(lens, lens, 4, 2, 64, torch.float32, 10)
    cu = borders(lens, q.device)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(packed_flash_attn_func(*leaves, cu, None, True), leaves, g)
    for i in range(3):
        d = torch.randn(leaves[i].shape, generator=torch.Generator().manual_seed(i)).to(q.device)
        d = d / d.norm()
        along = [(grads[i] * d).sum().double()]
        h, vals = 1e-2, []
        for s in (1, -1):
            moved = [x.detach().clone() for x in leaves]
            moved[i] += s * h * d
            vals.append((packed_flash_attn_func(*moved, cu, None, True).double() * g.double()).sum())
        along.append((vals[0] - vals[1]) / (2 * h))
        size = grads[i].norm().double() / math.sqrt(grads[i].numel())
        assert (along[0] - along[1]).abs() <= 2e-3 * (along[1].abs() + size * math.sqrt(d.numel()) * 0.5)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float16, 128), (torch.bfloat16, 24), (torch.float32, 64)])
def test_a_few_hundred_rows_against_long_key_sequences(dtype, D, causal):
    """The keys of a row tile are divided among blocks: parts that end inside a tile, rows that see only the first parts or none, a
    sequence that is shorter than its neighbours' parts, rows behind the last sequence."""
    _check([130], [5003], 4, 2, D, dtype, causal, seed=60, train=True)
    _check([300, 17], [4100, 9], 2, 1, D, dtype, causal, seed=61, tail_q=200, tail_k=90)
    _check([700, 40, 1], [600, 2600, 3000], 2, 2, D, dtype, causal, seed=62)
    _check([20, 0], [0, 6000], 1, 1, D, dtype, causal, seed=63, train=False)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D", [64, 128])
def test_long_rows_of_grouped_heads(D, causal):
    """Few key tiles with many query tiles each, which two blocks share: even and odd numbers of pairs, one pair, none."""
    _check([1600], [200], 8, 1, D, torch.bfloat16, causal, seed=50)
    _check([1700, 1], [130, 300], 6, 2, D, torch.float16, causal, seed=51)
    _check([2900, 64], [1, 700], 4, 2, D, torch.bfloat16, causal, seed=52)
    _check([0, 3000], [90, 129], 4, 2, D, torch.float16, causal, seed=53, tail_k=300)


@pytest.mark.parametrize("dtype", DTYPES)
def test_runs_are_reproducible_and_a_graph_replays_with_other_borders(dtype):
    from geoweave_b200 import check_status
    from geoweave_b200.custom_flash_attn import packed_flash_attn_inference_func
    from geoweave_b200.custom_flash_attn.packed_flash_attn import packed_attention_backward, packed_attention_forward

    lens = [200, 100, 300]
    q, k, v, g = _inputs(lens, lens, 4, 2, 64, dtype, 11)
    cu = borders(lens, q.device)

    def step():
        o, lse = packed_attention_forward(q, k, v, cu, cu, True, return_lse=True)
        return (o, *packed_attention_backward(q, k, v, cu, cu, o, lse, g, True))

    first = step()
    for a, b in zip(first, step()):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    graph.replay()
    for a, b in zip(first, captured):
        assert torch.equal(a, b)
    cu.copy_(borders([10, 500, 60], q.device))
    graph.replay()
    expect = step()
    for a, b in zip(expect, captured):
        assert torch.equal(a, b)
    check_status()


def test_two_streams_at_once():
    from geoweave_b200.custom_flash_attn import packed_flash_attn_func

    lens = [500, 700]
    sets = [_inputs(lens, lens, 4, 4, 64, torch.bfloat16, s) for s in (20, 21)]
    cu = borders(lens, sets[0][0].device)

    def step(q, k, v, g):
        q, k, v = [x.detach().requires_grad_() for x in (q, k, v)]
        o = packed_flash_attn_func(q, k, v, cu, None, False)
        return (o, *torch.autograd.grad(o, (q, k, v), g))

    alone = [step(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    together = []
    for _ in range(3):
        for st, s in zip(streams, sets):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                together.append(step(*s))
    torch.cuda.synchronize()
    for i, got in enumerate(together):
        for a, b in zip(alone[i % 2], got):
            assert torch.equal(a, b)


@pytest.mark.parametrize("H,Hk,D", [(16, 16, 64), (16, 4, 64), (16, 1, 64), (8, 2, 128), (4, 4, 96), (2, 1, 8)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_single_tokens_against_long_key_sequences(H, Hk, D, dtype):
    lens_k = [1, 700, 0, 64, 65, 2500, 333, 127]
    _check([1] * len(lens_k), lens_k, H, Hk, D, dtype, True, seed=12, train=False, max_q=1)
    _check([1, 0, 1, 1, 0, 1, 1, 1], lens_k, H, Hk, D, dtype, False, seed=13, train=False, max_q=1, tail_q=3, tail_k=40)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
def test_a_few_queries_against_long_key_sequences(dtype, causal):
    _check([3, 2, 0, 4, 1], [900, 1, 50, 2, 1300], 8, 2, 64, dtype, causal, seed=14, train=True, max_q=4)


def test_single_tokens_non_finite_neighbours():
    lens_k = [100, 130, 61]
    q, k, v, _ = _inputs([1] * 3, lens_k, 8, 2, 64, torch.bfloat16, 15, 0, 100)
    ref = packed_reference(q, k, v, [1] * 3, lens_k, True, 0.125)
    k[100:230], v[100:230] = float("nan"), float("inf")
    k[291:], v[291:] = float("inf"), float("nan")
    o, _ = _forward(q, k, v, [1] * 3, lens_k, True, max_q=1)
    for b in (0, 2):
        assert_within("o", o[b:b + 1], tuple(x[b:b + 1] for x in ref["o"]))


def test_a_bound_on_the_queries_that_is_too_small_is_reported():
    import geoweave_b200
    from geoweave_b200.custom_flash_attn import packed_flash_attn_inference_func

    q, k, v, _ = _inputs([1, 3, 1], [50, 60, 70], 4, 4, 64, torch.bfloat16, 19)
    ref = packed_reference(q, k, v, [1, 3, 1], [50, 60, 70], False, 0.125)
    o, _ = packed_flash_attn_inference_func(q, k, v, borders([1, 3, 1], q.device), borders([50, 60, 70], q.device), max_seqlen_q=1)
    with pytest.raises(geoweave_b200.GeoWeaveError):
        geoweave_b200.check_status()
    for row in (0, 4):  # the sequences that keep to it
        assert_within("o", o[row:row + 1], tuple(x[row:row + 1] for x in ref["o"]))
    _check([1, 3, 1], [50, 60, 70], 4, 4, 64, torch.bfloat16, False, train=False, max_q=3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_single_tokens_and_training_captured_and_replayed(dtype):
    """Through the public entry points, autograd included: what a captured program does must follow its inputs."""
    from geoweave_b200 import check_status
    from geoweave_b200.custom_flash_attn import packed_flash_attn_func, packed_flash_attn_inference_func

    lens_k = [700, 33, 1500]
    q1, k, v, _ = _inputs([1] * 3, lens_k, 8, 2, 64, dtype, 22)
    qs, ks, vs, g = _inputs([200, 90], [200, 90], 4, 2, 64, dtype, 23)
    cu1, cuk, cus = borders([1] * 3, q1.device), borders(lens_k, q1.device), borders([200, 90], q1.device)

    def step():
        token, _ = packed_flash_attn_inference_func(q1, k, v, cu1, cuk, True, max_seqlen_q=1)
        leaves = [x.detach().requires_grad_() for x in (qs, ks, vs)]
        o = packed_flash_attn_func(*leaves, cus, None, True)
        return (token, o.detach(), *torch.autograd.grad(o, leaves, g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (24, 25):
        for old, new in zip((q1, k, v), _inputs([1] * 3, lens_k, 8, 2, 64, dtype, seed)):
            old.copy_(new)
        for old, new in zip((qs, ks, vs, g), _inputs([200, 90], [200, 90], 4, 2, 64, dtype, seed + 10)):
            old.copy_(new)
        for _ in range(3):
            graph.replay()
        for a, b in zip(step(), captured):
            assert torch.equal(a, b)
    check_status()


def test_offsets_beyond_32_bits():
    """A key sequence of more than 4 GiB a tensor: its last keys count as its first do.  The scores are set up so that a few far keys
    carry all the weight, which makes the result known without touching the rest."""
    from geoweave_b200 import check_status
    from geoweave_b200.custom_flash_attn import packed_flash_attn_inference_func
    from tests.gpu_util import dev

    n, D = (1 << 24) + 77, 128
    k = torch.zeros(n, 1, D, dtype=torch.bfloat16, device=dev())
    v = torch.zeros(n, 1, D, dtype=torch.bfloat16, device=dev())
    far = torch.tensor([5, n // 2 + 3, n - 2, n - 1], device=dev())
    k[far] = 4.0
    v[far] = torch.arange(1, 5, device=dev(), dtype=torch.bfloat16)[:, None, None]
    q = torch.full((300, 1, D), 1.0, dtype=torch.bfloat16, device=dev())
    cu_k = borders([n], dev())
    # scores 512 / sqrt(128) = 45.25 for the four, 0 for the rest, whose share is n e^-45 < 1e-12: the mean of 1, 2, 3, 4
    for rows, most in ((1, 1), (16, 16), (300, None)):
        o, lse = packed_flash_attn_inference_func(q[:rows], k, v, borders([rows], dev()), cu_k, max_seqlen_q=most, return_lse=True)
        assert (o.float() - 2.5).abs().max() <= 2.5 * 2.0 ** -8
        assert (lse - (512 / math.sqrt(128) + math.log(4))).abs().max() <= 1e-4
    # causal: the row before the last does not see the last key
    o, _ = packed_flash_attn_inference_func(q[:2], k, v, borders([2], dev()), cu_k, True, max_seqlen_q=2)
    assert (o[0].float() - 2.0).abs().max() <= 2.0 ** -7 and (o[1].float() - 2.5).abs().max() <= 2.5 * 2.0 ** -8
    check_status()


def test_bad_borders_are_reported_and_nothing_is_lost():
    import geoweave_b200
    from geoweave_b200.custom_flash_attn import packed_flash_attn_func, packed_flash_attn_inference_func

    q, k, v, g = _inputs([100], [100], 2, 2, 64, torch.bfloat16, 16)
    for bad in ([0, 500], [0, 60, 40, 100], [5, 100], [-3, 100], [0, -7, 100]):
        cu = torch.tensor(bad, dtype=torch.int32, device=q.device)
        for most in (None, 1):
            packed_flash_attn_inference_func(q, k, v, cu, None, False, None, most)
            with pytest.raises(geoweave_b200.GeoWeaveError):
                geoweave_b200.check_status()
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        o = packed_flash_attn_func(*leaves, cu, None, True)
        torch.autograd.grad(o, leaves, g)
        with pytest.raises(geoweave_b200.GeoWeaveError):
            geoweave_b200.check_status()
    _check([100], [100], 2, 2, 64, torch.bfloat16, False)  # the next call is right again


def test_borders_that_name_more_tiles_than_there_are_rows_are_reported():
    """Overlapping sequences leave no spare block, which is where the rows behind the last sequence are dealt with."""
    import geoweave_b200
    from geoweave_b200.custom_flash_attn import packed_flash_attn_func, packed_flash_attn_inference_func

    for dtype in DTYPES:
        q, k, v, g = _inputs([2000], [2000], 2, 2, 64, dtype, 40)
        cu = torch.tensor([0, 2000] * 8, dtype=torch.int32, device=q.device)
        for most in (None, 1):
            packed_flash_attn_inference_func(q, k, v, cu, None, False, None, most)
            with pytest.raises(geoweave_b200.GeoWeaveError):
                geoweave_b200.check_status()
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        torch.autograd.grad(packed_flash_attn_func(*leaves, cu), leaves, g)
        with pytest.raises(geoweave_b200.GeoWeaveError):
            geoweave_b200.check_status()


def test_changes_between_forward_and_backward_are_noticed():
    from geoweave_b200.custom_flash_attn import packed_flash_attn_func
    from geoweave_b200.rotary import apply_rotary_axes, rotary_axes

    q, k, v, g = _inputs([50], [50], 2, 2, 64, torch.bfloat16, 41)
    cu = borders([50], q.device)
    leaf = q.clone().requires_grad_()
    o = packed_flash_attn_func(leaf, k, v, cu)
    k.add_(1)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(o, leaf, g)
    axes = rotary_axes((32, 32), 8, q.device)
    out, _ = apply_rotary_axes(leaf, None, torch.zeros(50, 2, dtype=torch.int64, device=q.device), axes)
    axes.cos.add_(1)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out, leaf, g)
    o = packed_flash_attn_func(leaf, k, v, cu)
    (first,) = torch.autograd.grad(o, leaf, g, create_graph=True)
    with pytest.raises(RuntimeError):  # no second derivative, and no silent zero in its place
        torch.autograd.grad(first.sum(), leaf)


def test_refusals():
    from geoweave_b200.custom_flash_attn import packed_flash_attn_func as f

    q, k, v, _ = _inputs([10], [10], 4, 2, 64, torch.bfloat16, 17)
    cu = borders([10], q.device)
    for call, error in [
        (lambda: f(q[None], k, v, cu), ValueError), (lambda: f(q, k, v[:5], cu), ValueError), (lambda: f(q, k[:5], v[:5], cu), ValueError),
        (lambda: f(q[:, :3], k, v, cu), ValueError), (lambda: f(q[..., :60], k[..., :60], v[..., :60], cu), ValueError),
        (lambda: f(q, k.float(), v, cu), TypeError), (lambda: f(q.double(), k.double(), v.double(), cu), TypeError),
        (lambda: f(q, k, v, cu.long()), TypeError), (lambda: f(q, k, v, cu.cpu()), ValueError), (lambda: f(q, k, v, cu[None]), ValueError),
        (lambda: f(q, k, v, cu, borders([5, 5], q.device)), ValueError), (lambda: f(q, k, v, cu, None, False, 0.0), ValueError),
        (lambda: f(q, k, v, cu, None, False, -1.0), ValueError), (lambda: f(q, k, v, cu, None, False, float("nan")), ValueError),
        (lambda: f(q, k, v, cu, None, False, None, -1), ValueError), (lambda: f(q.cpu(), k.cpu(), v.cpu(), cu.cpu()), ValueError),
    ]:
        with pytest.raises(error):
            call()
    empty = f(q[:0], k, v, borders([0], q.device), cu)
    assert empty.shape == (0, 4, 64)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rotary_then_attention_as_a_frame_block_uses_them(dtype):
    """q, k, v sliced from one projection, turned by time, height and width, attended view by view, and back again."""
    from geoweave_b200 import check_status
    from geoweave_b200.custom_flash_attn import packed_flash_attn_func
    from geoweave_b200.rotary import apply_rotary_axes, rotary_axes
    from tests.gpu_util import dev

    views, per, H, D, widths = 3, 5 + 6 * 7, 4, 64, (16, 24, 24)
    n = views * per
    g = torch.Generator().manual_seed(18)
    fused = torch.randn(n, 3 * H, D, generator=g).to(dtype).to(dev()).requires_grad_()
    up = torch.randn(n, H, D, generator=g).to(dtype).to(dev())
    pos = torch.randint(0, 40, (n, 3), generator=g).to(dev())
    axes = rotary_axes(widths, 40, dev())
    cu = borders([per] * views, dev())
    q, k = apply_rotary_axes(fused[:, :H], fused[:, H:2 * H], pos, axes)
    o = packed_flash_attn_func(q, k, fused[:, 2 * H:], cu)
    (grad,) = torch.autograd.grad(o, fused, up)
    check_status()

    x = fused.detach().double().requires_grad_()
    parts = []
    for lo in (0, H):
        at, cols = 0, []
        for a, w in enumerate(widths):
            z = torch.complex(x[:, lo:lo + H, at:at + w // 2], x[:, lo:lo + H, at + w // 2:at + w])
            ang = pos[:, a].double()[:, None] * 100.0 ** (-torch.arange(w // 2, device=dev()).double() * 2 / w)
            z = z * torch.polar(torch.ones_like(ang), ang)[:, None]
            cols += [z.real, z.imag]
            at += w
        parts.append(torch.cat(cols, -1))
    qs, ks, vs = [y.view(views, per, H, D).transpose(1, 2) for y in (*parts, x[:, 2 * H:])]
    ref = (torch.softmax(qs @ ks.transpose(-1, -2) / 8, -1) @ vs).transpose(1, 2).reshape(n, H, D)
    (gref,) = torch.autograd.grad(ref, x, up.double())
    # q and k are rounded on the way (scores move by a few u sum|q||k|/8), then P, o and dS: some twenty half steps of values near
    # one, against plain errors that are orders above
    u = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}[dtype]
    assert (o.double() - ref).norm() <= 8 * u * ref.norm()
    assert (grad.double() - gref).norm() <= 16 * u * gref.norm()
