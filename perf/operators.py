"""The operators of a dense attention block over several views, as measurable cases: rotary positions with several axes,
and attention over packed sequences (frames, a whole scene, ragged causal prompts, single query tokens), each with its
backward pass.

``listed()`` names the cases, ``draw(rng)`` makes more of the same ranges, ``prepare`` builds what a program has in hand
before the call, and ``run`` makes one pass: the plain torch form, or with ``own`` set the calls of geoweave_b200.
``exact`` is the definition in 64 bits, ``work`` the bytes and operations that a pass cannot do without.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_FREQUENCY = 100.0  # base of the rotary frequencies (the VGGT and Pi3 value)
_SPECIAL = 5        # special tokens in front of each view's patches (camera and registers); they stand at position 0


# ------------------------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------------------------
def _rotary(name, views, rows, cols, heads, kv_heads, dims, dtype, train):
    """`dims`: how many of the head's columns each axis turns (time, height, width); 0 = the axis is absent, columns
    behind the last axis are left alone."""
    return {"name": name, "op": "rotary", "views": views, "rows": rows, "cols": cols, "heads": heads, "kv_heads": kv_heads,
            "dim": dims[3], "time_dim": dims[0], "height_dim": dims[1], "width_dim": dims[2], "dtype": dtype, "train": train}


def _attn(name, seqs, shortest, longest, query, heads, kv_heads, dim, causal, dtype, train, empty=False):
    """`seqs` key sequences with lengths from `shortest` to `longest`; `query` query rows for each (0: as many as keys);
    `empty`: the second sequence has no token."""
    return {"name": name, "op": "attention", "seqs": seqs, "shortest": shortest, "longest": longest, "query": query,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "causal": causal, "dtype": dtype, "train": train, "empty": empty}


def listed():
    return [
        # one view of 37 x 28 patches: the frame blocks' two-axis rotary embedding, where the launch counts
        _rotary("rotary_view", 1, 37, 28, 16, 16, (0, 32, 32, 64), "bf16", False),
        # the 32-view stack with time, height and width, q and k sliced from one projection's output
        _rotary("rotary_video", 32, 37, 28, 16, 16, (16, 24, 24, 64), "bf16", False),
        # a training step of a grouped-head model over 16 odd-sized views, wide heads that the axes do not fill
        _rotary("rotary_train", 16, 23, 31, 16, 4, (32, 48, 40, 128), "fp16", True),
        # one short caption-sized sequence: latency
        _attn("attn_short", 1, 37, 37, 0, 16, 16, 64, False, "bf16", False),
        # frame attention of 32 views: every view attends to itself
        _attn("attn_views", 32, 1041, 1041, 0, 16, 16, 64, False, "bf16", False),
        # a dense global layer over 32 views
        _attn("attn_scene", 1, 33312, 33312, 0, 16, 16, 64, False, "bf16", False),
        # causal prompts of very different lengths in one batch, grouped wide heads, one of them empty
        _attn("attn_prompts", 9, 61, 7001, 0, 16, 4, 128, True, "fp16", False, True),
        # one new token for each of 24 sequences with caches of different lengths
        _attn("attn_token", 24, 129, 33312, 1, 16, 4, 64, True, "bf16", False),
        # full-precision tokens, four small views
        _attn("attn_fp32", 4, 333, 1041, 0, 16, 16, 64, False, "fp32", True),
        # training: frame attention of 16 views
        _attn("attn_views_train", 16, 1041, 1041, 0, 16, 16, 64, False, "bf16", True),
        # training: a global layer over 8 views
        _attn("attn_scene_train", 1, 8328, 8328, 0, 16, 16, 64, False, "bf16", True),
        # training: ragged causal prompts, grouped wide heads
        _attn("attn_prompts_train", 7, 45, 4099, 0, 16, 4, 128, True, "bf16", True),
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, evenly over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = ((16, 16), (16, 4), (16, 2), (12, 12), (8, 8), (8, 1), (4, 2))


def _pairs(case):
    """Allowed (query, key) pairs of a case, over all sequences."""
    total = 0
    for lq, lk in zip(*_lengths(case)):
        if case["causal"]:  # the last query sees every key; query i sees i + lk - lq + 1 keys
            first = max(0, lq - lk)
            rows = lq - first
            total += rows * (first + lk - lq + 1) + rows * (rows - 1) // 2
        else:
            total += lq * lk
    return total


def draw(rng):
    kind = rng.choice(("rotary", "rotary", "prompt", "prompt", "train", "train", "token"))
    heads, kv_heads = rng.choice(_HEADS)
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp16", "fp32"))
    if kind == "rotary":
        dims = rng.choice(((0, 32, 32, 64), (16, 24, 24, 64), (32, 48, 40, 128), (16, 56, 56, 128), (64, 0, 0, 64), (8, 12, 12, 32)))
        case = _rotary("", _spread(rng, 1, 32), _spread(rng, 4, 37), _spread(rng, 4, 37), heads, kv_heads, dims, dtype,
                       rng.random() < 0.4)
        del case["name"]
        return case
    dim = rng.choice((64, 64, 64, 128, 128, 96, 80, 32))
    while True:
        if kind == "token":
            seqs = _spread(rng, 1, 48)
            longest = _spread(rng, 1, 33312)
            case = _attn("", seqs, max(1, longest // rng.choice((1, 7, 200))), longest, 1, heads, kv_heads, dim, True, dtype, False)
            limit = 6e8
        else:
            seqs = _spread(rng, 1, 32)
            longest = _spread(rng, 16, 8328)
            query = 0 if rng.random() < 0.8 else _spread(rng, 2, 1041)
            case = _attn("", seqs, max(1, longest // rng.choice((1, 3, 40))), longest, query, heads, kv_heads, dim,
                         rng.random() < 0.5, dtype, kind == "train", seqs > 2 and rng.random() < 0.25)
            limit = 2e9 if dtype == "fp32" else 4e10
        tokens = sum(_lengths(case)[1])
        if _pairs(case) * heads * dim <= limit and 0 < tokens <= 400000:
            del case["name"]
            return case


def _lengths(case):
    """Query and key lengths of a case's sequences."""
    n, lo, hi = case["seqs"], case["shortest"], case["longest"]
    ladder = [int(round(lo * (hi / lo) ** (i / (n - 1)))) if n > 1 else hi for i in range(n)]
    keys = [ladder[(5 * i + 2) % n] if n % 5 else ladder[(3 * i + 2) % n] if n % 3 else ladder[i] for i in range(n)]
    if case["empty"] and n > 1:
        keys[1] = 0
    return [case["query"] or k for k in keys], keys


def _axes(case):
    return [(i, d) for i, d in enumerate((case["time_dim"], case["height_dim"], case["width_dim"])) if d]


def _tokens(case):
    return case["views"] * (_SPECIAL + case["rows"] * case["cols"])


# ------------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------------
def _positions(case):
    """int64 [tokens, axes]: (view, row + 1, column + 1) of each patch; a view's special tokens stand at row and column 0."""
    v, r, c = case["views"], case["rows"], case["cols"]
    t = np.repeat(np.arange(v), _SPECIAL + r * c)
    y = np.concatenate((np.zeros(_SPECIAL, np.int64), np.repeat(np.arange(r) + 1, c)))
    x = np.concatenate((np.zeros(_SPECIAL, np.int64), np.tile(np.arange(c) + 1, r)))
    full = np.stack((t, np.tile(y, v), np.tile(x, v)), 1)
    return torch.from_numpy(np.ascontiguousarray(full[:, [i for i, _ in _axes(case)]])).cuda()


def _normal(shape, generator, dtype, scale=1.0):
    return (torch.randn(shape, generator=generator, device="cuda") * scale).to(dtype)


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    state = {"case": case}
    if case["op"] == "rotary":
        n = _tokens(case)
        fused = _normal((n, h + 2 * hk, d), generator, dtype)  # one projection's output: q, k and v side by side
        state["q"], state["k"] = fused[:, :h], fused[:, h:h + hk]
        state["pos"] = _positions(case)
        if case["train"]:
            state["dq"] = _normal((n, h, d), generator, dtype)
            state["dk"] = _normal((n, hk, d), generator, dtype)
            state["q"], state["k"] = state["q"].detach().requires_grad_(), state["k"].detach().requires_grad_()
        if own:
            from geoweave_b200.rotary import rotary_axes
            state["axes"] = rotary_axes([w for _, w in _axes(case)], 1 + max(case["views"], case["rows"], case["cols"]), "cuda",
                                        frequency=_FREQUENCY)
        return state
    lq, lk = _lengths(case)
    tq, tk = sum(lq), sum(lk)
    q = _normal((tq, h, d), generator, dtype, 1.5)  # scores of about 1.5 standard deviations after the 1/sqrt(d)
    k, v = _normal((tk, hk, d), generator, dtype), _normal((tk, hk, d), generator, dtype)
    if case["train"]:
        state["do"] = _normal((tq, h, d), generator, dtype)
        q, k, v = q.requires_grad_(), k.requires_grad_(), v.requires_grad_()
    state.update(q=q, k=k, v=v)
    state["lens"] = (lq, lk)
    state["cu_q"] = torch.tensor(np.concatenate(((0,), np.cumsum(lq))), dtype=torch.int32).cuda()
    state["cu_k"] = torch.tensor(np.concatenate(((0,), np.cumsum(lk))), dtype=torch.int32).cuda()
    return state


# ------------------------------------------------------------------------------------------------------------------
# the plain forms
# ------------------------------------------------------------------------------------------------------------------
def _turn(x, cos, sin, widths, sign):
    """Rotate each axis's columns: column j of an axis pairs with column j + width / 2."""
    x = x.float()
    out, at, angle = x.clone(), 0, 0
    for w in widths:
        half = w // 2
        a, b = x[..., at:at + half], x[..., at + half:at + w]
        c, s = cos[:, None, angle:angle + half], sign * sin[:, None, angle:angle + half]
        out[..., at:at + half] = a * c - b * s
        out[..., at + half:at + w] = b * c + a * s
        at, angle = at + w, angle + half
    return out


def _plain_rotary(state):
    case, q, k = state["case"], state["q"].detach(), state["k"].detach()
    widths = [w for _, w in _axes(case)]
    angles = torch.cat([state["pos"][:, i:i + 1].double() * _FREQUENCY ** (-torch.arange(0, w, 2, device="cuda").double() / w)
                        for i, w in enumerate(widths)], 1)
    cos, sin = torch.cos(angles).float(), torch.sin(angles).float()
    out = [_turn(x, cos, sin, widths, 1.0).to(x.dtype) for x in (q, k)]
    if case["train"]:
        out += [_turn(x, cos, sin, widths, -1.0).to(x.dtype) for x in (state["dq"], state["dk"])]
    return out


def _plain_attention(state):
    case = state["case"]
    q, k, v = (state[n].detach() for n in "qkv")
    h, hk, d, train = case["heads"], case["kv_heads"], case["dim"], case["train"]
    g, scale = h // hk, 1.0 / math.sqrt(d)
    out = torch.zeros_like(q)
    grads = [torch.zeros_like(x) for x in (q, k, v)] if train else []
    aq = ak = 0
    for lq, lk in zip(*state["lens"]):
        if lq and lk:
            # [kv heads, group, rows, d] against [kv heads, 1, keys, d], a band of rows at a time
            ks = k[ak:ak + lk].float().transpose(0, 1).unsqueeze(1)
            vs = v[ak:ak + lk].float().transpose(0, 1).unsqueeze(1)
            band = max(1, min(lq, 400_000_000 // (h * lk)))
            if train:
                dks, dvs = torch.zeros_like(ks), torch.zeros_like(vs)
            for r0 in range(0, lq, band):
                r1 = min(lq, r0 + band)
                qs = q[aq + r0:aq + r1].float().view(r1 - r0, hk, g, d).permute(1, 2, 0, 3)
                s = torch.matmul(qs, ks.transpose(-1, -2)) * scale
                if case["causal"]:
                    row = torch.arange(r0, r1, device="cuda") + (lk - lq)
                    hidden = torch.arange(lk, device="cuda")[None, :] > row[:, None]
                    s = s.masked_fill(hidden, float("-inf"))
                top = s.amax(-1, keepdim=True)
                top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
                p = torch.exp(s - top)
                total = p.sum(-1, keepdim=True)
                p = p / torch.where(total == 0, torch.ones_like(total), total)
                o = torch.matmul(p, vs)
                out[aq + r0:aq + r1] = o.permute(2, 0, 1, 3).reshape(r1 - r0, h, d).to(q.dtype)
                if train:
                    do = state["do"][aq + r0:aq + r1].float().view(r1 - r0, hk, g, d).permute(1, 2, 0, 3)
                    dp = torch.matmul(do, vs.transpose(-1, -2))
                    ds = p * (dp - (do * o).sum(-1, keepdim=True)) * scale
                    grads[0][aq + r0:aq + r1] = torch.matmul(ds, ks).permute(2, 0, 1, 3).reshape(r1 - r0, h, d).to(q.dtype)
                    dks += torch.matmul(ds.transpose(-1, -2), qs).sum(1, keepdim=True)
                    dvs += torch.matmul(p.transpose(-1, -2), do).sum(1, keepdim=True)
            if train:
                grads[1][ak:ak + lk] = dks.squeeze(1).transpose(0, 1).to(k.dtype)
                grads[2][ak:ak + lk] = dvs.squeeze(1).transpose(0, 1).to(v.dtype)
        aq, ak = aq + lq, ak + lk
    return [out] + grads


# ------------------------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if not own:
        return _plain_rotary(state) if case["op"] == "rotary" else _plain_attention(state)
    if case["op"] == "rotary":
        from geoweave_b200.rotary import apply_rotary_axes
        q, k = apply_rotary_axes(state["q"], state["k"], state["pos"], state["axes"])
        if not case["train"]:
            return [q, k]
        return [q.detach(), k.detach(), *torch.autograd.grad((q, k), (state["q"], state["k"]), (state["dq"], state["dk"]))]
    from geoweave_b200.custom_flash_attn import packed_flash_attn_func, packed_flash_attn_inference_func
    q, k, v = state["q"], state["k"], state["v"]
    most = case["query"] or case["longest"]
    if not case["train"]:
        o, _ = packed_flash_attn_inference_func(q, k, v, state["cu_q"], state["cu_k"], causal=case["causal"], max_seqlen_q=most)
        return [o]
    o = packed_flash_attn_func(q, k, v, state["cu_q"], state["cu_k"], causal=case["causal"], max_seqlen_q=most)
    return [o.detach(), *torch.autograd.grad(o, (q, k, v), state["do"])]


def work(case):
    size, h, hk, d = _BYTES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "rotary":
        n, times = _tokens(case), 2 if case["train"] else 1  # q and k in and out; in training their gradients too
        turned = sum(w for _, w in _axes(case))
        return {"bytes": times * 2 * n * (h + hk) * d * size + n * 8 * len(_axes(case)), "flops": times * 3 * n * (h + hk) * turned}
    lq, lk = _lengths(case)
    tq, tk = sum(lq), sum(lk)
    # forward: q, k, v in, o out, two products; training: do in, dq, dk, dv out, four products more
    moved = 2 * tq * h * d + 2 * tk * hk * d
    if case["train"]:
        moved += 2 * tq * h * d + 2 * tk * hk * d
    return {"bytes": moved * size + 8 * (case["seqs"] + 1), "flops": (6 if case["train"] else 2) * 2 * _pairs(case) * h * d}


# ------------------------------------------------------------------------------------------------------------------
# the definition, in 64 bits
# ------------------------------------------------------------------------------------------------------------------
def _exact_rotary(case, state):
    axes = _axes(case)
    x = {n: state[n].detach().double() for n in ("q", "k", "dq", "dk") if n in state}
    out = []
    for name, sign in (("q", 1), ("k", 1), ("dq", -1), ("dk", -1)):
        if name not in x:
            continue
        y, at = x[name].clone(), 0
        for i, (_, w) in enumerate(axes):
            # the pair (j, j + w/2) as one complex number, turned by position * frequency^(-2j/w)
            z = torch.complex(x[name][..., at:at + w // 2], x[name][..., at + w // 2:at + w])
            rate = torch.exp(torch.arange(w // 2, device="cuda", dtype=torch.float64) * (-2.0 / w) * math.log(_FREQUENCY))
            turn = sign * state["pos"][:, i].double()[:, None] * rate
            z = z * torch.polar(torch.ones_like(turn), turn)[:, None, :]
            y[..., at:at + w // 2], y[..., at + w // 2:at + w] = z.real, z.imag
            at += w
        out.append(y)
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(case, state)
    q, k, v = (state[n].detach().double() for n in "qkv")
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    out = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    aq = ak = 0
    for lq, lk in zip(*state["lens"]):
        for head in range(h if lq and lk else 0):
            kv = head // (h // hk)
            keys, values = k[ak:ak + lk, kv], v[ak:ak + lk, kv]
            band = max(1, min(lq, 100_000_000 // lk))
            for r0 in range(0, lq, band):
                rows = slice(aq + r0, aq + min(lq, r0 + band))
                n = rows.stop - rows.start
                logits = (q[rows, head] @ keys.T) / math.sqrt(d)
                alive = torch.ones(n, dtype=torch.bool, device="cuda")
                if case["causal"]:
                    last = torch.arange(r0, r0 + n, device="cuda") + lk - lq
                    logits[torch.arange(lk, device="cuda")[None] > last[:, None]] = -math.inf
                    alive = last >= 0
                weight = torch.zeros_like(logits)
                weight[alive] = torch.softmax(logits[alive], -1)
                out[rows, head] = weight @ values
                if case["train"]:
                    do = state["do"][rows, head].double()
                    dv[ak:ak + lk, kv] += weight.T @ do
                    flow = do @ values.T
                    flow = weight * (flow - (flow * weight).sum(-1, keepdim=True)) / math.sqrt(d)
                    dq[rows, head] = flow @ keys
                    dk[ak:ak + lk, kv] += flow.T @ q[rows, head]
        aq, ak = aq + lq, ak + lk
    return [out, dq, dk, dv] if case["train"] else [out]
