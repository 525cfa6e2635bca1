"""Mixture-of-experts operators against plain 64-bit formulas (one GPU)."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)


def _within(got, want, bound):
    """|got - want| <= bound elementwise (NaNs nowhere)."""
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst " \
                          f"{err[bad].max().item():.3e} at bound {bound[bad].min().item():.3e}"


# ------------------------------------------------------------------------------ routing
def _route64(logits, k, score, bias, groups, top_groups, group_score, renormalize, scale, mask):
    """Row by row in Python floats; returns (weights, ids) as tensors."""
    T, E = logits.shape
    w = torch.zeros(T, k, dtype=torch.float64)
    ids = torch.full((T, k), -1, dtype=torch.int32)
    rows = logits.double().cpu()
    b = [0.0] * E if bias is None else bias.double().cpu().tolist()
    for t in range(T):
        if mask is not None and not bool(mask[t]):
            continue
        l = rows[t].tolist()
        if all(v == -math.inf for v in l):
            continue
        if score == "softmax":
            m = max(l)
            e = [math.exp(v - m) for v in l]
            s = math.fsum(e)
            p = [v / s for v in e]
        else:
            p = [1 / (1 + math.exp(-v)) if v > -700 else 0.0 for v in l]
        alive = {e: p[e] + b[e] for e in range(E) if l[e] != -math.inf and b[e] != -math.inf}
        if groups > 1:
            per = E // groups
            score_of = {}
            for e, key in alive.items():
                score_of.setdefault(e // per, []).append(key)
            rank = sorted(score_of, key=lambda g: (-sum(sorted(score_of[g])[-(1 if group_score == "max" else 2):]), g))
            alive = {e: key for e, key in alive.items() if e // per in rank[:top_groups]}
        best = sorted(alive, key=lambda e: (-alive[e], e))[:k]
        total = math.fsum(p[e] for e in best) if renormalize else 1.0
        for j, e in enumerate(best):
            ids[t, j] = e
            w[t, j] = scale * p[e] / total
    return w.cuda(), ids.cuda()


ROUTE_CASES = [
    # tokens, experts, k, score, bias, groups, top_groups, group_score, renorm, scale
    (1, 8, 2, "softmax", False, 1, 1, "top2", True, 1.0),
    (1, 1, 1, "sigmoid", True, 1, 1, "top2", True, 1.0),
    (7, 33, 5, "softmax", True, 1, 1, "top2", False, 1.0),
    (130, 64, 8, "sigmoid", False, 1, 1, "top2", False, 2.5),
    (65, 256, 8, "sigmoid", True, 8, 4, "top2", True, 2.5),
    (33, 160, 6, "softmax", False, 8, 3, "max", False, 16.0),
    (29, 96, 6, "softmax", False, 4, 2, "top2", True, 1.0),
    (17, 512, 32, "softmax", False, 1, 1, "top2", True, 1.0),
    (9, 32, 3, "sigmoid", True, 32, 5, "top2", True, 1.0),       # groups of one expert
]


@pytest.mark.parametrize("case", ROUTE_CASES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_route_matches_formula(case, dtype):
    from tileccl_b200 import ops

    T, E, k, score, with_bias, groups, top_groups, gs, renorm, scale = case
    g = _gen(T + E)
    logits = _randn(g, T, E, std=2.0).to(dtype)
    bias = _randn(g, E, std=0.1) if with_bias else None
    w, ids = ops.route_experts(logits, k, score=score, bias=bias, groups=groups,
                               top_groups=top_groups, group_score=gs, renormalize=renorm,
                               scale=scale)
    ref_w, ref_ids = _route64(logits, k, score, bias, groups, top_groups, gs, renorm, scale, None)
    assert w.dtype == torch.float32 and torch.equal(ids, ref_ids)
    # exp within 2 ulp, its argument's rounding |l - m| 2^-24 (< 20 here), a sum of at most 512
    # positive terms, a division and a product: below 2^-24 * (4 + 20 + 10 + 2)
    _within(w, ref_w, ref_w * 36 * 2 ** -24)


def test_route_tells_close_keys_apart():
    """Scores that agree in 32 bits are told apart; equal ones go to the lower index."""
    from tileccl_b200 import ops

    logits = torch.full((3, 16), -4.0, device="cuda")
    logits[0, 5], logits[0, 9] = 9.0, 9.0000019          # sigmoids differ by 2^-32 or so
    logits[1, 9], logits[1, 5] = 9.0, 9.0000019
    logits[2, 3] = logits[2, 11] = 1.0
    bias = torch.full((16,), 0.25, device="cuda")
    for score in ("sigmoid", "softmax"):
        _, ids = ops.route_experts(logits, 3, score=score, bias=bias)
        assert ids[:, :2].tolist() == [[9, 5], [5, 9], [3, 11]]
        assert ids[:, 2].tolist() == [0, 0, 0]


def test_route_masks_and_unavailable_experts():
    from tileccl_b200 import ops

    inf, nan = math.inf, math.nan
    logits = torch.tensor([[1.0, 2.0, 3.0, 4.0],
                           [nan, inf, nan, 2.0],          # masked row
                           [-inf, 1.0, -inf, -inf],       # fewer experts than k
                           [-inf, -inf, -inf, -inf],
                           [0.0, nan, 1.0, -inf],
                           [-200.0, -201.0, -300.0, -inf]], device="cuda")
    mask = torch.tensor([True, False, True, True, True, True], device="cuda")
    for score in ("softmax", "sigmoid"):
        w, ids = ops.route_experts(logits, 3, score=score, mask=mask)
        assert ids.tolist() == [[3, 2, 1], [-1] * 3, [1, -1, -1], [-1] * 3, [2, 0, 1], [0, 1, 2]]
        assert w[1].tolist() == [0.0] * 3 and w[3].tolist() == [0.0] * 3
        assert w[2].tolist() == [1.0, 0.0, 0.0]
        assert torch.isnan(w[4]).all()
        # renormalised scores keep their ratio e where the scores themselves underflow
        assert abs(w[5, 0].item() - 1 / (1 + math.exp(-1))) < 1e-6
    bias = torch.tensor([0.0, 0.0, -inf, -inf], device="cuda")
    _, ids = ops.route_experts(logits[:1], 3, bias=bias)
    assert ids.tolist() == [[1, 0, -1]]
    # groups without an available expert stay behind
    grouped = torch.tensor([[-inf, -inf, -5.0, -inf]], device="cuda")
    _, ids = ops.route_experts(grouped, 2, score="sigmoid", groups=2, top_groups=1)
    assert ids.tolist() == [[2, -1]]
    w, ids = ops.route_experts(logits[:0], 2)
    assert tuple(w.shape) == tuple(ids.shape) == (0, 2)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("shape", [(1, 8, 2), (67, 33, 5), (40, 300, 8), (5, 64, 1)])
def test_route_backward(score, renorm, shape):
    from tileccl_b200 import ops

    T, E, k = shape
    g = _gen(E)
    big = _randn(g, T, E + 5, std=1.5)
    logits = big[:, :E]                                   # strided rows
    _, ids = ops.route_experts(logits, k, score=score, renormalize=renorm, scale=1.5)
    grad = _randn(g, T, k)
    if T > 2:
        ids[2, -1] = -1                                   # a place without an expert
    got = ops.route_experts_backward(grad, logits, ids, score=score, renormalize=renorm, scale=1.5)
    l = logits.double().requires_grad_(True)
    p = torch.softmax(l, 1) if score == "softmax" else torch.sigmoid(l)
    here = ids >= 0
    c = p.gather(1, ids.clamp(min=0).long()) * here
    none = ~here.any(1, keepdim=True)                     # (a token without any expert: 0 / 1)
    w = 1.5 * (c / (c.sum(1, keepdim=True) + none) if renorm else c)
    (w * grad.double()).sum().backward()
    # terms are at most scale * |p| * (|g| + sum |g w|); each carries the 36 half steps of a
    # weight and as many again for the dot product
    size = 1.5 * p.detach() * (2 + grad.double().abs().sum(1, keepdim=True))
    if renorm:
        size = size / (c.detach().sum(1, keepdim=True) + none)
    _within(got, l.grad, 80 * 2 ** -24 * size)
    # and against differences of the forward pass in 64 bits, in one direction
    d = _randn(g, T, E).double() * 1e-5

    def loss(x):
        q = torch.softmax(x, 1) if score == "softmax" else torch.sigmoid(x)
        cc = q.gather(1, ids.clamp(min=0).long()) * here
        return (1.5 * (cc / (cc.sum(1, keepdim=True) + none) if renorm else cc) * grad.double()).sum()

    diff = (loss(logits.double() + d) - loss(logits.double() - d)) / 2
    want = (got.double() * d).sum()
    assert abs(diff - want) <= 1e-5 * (got.double().abs() * d.abs()).sum()


def test_route_backward_unrouted_rows_are_zero():
    from tileccl_b200 import ops

    logits = torch.full((2, 40), math.nan, device="cuda")
    logits[1] = 0.5
    logits[1, 3] = -math.inf
    ids = torch.tensor([[-1, -1], [4, 7]], dtype=torch.int32, device="cuda")
    for score in ("softmax", "sigmoid"):
        for renorm in (False, True):
            d = ops.route_experts_backward(torch.ones(2, 2, device="cuda"), logits, ids, score=score,
                                           renormalize=renorm)
            assert (d[0] == 0).all() and d[1, 3] == 0 and torch.isfinite(d).all()


# ------------------------------------------------------------------------------ slot map
def test_slots_of_a_very_large_batch():
    """Beyond 256 CTAs the counts are summed by a kernel of their own."""
    from tileccl_b200 import ops

    tokens, k, experts = 150_003, 8, 300
    ids = torch.randint(-3, experts, (tokens, k), device="cuda", generator=_gen(77)).int()
    s = ops.expert_slots(ids, 290, first_expert=5)
    flat = ids.reshape(-1).long() - 5
    here = (flat >= 0) & (flat < 290)
    key = torch.where(here, flat, torch.full_like(flat, 290))
    order = torch.sort(key, stable=True).indices
    used = int(here.sum())
    counts = torch.bincount(key, minlength=291)[:290]
    assert s.offsets.tolist() == [0] + counts.cumsum(0).tolist()
    assert torch.equal(s.token_of_slot[:used].long(), order[:used] // k)
    assert (s.token_of_slot[used:] == -1).all()
    want = torch.full_like(flat, -1)
    want[order[:used]] = torch.arange(used, device="cuda")
    assert torch.equal(s.slot_of.reshape(-1).long(), want)


@pytest.mark.parametrize("tokens, k, experts, first, local", [
    (0, 2, 4, 0, 4), (1, 1, 1, 0, 1), (1, 8, 64, 0, 64), (37, 3, 5, 1, 3), (512, 8, 8, 0, 8),
    (513, 8, 8, 2, 2), (2049, 2, 1024, 0, 1024), (5000, 6, 61, 60, 1), (20011, 8, 256, 128, 128)])
def test_slots(tokens, k, experts, first, local):
    from tileccl_b200 import ops

    g = _gen(tokens + 1)
    ids = torch.randint(-1, experts, (tokens, k), device="cuda", generator=g).int()
    s = ops.expert_slots(ids, local, first_expert=first)
    flat = ids.reshape(-1).long().cpu() - first
    here = (flat >= 0) & (flat < local)
    order = sorted(torch.nonzero(here).flatten().tolist(), key=lambda i: (int(flat[i]), i))
    counts = torch.bincount(flat[here], minlength=local)
    assert s.offsets.tolist() == [0] + counts.cumsum(0).tolist()
    tok = torch.full((tokens * k,), -1, dtype=torch.int32)
    tok[:len(order)] = torch.tensor([i // k for i in order], dtype=torch.int32)
    slot = torch.full((tokens * k,), -1, dtype=torch.int32)
    if order:
        slot[torch.tensor(order)] = torch.arange(len(order), dtype=torch.int32)
    assert torch.equal(s.token_of_slot.cpu(), tok)
    assert torch.equal(s.slot_of.cpu().reshape(-1), slot)


# ----------------------------------------------------------------------------- products
def _make_slots(g, tokens, k, experts, lost=0.0):
    from tileccl_b200 import ops

    ids = _randn(g, tokens, experts).topk(k, 1).indices.int()
    if lost:
        drop = torch.rand(tokens, k, device="cuda", generator=g) < lost
        ids = torch.where(drop, torch.full_like(ids, -1), ids)
    return ops.expert_slots(ids, experts)


def _sum_bound(a, b, terms):
    """Error of an fp32 sum of `terms` products in any order, the tensor cores' truncating
    additions (2^-23 each) included."""
    return terms * 2 ** -23 * (a.abs() @ b.abs())


def _pairs(N):
    """Columns of gate and up in packed order."""
    c = torch.arange(N // 2, device="cuda")
    gate = (c // 128) * 256 + c % 128
    return gate, gate + 128


def _ref_product(x, w, gate):
    """(out, bound before rounding) of one expert in 64 bits; w is [K, N]."""
    x, w = x.double(), w.double()
    y, dy = x @ w, _sum_bound(x, w, x.shape[1])
    if not gate:
        return y, dy
    cg, cu = _pairs(w.shape[1])
    a, u, da, du = y[:, cg], y[:, cu], dy[:, cg], dy[:, cu]
    s = torch.sigmoid(a)
    out = a * s * u
    # |silu'| < 1.1; exp and the division of the epilogue carry a few 2^-22 of relative error
    # (the fast exponential's grows with its argument: |a| 2^-23)
    return out, 1.1 * u.abs() * da + (a * s).abs() * du + da * du * 1.1 + \
        out.abs() * (8 + a.abs()) * 2 ** -22


PRODUCT_CASES = [
    # tokens, k, experts, K, N, lost
    (1, 1, 1, 8, 256, 0.0),
    (1, 2, 8, 64, 256, 0.0),
    (3, 2, 4, 72, 512, 0.3),
    (40, 4, 16, 136, 256, 0.0),
    (200, 2, 3, 320, 768, 0.0),
    (700, 3, 5, 1024, 512, 0.1),
    (1100, 1, 2, 512, 1024, 0.0),
    # long contractions of few rows: tiles shared among the SMs
    (1, 2, 8, 4096, 768, 0.0),
    (5, 2, 8, 4168, 1280, 0.2),
    (60, 2, 3, 4096, 256, 0.0),
]


@pytest.mark.parametrize("case", PRODUCT_CASES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b_is_nk", [False, True])
@pytest.mark.parametrize("rows", ["tokens", "slots"])
@pytest.mark.parametrize("epilogue", ["none", "silu_gate"])
def test_expert_gemm(case, dtype, b_is_nk, rows, epilogue):
    from tileccl_b200 import ops

    T, k, E, K, N, lost = case
    gate = epilogue == "silu_gate"
    if not gate:
        N -= 8 * (E % 4)                                  # odd widths without the gate
    g = _gen(T + K)
    slots = _make_slots(g, T, k, E, lost)
    X = _randn(g, T if rows == "tokens" else T * k, K, std=K ** -0.5, dtype=dtype)
    W = _randn(g, E, N, K, dtype=dtype) if b_is_nk else _randn(g, E, K, N, dtype=dtype)
    out = torch.full((T * k, N // 2 if gate else N), 7.0, dtype=dtype, device="cuda")
    got = ops.expert_gemm(X, W, slots, out, rows=rows, b_is_nk=b_is_nk, epilogue=epilogue)
    assert got is out
    off, tok = slots.offsets.tolist(), slots.token_of_slot.long()
    for e in range(E):
        a, b = off[e], off[e + 1]
        x = X[tok[a:b]] if rows == "tokens" else X[a:b]
        want, bound = _ref_product(x, W[e].t() if b_is_nk else W[e], gate)
        _within(out[a:b], want, bound + (want.abs() + bound) * _half_step(dtype) + 2 ** -25)
    assert (out[off[E]:] == 7.0).all()                    # behind the last slot


def test_expert_gemm_strided_operands_and_poisoned_neighbours():
    """Row pitches and expert pitches beyond the width; NaN in every place that must not be
    read into a result: other tokens' rows, rows behind the last slot, columns beside a view."""
    from tileccl_b200 import ops

    dtype, T, k, E, K, N = torch.bfloat16, 50, 2, 4, 200, 264
    g = _gen(3)
    ids = torch.randint(0, E, (T, k), device="cuda", generator=g).int()
    ids[:, 1] = -1
    ids[10:20] = -1                                       # tokens that no expert takes
    slots = ops.expert_slots(ids, E)
    big_x = torch.full((T, K + 64), math.nan, dtype=dtype, device="cuda")
    big_w = torch.full((E, K + 8, N + 24), math.nan, dtype=dtype, device="cuda")
    X, W = big_x[:, 8:8 + K], big_w[:, 8:, 8:8 + N]
    X.copy_(_randn(g, T, K, std=K ** -0.5))
    X[10:20] = math.nan
    W.copy_(_randn(g, E, K, N))
    big_out = torch.full((T * k, N + 16), 5.0, dtype=dtype, device="cuda")
    out = big_out[:, 8:8 + N]
    ops.expert_gemm(X, W, slots, out)
    off, tok = slots.offsets.tolist(), slots.token_of_slot.long()
    for e in range(E):
        a, b = off[e], off[e + 1]
        want, bound = _ref_product(X[tok[a:b]], W[e], False)
        _within(out[a:b], want, bound + (want.abs() + bound) * _half_step(dtype))
    assert (big_out[:, :8] == 5.0).all() and (big_out[:, 8 + N:] == 5.0).all()
    assert (out[off[E]:] == 5.0).all()
    # slot rows: the same with NaN behind the last slot and in the neighbours' rows
    Xs = torch.full((T * k, K), math.nan, dtype=dtype, device="cuda")
    Xs[:off[E]] = X[tok[:off[E]]]
    again = ops.expert_gemm(Xs, W, slots, rows="slots")
    assert torch.equal(again[:off[E]], out[:off[E]])


def test_expert_gemm_empty_experts_and_tokens():
    from tileccl_b200 import ops

    W = torch.randn(3, 64, 256, device="cuda").half()
    none = ops.expert_slots(torch.empty(0, 2, dtype=torch.int32, device="cuda"), 3)
    X = torch.empty(0, 64, device="cuda").half()
    assert tuple(ops.expert_gemm(X, W, none).shape) == (0, 256)
    gx, gw = ops.expert_gemm_backward(torch.empty(0, 256, device="cuda").half(), X, W, none)
    assert tuple(gx.shape) == (0, 64) and (gw == 0).all()
    assert tuple(ops.expert_combine(torch.empty(0, 256, device="cuda").half(), none).shape) == (0, 256)
    lost = ops.expert_slots(torch.full((5, 2), -1, dtype=torch.int32, device="cuda"), 3)
    X = torch.randn(5, 64, device="cuda").half()
    out = torch.ones(10, 256, device="cuda").half()
    ops.expert_gemm(X, W, lost, out)
    assert (out == 1).all()
    gx, gw = ops.expert_gemm_backward(out, X, W, lost)
    assert (gx == 0).all() and (gw == 0).all()


@pytest.mark.parametrize("case", [(1, 1, 1, 64, 256, 0.0), (70, 2, 4, 136, 512, 0.2),
                                  (300, 3, 7, 256, 256, 0.0), (900, 2, 3, 512, 768, 0.0),
                                  # few rows per expert: every block is an expert's last one
                                  (150, 4, 40, 264, 1024, 0.0)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b_is_nk", [False, True])
@pytest.mark.parametrize("rows", ["tokens", "slots"])
@pytest.mark.parametrize("epilogue", ["none", "silu_gate"])
def test_expert_gemm_backward(case, dtype, b_is_nk, rows, epilogue):
    from tileccl_b200 import ops

    T, k, E, K, N, lost = case
    gate = epilogue == "silu_gate"
    if not gate:
        N -= 8 * (E % 4)
    g = _gen(T + K + 1)
    slots = _make_slots(g, T, k, E, lost)
    S = T * k
    X = _randn(g, T if rows == "tokens" else S, K, std=K ** -0.5, dtype=dtype)
    W = _randn(g, E, N, K, dtype=dtype) if b_is_nk else _randn(g, E, K, N, dtype=dtype)
    dY = _randn(g, S, N // 2 if gate else N, std=0.25, dtype=dtype)
    off, tok = slots.offsets.tolist(), slots.token_of_slot.long()
    dY[off[E]:] = math.nan                                # behind the last slot: never read
    gx, gw = ops.expert_gemm_backward(dY, X, W, slots, rows=rows, b_is_nk=b_is_nk,
                                      epilogue=epilogue)
    u = _half_step(dtype)
    want_x = torch.zeros(X.shape, dtype=torch.float64, device="cuda")
    bound_x = torch.zeros_like(want_x)
    for e in range(E):
        a, b = off[e], off[e + 1]
        w = (W[e].t() if b_is_nk else W[e]).double()
        at = tok[a:b] if rows == "tokens" else torch.arange(a, b, device="cuda")
        x, dy = X[at].double(), dY[a:b].double()
        err = torch.zeros(b - a, N, dtype=torch.float64, device="cuda")
        if gate:
            y, ey = x @ w, _sum_bound(x, w, K)
            cg, cu = _pairs(N)
            ga, up, eg, eu = y[:, cg], y[:, cu], ey[:, cg], ey[:, cu]
            s = torch.sigmoid(ga)
            d = torch.zeros(b - a, N, dtype=torch.float64, device="cuda")
            d[:, cg] = dy * up * s * (1 + ga * (1 - s))
            d[:, cu] = dy * ga * s
            # |silu'| < 1.1, |silu''| <= 0.5; then the rounding of the operand to 16 bits
            fast = (8 + ga.abs()) * 2 ** -22
            err[:, cg] = dy.abs() * (1.1 * eu + 0.5 * up.abs() * eg
                                     + up.abs() * (1 + ga.abs()) * fast)
            err[:, cu] = dy.abs() * (1.1 * eg + (ga * s).abs() * fast)
            dy, err = d, err * 1.01 + (d.abs() + err) * u + 2 ** -25
        dx = dy @ w.t()
        bx = _sum_bound(dy.abs() + err, w.t(), N) + err @ w.t().abs()
        if rows == "slots":
            bx = bx + (dx.abs() + bx) * u                 # the result; token rows are summed in fp32
        dw = x.t() @ dy
        bw = _sum_bound(x.t(), dy.abs() + err, b - a) + x.t().abs() @ err
        got_w = gw[e].t() if b_is_nk else gw[e]
        _within(got_w, dw, bw + (dw.abs() + bw) * u + 2 ** -25)
        if rows == "tokens":
            want_x.index_add_(0, at, dx)
            bound_x.index_add_(0, at, bx)
        else:
            want_x[a:b], bound_x[a:b] = dx, bx
    if rows == "tokens":
        # (the bound of the fp32 products covers the sum of at most three of them)
        _within(gx, want_x, bound_x + (want_x.abs() + bound_x) * u + 2 ** -25)
    else:
        _within(gx[:off[E]], want_x[:off[E]], bound_x[:off[E]] + 2 ** -25)


def test_backward_against_differences():
    """Directional derivative of a scalar of the gated product against the gradients."""
    from tileccl_b200 import ops

    g = _gen(11)
    T, k, E, K, N, dtype = 60, 2, 3, 64, 256, torch.float16
    slots = _make_slots(g, T, k, E)
    X, W = _randn(g, T, K, std=K ** -0.5, dtype=dtype), _randn(g, E, K, N, dtype=dtype)
    dY = _randn(g, T * k, N // 2, dtype=dtype)
    gx, gw = ops.expert_gemm_backward(dY, X, W, slots, epilogue="silu_gate")
    off, tok = slots.offsets.tolist(), slots.token_of_slot.long()
    cg, cu = _pairs(N)

    def loss(x, w):
        total = 0.0
        for e in range(E):
            y = x[tok[off[e]:off[e + 1]]] @ w[e]
            total += (torch.nn.functional.silu(y[:, cg]) * y[:, cu] * dY[off[e]:off[e + 1]].double()).sum()
        return total

    x, w = X.double(), W.double()
    dx, dw = _randn(g, T, K).double() * 1e-4, _randn(g, E, K, N).double() * 1e-4
    diff = (loss(x + dx, w + dw) - loss(x - dx, w - dw)) / 2
    mine = (gx.double() * dx).sum() + (gw.double() * dw).sum()
    # two 16-bit roundings on the way to every gradient, signs at random over many terms
    size = math.sqrt((gx.double() * dx).square().sum() + (gw.double() * dw).square().sum())
    assert abs(diff - mine) <= 8 * 2 * _half_step(dtype) * size


# ------------------------------------------------------------------------------ combine
@pytest.mark.parametrize("tokens, k, n, lost, weighted, add", [
    (1, 1, 8, 0.0, True, False), (1, 8, 4096, 0.0, True, True), (5, 3, 264, 0.5, False, False),
    (300, 6, 1032, 0.2, True, True), (33, 2, 9000, 0.0, True, False)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_combine(tokens, k, n, lost, weighted, add, dtype):
    from tileccl_b200 import ops

    g = _gen(tokens + n)
    slots = _make_slots(g, tokens, k, 16, lost)
    used = int(slots.offsets[-1])
    H = _randn(g, tokens * k, n, dtype=dtype)
    H[used:] = math.nan
    w = _randn(g, tokens, k) if weighted else None
    base = _randn(g, tokens, n, dtype=dtype) if add else None
    keep = None if base is None else base.clone()
    got = ops.expert_combine(H, slots, w, add=base)
    here = slots.slot_of >= 0
    ww = (torch.ones(tokens, k, device="cuda") if w is None else w).double() * here
    rows = H[slots.slot_of.clamp(min=0).long()].double()
    rows = torch.where(here[:, :, None], rows, torch.zeros_like(rows))
    want = torch.einsum("tj,tjn->tn", ww, rows)
    size = torch.einsum("tj,tjn->tn", ww.abs(), rows.abs())
    if base is not None:
        want, size = want + base.double(), size + base.double().abs()
    bound = (k + 1) * 2 ** -24 * size
    bound = bound + (want.abs() + bound) * _half_step(dtype) + 2 ** -25
    _within(got, want, bound)
    if base is not None:                                  # in place over the residual
        ops.expert_combine(H, slots, w, base, add=base)
        assert torch.equal(base, got) and not torch.equal(base, keep)


@pytest.mark.parametrize("tokens, k, n, lost", [(1, 1, 8, 0.0), (3, 8, 4096, 0.0),
                                               (200, 6, 1032, 0.3), (17, 2, 20000, 0.0)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_combine_backward(tokens, k, n, lost, dtype):
    from tileccl_b200 import ops

    g = _gen(tokens + n)
    slots = _make_slots(g, tokens, k, 16, lost)
    used = int(slots.offsets[-1])
    big = _randn(g, tokens * k, n + 16, dtype=dtype)
    H = big[:, 8:8 + n]
    H[used:] = math.nan
    w = _randn(g, tokens, k)
    w[slots.slot_of < 0] = math.nan
    dy = _randn(g, tokens, n, dtype=dtype)
    gh, gw = ops.expert_combine_backward(dy, H, slots, w)
    here = slots.slot_of >= 0
    at = slots.slot_of[here].long()
    want_h = torch.zeros(tokens * k, n, dtype=torch.float64, device="cuda")
    tok = torch.arange(tokens, device="cuda")[:, None].expand(tokens, k)[here]
    want_h[at] = w[here].double()[:, None] * dy[tok].double()
    u = _half_step(dtype)
    _within(gh[:used], want_h[:used], want_h[:used].abs() * (u + 2 ** -23) + 2 ** -25)
    want_w = torch.zeros(tokens, k, dtype=torch.float64, device="cuda")
    prod = dy[tok].double() * H[at].double()
    want_w[here] = prod.sum(1)
    size = torch.zeros_like(want_w)
    size[here] = prod.abs().sum(1)
    _within(gw, want_w, n * 2 ** -24 * size)


# --------------------------------------------------------------------- as used together
def _layer(ops, logits, x, w_gu, w_down, k):
    weights, ids = ops.route_experts(logits, k)
    slots = ops.expert_slots(ids, w_gu.shape[0])
    h = ops.expert_gemm(x, w_gu, slots, epilogue="silu_gate")
    y = ops.expert_gemm(h, w_down, slots, rows="slots")
    return ops.expert_combine(y, slots, weights, add=x), weights, slots, h, y


def _layer_ref(logits, x, w_gu, w_down, k):
    """The layer in 64 bits, differentiable, every expert applied to every token."""
    p = torch.softmax(logits, 1)
    top = p.topk(k, 1)
    w = torch.zeros_like(p).scatter(1, top.indices, top.values / top.values.sum(1, keepdim=True))
    cg, cu = _pairs(w_gu.shape[2])
    out = x
    for e in range(w_gu.shape[0]):
        y = x @ w_gu[e]
        out = out + w[:, e:e + 1] * ((torch.nn.functional.silu(y[:, cg]) * y[:, cu]) @ w_down[e])
    return out


@pytest.mark.parametrize("tokens", [1, 3, 257])
def test_layer_forward_and_backward(tokens):
    from tileccl_b200 import ops

    dtype, k, E, H, F = torch.float16, 2, 6, 256, 384
    g = _gen(tokens)
    logits, x = _randn(g, tokens, E, std=1.5), _randn(g, tokens, H, dtype=dtype)
    w_gu, w_down = _randn(g, E, H, 2 * F, std=H ** -0.5, dtype=dtype), _randn(g, E, F, H, std=F ** -0.5, dtype=dtype)
    out, weights, slots, h, y = _layer(ops, logits, x, w_gu, w_down, k)
    leaves = [t.double().requires_grad_(True) for t in (logits, x, w_gu, w_down)]
    ref = _layer_ref(*leaves, k)
    dout = _randn(g, tokens, H, dtype=dtype)
    ref.backward(dout.double())
    dy, dweights = ops.expert_combine_backward(dout, y, slots, weights)
    dh, dw_down = ops.expert_gemm_backward(dy, h, w_down, slots, rows="slots")
    dx, dw_gu = ops.expert_gemm_backward(dh, x, w_gu, slots, epilogue="silu_gate")
    dx = dx.double() + dout.double()
    dlogits = ops.route_experts_backward(dweights, logits, ops.route_experts(logits, k)[1])
    # at most five 16-bit roundings lie on any path, each half a step of a value that the
    # following sums mix with random signs: five half steps of the result's size, times 4
    # for the largest of some 10^5 normal deviates
    for got, want in ((out, ref.detach()), (dx, leaves[1].grad), (dw_gu, leaves[2].grad),
                      (dw_down, leaves[3].grad), (dlogits, leaves[0].grad)):
        rms = want.square().mean().sqrt()
        err = (got.double() - want).abs()
        assert (err <= 5 * 4 * _half_step(dtype) * (want.abs() + rms) + 1e-9).all(), err.max().item()


def test_layer_in_a_graph_on_another_stream_and_twice_at_once():
    """Captured and replayed on new inputs; two graphs and an eager layer at the same time."""
    from tileccl_b200 import ops

    dtype, k, E, H, F, T = torch.bfloat16, 2, 8, 512, 256, 40
    g = _gen(9)
    w_gu, w_down = _randn(g, E, H, 2 * F, std=H ** -0.5, dtype=dtype), _randn(g, E, F, H, std=F ** -0.5, dtype=dtype)
    data = [(_randn(g, T, E), _randn(g, T, H, dtype=dtype)) for _ in range(6)]
    want = [_layer(ops, l, x, w_gu, w_down, k)[0].clone() for l, x in data]
    graphs = []
    for i in range(2):
        l, x = data[i][0].clone(), data[i][1].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _layer(ops, l, x, w_gu, w_down, k)[0]
        graphs.append((graph, l, x, out))
    streams = [torch.cuda.Stream() for _ in range(3)]
    for rep in range(3):
        for i, (graph, l, x, out) in enumerate(graphs):
            with torch.cuda.stream(streams[i]):
                l.copy_(data[2 * rep + i][0])
                x.copy_(data[2 * rep + i][1])
        torch.cuda.synchronize()
        eager = []
        for i, (graph, l, x, out) in enumerate(graphs):
            with torch.cuda.stream(streams[i]):
                graph.replay()
        for l, x in data[:2]:
            weights, ids = ops.route_experts(l, k, stream=streams[2])
            s = ops.expert_slots(ids, E, stream=streams[2])
            h = ops.expert_gemm(x, w_gu, s, epilogue="silu_gate", stream=streams[2])
            y = ops.expert_gemm(h, w_down, s, rows="slots", stream=streams[2])
            eager.append(ops.expert_combine(y, s, weights, add=x, stream=streams[2]))
        torch.cuda.synchronize()
        for i, (graph, l, x, out) in enumerate(graphs):
            assert torch.equal(out, want[2 * rep + i])
        assert torch.equal(eager[0], want[0]) and torch.equal(eager[1], want[1])


def test_backward_repeats_and_captures():
    from tileccl_b200 import ops

    g = _gen(21)
    T, k, E, K, N, dtype = 300, 2, 4, 256, 512, torch.bfloat16
    slots = _make_slots(g, T, k, E)
    X, W = _randn(g, T, K, dtype=dtype), _randn(g, E, K, N, std=K ** -0.5, dtype=dtype)
    dY = _randn(g, T * k, N // 2, dtype=dtype)
    first = [t.clone() for t in ops.expert_gemm_backward(dY, X, W, slots, epilogue="silu_gate")]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gx, gw = ops.expert_gemm_backward(dY, X, W, slots, epilogue="silu_gate")
    for _ in range(3):
        graph.replay()
        again = ops.expert_gemm_backward(dY, X, W, slots, epilogue="silu_gate")
        torch.cuda.synchronize()
        assert torch.equal(gx, first[0]) and torch.equal(gw, first[1])
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups, top_groups", [(1, 1), (4, 2), (8, 3), (5, 2)])
def test_route_decides_crowded_rows_exactly(score, groups, top_groups):
    """Many keys within a few 2^-24 of one another, and many that are equal: at the border of
    the choice, inside it, and between groups; also more near-equal keys than lanes."""
    from tileccl_b200 import ops

    E, k, T = 40 * groups if groups != 5 else 100, 6, 48
    g = _gen(groups)
    level = torch.randint(0, 3, (T, E), device="cuda", generator=g).float()
    tiny = torch.randint(-2, 3, (T, E), device="cuda", generator=g).float() * 2 ** -22
    logits = level + tiny
    logits[::4] = level[::4]                              # exact ties only
    bias = torch.where(torch.rand(E, device="cuda", generator=g) < 0.5, 0.0, 2 ** -23)
    for b in (bias, torch.zeros_like(bias), None):
        w, ids = ops.route_experts(logits, k, score=score, bias=b, groups=groups, top_groups=top_groups)
        _, want = _route64(logits, k, score, b, groups, top_groups, "top2", True, 1.0, None)
        same = ids == want
        # Keys that differ by less than 2^-50 depend on the last bit of a 64-bit exponential: there
        # either order is right, so compare the keys of the chosen, in order.
        p = (torch.softmax(logits.double(), 1) if score == "softmax" else torch.sigmoid(logits.double()))
        key = p + (0.0 if b is None else b.double())
        got_k, want_k = key.gather(1, ids.long()), key.gather(1, want.long())
        assert ((got_k - want_k).abs() <= 2 ** -50)[~same].all()
        assert same.float().mean() > 0.99


def test_expert_gemm_fp32_result():
    from tileccl_b200 import ops

    g = _gen(31)
    T, E, K, N = 300, 3, 136, 72
    slots = _make_slots(g, T, 2, E)
    X, W = _randn(g, T, K, dtype=torch.bfloat16), _randn(g, E, K, N, dtype=torch.bfloat16)
    big = torch.full((2 * T, N + 8), 3.0, device="cuda")
    out = big[:, 4:4 + N]
    got = ops.expert_gemm(X, W, slots, out)               # (the type of `out` counts)
    again = ops.expert_gemm(X, W, slots, out_dtype=torch.float32)
    assert got is out and torch.equal(again, out) and (big[:, :4] == 3).all() and (big[:, 4 + N:] == 3).all()
    off, tok = slots.offsets.tolist(), slots.token_of_slot.long()
    for e in range(E):
        x = X[tok[off[e]:off[e + 1]]].double()
        _within(out[off[e]:off[e + 1]], x @ W[e].double(), _sum_bound(x, W[e].double(), K))


@pytest.mark.parametrize("ws", [1, 2, 4])
def test_tp_moe_matches_fp32_reference(ws):
    import tileccl_b200 as tccl
    from tileccl_b200.models.tp_moe import smoke_moe_forward

    ctxs = tccl.init_local(ws, 256 << 20)
    try:
        smoke_moe_forward(ctxs)
        smoke_moe_forward(ctxs, tokens=ws, experts=16, top_k=3)       # one token per rank
    finally:
        for d in range(torch.cuda.device_count()):
            torch.cuda.synchronize(d)
        for c in ctxs:
            c.heap.cleanup()


def test_tp_moe_in_a_graph():
    import tileccl_b200 as tccl
    from tileccl_b200.models import TPMoE

    ctx = tccl.init_local(1, 64 << 20)[0]
    try:
        moe = TPMoE(ctx, tokens=48, hidden=256, ffn=512, experts=8, top_k=2, balance=True, groups=4,
                    top_groups=2, score="sigmoid")
        xs = [_randn(_gen(i), 48, 256, dtype=torch.bfloat16) for i in range(3)]
        want = [moe(x).clone() for x in xs]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            moe.forward()
        for x, y in zip(xs, want):
            moe.x_local.copy_(x)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(moe.y, y)
    finally:
        torch.cuda.synchronize()
        ctx.heap.cleanup()


def test_shared_tiles_repeat_in_graphs_and_beside_each_other():
    """Products whose tiles are shared (few rows, long contraction) leave their counters as they
    found them: repeated, captured twice, replayed beside one another and beside eager calls."""
    from tileccl_b200 import ops

    g = _gen(41)
    dtype, T, E, K, N = torch.bfloat16, 3, 8, 4608, 512
    W = _randn(g, E, K, N, std=K ** -0.5, dtype=dtype)
    data = [(_randn(g, T, K, dtype=dtype), _make_slots(g, T, 2, E)) for _ in range(3)]
    want = [ops.expert_gemm(x, W, s).clone() for x, s in data]
    graphs = []
    for x, s in data[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = [ops.expert_gemm(x, W, s) for _ in range(3)]
        graphs.append((graph, outs))
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(20):
        for (graph, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        eager = [ops.expert_gemm(*[data[2][0], W, data[2][1]], stream=streams[2]) for _ in range(3)]
        torch.cuda.synchronize()
        for (_, outs), y in zip(graphs, want):
            assert all(torch.equal(o, y) for o in outs)
        assert all(torch.equal(o, want[2]) for o in eager)
    ops.check_expert_status()


def test_counters_run_out(monkeypatch):
    """Captured products beyond the prepared counters zero their own."""
    from tileccl_b200 import ops
    from tileccl_b200.kernels import experts

    g = _gen(43)
    x, W = _randn(g, 2, 4096, dtype=torch.float16), _randn(g, 4, 4096, 256, std=1 / 64, dtype=torch.float16)
    slots = _make_slots(g, 2, 2, 4)
    want = ops.expert_gemm(x, W, slots).clone()
    arena = experts._ARENAS[x.device.index]
    monkeypatch.setattr(arena, "used", arena.BYTES)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [ops.expert_gemm(x, W, slots) for _ in range(2)]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)
    stream = torch.cuda.Stream()                          # a stream that has no piece yet
    stream.wait_stream(torch.cuda.current_stream())
    got = ops.expert_gemm(x, W, slots, stream=stream)
    stream.synchronize()
    assert torch.equal(got, want)


def test_the_same_expert_twice():
    """A token that names an expert twice has two slots of it; gradients add up."""
    from tileccl_b200 import ops

    g = _gen(51)
    ids = torch.tensor([[1, 1], [0, 1], [2, 2]], dtype=torch.int32, device="cuda")
    slots = ops.expert_slots(ids, 3)
    assert slots.offsets.tolist() == [0, 1, 4, 6] and slots.slot_of.tolist() == [[1, 2], [0, 3], [4, 5]]
    X, W = _randn(g, 3, 64, dtype=torch.float16), _randn(g, 3, 64, 72, std=0.125, dtype=torch.float16)
    y = ops.expert_gemm(X, W, slots)
    assert torch.equal(y[1], y[2]) and torch.equal(y[4], y[5])
    w = torch.tensor([[0.25, 0.75], [1.0, 1.0], [2.0, -1.0]], device="cuda")
    out = ops.expert_combine(y, slots, w)
    once = ops.expert_combine(y, slots, w.sum(1, keepdim=True) * torch.tensor([[1.0, 0.0]], device="cuda"))
    assert torch.equal(out[0], once[0]) and torch.equal(out[2], once[2])
    logits = _randn(g, 3, 8)
    grad = torch.ones(3, 2, device="cuda")
    d = ops.route_experts_backward(grad, logits, ids, score="sigmoid", renormalize=False)
    p = torch.sigmoid(logits.double())
    want = torch.zeros_like(p)
    for t in range(3):
        for j in range(2):
            e = int(ids[t, j])
            want[t, e] += p[t, e] * (1 - p[t, e])
    _within(d, want, want * 2 ** -20)


def test_malformed_maps_stay_in_bounds():
    """Indices that no expert_slots would give are skipped or clamped, never followed."""
    from tileccl_b200 import ops

    T, k, E, K, N = 6, 2, 3, 64, 72
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    bad = ops.ExpertSlots(i32([5, -3, 400, 7]), i32([900, -7] + [0] * 10), i32([[99, -5]] * T))
    X, W = torch.ones(T, K, device="cuda").half(), torch.ones(E, K, N, device="cuda").half()
    guard = torch.full((T * k + 16, N), 4.0, device="cuda").half()
    out = guard[8:8 + T * k]
    ops.expert_gemm(X, W, bad, out)
    gx, gw = ops.expert_gemm_backward(torch.ones(T * k, N, device="cuda").half(), X, W, bad)
    assert (ops.expert_combine(out, bad, torch.ones(T, k, device="cuda")) == 0).all()
    _, dw = ops.expert_combine_backward(torch.ones(T, N, device="cuda").half(), out, bad,
                                        torch.ones(T, k, device="cuda"))
    torch.cuda.synchronize()
    ops.check_expert_status()
    assert (guard[:8] == 4).all() and (guard[8 + T * k:] == 4).all() and (dw == 0).all()
    d = ops.route_experts_backward(torch.ones(1, 2, device="cuda"), torch.zeros(1, 8, device="cuda"),
                                   i32([[8, -9]]))
    assert (d == 0).all()


def test_weights_with_interleaved_experts():
    """W[e] may lie between the rows of the others ([K, E, N] in memory)."""
    from tileccl_b200 import ops

    g = _gen(61)
    base = _randn(g, 64, 3, 72, dtype=torch.float16)
    W = base.transpose(0, 1)
    slots = _make_slots(g, 20, 2, 3)
    X = _randn(g, 20, 64, std=0.125, dtype=torch.float16)
    assert torch.equal(ops.expert_gemm(X, W, slots), ops.expert_gemm(X, W.contiguous(), slots))
    gx, gw = ops.expert_gemm_backward(_randn(g, 40, 72, dtype=torch.float16), X, W, slots)
    assert gw.is_contiguous() and gw.shape == W.shape


def test_offsets_beyond_32_bits():
    """Matrices of more than 2^31 elements: their last rows are the ones that are computed."""
    from tileccl_b200 import ops

    g = _gen(71)
    T, K, N = 75_000, 64, 28_672                          # 2.15e9 elements of 16 bits
    ids = torch.zeros(T, 1, dtype=torch.int32, device="cuda")
    slots = ops.expert_slots(ids, 1)
    x, w = _randn(g, T, K, std=0.125, dtype=torch.float16), _randn(g, 1, K, N, dtype=torch.float16)
    y = ops.expert_gemm(x, w, slots)
    assert y.numel() > 1 << 31
    want = x[-300:].double() @ w[0].double()
    bound = _sum_bound(x[-300:].double(), w[0].double(), K)
    _within(y[-300:], want, bound + (want.abs() + bound) * _half_step(torch.float16))
    weights = torch.rand(T, 1, device="cuda", generator=g)
    out = ops.expert_combine(y, slots, weights)
    want = weights[-5:].double() * y[-5:].double()
    _within(out[-5:], want, want.abs() * (_half_step(torch.float16) + 2 ** -23) + 2 ** -25)
    dh, dw = ops.expert_combine_backward(out, y, slots, weights)
    want = weights[-5:].double() * out[-5:].double()
    _within(dh[-5:], want, want.abs() * (_half_step(torch.float16) + 2 ** -23) + 2 ** -25)
    prod = out[-5:].double() * y[-5:].double()
    _within(dw[-5:], prod.sum(1, keepdim=True), N * 2 ** -24 * prod.abs().sum(1, keepdim=True))
    # the wide matrix as the left operand, gathered and in slot order, and in the weight gradient
    back = w.transpose(1, 2).contiguous()
    del dh, out
    z = ops.expert_gemm(y, back, slots)
    assert torch.equal(z[-300:], ops.expert_gemm(y, back, slots, rows="slots")[-300:])
    want = y[-300:].double() @ back[0].double()
    bound = _sum_bound(y[-300:].double(), back[0].double(), N)
    _within(z[-300:], want, bound + (want.abs() + bound) * _half_step(torch.float16))
    few = torch.zeros_like(z)
    few[-3:] = 1.0                                        # only the last rows reach the gradient
    _, gw = ops.expert_gemm_backward(few, y, back, slots, rows="slots")
    want = y[-3:].double().sum(0)[:, None].expand(N, K)
    _within(gw[0], want, 3 * 2 ** -23 * y[-3:].double().abs().sum(0)[:, None]
            + want.abs() * _half_step(torch.float16) + 2 ** -25)


def test_padded_batch():
    """Masked tokens take no part: NaN in their logits and rows reaches nothing, their result is
    the residual alone, and the unmasked ones are those of the batch without them."""
    from tileccl_b200 import ops

    g = _gen(73)
    T, E, H, F, k = 50, 8, 128, 128, 3
    keep = torch.rand(T, device="cuda", generator=g) < 0.6
    logits, x = _randn(g, T, E), _randn(g, T, H, dtype=torch.bfloat16)
    w_gu = _randn(g, E, H, 2 * F, std=H ** -0.5, dtype=torch.bfloat16)
    w_down = _randn(g, E, F, H, std=F ** -0.5, dtype=torch.bfloat16)

    def layer(logits, x, mask):
        weights, ids = ops.route_experts(logits, k, score="sigmoid", mask=mask)
        slots = ops.expert_slots(ids, E)
        h = ops.expert_gemm(x, w_gu, slots, epilogue="silu_gate")
        y = ops.expert_gemm(h, w_down, slots, rows="slots")
        return weights, ids, slots, y, ops.expert_combine(y, slots, weights)

    alone = layer(logits[keep], x[keep], None)
    logits[~keep], x[~keep] = math.nan, math.nan
    weights, ids, slots, y, out = layer(logits, x, keep)
    assert torch.equal(out[keep], alone[4]) and (out[~keep] == 0).all()
    assert (ids[~keep] == -1).all() and (weights[~keep] == 0).all()
    dout = _randn(g, T, H, dtype=torch.bfloat16)
    dout[~keep] = math.nan
    dy, dw = ops.expert_combine_backward(dout, y, slots, weights)
    gx, gw = ops.expert_gemm_backward(dy, torch.zeros(T * k, F, device="cuda").bfloat16(), w_down, slots,
                                      rows="slots")
    dl = ops.route_experts_backward(dw, logits, ids, score="sigmoid")
    assert (dw[~keep] == 0).all() and (dl[~keep] == 0).all() and torch.isfinite(dl).all()
    assert torch.isfinite(gw).all() and torch.isfinite(gx[:int(slots.offsets[-1])]).all()


def test_first_calls_of_a_process_may_be_captured():
    """No call before the capture: kernels, counters and status words are not there yet."""
    import os
    import subprocess
    import sys

    code = """
import torch
from tileccl_b200 import ops
g = torch.Generator(device='cuda'); g.manual_seed(0)
r = lambda *s: torch.randn(*s, device='cuda', generator=g)
logits, x = r(5, 8), r(5, 4096).bfloat16()
w_gu, w_down = (r(8, 4096, 256) / 64).bfloat16(), (r(8, 128, 4096) / 12).bfloat16()
def layer():
    w, ids = ops.route_experts(logits, 2)
    s = ops.expert_slots(ids, 8)
    h = ops.expert_gemm(x, w_gu, s, epilogue='silu_gate')
    y = ops.expert_gemm(h, w_down, s, rows='slots')
    out = ops.expert_combine(y, s, w, add=x)
    dy, dw = ops.expert_combine_backward(out, y, s, w)
    dx, dg = ops.expert_gemm_backward(dy, h, w_down, s, rows='slots')
    return out, dx, dg, ops.route_experts_backward(dw, logits, ids)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    captured = layer()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(captured, layer()))
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_waits_grow_with_the_work(monkeypatch):
    """Products that run for far longer than the budget of their waits end well: the kernels add
    100 us per K block and tile of an SM pair to it."""
    from tileccl_b200 import ops
    from tileccl_b200.kernels import experts

    g = _gen(81)
    dtype, T, E, K, N = torch.bfloat16, 4096, 4, 2048, 8192
    slots = _make_slots(g, T, 2, E)
    X, W = _randn(g, T, K, dtype=dtype), _randn(g, E, K, N, std=K ** -0.5, dtype=dtype)
    dY = _randn(g, T * 2, N, dtype=dtype)
    want = [ops.expert_gemm(X, W, slots), *ops.expert_gemm_backward(dY, X, W, slots)]
    monkeypatch.setattr(experts, "_wait_budget_ns", lambda: 1)          # (0 would be two seconds)
    got = [ops.expert_gemm(X, W, slots), *ops.expert_gemm_backward(dY, X, W, slots)]
    ops.check_expert_status()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_captured_first_product_has_status_words():
    """A graph captured before any eager product reports to the words that eager calls report to,
    and its counters are the device's own."""
    import os
    import subprocess
    import sys

    code = """
import torch
from tileccl_b200 import ops
from tileccl_b200.kernels import experts
x, w = torch.ones(2, 4096, device='cuda').half(), torch.ones(2, 4096, 256, device='cuda').half()
slots = ops.expert_slots(torch.tensor([[0], [1]], dtype=torch.int32, device='cuda'), 2)
seen, launch = [], experts._launch
def record(fn, *args):
    if fn == 'tccl_expert_gemm':
        seen.append((args[0]._obj.status, args[0]._obj.counters))
    launch(fn, *args)
experts._launch = record
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = ops.expert_gemm(x, w, slots)
for _ in range(2):
    graph.replay()
z = ops.expert_gemm(x, w, slots)
ops.check_expert_status()
assert torch.equal(y, z) and (y == 4096).all()
(s0, c0), (s1, c1) = seen
assert s0 == s1 != 0 and c0 != c1 and abs(c0 - c1) < 1 << 20
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_a_reported_wait_is_raised_once_and_counters_are_cleared():
    """What a product that gave up leaves behind (written here by hand: a status word and arrival
    counters) is raised by the check and gone afterwards."""
    from tileccl_b200 import ops
    from tileccl_b200.kernels import experts

    g = _gen(83)
    x, W = _randn(g, 2, 4096, dtype=torch.float16), _randn(g, 4, 4096, 256, std=1 / 64, dtype=torch.float16)
    slots = _make_slots(g, 2, 2, 4)
    want = ops.expert_gemm(x, W, slots).clone()
    ops.check_expert_status()

    def words(address, n):
        class Memory:
            __cuda_array_interface__ = dict(shape=(n,), typestr="<i4", data=(address, False), version=3)

        return torch.as_tensor(Memory(), device="cuda")

    arena = experts._ARENAS[x.device.index]
    counters = words(arena.address, arena.BYTES // 4)
    assert (counters == 0).all()
    counters[:arena.used // 4] = 1
    words(experts._STATUS[x.device.index], 8)[0] = 2
    with pytest.raises(ops.TileCCLTimeoutError):
        ops.check_expert_status()
    assert (counters == 0).all()
    ops.check_expert_status()
    assert torch.equal(ops.expert_gemm(x, W, slots), want)


def test_streams_have_numbers_of_their_own():
    """Also where the driver gives a destroyed stream's handle out again; products on the streams
    of two host threads that are made and destroyed agree with the others."""
    import ctypes as C
    import threading

    from tileccl_b200 import ops
    from tileccl_b200.kernels import experts

    torch.cuda.synchronize()
    cudart = torch.cuda.cudart()

    def key(stream):
        with torch.cuda.stream(stream):
            return experts._stream_key(stream.device.index, stream.cuda_stream)

    lasting = [torch.cuda.default_stream(), torch.cuda.Stream(), torch.cuda.Stream(priority=-1)]
    keys = [key(s) for s in lasting]
    assert keys == [s.cuda_stream for s in lasting]
    for _ in range(4):
        handle = C.c_uint64()
        assert int(cudart.cudaStreamCreate(C.addressof(handle))) == 0
        stream = torch.cuda.ExternalStream(handle.value)
        keys.append(key(stream))
        assert key(stream) == keys[-1] != handle.value
        assert int(cudart.cudaStreamDestroy(handle.value)) == 0
    assert len(set(keys)) == len(keys)

    g = _gen(87)
    dtype, T, E, K, N = torch.bfloat16, 3, 8, 4608, 512
    W = _randn(g, E, K, N, std=K ** -0.5, dtype=dtype)
    data = [(_randn(g, T, K, dtype=dtype), _make_slots(g, T, 2, E)) for _ in range(2)]
    want = [ops.expert_gemm(x, W, s).clone() for x, s in data]
    torch.cuda.synchronize()
    off = []

    def work(i, stream):
        with torch.cuda.stream(stream):
            for _ in range(100):
                got = ops.expert_gemm(data[i][0], W, data[i][1])
                if not torch.equal(got, want[i]):
                    off.append(i)

    for streams in ([torch.cuda.Stream(), torch.cuda.Stream()], [torch.cuda.default_stream()] * 2):
        threads = [threading.Thread(target=work, args=(i, s)) for i, s in enumerate(streams)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    assert off == []
    ops.check_expert_status()


# ------------------------------------------- the larger forms of every launch, and their seams
def _pairs_of_sms():
    return torch.cuda.get_device_properties(0).multi_processor_count // 2


@pytest.mark.parametrize("extra", [0.0, 0.2, 0.34])
@pytest.mark.parametrize("form", ["plain", "float", "silu_gate"])
@pytest.mark.parametrize("b_is_nk", [False, True])
def test_shared_tiles_before_whole_ones(extra, form, b_is_nk):
    """A few tiles more than pairs of SMs: the tiles of a round and of the rest are cut up, so that
    a pair's run may hold the end of a tile, whole tiles and the start of another.  From a third
    of the pairs more they stay whole."""
    from tileccl_b200 import ops

    P = _pairs_of_sms()
    tiles = P + max(1, int(extra * P))
    dtype, T, K, N = torch.bfloat16, 3, 4096, 256 * tiles
    gate = form == "silu_gate"
    g = _gen(91)
    slots = _make_slots(g, T, 1, 1)
    X = _randn(g, T, K, std=K ** -0.5, dtype=dtype)
    W = _randn(g, 1, N, K, dtype=dtype) if b_is_nk else _randn(g, 1, K, N, dtype=dtype)
    kw = dict(b_is_nk=b_is_nk, epilogue="silu_gate" if gate else "none",
              out_dtype=torch.float32 if form == "float" else None)
    got = ops.expert_gemm(X, W, slots, **kw)
    for _ in range(3):
        assert torch.equal(ops.expert_gemm(X, W, slots, **kw), got)
    want, bound = _ref_product(X[slots.token_of_slot.long()], W[0].t() if b_is_nk else W[0], gate)
    if form != "float":
        bound = bound + (want.abs() + bound) * _half_step(dtype) + 2 ** -25
    _within(got, want, bound)
    ops.check_expert_status()


@pytest.mark.parametrize("more", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", ["tokens", "slots"])
@pytest.mark.parametrize("epilogue", ["none", "silu_gate"])
def test_backward_of_shared_tiles(more, dtype, rows, epilogue):
    """Few rows, contractions of 4096 and more: the gate's gradient (16 tiles, or one more than there
    are pairs) and the token gradients come from shared tiles, too."""
    tiles = _pairs_of_sms() + 1 if more else 17
    test_expert_gemm_backward((3, 1, 1, 4096, 256 * tiles, 0.0), dtype, False, rows, epilogue)


@pytest.fixture
def many_choices(monkeypatch):
    """Lets the tests above take more choices than they have experts for, with room for sums of that
    many terms in the bounds of the products."""
    slots, bound = _make_slots, _sum_bound
    here = globals()
    monkeypatch.setitem(here, "_make_slots", lambda g, t, k, e, lost=0.0: slots(g, t, k, max(e, k), lost))
    # (|a sum of k products' results| <= sum of |a| |b|: k additions of 2^-24 each)
    monkeypatch.setitem(here, "_sum_bound", lambda a, b, terms: bound(a, b, terms + 16))


@pytest.mark.parametrize("tokens, k, n, lost", [
    (300, 2, 9000, 0.1), (300, 4, 4104, 0.0), (300, 3, 264, 0.3), (256, 4, 8, 0.0), (5, 11, 1032, 0.2),
    (300, 20, 264, 0.1), (257, 9, 2056, 0.0), (2, 32, 8200, 0.0)])
@pytest.mark.parametrize("weighted, add", [(True, True), (False, False)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_combine_of_every_batch(many_choices, tokens, k, n, lost, weighted, add, dtype):
    test_combine(tokens, k, n, lost, weighted, add, dtype)


@pytest.mark.parametrize("tokens, k, n, lost", [
    (300, 3, 264, 0.0), (40, 4, 4104, 0.2), (300, 9, 1032, 0.0), (7, 20, 2056, 0.3), (2, 32, 8, 0.0)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_combine_backward_of_every_batch(many_choices, tokens, k, n, lost, dtype):
    test_combine_backward(tokens, k, n, lost, dtype)


@pytest.mark.parametrize("case", [(300, 2, 4, 2568, 256, 0.0),         # two choices, several pieces
                                  (300, 3, 4, 1032, 256, 0.1), (40, 6, 8, 264, 256, 0.2),
                                  (270, 12, 16, 136, 256, 0.0)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("epilogue", ["none", "silu_gate"])
def test_backward_sums_of_many_choices(many_choices, case, dtype, epilogue):
    """Token gradients summed over more choices than one batch of the fp32 combine holds."""
    test_expert_gemm_backward(case, dtype, False, "tokens", epilogue)


@pytest.mark.parametrize("case", [(300, 8, 64, 64, 256, 0.0), (90, 6, 200, 72, 512, 0.2),
                                  (50, 4, 129, 4096, 256, 0.0), (700, 4, 1024, 64, 256, 0.1),
                                  (3, 8, 1024, 136, 256, 0.0)])
@pytest.mark.parametrize("b_is_nk", [False, True])
@pytest.mark.parametrize("epilogue", ["none", "silu_gate"])
def test_products_of_many_experts(case, b_is_nk, epilogue):
    test_expert_gemm(case, torch.bfloat16, b_is_nk, "tokens", epilogue)
    if case[3] < 4096:
        test_expert_gemm_backward(case, torch.bfloat16, b_is_nk, "slots", epilogue)


def test_products_of_a_part_of_the_experts():
    """A rank that holds the experts 24 .. 40 of 64: the same rows as in the whole map, and nothing
    behind the last of them."""
    from tileccl_b200 import ops

    g = _gen(93)
    T, k, E, first, local, K, N, dtype = 120, 6, 64, 24, 16, 136, 256, torch.float16
    ids = _randn(g, T, E).topk(k, 1).indices.int()
    X, W = _randn(g, T, K, std=K ** -0.5, dtype=dtype), _randn(g, E, K, N, dtype=dtype)
    dY = _randn(g, T * k, N, dtype=dtype)
    whole, part = ops.expert_slots(ids, E), ops.expert_slots(ids, local, first_expert=first)
    a, b = int(whole.offsets[first]), int(whole.offsets[first + local])
    y = ops.expert_gemm(X, W, whole)
    out = torch.full((T * k, N), 7.0, dtype=dtype, device="cuda")
    ops.expert_gemm(X, W[first:first + local], part, out)
    assert torch.equal(out[:b - a], y[a:b]) and (out[b - a:] == 7.0).all()
    _, gw = ops.expert_gemm_backward(dY, X, W, whole)
    dY_part = torch.full_like(dY, math.nan)
    dY_part[:b - a] = dY[a:b]
    gx, gw_part = ops.expert_gemm_backward(dY_part, X, W[first:first + local], part)
    assert torch.equal(gw_part, gw[first:first + local]) and torch.isfinite(gx).all()
    here = ((ids >= first) & (ids < first + local)).any(1)
    assert (gx[~here] == 0).all() and (gx[here] != 0).any(1).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("E, k, kw", [
    (8, 2, {}), (64, 8, {}), (256, 8, dict(groups=8, top_groups=3, group_score="max")),
    (256, 8, dict(score="sigmoid", biased=True, groups=8, top_groups=4, scale=2.5)),
    (33, 5, dict(biased=True, renormalize=False)), (500, 32, dict(score="sigmoid", biased=True)),
    (40, 3, dict(score="sigmoid", groups=5, top_groups=2))])
def test_route_of_a_large_batch(dtype, E, k, kw):
    """More tokens than there are warps in a launch: every row as in a small batch."""
    from tileccl_b200 import ops

    g = _gen(95 + E)
    kw = dict(kw)
    T, step = 10_007, 251
    logits = _randn(g, T, E, std=1.5).to(dtype)
    logits[::7, 1] = -math.inf
    mask = torch.rand(T, device="cuda", generator=g) < 0.9
    bias = _randn(g, E, std=0.1) if kw.pop("biased", False) else None
    w, ids = ops.route_experts(logits, k, bias=bias, mask=mask, **kw)
    assert (ids[~mask] == -1).all() and (ids[mask][:, 0] >= 0).all()
    grad = _randn(g, T, k)
    options = {n: kw[n] for n in ("score", "renormalize", "scale") if n in kw}
    dl = ops.route_experts_backward(grad, logits, ids, **options)
    for a in range(0, T, step):
        b = a + step
        w1, ids1 = ops.route_experts(logits[a:b], k, bias=bias, mask=mask[a:b], **kw)
        assert torch.equal(ids1, ids[a:b]) and torch.equal(w1, w[a:b])
        assert torch.equal(ops.route_experts_backward(grad[a:b], logits[a:b], ids1, **options), dl[a:b])


@pytest.mark.parametrize("b_is_nk", [False, True])
@pytest.mark.parametrize("N, epilogue", [(72, "none"), (192, "none"), (512, "silu_gate")])
def test_interleaved_experts_give_the_results_of_separate_ones(b_is_nk, N, epilogue):
    """W[e] between the rows of the others, in every form of the weights' map, forward and back."""
    from tileccl_b200 import ops

    g = _gen(97)
    dtype, T, k, E, K = torch.float16, 40, 2, 3, 136
    slots = _make_slots(g, T, k, E)
    X = _randn(g, T, K, std=K ** -0.5, dtype=dtype)
    W = _randn(g, *((N, E, K) if b_is_nk else (K, E, N)), dtype=dtype).transpose(0, 1)
    dY = _randn(g, T * k, N // 2 if epilogue == "silu_gate" else N, dtype=dtype)
    kw = dict(b_is_nk=b_is_nk, epilogue=epilogue)
    assert not W.is_contiguous()
    assert torch.equal(ops.expert_gemm(X, W, slots, **kw), ops.expert_gemm(X, W.contiguous(), slots, **kw))
    got = ops.expert_gemm_backward(dY, X, W, slots, **kw)
    want = ops.expert_gemm_backward(dY, X, W.contiguous(), slots, **kw)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and got[1].is_contiguous()


def test_layers_of_two_host_threads():
    """Whole layers and their gradients, on a stream per thread and on one for both."""
    import threading

    from tileccl_b200 import ops

    dtype, k, E, H, F, T = torch.bfloat16, 2, 8, 4096, 256, 24
    g = _gen(99)
    w_gu, w_down = _randn(g, E, H, 2 * F, std=H ** -0.5, dtype=dtype), _randn(g, E, F, H, std=F ** -0.5, dtype=dtype)
    data = [(_randn(g, T, E), _randn(g, T, H, dtype=dtype)) for _ in range(2)]

    def step(l, x):
        out, weights, slots, h, y = _layer(ops, l, x, w_gu, w_down, k)
        dy, dw = ops.expert_combine_backward(out, y, slots, weights)
        dh, dw_down = ops.expert_gemm_backward(dy, h, w_down, slots, rows="slots")
        dx, dw_gu = ops.expert_gemm_backward(dh, x, w_gu, slots, epilogue="silu_gate")
        return out, dw, dh, dw_down, dx, dw_gu

    want = [step(*d) for d in data]
    torch.cuda.synchronize()
    off = []

    def work(i, stream):
        with torch.cuda.stream(stream):
            for _ in range(20):
                got = step(*data[i])
                off.extend((i, n) for n, (a, b) in enumerate(zip(got, want[i])) if not torch.equal(a, b))

    for streams in ([torch.cuda.Stream(), torch.cuda.Stream()], [torch.cuda.default_stream()] * 2):
        threads = [threading.Thread(target=work, args=(i, s)) for i, s in enumerate(streams)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    assert off == []
    ops.check_expert_status()
