"""Cases of the mixture-of-experts operators: routing, slot map, grouped GEMM, combine.

``run`` computes a case in elementary torch operations (``own`` false) or through
``tileccl_b200.ops`` (``own`` true).  Widths are those of the tensor-parallel MLP block
(hidden 4096, FFN 14336, a 1/8 shard of it 1792) or generic.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # one token of a decode step: pure latency
        dict(name="route_decode", op="route", tokens=1, experts=64, top_k=8, score="softmax",
             bias=False, groups=1, top_groups=1, renormalize=True, scale=1.0, dtype="bf16"),
        # a prefill batch, sigmoid scores steered by a balance bias, choice limited to groups
        dict(name="route_grouped_sigmoid", op="route", tokens=16384, experts=256, top_k=8,
             score="sigmoid", bias=True, groups=8, top_groups=4, renormalize=True, scale=2.5,
             dtype="fp32"),
        # the router's training step: gradient of the logits
        dict(name="route_backward", op="route_backward", tokens=16384, experts=128, top_k=6,
             score="softmax", renormalize=False, scale=1.0, dtype="fp32"),
        # a decode batch
        dict(name="slots_decode", op="slots", tokens=16, experts=64, top_k=8, first=0, local=64),
        # a large prefill batch whose experts are split over two ranks: this rank holds the upper half
        dict(name="slots_prefill", op="slots", tokens=65536, experts=256, top_k=8, first=128,
             local=128),
        # up projection of a decode batch: every weight of the touched experts once
        dict(name="gemm_decode_up", op="gemm", tokens=8, experts=64, top_k=8, k=4096, n=3584,
             epilogue="silu_gate", rows="tokens", b_is_nk=False, dtype="bf16"),
        # up projection of a prefill batch at the full FFN width
        dict(name="gemm_prefill_up", op="gemm", tokens=8192, experts=8, top_k=2, k=4096, n=28672,
             epilogue="silu_gate", rows="tokens", b_is_nk=False, dtype="bf16"),
        # down projection of a mid-size ragged batch over an odd number of experts
        dict(name="gemm_ragged_down", op="gemm", tokens=1003, experts=61, top_k=6, k=1792, n=4096,
             epilogue="none", rows="slots", b_is_nk=True, dtype="fp16"),
        # training step of the gated up projection: gradients of tokens and weights
        dict(name="gemm_backward_up", op="gemm_backward", tokens=4096, experts=8, top_k=2, k=4096,
             n=3584, epilogue="silu_gate", rows="tokens", b_is_nk=False, dtype="bf16"),
        # end of a decode step
        dict(name="combine_decode", op="combine", tokens=4, experts=64, top_k=8, n=4096, add=True,
             dropped=0.0, dtype="bf16"),
        # end of a prefill batch when a part of the chosen experts lives on other ranks
        dict(name="combine_prefill", op="combine", tokens=16384, experts=64, top_k=8, n=4096,
             add=False, dropped=0.25, dtype="bf16"),
        # training step of the combine
        dict(name="combine_backward", op="combine_backward", tokens=4096, experts=64, top_k=8,
             n=4096, dropped=0.0, dtype="fp16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["route", "route", "route_backward", "slots", "gemm", "gemm", "gemm_backward",
                     "combine", "combine_backward"])
    dtype16 = rng.choice(["bf16", "fp16"])
    if op in ("route", "route_backward"):
        groups = rng.choice([1, 1, 4, 8]) if op == "route" else 1
        experts = groups * _log_int(rng, 8, 256 // groups) if groups > 1 else _log_int(rng, 8, 256)
        top_groups = rng.randint(max(1, groups // 4), groups)
        top_k = rng.randint(1, min(8, top_groups * (experts // groups)))
        case = dict(op=op, tokens=_log_int(rng, 1, 16384), experts=experts, top_k=top_k,
                    score=rng.choice(["softmax", "sigmoid"]), renormalize=rng.random() < 0.5,
                    scale=rng.choice([1.0, 2.5]), dtype=rng.choice(["fp32", "bf16", "fp16"]))
        if op == "route":
            case.update(bias=rng.random() < 0.5, groups=groups, top_groups=top_groups)
        return case
    experts = _log_int(rng, 4, 128)
    top_k = rng.randint(1, min(8, experts))
    if op == "slots":
        local = rng.randint(1, experts)
        return dict(op=op, tokens=_log_int(rng, 1, 65536), experts=experts, top_k=top_k,
                    first=rng.randint(0, experts - local), local=local)
    if op.startswith("combine"):
        case = dict(op=op, tokens=_log_int(rng, 1, 4096), experts=experts, top_k=top_k,
                    n=8 * _log_int(rng, 8, 512), dropped=0.0, dtype=dtype16)
        if op == "combine":
            case.update(add=rng.random() < 0.5, dropped=rng.choice([0.0, 0.25]))
        return case
    backward = op == "gemm_backward"
    gate = rng.random() < 0.5
    case = dict(op=op, tokens=_log_int(rng, 1, 2048), experts=_log_int(rng, 4, 64), top_k=0,
                k=8 * _log_int(rng, 16, 512),
                n=256 * _log_int(rng, 1, 14) if gate else 8 * _log_int(rng, 16, 512),
                epilogue="silu_gate" if gate else "none",
                rows=rng.choice(["tokens", "slots"]), b_is_nk=rng.random() < 0.5, dtype=dtype16)
    case["top_k"] = rng.randint(1, min(4 if backward else 8, case["experts"]))
    return case


# -------------------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)


def _choice(g, tokens, experts, top_k):
    """Distinct expert ids per token; some experts are more popular than others."""
    liking = _normal(g, tokens, experts) + _normal(g, experts, std=0.5)
    return liking.topk(top_k, dim=1).indices.to(torch.int32)


def _slot_map(ids, experts, first=0):
    """(offsets, token_of_slot, slot_of): (token, choice) pairs sorted by expert, stably."""
    tokens, top_k = ids.shape
    local = ids.reshape(-1).long() - first
    here = (local >= 0) & (local < experts)
    key = torch.where(here, local, torch.full_like(local, experts))
    order = torch.sort(key, stable=True).indices
    counts = (key[:, None] == torch.arange(experts, device=ids.device)).sum(0) \
        if key.numel() * experts < (1 << 26) else torch.bincount(key, minlength=experts + 1)[:experts]
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device=ids.device)
    offsets[1:] = counts.cumsum(0)
    sorted_here = here[order]
    token_of_slot = torch.where(sorted_here, order // top_k, torch.full_like(order, -1)).int()
    slot_of = torch.empty_like(order)
    slot_of[order] = torch.arange(order.numel(), device=ids.device)
    slot_of = torch.where(here, slot_of, torch.full_like(slot_of, -1)).int().reshape(tokens, top_k)
    return offsets, token_of_slot, slot_of


def prepare(case, seed):
    g = _generator(seed)
    op, T, k = case["op"], case["tokens"], case["top_k"]
    E = case["experts"]
    st = {"case": case}
    if op in ("route", "route_backward"):
        # a normalised activation times the router's weights, some experts liked more than others
        logits = _normal(g, T, E, std=1.5) + _normal(g, E, std=0.5)
        st["logits"] = logits.to(_DTYPES[case["dtype"]])
        if op == "route":
            st["bias"] = _normal(g, E, std=0.1) if case["bias"] else None
        else:
            # the forward pass chose the largest logits
            st["ids"] = torch.sort(st["logits"], dim=1, descending=True, stable=True) \
                .indices[:, :k].to(torch.int32).contiguous()
            st["grad_weights"] = _normal(g, T, k)
        return st
    st["ids"] = _choice(g, T, E, k)
    if op == "slots":
        return st
    dt = _DTYPES[case["dtype"]]
    if case.get("dropped", 0.0) > 0:
        lost = torch.rand(T, k, device="cuda", generator=g) < case["dropped"]
        st["ids"] = torch.where(lost, torch.full_like(st["ids"], -1), st["ids"])
    st["offsets"], st["token_of_slot"], st["slot_of"] = _slot_map(st["ids"], E)
    S = T * k
    if op.startswith("combine"):
        st["weights"] = torch.rand(T, k, device="cuda", generator=g) * (2.0 / k)
        st["hidden"] = _normal(g, S, case["n"], dtype=dt)
        if op == "combine":
            st["add"] = _normal(g, T, case["n"], dtype=dt) if case["add"] else None
        else:
            st["grad_out"] = _normal(g, T, case["n"], dtype=dt)
        return st
    K, N = case["k"], case["n"]
    st["x"] = _normal(g, T if case["rows"] == "tokens" else S, K, dtype=dt)
    w = torch.empty((E, N, K) if case["b_is_nk"] else (E, K, N), dtype=dt, device="cuda")
    for e in range(E):
        w[e] = _normal(g, *w.shape[1:], std=0.02, dtype=dt)
    st["w"] = w
    if op == "gemm_backward":
        n_out = N // 2 if case["epilogue"] == "silu_gate" else N
        st["grad_out"] = _normal(g, S, n_out, dtype=dt)
    return st


# ----------------------------------------------------------------------- plain forms
def _plain_route(st):
    c = st["case"]
    # (the choice between nearly equal keys is made in 64 bits)
    l64 = st["logits"].double()
    if c["score"] == "softmax":
        e = (l64 - l64.amax(1, keepdim=True)).exp()
        p = e / e.sum(1, keepdim=True)
    else:
        p = 1.0 / (1.0 + (-l64).exp())
    key = p if st["bias"] is None else p + st["bias"].double()
    T, E = key.shape
    if c["groups"] > 1:
        per = key.reshape(T, c["groups"], E // c["groups"])
        top2 = per.sort(dim=2, descending=True).values[:, :, :2].sum(2)
        best = torch.sort(top2, dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        keep = (best[:, :, None] == torch.arange(c["groups"], device=key.device)).any(1)
        keep = keep[:, :, None].expand(per.shape).reshape(T, E)
        key = torch.where(keep, key, torch.full_like(key, -math.inf))
    ids = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :c["top_k"]]
    w = p.gather(1, ids).float()
    if c["renormalize"]:
        w = w / w.sum(1, keepdim=True)
    return w * c["scale"], ids.int()


def _plain_route_backward(st):
    c = st["case"]
    logits, ids, g = st["logits"].float(), st["ids"].long(), st["grad_weights"]
    if c["score"] == "softmax":
        e = (logits - logits.amax(1, keepdim=True)).exp()
        p = e / e.sum(1, keepdim=True)
    else:
        p = 1.0 / (1.0 + (-logits).exp())
    chosen = p.gather(1, ids)
    gp = g * c["scale"]
    if c["renormalize"]:
        total = chosen.sum(1, keepdim=True)
        gp = (gp - (gp * chosen).sum(1, keepdim=True) / total) / total
    dp = torch.zeros_like(p).scatter_(1, ids, gp)
    if c["score"] == "softmax":
        dl = p * (dp - (dp * p).sum(1, keepdim=True))
    else:
        dl = dp * p * (1.0 - p)
    return dl.to(st["logits"].dtype)


def _experts_of(st):
    bounds = st["offsets"].tolist()
    return [(e, bounds[e], bounds[e + 1]) for e in range(len(bounds) - 1)]


def _slot_rows(st, a, b):
    x = st["x"]
    return x[st["token_of_slot"][a:b].long()].float() if st["case"]["rows"] == "tokens" \
        else x[a:b].float()


def _unpack_gate(gu):
    """Columns come as 128 gate columns followed by 128 up columns."""
    blocks = gu.reshape(gu.shape[0], -1, 2, 128)
    return blocks[:, :, 0].reshape(gu.shape[0], -1), blocks[:, :, 1].reshape(gu.shape[0], -1)


def _pack_gate(g, u):
    n = g.shape[0]
    return torch.stack([g.reshape(n, -1, 128), u.reshape(n, -1, 128)], 2).reshape(n, -1)


def _plain_gemm(st):
    c = st["case"]
    gate = c["epilogue"] == "silu_gate"
    S = c["tokens"] * c["top_k"]
    out = torch.empty(S, c["n"] // 2 if gate else c["n"], dtype=st["x"].dtype, device="cuda")
    for e, a, b in _experts_of(st):
        if a == b:
            continue
        w = st["w"][e].float()
        y = _slot_rows(st, a, b) @ (w.t() if c["b_is_nk"] else w)
        if gate:
            g, u = _unpack_gate(y)
            y = g / (1.0 + (-g).exp()) * u
        out[a:b] = y.to(out.dtype)
    return out


def _plain_gemm_backward(st):
    c = st["case"]
    x, dt = st["x"], st["x"].dtype
    dx = torch.zeros(x.shape, dtype=torch.float32, device="cuda")
    dw = torch.zeros_like(st["w"])
    for e, a, b in _experts_of(st):
        if a == b:
            continue
        w = st["w"][e].float()
        w = w.t() if c["b_is_nk"] else w
        rows, dy = _slot_rows(st, a, b), st["grad_out"][a:b].float()
        if c["epilogue"] == "silu_gate":
            g, u = _unpack_gate(rows @ w)
            s = 1.0 / (1.0 + (-g).exp())
            dy = _pack_gate(dy * u * s * (1.0 + g * (1.0 - s)), dy * g * s)
        d = dy @ w.t()
        if c["rows"] == "tokens":
            dx.index_add_(0, st["token_of_slot"][a:b].long(), d)
        else:
            dx[a:b] = d
        dwe = rows.t() @ dy
        dw[e] = (dwe.t() if c["b_is_nk"] else dwe).to(dt)
    return dx.to(dt), dw


def _plain_combine(st):
    c = st["case"]
    T, k = c["tokens"], c["top_k"]
    y = torch.zeros(T, c["n"], device="cuda") if st["add"] is None else st["add"].float()
    for j in range(k):
        slot = st["slot_of"][:, j].long()
        rows = st["hidden"][slot.clamp(min=0)].float() * st["weights"][:, j:j + 1]
        y = y + torch.where(slot[:, None] >= 0, rows, torch.zeros_like(rows))
    return y.to(st["hidden"].dtype)


def _plain_combine_backward(st):
    c = st["case"]
    dy, dt = st["grad_out"].float(), st["hidden"].dtype
    dh = torch.zeros(st["hidden"].shape, dtype=dt, device="cuda")
    dw = torch.zeros_like(st["weights"])
    for j in range(c["top_k"]):
        slot = st["slot_of"][:, j].long()
        dh[slot] = (dy * st["weights"][:, j:j + 1]).to(dt)
        dw[:, j] = (dy * st["hidden"][slot].float()).sum(1)
    return dh, dw


_PLAIN = {"route": _plain_route, "route_backward": _plain_route_backward,
          "gemm": _plain_gemm, "gemm_backward": _plain_gemm_backward,
          "combine": _plain_combine, "combine_backward": _plain_combine_backward}


# ------------------------------------------------------------------------------ run
def run(state):
    c = state["case"]
    op = c["op"]
    if not own:
        if op == "slots":
            return _slot_map(state["ids"], c["local"], c["first"])
        return _PLAIN[op](state)
    from tileccl_b200 import ops

    if op == "route":
        return ops.route_experts(state["logits"], c["top_k"], score=c["score"], bias=state["bias"],
                                 groups=c["groups"], top_groups=c["top_groups"],
                                 renormalize=c["renormalize"], scale=c["scale"])
    if op == "route_backward":
        return ops.route_experts_backward(state["grad_weights"], state["logits"], state["ids"],
                                          score=c["score"], renormalize=c["renormalize"],
                                          scale=c["scale"])
    if op == "slots":
        s = ops.expert_slots(state["ids"], c["local"], first_expert=c["first"])
        return s.offsets, s.token_of_slot, s.slot_of
    slots = ops.ExpertSlots(state["offsets"], state["token_of_slot"], state["slot_of"])
    if op == "gemm":
        return ops.expert_gemm(state["x"], state["w"], slots, rows=c["rows"],
                               b_is_nk=c["b_is_nk"], epilogue=c["epilogue"])
    if op == "gemm_backward":
        return ops.expert_gemm_backward(state["grad_out"], state["x"], state["w"], slots,
                                        rows=c["rows"], b_is_nk=c["b_is_nk"],
                                        epilogue=c["epilogue"])
    if op == "combine":
        return ops.expert_combine(state["hidden"], slots, state["weights"], add=state["add"])
    return ops.expert_combine_backward(state["grad_out"], state["hidden"], slots,
                                       state["weights"])


# ---------------------------------------------------------------------------- exact
def _exact_probabilities(c, l):
    if c["score"] == "softmax":
        return (l - torch.logsumexp(l, dim=1, keepdim=True)).exp()
    return torch.sigmoid(l)


def _exact_route(c, st):
    p = _exact_probabilities(c, st["logits"].double().cpu()).numpy()
    key = p + (0.0 if st["bias"] is None else st["bias"].double().cpu().numpy())
    T, E = key.shape
    if T * E > (1 << 22):
        return None
    per = E // c["groups"]
    ids = torch.empty(T, c["top_k"], dtype=torch.int32)
    w = torch.empty(T, c["top_k"], dtype=torch.float64)
    for t in range(T):
        row = [(-float(v), e) for e, v in enumerate(key[t])]
        if c["groups"] > 1:
            scores = []
            for gi in range(c["groups"]):
                members = sorted(row[gi * per:(gi + 1) * per])
                scores.append((sum(m[0] for m in members[:2]), gi))
            allowed = {gi for _, gi in sorted(scores)[:c["top_groups"]]}
            row = [r for r in row if r[1] // per in allowed]
        best = [e for _, e in sorted(row)[:c["top_k"]]]
        total = math.fsum(p[t][e] for e in best) if c["renormalize"] else 1.0
        for j, e in enumerate(best):
            ids[t, j] = e
            w[t, j] = c["scale"] * p[t][e] / total
    return w.cuda(), ids.cuda()


def _exact_route_backward(c, st):
    l = st["logits"].double().requires_grad_(True)
    with torch.enable_grad():
        w = _exact_probabilities(c, l).gather(1, st["ids"].long())
        if c["renormalize"]:
            w = w / w.sum(1, keepdim=True)
        (w * c["scale"] * st["grad_weights"].double()).sum().backward()
    return l.grad


def _exact_expert(c, st, e, rows, dy=None):
    """One expert's outputs, or its (row gradients, weight gradient), by autograd in 64 bits."""
    w = st["w"][e].double()
    x = rows.double()
    if dy is not None:
        w.requires_grad_(True)
        x.requires_grad_(True)
    with torch.set_grad_enabled(dy is not None):
        y = torch.einsum("rk,nk->rn" if c["b_is_nk"] else "rk,kn->rn", x, w)
        if c["epilogue"] == "silu_gate":
            y = y.reshape(y.shape[0], -1, 256)
            y = (y[:, :, :128] * torch.sigmoid(y[:, :, :128]) * y[:, :, 128:]).flatten(1)
        if dy is None:
            return y
        return torch.autograd.grad(y, (x, w), dy.double())


def _exact_gemm(c, st, backward):
    S = c["tokens"] * c["top_k"]
    by_expert = {}
    for i, e in enumerate(st["ids"].reshape(-1).tolist()):
        by_expert.setdefault(e, []).append(i)
    place = 0
    n_out = c["n"] // 2 if c["epilogue"] == "silu_gate" else c["n"]
    if backward:
        dx = torch.zeros(st["x"].shape, dtype=torch.float64, device="cuda")
        dw = torch.zeros(st["w"].shape, dtype=torch.float64, device="cuda")
    else:
        out = torch.zeros(S, n_out, dtype=torch.float64, device="cuda")
    for e in sorted(by_expert):
        entries = torch.tensor(by_expert[e], device="cuda")
        n = entries.numel()
        at = entries // c["top_k"] if c["rows"] == "tokens" \
            else torch.arange(place, place + n, device="cuda")
        if backward:
            dxe, dwe = _exact_expert(c, st, e, st["x"][at], st["grad_out"][place:place + n])
            dx.index_add_(0, at, dxe)
            dw[e] = dwe
        else:
            out[place:place + n] = _exact_expert(c, st, e, st["x"][at])
        place += n
    return (dx, dw) if backward else out


def _exact_combine(c, st):
    h = st["hidden"].double()
    slot = st["slot_of"].long()
    w = torch.where(slot >= 0, st["weights"].double(), torch.zeros((), device="cuda",
                                                                   dtype=torch.float64))
    out = torch.empty(c["tokens"], c["n"], dtype=torch.float64, device="cuda")
    for a in range(0, c["tokens"], 512):
        s = slot[a:a + 512].clamp(min=0)
        out[a:a + 512] = torch.einsum("tj,tjn->tn", w[a:a + 512], h[s])
    return out if st["add"] is None else out + st["add"].double()


def _exact_combine_backward(c, st):
    slot = st["slot_of"].long()
    dh = torch.zeros(st["hidden"].shape, dtype=torch.float64, device="cuda")
    dw = torch.empty(c["tokens"], c["top_k"], dtype=torch.float64, device="cuda")
    for a in range(0, c["tokens"], 512):
        s, dy = slot[a:a + 512], st["grad_out"][a:a + 512].double()
        dh[s] = torch.einsum("tj,tn->tjn", st["weights"][a:a + 512].double(), dy)
        dw[a:a + 512] = torch.einsum("tn,tjn->tj", dy, st["hidden"][s].double())
    return dh, dw


def exact(case, seed):
    if case["op"] == "slots":
        return None                                   # whole numbers
    st = prepare(case, seed)
    return {"route": lambda: _exact_route(case, st),
            "route_backward": lambda: _exact_route_backward(case, st),
            "gemm": lambda: _exact_gemm(case, st, False),
            "gemm_backward": lambda: _exact_gemm(case, st, True),
            "combine": lambda: _exact_combine(case, st),
            "combine_backward": lambda: _exact_combine_backward(case, st)}[case["op"]]()


# ----------------------------------------------------------------------------- work
def work(case):
    op, T, k, E = case["op"], case["tokens"], case["top_k"], case["experts"]
    S = T * k
    if op == "route":
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": T * E * size + S * 8 + (E * 4 if case["bias"] else 0), "flops": 4 * T * E}
    if op == "route_backward":
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": 2 * T * E * size + S * 8, "flops": 6 * T * E}
    if op == "slots":
        return {"bytes": S * 12 + 4 * (case["local"] + 1), "flops": S}
    if op == "combine":
        here = S * (1.0 - case["dropped"])
        rows = int(here) + T * (2 if case["add"] else 1)
        return {"bytes": rows * case["n"] * 2 + S * 8, "flops": int(2 * here * case["n"])}
    if op == "combine_backward":
        return {"bytes": (2 * S + T) * case["n"] * 2 + S * 12, "flops": 3 * S * case["n"]}
    K, N = case["k"], case["n"]
    n_out = N // 2 if case["epilogue"] == "silu_gate" else N
    touched = E * (1.0 - (1.0 - k / E) ** T)
    x_bytes = (T if case["rows"] == "tokens" else S) * K * 2
    if op == "gemm":
        return {"bytes": int(touched * K * N * 2) + x_bytes + S * n_out * 2, "flops": 2 * S * K * N}
    # gradient rows in, token and weight gradients out (every expert's, zeros included)
    products = 3 if case["epilogue"] == "silu_gate" else 2
    return {"bytes": int(touched * K * N * 2) + E * K * N * 2 + 2 * x_bytes + S * n_out * 2,
            "flops": products * 2 * S * K * N}
