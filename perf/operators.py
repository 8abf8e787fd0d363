"""The expert-layer operators and the 4-bit weight products: cases, inputs, plain forms.

`run` computes an operator in elementary torch operations, or through maia_b200 where `own` is true.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def route_case(tokens, experts, k, dtype, renormalize, padded, masked, train):
    return {"op": "route", "tokens": tokens, "experts": experts, "k": k, "dtype": dtype, "renormalize": renormalize,
            "padded": padded, "masked": masked, "train": train}


def dispatch_case(tokens, experts, k, width, dtype, block, dropped):
    return {"op": "dispatch", "tokens": tokens, "experts": experts, "k": k, "width": width, "dtype": dtype,
            "block": block, "dropped": dropped}


def combine_case(tokens, experts, k, width, dtype, block, dropped, train):
    # block 0: the rows lie in slot order [tokens, k, width], as a decode step leaves them.
    return {"op": "combine", "tokens": tokens, "experts": experts, "k": k, "width": width, "dtype": dtype,
            "block": block, "dropped": dropped, "train": train}


def gemv_case(tokens, n, k, group, dtype, zeros, experts=0, topk=0, down=False):
    # experts 0: one matrix. down: every slot has its own input row (the second product of an expert).
    return {"op": "gemv", "tokens": tokens, "n": n, "k": k, "group": group, "dtype": dtype, "zeros": zeros,
            "experts": experts, "topk": topk, "down": down}


def listed():
    return [
        # One decoded token through a router whose logits are kept in fp32.
        {"name": "route_one_token", **route_case(1, 64, 8, "f32", True, False, False, False)},
        # A prefill batch, a part of its tokens padding, some experts masked for each token.
        {"name": "route_prefill", **route_case(8192, 128, 8, "bf16", True, True, True, False)},
        # A training step's tokens: the routing, the balance loss and the gradient of the logits.
        {"name": "route_train", **route_case(131072, 256, 8, "bf16", False, False, False, True)},
        # A short ragged prompt, rows of an odd width, some slots dropped.
        {"name": "dispatch_ragged", **dispatch_case(331, 16, 2, 1001, "f16", 128, True)},
        # Prefill of 8192 tokens into the m-grouped layout of the CTA-pair kernel.
        {"name": "dispatch_prefill", **dispatch_case(8192, 64, 4, 4096, "bf16", 256, False)},
        # The end of a decode step: 16 tokens, 8 experts each, rows in slot order.
        {"name": "combine_decode", **combine_case(16, 64, 8, 8192, "bf16", 0, False, False)},
        # A training step: the weighted sum and the gradients of the experts' rows and of the weights.
        {"name": "combine_train", **combine_case(8192, 64, 4, 4096, "bf16", 128, True, True)},
        # One token on the benchmark's decode weights, 28672 x 8192.
        {"name": "gemv_one_token", **gemv_case(1, 28672, 8192, 128, "bf16", False)},
        # A small square layer, one token: the call's latency counts.
        {"name": "gemv_small", **gemv_case(1, 4096, 4096, 128, "f16", True)},
        # A handful of sequences, odd sizes, short groups with zero points.
        {"name": "gemv_ragged_batch", **gemv_case(13, 10007, 4128, 64, "f16", True)},
        # One token's eight experts, the first product of each.
        {"name": "experts_one_token", **gemv_case(1, 4096, 2048, 128, "bf16", False, 64, 8)},
        # 16 sequences, the second product of their experts: every slot has its own input row.
        {"name": "experts_batch", **gemv_case(16, 4096, 1536, 32, "bf16", True, 64, 4, True)},
    ]


def spread(rng, low, high):
    """A whole number between the two, even over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1)) - 1e-9))))


def draw(rng):
    op = rng.choice(["route", "dispatch", "combine", "gemv", "gemv"])
    if op == "route":
        experts = rng.choice([8, 16, 60, 64, 100, 128, 160, 256, 384, 512])
        tokens = spread(rng, 1, min(131072, 131072 * 256 // experts))
        return route_case(tokens, experts, rng.randint(1, 8), rng.choice(["bf16", "f16", "f32"]), rng.random() < 0.5,
                          rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.5)
    if op in ("dispatch", "combine"):
        experts, k = rng.choice([4, 8, 16, 60, 64]), rng.randint(1, 4)
        width = rng.choice([spread(rng, 64, 4096), 8 * spread(rng, 8, 512)])
        tokens = spread(rng, 1, 8192)
        dtype = rng.choice(["bf16", "f16", "f32"]) if tokens <= 4096 else rng.choice(["bf16", "f16"])
        if op == "dispatch":
            return dispatch_case(tokens, experts, k, width, dtype, rng.choice([128, 256]), rng.random() < 0.5)
        return combine_case(tokens, experts, k, width, dtype, rng.choice([0, 128]), rng.random() < 0.5,
                            rng.random() < 0.5)
    group, dtype, zeros = rng.choice([32, 64, 128, 256]), rng.choice(["bf16", "f16"]), rng.random() < 0.5
    k = 32 * spread(rng, 2, 256)
    if rng.random() < 0.5:
        return gemv_case(spread(rng, 1, 32), spread(rng, 64, 28672), k, group, dtype, zeros)
    k = min(k, 4096)
    n = spread(rng, 64, 4096)
    return gemv_case(rng.randint(1, 16), n, k, group, dtype, zeros, rng.choice([8, 16, 64]), rng.randint(1, 4),
                     rng.random() < 0.5)


def padded_rows(slots, experts, block):
    """Rows of the grouped layout that hold any split of `slots` rows over the experts."""
    return (slots + min(experts, slots) * (block - 1)) // block * block


def plain_plan(ids, experts, block):
    """(rows, slots, m_block_group): every slot's row in the grouped layout, every row's slot, every 128-row block's
    expert; -1 = none. Within an expert the slots keep their order."""
    flat = ids.reshape(-1).long()
    total = flat.numel()
    room = padded_rows(total, experts, block)
    key = torch.where(flat >= 0, flat, experts)
    counts = torch.zeros(experts + 1, dtype=torch.long, device=flat.device).scatter_add_(0, key, torch.ones_like(key))
    sizes = (counts[:experts] + block - 1) // block * block
    ends = sizes.cumsum(0)
    starts = torch.cat([ends - sizes, torch.full_like(ends[:1], room)])
    ordered, order = torch.sort(key, stable=True)
    rank = torch.arange(total, device=flat.device) - (counts.cumsum(0) - counts)[ordered]
    place = torch.where(ordered < experts, starts[ordered] + rank, room)
    slots = torch.full((room + 1,), -1, dtype=torch.int32, device=flat.device)
    slots[place] = order.to(torch.int32)
    rows = torch.empty_like(flat, dtype=torch.int32)
    rows[order] = torch.where(ordered < experts, place, -1).to(torch.int32)
    first = torch.arange(0, room, 128, device=flat.device)
    owner = (first[:, None] >= ends[None, :]).sum(1)
    return rows.view_as(ids), slots[:room], torch.where(owner < experts, owner, -1).to(torch.int32)


def routed_ids(case, gen, device):
    """Distinct experts for each token, some far more liked than others; dropped slots are -1."""
    t, e, k = case["tokens"], case["experts"], case["k"] if "k" in case and case["op"] != "gemv" else case["topk"]
    liked = torch.randn((1, e), generator=gen, device=device)
    ids = torch.sort(torch.randn((t, e), generator=gen, device=device) + liked, dim=1, descending=True)[1][:, :k]
    if case.get("dropped"):
        ids = torch.where(torch.rand((t, k), generator=gen, device=device) < 0.1, -1, ids)
    return ids.to(torch.int32).contiguous()


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=gen, device=device)  # noqa: E731
    s = {"case": case}
    if case["op"] == "route":
        t, e, dtype = case["tokens"], case["experts"], DTYPES[case["dtype"]]
        logits = normal(t, e) * 1.5 + normal(1, e) * 0.7
        if case["masked"]:  # half of the experts are open to each token, as in group-limited routing
            shut = torch.rand((t, e), generator=gen, device=device) < 0.5
            logits = logits.masked_fill(shut, -math.inf)
        s["valid"] = None
        if case["padded"]:
            s["valid"] = torch.rand((t,), generator=gen, device=device) < 0.9
            logits = torch.where(s["valid"][:, None], logits, math.nan)  # what padding holds is nobody's
        s["logits"] = logits.to(dtype)
        if case["train"]:
            s["dweights"] = normal(t, case["k"]) * 1e-2
            s["dloss"] = torch.tensor(0.01, device=device)
        return s
    if case["op"] in ("dispatch", "combine"):
        t, k, dtype = case["tokens"], case["k"], DTYPES[case["dtype"]]
        s["ids"] = routed_ids(case, gen, device)
        if case["op"] == "dispatch":
            s["x"] = normal(t, case["width"]).to(dtype)
            return s
        weights = torch.rand((t, k), generator=gen, device=device) + 0.05
        s["weights"] = weights / weights.sum(1, keepdim=True)
        if case["block"]:
            s["rows"], s["slots"], _ = plain_plan(s["ids"], case["experts"], case["block"])
            s["y"] = normal(s["slots"].numel(), case["width"]).to(dtype)
        else:
            s["rows"] = s["slots"] = None
            s["y"] = normal(t, k, case["width"]).to(dtype)
        if case["train"]:
            s["dout"] = (normal(t, case["width"]) * 1e-2).to(dtype)
        return s
    t, n, k, group, e, dtype = (case[x] for x in ("tokens", "n", "k", "group", "experts", "dtype"))
    many, groups = max(1, e), -(-k // group)
    # Weights as a quantiser leaves them: codes around the middle, positive group scales, zero points near 8.
    codes = torch.randint(0, 6, (2, many, n, k // 2), generator=gen, device=device, dtype=torch.uint8)
    codes += torch.randint(0, 6, codes.shape, generator=gen, device=device, dtype=torch.uint8)
    codes += torch.randint(0, 6, codes.shape, generator=gen, device=device, dtype=torch.uint8)
    q = codes[0] | codes[1] << 4
    scales = ((torch.rand((many, n, groups), generator=gen, device=device) + 0.5) * 0.01).to(DTYPES[dtype])
    zeros = None
    if case["zeros"]:
        zeros = torch.randint(6, 11, (many, n, groups), generator=gen, device=device, dtype=torch.uint8)
    if not e:
        q, scales, zeros = q[0], scales[0], None if zeros is None else zeros[0]
    else:
        s["ids"] = routed_ids(case, gen, device)
    s["q"], s["scales"], s["zeros"] = q, scales, zeros
    s["x"] = (normal(t, case["topk"], k) if case["down"] else normal(t, k)).to(DTYPES[dtype])
    return s


def work(case):
    if case["op"] == "route":
        t, e, k, b = case["tokens"], case["experts"], case["k"], BYTES[case["dtype"]]
        moved, flops = t * e * b + t * k * 8 + e * 4 + 8 + (t if case["padded"] else 0), 6 * t * e
        if case["train"]:
            moved, flops = moved + t * e * b + t * k * 4, flops + 6 * t * e
        return {"bytes": moved, "flops": flops}
    if case["op"] in ("dispatch", "combine"):
        t, k, w, b = case["tokens"], case["k"], case["width"], BYTES[case["dtype"]]
        room = padded_rows(t * k, case["experts"], case["block"]) if case["block"] else t * k
        if case["op"] == "dispatch":
            return {"bytes": t * w * b + room * w * b + t * k * 8 + room * 4 + room // 128 * 4, "flops": 0}
        moved, flops = t * k * w * b + t * w * b + t * k * 8, 2 * t * k * w
        if case["train"]:
            moved, flops = moved + t * w * b + room * w * b + t * k * 4, flops + 3 * t * k * w
        return {"bytes": moved, "flops": flops}
    t, n, k, e = case["tokens"], case["n"], case["k"], case["experts"]
    slots = t * case["topk"] if e else t
    used = e * (1 - (1 - 1 / e) ** slots) if e else 1
    groups = -(-k // case["group"])
    matrix = n * k // 2 + n * groups * (3 if case["zeros"] else 2)
    rows = slots if case["down"] else t
    return {"bytes": int(used * matrix) + rows * k * 2 + slots * n * 2, "flops": 2 * slots * n * k}


def plain_route(s):
    c, valid = s["case"], s["valid"]
    e, k = c["experts"], c["k"]
    logits = s["logits"].float()
    routed = (logits > -math.inf).any(1)
    if valid is not None:
        routed = routed & valid
    logits = torch.where(routed[:, None], logits, 0.0)
    top = logits.max(1, keepdim=True)[0]
    exps = torch.exp(logits - top)
    probs = exps / exps.sum(1, keepdim=True)
    value, ids = torch.sort(logits, dim=1, descending=True, stable=True)
    value, ids = value[:, :k], ids[:, :k]
    live = routed[:, None] & (value > -math.inf)
    chosen = torch.where(live, torch.exp(value - top), 0.0)
    weights = chosen / (chosen.sum(1, keepdim=True) if c["renormalize"] else exps.sum(1, keepdim=True))
    weights = torch.where(live, weights, 0.0)
    key = torch.where(live, ids, e).reshape(-1)
    counts = torch.zeros(e + 1, dtype=torch.int32, device=key.device)
    counts = counts.scatter_add_(0, key, torch.ones_like(key, dtype=torch.int32))[:e]
    tokens = routed.sum(dtype=torch.int32)
    share = torch.where(routed[:, None], probs, 0.0).sum(0)
    n = tokens.clamp(min=1).float()
    loss = e * (counts / (k * n) * (share / n)).sum()
    out = {"ids": torch.where(live, ids, -1).to(torch.int32), "weights": weights, "counts": counts, "tokens": tokens,
           "loss": loss}
    if c["train"]:
        pull = torch.where(live, s["dweights"], 0.0) * weights
        total = pull.sum(1, keepdim=True)
        push = s["dloss"] * e * counts / (k * n * n)
        level = (probs * push).sum(1, keepdim=True)
        grad = probs * (push - level - (0.0 if c["renormalize"] else total))
        grad = grad.scatter_add(1, ids, pull - weights * total if c["renormalize"] else pull)
        out["dlogits"] = torch.where(routed[:, None], grad, 0.0).to(s["logits"].dtype)
    return out


def plain_dispatch(s):
    c = s["case"]
    rows, slots, blocks = plain_plan(s["ids"], c["experts"], c["block"])
    a = s["x"][slots.clamp(min=0).long() // c["k"]]
    return {"rows": rows, "slots": slots, "blocks": blocks, "a": torch.where(slots[:, None] >= 0, a, 0.0).to(a.dtype)}


def plain_combine(s):
    c, y, weights = s["case"], s["y"], s["weights"]
    if s["rows"] is None:
        picked = y.float()
    else:
        picked = torch.where(s["rows"][..., None] >= 0, y[s["rows"].clamp(min=0).long()].float(), 0.0)
    out = {"out": (weights[..., None] * picked).sum(1).to(y.dtype)}
    if c["train"]:
        dout = s["dout"].float()
        out["dweights"] = (dout[:, None, :] * picked).sum(2)
        if s["slots"] is None:
            out["dy"] = (weights[..., None] * dout[:, None, :]).to(y.dtype)
        else:
            at = s["slots"].clamp(min=0).long()
            dy = weights.reshape(-1)[at][:, None] * dout[at // c["k"]]
            out["dy"] = torch.where(s["slots"][:, None] >= 0, dy, 0.0).to(y.dtype)
    return out


def plain_weights(q, scales, zeros, group):
    """The matrix or matrices that the codes, scales and zero points stand for, in fp32."""
    k = q.shape[-1] * 2
    codes = torch.stack([q & 15, q >> 4], dim=-1).flatten(-2).float()
    at = torch.arange(k, device=q.device) // group
    return (codes - (8.0 if zeros is None else zeros.float()[..., at])) * scales.float()[..., at]


def plain_gemv(s):
    c, x = s["case"], s["x"]
    if not c["experts"]:
        return (x.float() @ plain_weights(s["q"], s["scales"], s["zeros"], c["group"]).T).to(x.dtype)
    ids = s["ids"].reshape(-1).long()
    zeros = None if s["zeros"] is None else s["zeros"][ids]
    w = plain_weights(s["q"][ids], s["scales"][ids], zeros, c["group"])
    rows = x.reshape(-1, c["k"]) if c["down"] else x.repeat_interleave(c["topk"], 0)
    return torch.bmm(w, rows.float()[:, :, None])[:, :, 0].view(c["tokens"], c["topk"], c["n"]).to(x.dtype)


def run(state):
    s = state
    c = s["case"]
    if not own:
        return {"route": plain_route, "dispatch": plain_dispatch, "combine": plain_combine, "gemv": plain_gemv}[c["op"]](s)
    import maia_b200 as kl

    if c["op"] == "route":
        r = kl.moe_route(s["logits"], c["k"], renormalize=c["renormalize"], valid=s["valid"])
        out = {"ids": r.ids, "weights": r.weights, "counts": r.counts, "tokens": r.tokens, "loss": r.loss}
        if c["train"]:
            out["dlogits"] = kl.moe_route_grad(s["logits"], r, s["dweights"], s["dloss"], renormalize=c["renormalize"],
                                               valid=s["valid"])
        return out
    if c["op"] == "dispatch":
        plan = kl.moe_plan(s["ids"], c["experts"], block=c["block"])
        return {"rows": plan.rows, "slots": plan.slots, "blocks": plan.m_block_group, "a": kl.moe_dispatch(s["x"], plan)}
    if c["op"] == "combine":
        out = {"out": kl.moe_combine(s["y"], s["weights"], rows=s["rows"])}
        if c["train"]:
            out["dy"], out["dweights"] = kl.moe_combine_grad(s["dout"], s["y"], s["weights"], rows=s["rows"],
                                                             slots=s["slots"])
        return out
    return kl.gemv_int4(s["x"], s["q"], s["scales"], s["zeros"], group=c["group"], ids=s.get("ids"))


def exact(case, seed):
    """The same outputs from the definitions, token by token or expert by expert, in float64; None where an output is
    whole numbers or copies."""
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "dispatch":
        return None
    if case["op"] == "route":
        logits, e, k = s["logits"].to(f64), case["experts"], case["k"]
        logits = torch.nan_to_num(logits, nan=0.0, neginf=-math.inf)
        keep = torch.isfinite(logits).any(1)
        if s["valid"] is not None:
            keep &= s["valid"]
        p = torch.softmax(logits[keep], 1)
        # Stable order: a value's rank is the number of experts that come before it.
        ids = torch.argsort(-logits[keep], dim=1, stable=True)[:, :k]
        chosen = torch.gather(p, 1, ids)
        live = torch.gather(logits[keep], 1, ids) > -math.inf
        w = chosen / chosen.sum(1, keepdim=True) if case["renormalize"] else chosen
        weights = torch.zeros((case["tokens"], k), dtype=f64, device=p.device)
        weights[keep] = w
        n = int(keep.sum())
        counts = torch.bincount(ids[live], minlength=e).to(f64)
        loss = e * torch.dot(counts, p.mean(0)) / (k * n) if n else torch.zeros((), dtype=f64, device=p.device)
        out = {"ids": None, "weights": weights, "counts": None, "tokens": None, "loss": loss}
        if case["train"]:
            grad = torch.zeros(logits.shape, dtype=f64, device=p.device)
            if n:
                # d loss / d p and d weights / d p, then the softmax's Jacobian.
                dp = (s["dloss"].to(f64) * e * counts / (k * n * n)).expand(n, e).clone()
                dw = torch.where(live, s["dweights"][keep].to(f64), 0.0)
                if case["renormalize"]:
                    dw = (dw - (dw * w).sum(1, keepdim=True)) / chosen.sum(1, keepdim=True)
                dp.scatter_add_(1, ids, torch.where(live, dw, 0.0))
                grad[keep] = p * (dp - (dp * p).sum(1, keepdim=True))
            out["dlogits"] = grad
        return out
    if case["op"] == "combine":
        y, w, t, k = s["y"].to(f64), s["weights"].to(f64), case["tokens"], case["k"]
        flat = y.reshape(-1, case["width"])
        rows = torch.arange(t * k, device=y.device).view(t, k) if s["rows"] is None else s["rows"].long()
        out = torch.zeros((t, case["width"]), dtype=f64, device=y.device)
        dweights = torch.zeros((t, k), dtype=f64, device=y.device)
        dy = torch.zeros_like(flat)
        for j in range(k):
            has = rows[:, j] >= 0
            at = rows[has, j]
            out[has] += w[has, j, None] * flat[at]
            if case["train"]:
                dout = s["dout"][has].to(f64)
                dweights[has, j] = torch.einsum("tn,tn->t", dout, flat[at])
                dy[at] = w[has, j, None] * dout
        if case["train"]:
            return {"out": out, "dweights": dweights, "dy": dy.view_as(y)}
        return {"out": out}
    t, n, k, e, top = case["tokens"], case["n"], case["k"], case["experts"], case["topk"]
    many = max(1, e)
    q = s["q"].view(many, n, k // 2)
    scales = s["scales"].view(many, n, -1).to(f64)
    zeros = torch.full_like(scales, 8.0) if s["zeros"] is None else s["zeros"].view(many, n, -1).to(f64)
    if e:
        x = (s["x"].reshape(t * top, k) if case["down"] else s["x"].repeat_interleave(top, 0)).to(f64)
        pick = s["ids"].reshape(-1)
    else:
        x, pick = s["x"].to(f64), torch.zeros(t, dtype=torch.int32, device=q.device)
    out = torch.zeros((x.shape[0], n), dtype=f64, device=q.device)
    for m in range(many):
        mine = (pick == m).nonzero()[:, 0]
        if not mine.numel():
            continue
        for at in range(0, n, 4096):
            code = q[m, at:at + 4096]
            w = torch.empty((code.shape[0], k), dtype=f64, device=q.device)
            w[:, 0::2] = (code % 16).to(f64)
            w[:, 1::2] = torch.div(code, 16, rounding_mode="floor").to(f64)
            wide = lambda v: v[m, at:at + 4096].repeat_interleave(case["group"], 1)[:, :k]  # noqa: E731
            out[mine, at:at + 4096] = x[mine] @ ((w - wide(zeros)) * wide(scales)).T
    return out.view(t, top, n) if e else out
