"""The expert layer's definitions in 64 bits on the host, element by element where order matters."""

import math

import torch

F64 = torch.float64


def route(logits, k, renormalize=True, valid=None):
    """(ids, weights, counts, routed, loss, probabilities) in float64."""
    x = logits.detach().cpu().to(F64)
    tokens, experts = x.shape
    ids = torch.full((tokens, k), -1, dtype=torch.int32)
    weights = torch.zeros((tokens, k), dtype=F64)
    probs = torch.zeros((tokens, experts), dtype=F64)
    counts = torch.zeros(experts, dtype=torch.int32)
    routed = 0
    for t in range(tokens):
        row = x[t].tolist()
        open_ = [e for e in range(experts) if not row[e] == -math.inf]
        if (valid is not None and not bool(valid[t])) or not open_:
            continue
        routed += 1
        probs[t] = torch.softmax(x[t], 0)
        order = sorted(open_, key=lambda e: (0 if math.isnan(row[e]) else 1, -row[e] if not math.isnan(row[e]) else 0, e))[:k]
        total = sum(probs[t, e].item() for e in order)
        for j, e in enumerate(order):
            ids[t, j] = e
            weights[t, j] = probs[t, e] / total if renormalize else probs[t, e]
            counts[e] += 1
    loss = experts * (counts.to(F64) / (k * routed) * probs.sum(0) / routed).sum().item() if routed else 0.0
    return ids, weights, counts, routed, loss, probs


def route_grad(logits, k, dweights, dloss, renormalize=True, valid=None):
    """d(sum weights dweights + loss dloss) / d logits by autograd through the float64 definition, with
    the choice and the counts held fixed."""
    ids, _, counts, routed, _, _ = route(logits, k, renormalize, valid)
    x = logits.detach().cpu().to(F64)
    live = ids >= 0
    on = live.any(1)
    grad = torch.zeros_like(x)
    if not routed:
        return grad
    leaf = x[on].clone().requires_grad_()
    p = torch.softmax(leaf, 1)
    sel = torch.where(live[on], p.gather(1, ids[on].clamp(min=0).long()), 0.0)
    w = sel / sel.sum(1, keepdim=True) if renormalize else sel
    total = leaf.sum() * 0
    if dweights is not None:
        total = total + torch.where(live[on], w * dweights.cpu().to(F64)[on], 0.0).sum()
    if dloss is not None:
        f = counts.to(F64) / (k * routed)
        total = total + float(dloss) * x.shape[1] * (f * p.sum(0) / routed).sum()
    grad[on] = torch.autograd.grad(total, leaf)[0]
    return grad


def plan(ids, experts, block, m):
    """rows, slots, m_block_group by walking the slots in order."""
    flat = ids.cpu().reshape(-1).tolist()
    of = {e: [s for s, x in enumerate(flat) if x == e] for e in range(experts)}
    rows = torch.full((len(flat),), -1, dtype=torch.int32)
    slots = torch.full((m,), -1, dtype=torch.int32)
    groups = torch.full((m // 128,), -1, dtype=torch.int32)
    at = 0
    for e in range(experts):
        for i, s in enumerate(of[e]):
            rows[s] = at + i
            slots[at + i] = s
        size = -(-len(of[e]) // block) * block
        groups[at // 128:(at + size) // 128] = e
        at += size
    return rows.view(ids.shape), slots, groups


def int4_weights(q, scales, zeros, group):
    q = q.cpu()
    codes = torch.stack([q % 16, q // 16], -1).flatten(-2).to(F64)
    at = torch.arange(codes.shape[-1]) // group
    z = 8.0 if zeros is None else zeros.cpu().to(F64)[..., at]
    return (codes - z) * scales.cpu().to(F64)[..., at]
