"""Plain 64-bit forms of the mixture-of-experts operations, for the tests."""
from __future__ import annotations

import math

import torch

EPS32 = 2.0 ** -24          # half a step of fp32, relative
STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}     # half steps
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # half the smallest step


def plan_ref(experts: torch.Tensor, E: int):
    """offsets, tiles, wide_tiles, rows, slots, source of int choices [T, k], by counting (CPU, int64)."""
    ids = experts.cpu().reshape(-1).tolist()
    by = [[i for i, e in enumerate(ids) if e == x] for x in range(E)]
    offsets, tiles, wide = [0], [0], [0]
    rows, slots, source = [-1] * len(ids), [-1] * len(ids), []
    for copies in by:
        for n, i in enumerate(copies):
            rows[i], slots[i] = offsets[-1] + n, tiles[-1] * 128 + n
        source += copies
        offsets.append(offsets[-1] + len(copies))
        tiles.append(tiles[-1] + (len(copies) + 127) // 128)
        wide.append(wide[-1] + (len(copies) + 255) // 256)
    source += [-1] * (len(ids) - len(source))
    t = lambda v: torch.tensor(v, dtype=torch.int64)  # noqa: E731
    return t(offsets), t(tiles), t(wide), t(rows).view(experts.shape), t(slots).view(experts.shape), t(source)


def check_plan(plan, experts, E):
    assert (plan.num_tokens, plan.top_k, plan.num_experts) == (*experts.shape, E)
    for name, want in zip(("offsets", "tiles", "wide_tiles", "rows", "slots", "source"), plan_ref(experts, E)):
        got = getattr(plan, name)
        assert got.dtype == torch.int32 and torch.equal(got.cpu().long(), want), name


def route_ref(logits: torch.Tensor, k: int, renormalize: bool, mask=None):
    """(weights float64, experts) of [T, E], on the CPU, one entry after the other."""
    l = logits.double().cpu()
    T, E = l.shape
    weights, experts = torch.zeros((T, k), dtype=torch.float64), torch.full((T, k), -1, dtype=torch.int64)
    for t in range(T):
        if mask is not None and not bool(mask[t]):
            continue
        row = [(float(v), e) for e, v in enumerate(l[t].tolist()) if not math.isnan(v) and v > -math.inf]
        if not row:
            continue
        row.sort(key=lambda x: (-x[0], x[1]))
        top = row[0][0]
        p = [1.0 if v == top else math.exp(v - top) for v, _ in row]
        total = sum(p[:k]) if renormalize else sum(p)
        for j in range(min(k, len(row))):
            weights[t, j], experts[t, j] = p[j] / total, row[j][1]
    return weights, experts


def dequant(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """[..., K/2] bytes and [..., K/16] e4m3 -> float64 [..., K]."""
    values = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64,
                          device=codes.device)
    c = codes.int()
    v = values[torch.stack([c & 15, c >> 4], dim=-1).flatten(-2)]
    return (v.unflatten(-1, (-1, 16)) * scales.double()[..., None]).flatten(-2)


def choices(T, E, k, drop=0.0, seed=0, device="cuda"):
    """k different experts for each token, some of them dropped."""
    g = torch.Generator().manual_seed(seed)
    ids = (torch.rand((T, E), generator=g) + torch.rand((1, E), generator=g)).topk(k, dim=1).indices.int()
    ids[torch.rand((T, k), generator=g) < drop] = -1
    return ids.to(device)
