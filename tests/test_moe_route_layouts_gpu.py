"""The router and its gradient in every layout of a token's entries over lanes (up to 64, 128, 256, 512 and 1024 experts; a
launch of its own, or fused with the sort), with excluded entries among the others, against 64-bit forms.  The bounds
follow each row's own entries."""
import math

import pytest
import torch

from _moe import EPS32, STEP, TINY

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
MORE = 1 + 2.0 ** -10           # products of the bounds' own terms
# experts and choices: both sides of every layout's limit, widths that no vector divides, more choices than lanes
WIDTHS = [(8, 3), (64, 9), (65, 4), (128, 32), (129, 5), (200, 17), (255, 2), (256, 8), (257, 3), (400, 20), (512, 32), (513, 1), (770, 6)]


def _logits(T, E, dtype, seed, kind):
    g = torch.Generator().manual_seed(seed)
    if kind == "normal":
        return (torch.randn((T, E), generator=g) * 2).to(dtype).cuda(), None
    l = torch.randint(-3, 4, (T, E), generator=g).float()           # ties everywhere
    l[l == 0] = -0.0                                                # equal to +0
    l[:, 1] = 0.0
    l += torch.randn((T, E), generator=g) * (torch.rand((T, 1), generator=g) < 0.5)
    l = l.to(dtype)
    l[torch.rand((T, E), generator=g) < 0.2] = math.nan
    l[torch.rand((T, E), generator=g) < 0.2] = -math.inf
    row = torch.arange(T) % 8
    l[row == 1] = -math.inf                                         # nothing to choose
    l[(row == 2)[:, None] & (torch.arange(E) > 1)[None, :]] = -math.inf    # fewer than k
    l[(row == 3)[:, None] & (torch.arange(E) % 5 == 1)[None, :]] = math.inf    # share the weight
    l[(row == 4)[:, None] & (torch.arange(E) % 3 == 0)[None, :]] = torch.finfo(dtype).min    # a value like others ...
    l[row == 5] = torch.finfo(dtype).min                            # ... and the row's largest
    mask = torch.rand((T,), generator=g) < 0.8
    mask[:6] = True
    l[~mask] = torch.where(torch.rand((int((~mask).sum()), E), generator=g) < 0.5, math.nan, math.inf).to(dtype)
    return l.cuda(), mask.cuda()


def _exact(l, k, renormalize, mask):
    """64-bit weights and choices, the share p of every entry, and the bounds of both over EPS32."""
    l = l.double()
    out = torch.isnan(l) if mask is None else torch.isnan(l) | ~mask[:, None]
    l = torch.where(out, -math.inf, l)
    v, e = torch.sort(l, dim=1, descending=True, stable=True)       # equal ones: the lowest index first
    e = torch.where(v > -math.inf, e, -1)[:, :k]
    top = v[:, :1]
    chosen = torch.zeros((l.shape[0], l.shape[1] + 1), dtype=torch.bool, device=l.device)
    chosen = chosen.scatter_(1, torch.where(e < 0, l.shape[1], e), True)[:, :-1]
    p = torch.where((l == top) & (l > -math.inf), 1.0, torch.exp(l - top)).nan_to_num(0.0)
    gap = torch.where(p > 0, top - l, 0.0).nan_to_num(0.0)          # (equal infinities: no difference is taken)
    if renormalize:
        p = torch.where(chosen, p, 0.0)
    total = p.sum(1, keepdim=True).clamp(min=1.0)                   # (the largest term is 1)
    # an exponential: its argument is rounded once (the difference times half a step), then up to two steps of its own;
    # the sum: its terms' errors and a half step for each addition, k of them one after the other or up to 32 in a lane
    # and a tree of 5; a division
    term = gap + 4
    rel = term + (p * term).sum(1, keepdim=True) / total + (k if renormalize else 37) + 1
    p = p / total
    w = torch.where(e < 0, 0.0, p.gather(1, e.clamp(min=0)))
    return w, e, p, rel


LOST = 2.0 ** -147              # of an exponential below the smallest normal number: two of its steps, and the rest rounded


@pytest.mark.parametrize("E,k", WIDTHS)
@pytest.mark.parametrize("T", [6, 300, 512, 513, 1300])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("kind", ["normal", "odd"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_and_its_gradient(T, E, k, dtype, kind, renormalize):
    from eval_test_b200 import moe
    l, mask = _logits(T, E, dtype, T + 7 * E, kind)
    r = moe.route(l, k, renormalize=renormalize, mask=mask)
    w, e, p, rel = _exact(l, k, renormalize, mask)
    assert torch.equal(r.experts.long(), e)
    rel_w = torch.where(w > 0, rel.gather(1, e.clamp(min=0)), 0.0)
    assert float(rel_w.max()) * EPS32 < 2.0 ** -15                  # the bound says something
    assert torch.all((r.weights.double() - w).abs() <= rel_w * EPS32 * MORE * w + LOST)
    # the plan is that of these choices
    ids = torch.where(e < 0, E, e).reshape(-1)
    source = torch.sort(ids, stable=True).indices
    live = int((ids < E).sum())
    assert torch.equal(r.plan.source[:live].long(), source[:live]) and bool((r.plan.source[live:] == -1).all())
    assert torch.equal(r.plan.offsets.long(), torch.cat([ids.new_zeros(1), torch.bincount(ids, minlength=E + 1)[:E].cumsum(0)]))

    dw = torch.randn((T, k), generator=torch.Generator().manual_seed(9)).cuda()
    dw[e < 0] = math.nan                                            # gradients of weights that do not exist
    got = moe.route_backward(dw, l, r.weights, r.experts, renormalize=renormalize)
    assert got.dtype == dtype and got.shape == l.shape
    d64 = torch.where(e < 0, 0.0, dw.double())
    g = torch.zeros((T, E + 1), dtype=torch.float64, device="cuda").scatter_(1, torch.where(e < 0, E, e), d64)[:, :E]
    dot, sizes = (w * d64).sum(1, keepdim=True), (w * d64).abs().sum(1, keepdim=True)
    want = p * (g - dot)
    # p with a reciprocal and a product in the place of the division, the weights' own errors and the roundings of the
    # dot product (a product and an addition for each choice, 5 steps of a tree), a difference and a product
    bound = (rel + 2 + rel_w.amax(1, keepdim=True) + k + 10) * EPS32 * MORE * p * (g.abs() + sizes)
    bound = bound + 2 * LOST * (g.abs() + sizes + 1) + STEP[dtype] * want.abs() * (1 + 2.0 ** -7) + TINY[dtype]
    assert torch.all((got.double() - want).abs() <= bound)
    assert not got[p == 0].any()


def test_a_wrong_sum_would_be_seen():
    """An excluded entry that was counted, or a choice left out of the sum, is far outside of the bound (on the oracle)."""
    l, mask = _logits(300, 48, F32, 3, "odd")
    w, e, p, rel = _exact(l, 6, False, mask)
    few = (e[:, 1] >= 0) & (w[:, 0] < 1)
    wrong = w / (1 + p.amin(1, keepdim=True).clamp(min=1e-3))       # one more entry in the sum
    rel_w = rel.gather(1, e.clamp(min=0))
    assert bool(((wrong - w).abs() > 10 * rel_w * EPS32 * w + LOST)[few, 0].all()) and int(few.sum()) > 100
