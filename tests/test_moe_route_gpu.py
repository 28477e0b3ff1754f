"""Router, its gradient and the plan of sorted copies against plain 64-bit forms."""
import math

import pytest
import torch

from _moe import EPS32, STEP, TINY, check_plan, choices, route_ref

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _logits(T, E, dtype, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((T, E), generator=g) * spread).to(dtype).cuda()


def _weight_bound(logits, E):
    """Relative bound of a weight: exp of a difference rounded to fp32 (its size times half a step) with an error of up
    to two steps, a sum of E terms (32 lanes, E / 32 in a lane, 5 steps of the tree) twice, one division."""
    l = logits.float().cpu()
    fin = torch.where(torch.isfinite(l), l, 0.0)
    gap = float((fin.max() - fin.min()).abs()) if l.numel() else 0.0
    return (gap + 4 + 2 * (math.ceil(E / 32) + 5) + 2) * EPS32


def _check(logits, k, renormalize, mask=None):
    from eval_test_b200 import moe
    r = moe.route(logits, k, renormalize=renormalize, mask=mask)
    torch.cuda.synchronize()
    want_w, want_e = route_ref(logits, k, renormalize, mask)
    assert torch.equal(r.experts.cpu().long(), want_e)
    bound = _weight_bound(logits, logits.shape[1])
    assert torch.all((r.weights.cpu().double() - want_w).abs() <= bound * want_w + 2.0 ** -149)
    check_plan(r.plan, r.experts, logits.shape[1])
    return r


@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 8), (3, 33, 5), (33, 64, 8), (256, 40, 3), (257, 64, 8), (1000, 300, 32),
                                   (70, 1024, 16), (2001, 128, 2), (300, 31, 31)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_against_the_definition(T, E, k, dtype, renormalize):
    _check(_logits(T, E, dtype, T + E + k), k, renormalize)


@pytest.mark.parametrize("T", [7, 300])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_ties_infinities_nan_and_empty_rows(T, renormalize):
    g = torch.Generator().manual_seed(T)
    l = torch.randint(-2, 3, (T, 48), generator=g).float()          # ties everywhere
    l[l == 0] = -0.0                                                # equal to +0
    l[:, 5] = 0.0
    l[1] = -math.inf                                                # nothing to choose
    l[2, 3:] = -math.inf                                            # fewer than k
    l[3, ::2] = math.nan
    l[4, 10] = l[4, 40] = math.inf                                  # share the weight
    l[5] = torch.finfo(F32).min                                     # the type's lowest value is a value
    l[6] = math.nan
    mask = torch.rand((T,), generator=g) < 0.7
    mask[:6] = True
    mask[6] = False                                                 # NaN in a masked place
    r = _check(l.cuda(), 6, renormalize, mask.cuda())
    assert r.weights[4, 0] == 0.5 and r.weights[4, 1] == 0.5 and r.experts[4, :2].tolist() == [10, 40]
    assert not r.weights[1].any() and (r.experts[1] == -1).all()
    assert torch.isfinite(r.weights).all()


def test_route_rows_with_a_pitch_and_without_alignment():
    from eval_test_b200 import moe
    big = _logits(50, 201, BF16, 3)
    _check(big[:, 1:100], 4, True)
    _check(big[::3, 7:8], 1, False)
    _check(big[5:6, :].expand(9, 201), 3, True)                     # one row for all tokens
    with pytest.raises(ValueError, match="at most"):                # (and for more than 32 bits count)
        moe.route(big[5:6, :].expand((1 << 32) + 5, 201), 3)


def test_route_of_no_tokens():
    from eval_test_b200 import moe
    r = moe.route(torch.empty((0, 16), device="cuda"), 4)
    assert r.weights.shape == (0, 4) and r.plan.rows.shape == (0, 4)
    assert not r.plan.offsets.any() and not r.plan.tiles.any()
    assert moe.route_backward(r.weights, torch.empty((0, 16), device="cuda"), r.weights, r.experts).shape == (0, 16)


def _forward64(l, experts, renormalize):
    """Weights of given choices of float64 logits [T, E] (all finite)."""
    chosen = l.gather(1, experts)
    return torch.softmax(chosen, 1) if renormalize else torch.softmax(l, 1).gather(1, experts)


@pytest.mark.parametrize("T,E,k", [(1, 8, 2), (5, 1, 1), (40, 33, 5), (300, 128, 8), (20, 1024, 32), (2000, 64, 4)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_backward_against_formula_and_differences(T, E, k, dtype, renormalize):
    from eval_test_b200 import moe
    l = _logits(T, E, dtype, T * 7 + E)
    r = moe.route(l, k, renormalize=renormalize)
    dw = torch.randn((T, k), generator=torch.Generator().manual_seed(9)).cuda()
    got = moe.route_backward(dw, l, r.weights, r.experts, renormalize=renormalize)
    assert got.dtype == dtype and got.shape == l.shape
    l64, e64, d64 = l.double(), r.experts.long(), dw.double()
    w = _forward64(l64, e64, renormalize)
    g = torch.zeros_like(l64).scatter_(1, e64, d64)
    p = torch.softmax(l64, 1) if not renormalize else torch.zeros_like(l64).scatter_(1, e64, w)
    dot = (w * d64).sum(1, keepdim=True)
    want = p * (g - dot)
    # the weight's own bound, the k products of the dot with the 5 steps of its tree, three more roundings
    size = p * (g.abs() + (w * d64.abs()).sum(1, keepdim=True))
    bound = 2 * (_weight_bound(l, E) + (k + 8) * EPS32) * size + STEP[dtype] * want.abs() + TINY[dtype]
    assert torch.all((got.double() - want).abs() <= bound)
    if dtype == F32:
        # differences of the 64-bit forward pass along one direction
        v = torch.randn((T, E), generator=torch.Generator().manual_seed(10), dtype=torch.float64).cuda()
        h = 1e-5
        up, down = (_forward64(l64 + s * h * v, e64, renormalize) for s in (1, -1))
        slope = ((up - down) * d64).sum() / (2 * h)
        # third derivatives of a softmax are below 6 in size: h^2 of them, and 64-bit cancellation over 2h
        room = (bound * v.abs()).sum() + (d64.abs().sum() * float(v.abs().max()) ** 3) * h * h * 6 + d64.abs().sum() * 1e-15 / h
        assert abs(float((got.double() * v).sum() - slope)) <= float(room)


@pytest.mark.parametrize("renormalize", [True, False])
def test_route_backward_of_rows_without_choices(renormalize):
    from eval_test_b200 import moe
    l = _logits(6, 40, F32, 1)
    l[0] = -math.inf
    l[1, 2:] = -math.inf
    l[2, ::3] = math.nan
    l[3] = math.nan
    mask = torch.tensor([True, True, True, False, False, True]).cuda()
    r = moe.route(l, 4, renormalize=renormalize, mask=mask)
    dw = torch.randn((6, 4), generator=torch.Generator().manual_seed(2)).cuda()
    dw[0] = dw[3] = math.nan                                        # gradients of weights that do not exist
    d = moe.route_backward(dw, l, r.weights, r.experts, renormalize=renormalize)
    assert torch.isfinite(d).all()
    assert not d[0].any() and not d[3].any() and not d[4].any() and not d[1, 2:].any() and not d[2, ::3].any()
    assert d[1, :2].any() and d[5].any()


# ------------------------------------------------------------------------------------------------ plan
@pytest.mark.parametrize("T,E,k,drop", [(1, 1, 1, 0.0), (1, 64, 8, 0.0), (5, 3, 2, 0.5), (129, 7, 1, 0.0), (1025, 1024, 3, 0.1),
                                        (3000, 33, 5, 0.3), (20011, 64, 8, 0.0), (5500, 1024, 3, 0.2), (16385, 1, 1, 0.1),
                                        (4096, 300, 4, 0.0), (70001, 129, 1, 0.0)])
def test_plan_sorts_stably(T, E, k, drop):
    from eval_test_b200 import moe
    ids = choices(T, E, k, drop, seed=T)
    check_plan(moe.plan(ids, E), ids, E)


def test_plan_of_odd_choices():
    from eval_test_b200 import moe
    ids = torch.full((400, 3), -1, dtype=torch.int32, device="cuda")
    check_plan(moe.plan(ids, 5), ids, 5)                            # nothing is routed
    ids[:] = 4
    check_plan(moe.plan(ids, 5), ids, 5)                            # every copy to one expert, three times a token
    g = torch.Generator().manual_seed(0)
    ids = torch.randint(-3, 9, (777, 4), generator=g, dtype=torch.int32)
    ids[0] = torch.tensor([2 ** 31 - 1, -2 ** 31, 5, 6])
    ids = ids.cuda()
    check_plan(moe.plan(ids, 6), ids, 6)                            # ids out of range are not routed
    empty = moe.plan(torch.empty((0, 2), dtype=torch.int32, device="cuda"), 3)
    assert not empty.offsets.any() and empty.most_tiles == 0


def test_refusals():
    from eval_test_b200 import moe
    l = torch.zeros((4, 16), device="cuda")
    for k in (0, 17):
        with pytest.raises(ValueError, match="top_k"):
            moe.route(l, k)
    with pytest.raises(ValueError, match="experts"):
        moe.route(torch.zeros((2, 1025), device="cuda"), 2)
    with pytest.raises(ValueError, match="contiguous"):
        moe.route(l.t(), 2)
    with pytest.raises(ValueError, match="logits"):
        moe.route(l.double(), 2)
    with pytest.raises(ValueError, match="mask"):
        moe.route(l, 2, mask=torch.ones(5, dtype=torch.bool, device="cuda"))
    with pytest.raises(ValueError, match="mask"):
        moe.route(l, 2, mask=torch.ones(4, device="cuda"))
    ids = torch.zeros((4, 2), dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="num_experts"):
        moe.plan(ids, 0)
    with pytest.raises(ValueError, match="experts"):
        moe.plan(ids.long(), 4)
    with pytest.raises(ValueError, match="choices"):
        moe.plan(torch.zeros((4, 33), dtype=torch.int32, device="cuda"), 64)
    with pytest.raises(ValueError, match="weights"):
        moe.route_backward(torch.zeros((4, 2), device="cuda"), l, torch.zeros((4, 3), device="cuda"), ids)
