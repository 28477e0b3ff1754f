"""Tokens sorted by expert and back, their gradients and the quantising dispatch, against plain 64-bit forms."""
import math

import pytest
import torch

from _moe import EPS32, STEP, TINY, choices

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
# T, E, k, H; the last two: a warp per token, and four vectors of two rows at a time
SIZES = [(1, 1, 1, 8), (1, 64, 8, 4096), (5, 3, 2, 1), (40, 7, 3, 100), (33, 16, 4, 1001), (300, 8, 2, 64), (129, 40, 10, 1032),
         (2, 5, 5, 8200), (2500, 3, 2, 1304), (2400, 9, 3, 1040)]


def _normal(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def _gathered(rows, y):
    """float64 [T, k, H]: the row of each copy, zero where it has none."""
    return torch.where((rows >= 0)[..., None], y.double()[rows.clamp(min=0).long()], 0.0)


@pytest.mark.parametrize("T,E,k,H", SIZES)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("drop", [0.0, 0.4])
def test_dispatch_and_its_gradient(T, E, k, H, dtype, drop):
    from eval_test_b200 import moe
    plan = moe.plan(choices(T, E, k, drop, seed=H), E)
    x = _normal((T, H), dtype, 1)
    xs = moe.dispatch(x, plan)
    want = torch.where((plan.source >= 0)[:, None], x[plan.source.clamp(min=0).long() // k], 0)
    assert torch.equal(xs, want)
    d = _normal((T * k, H), dtype, 2)
    d[int(plan.offsets[-1]):] = math.nan                            # rows of no copy
    got = moe.dispatch_backward(d, plan)
    parts = _gathered(plan.rows, d)
    exact = parts.sum(1)
    assert got.dtype == dtype
    assert torch.all((got.double() - exact).abs() <= k * EPS32 * parts.abs().sum(1) + STEP[dtype] * exact.abs() * (1 + 2 ** -10) + TINY[dtype])


@pytest.mark.parametrize("T,E,k,H", SIZES)
@pytest.mark.parametrize("dtype,out", [(F32, F32), (F16, F16), (BF16, BF16), (F16, BF16), (F16, F32), (F32, F16), (BF16, F32)])
def test_combine_and_its_gradients(T, E, k, H, dtype, out):
    from eval_test_b200 import moe
    plan = moe.plan(choices(T, E, k, 0.2, seed=H + 1), E)
    y, w, dout = _normal((T * k, H), dtype, 3), _normal((T, k), F32, 4), _normal((T, H), out, 5)
    live = int(plan.offsets[-1])
    y[live:] = math.nan                                             # rows of no copy
    w[plan.rows < 0] = math.nan                                     # weights of choices that are not routed
    w64 = torch.where(plan.rows >= 0, w.double(), 0.0)
    parts = w64[..., None] * _gathered(plan.rows, y)
    exact = parts.sum(1)
    got = moe.combine(y, plan, w, dtype=out)
    assert got.dtype == out
    # k fused multiply-adds, one rounding to the output type (2^-10: of the rounded value, not of the exact one)
    assert torch.all((got.double() - exact).abs() <= k * EPS32 * parts.abs().sum(1) + STEP[out] * exact.abs() * (1 + 2 ** -10) + TINY[out])

    dy, dw = moe.combine_backward(dout, y, plan, w)
    assert dy.dtype == dtype and dy.shape == y.shape
    src = plan.source.clamp(min=0).long()
    exact_dy = torch.where((plan.source >= 0)[:, None], w64.reshape(-1)[src][:, None] * dout.double()[src // k], 0.0)
    assert torch.all((dy.double() - exact_dy).abs() <= (EPS32 + STEP[dtype] * (1 + 2 ** -10)) * exact_dy.abs() + TINY[dtype] + TINY[F32])
    assert not dy[live:].any()
    terms = dout.double()[:, None, :] * _gathered(plan.rows, y)
    # at most H / 32 products of a thread one after the other, then a tree of 5 and a sum of 8
    assert torch.all((dw.double() - terms.sum(2)).abs() <= (H / 32 + 16) * EPS32 * terms.abs().sum(2))
    assert not dw[plan.rows < 0].any()


def test_gradients_are_slopes():
    """combine is linear in y and in the weights, dispatch in x: the gradient's product with a direction is the change."""
    from eval_test_b200 import moe
    T, E, k, H = 30, 6, 3, 96
    plan = moe.plan(choices(T, E, k, 0.1, seed=5), E)
    y, w, d = _normal((T * k, H), F32, 1), _normal((T, k), F32, 2), _normal((T, H), F32, 3)
    vy, vw = _normal((T * k, H), F32, 4), _normal((T, k), F32, 5)
    dy, dw = moe.combine_backward(d, y, plan, w)
    for slope, there, size in ((dy.double() * vy.double(), moe.combine(vy, plan, w), vy), (dw.double() * vw.double(), moe.combine(y, plan, vw), y)):
        change = d.double() * there.double()
        # sums in 64 bits of values that each carry at most k + H / 32 + 16 half steps of fp32
        assert abs(float(slope.sum() - change.sum())) <= (k + H / 32 + 16) * EPS32 * k * float(
            slope.abs().sum() + change.abs().sum() + size.abs().double().sum())
    v = _normal((T, H), F32, 6)
    left = (moe.dispatch(v, plan).double() * y.double()).sum()
    right = (moe.dispatch_backward(y, plan).double() * v.double())
    assert abs(float(left - right.sum())) <= k * EPS32 * k * float((right.abs() + v.double().abs() * 6).sum())


def test_an_expert_twice_in_a_token():
    from eval_test_b200 import moe
    ids = torch.tensor([[1, 1, 0], [2, 1, 2]], dtype=torch.int32, device="cuda")
    plan = moe.plan(ids, 3)
    x = _normal((2, 16), F32, 1)
    xs = moe.dispatch(x, plan)
    assert torch.equal(moe.dispatch_backward(xs, plan), (x + x) + x)
    w = torch.tensor([[.5, .25, .25], [.25, .5, .25]], device="cuda")
    assert torch.equal(moe.combine(xs, plan, w), torch.addcmul(torch.addcmul(w[:, :1] * x, w[:, 1:2], x), w[:, 2:], x))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_rows_with_a_pitch_and_without_alignment(dtype):
    from eval_test_b200 import moe
    T, E, k, H = 37, 5, 2, 72
    plan = moe.plan(choices(T, E, k, 0.1, seed=1), E)
    w = _normal((T, k), F32, 2)
    wide, tall = _normal((T, 90), dtype, 3), _normal((T * k, 90), dtype, 4)
    for at in (0, 1, 2, 8):
        x, y = wide[:, at:at + H], tall[:, at:at + H]
        assert torch.equal(moe.dispatch(x, plan), moe.dispatch(x.contiguous(), plan))
        assert torch.equal(moe.combine(y, plan, w), moe.combine(y.contiguous(), plan, w))
        got, want = moe.combine_backward(x, y, plan, w), moe.combine_backward(x.contiguous(), y.contiguous(), plan, w)
        assert torch.equal(got[0], want[0])
        # another vector width sums a dot product in another order
        assert torch.all((got[1].double() - want[1].double()).abs() <= 2 * (H / 32 + 16) * EPS32 * 40 * H)
    one = wide[3:4, :H].expand(T, H)                                # one row for all tokens
    assert torch.equal(moe.dispatch(one, plan), moe.dispatch(one.contiguous(), plan))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_dispatch_nvfp4_of_rows_with_a_pitch(dtype):
    from eval_test_b200 import moe
    plan = moe.plan(choices(37, 5, 2, 0.1, seed=1), 5)
    wide = _normal((37, 320), dtype, 3)
    live = plan.slots.reshape(-1)[plan.slots.reshape(-1) >= 0].long()
    for x in (wide[:, 64:256], wide[3:4, :192].expand(37, 192)):
        (a, sfa), (b, sfb) = moe.dispatch_nvfp4(x, plan), moe.dispatch_nvfp4(x.contiguous(), plan)
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        s, t = (v.view(torch.uint8).permute(5, 2, 1, 0, 4, 3).reshape(plan.most_tiles * 128, -1)[live] for v in (sfa, sfb))
        assert torch.equal(s, t)


def test_the_same_call_gives_the_same_bits():
    from eval_test_b200 import moe
    T, E, k, H = 3000, 40, 6, 1000
    ids = choices(T, E, k, 0.1, seed=8)
    y, w, d = _normal((T * k, H), BF16, 1), _normal((T, k), F32, 2), _normal((T, H), BF16, 3)

    def once():
        plan = moe.plan(ids, E)
        return (plan.buffer[:3 * (E + 1) + 3 * T * k], moe.combine(y, plan, w), *moe.combine_backward(d, y, plan, w), moe.dispatch_backward(y, plan))

    first = once()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, once()))


def test_of_no_tokens_and_no_columns():
    from eval_test_b200 import moe
    plan = moe.plan(torch.empty((0, 2), dtype=torch.int32, device="cuda"), 3)
    x = torch.empty((0, 64), device="cuda")
    assert moe.dispatch(x, plan).shape == (0, 64) and moe.combine(x, plan).shape == (0, 64)
    a, sfa = moe.dispatch_nvfp4(x, plan)
    assert a.shape == (0, 32, 1) and sfa.numel() == 0
    plan = moe.plan(choices(4, 3, 2), 3)
    x = torch.empty((4, 0), device="cuda")
    assert moe.dispatch(x, plan).shape == (8, 0)
    dy, dw = moe.combine_backward(x, torch.empty((8, 0), device="cuda"), plan, torch.ones((4, 2), device="cuda"))
    assert dy.shape == (8, 0) and not dw.any()


@pytest.mark.parametrize("T,E,k,K", [(1, 1, 1, 64), (1, 64, 8, 4096), (40, 7, 3, 192), (300, 2, 2, 256), (33, 300, 4, 1024),
                                     (1030, 1000, 8, 2304), (9000, 3, 2, 1024), (17000, 9, 8, 320), (10300, 37, 8, 2048),
                                     (128, 40, 8, 163840)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("drop", [0.0, 0.4])
def test_dispatch_nvfp4_is_the_quantiser_of_the_sorted_rows(T, E, k, K, dtype, drop):
    from eval_test_b200 import formats as F, moe
    plan = moe.plan(choices(T, E, k, drop, seed=K), E)
    x = _normal((T, K), dtype, 7)
    x[0, :16] = 0                                                   # an all-zero block
    x[-1, 16:32] *= 1e4                                             # a scale that saturates
    x = torch.nan_to_num(x)                                         # (fp16: 65504 in the place of an infinity)
    a, sfa = moe.dispatch_nvfp4(x, plan)
    codes, scales = F.quantize_nvfp4(x.float())
    src = plan.source.clamp(min=0).long()
    live = (plan.source >= 0)[:, None]
    got = a.view(torch.uint8)[:, :, 0]
    assert a.shape == (T * k, K // 2, 1)
    assert torch.equal(got, torch.where(live, codes[src // k], 0))
    flat = F.unswizzle_scales(sfa.view(torch.uint8).permute(5, 2, 4, 0, 1, 3).reshape(-1), plan.most_tiles * 128, K, 1)[0]
    kept = plan.rows.reshape(-1) >= 0
    copies = torch.arange(T * k, device="cuda")[kept]
    assert torch.equal(flat[plan.slots.reshape(-1)[kept].long()], scales[copies // k])


def test_refusals():
    from eval_test_b200 import moe
    plan = moe.plan(choices(4, 3, 2), 3)
    x, y, w = _normal((4, 64), F32, 1), _normal((8, 64), F32, 2), _normal((4, 2), F32, 3)
    for f in (moe.dispatch, moe.dispatch_nvfp4):
        with pytest.raises(ValueError, match="shape"):
            f(y, plan)
        with pytest.raises(ValueError, match="contiguous"):
            f(_normal((64, 4), F32, 1).t(), plan)
        with pytest.raises(ValueError, match="matrix"):
            f(x.double(), plan)
    with pytest.raises(ValueError, match="multiple of 64"):
        moe.dispatch_nvfp4(_normal((4, 96), F32, 1), plan)
    with pytest.raises(RuntimeError, match="aligned"):
        moe.dispatch_nvfp4(_normal((4, 65), F32, 1)[:, 1:], plan)
    with pytest.raises(ValueError, match="shape"):
        moe.combine(x, plan, w)
    with pytest.raises(ValueError, match="weights"):
        moe.combine(y, plan, w.half())
    with pytest.raises(ValueError, match="weights"):
        moe.combine(y, plan, w[:, :1])
    with pytest.raises(ValueError, match="dtype"):
        moe.combine(y, plan, w, dtype=torch.float64)
    with pytest.raises(ValueError, match="shape"):
        moe.combine_backward(x, _normal((8, 32), F32, 2), plan, w)
