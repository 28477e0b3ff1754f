"""combine and its gradient on rows that lie 2^32 bytes and more apart, and on rows as long as that."""
import pytest
import torch

from _moe import EPS32, choices

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


# vectors of 16 bytes, pairs of 16-bit elements, single elements
@pytest.mark.parametrize("dtype,pitch", [(F32, (1 << 30) + 4), (F32, (1 << 30) + 1), (BF16, (1 << 31) + 8), (F16, (1 << 31) + 2), (BF16, (1 << 31) + 1)])
def test_rows_far_apart(dtype, pitch):
    from eval_test_b200 import moe
    T, E, k, H = 2, 3, 2, 72
    plan = moe.plan(choices(T, E, k, seed=1), E)
    g = torch.Generator().manual_seed(2)
    near = torch.randn((T * k, H), generator=g).to(dtype).cuda()
    far = torch.empty((T * k - 1) * pitch + H, dtype=dtype, device="cuda").as_strided((T * k, H), (pitch, 1))
    far.copy_(near)
    w, d = torch.randn((T, k), generator=g).cuda(), torch.randn((T, H), generator=g).to(dtype).cuda()
    assert torch.equal(moe.combine(far, plan, w), moe.combine(near, plan, w))
    assert torch.equal(moe.dispatch_backward(far, plan), moe.dispatch_backward(near, plan))
    got, want = moe.combine_backward(d, far, plan, w), moe.combine_backward(d, near, plan, w)
    assert torch.equal(got[0], want[0])
    # another vector width sums a dot product in another order: at most H products one after the other on either side
    size = (d.double()[:, None, :] * near.double()[plan.rows.long()]).abs().sum(2)
    assert torch.all((got[1].double() - want[1].double()).abs() <= 2 * H * EPS32 * size)


def test_gradient_of_a_row_of_more_than_32_bits_of_bytes():
    from eval_test_b200 import moe
    H = (1 << 30) + 8
    plan = moe.plan(torch.zeros((1, 1), dtype=torch.int32, device="cuda"), 1)
    y, d = torch.ones((1, H), device="cuda"), torch.zeros((1, H), device="cuda")
    d[0, 0], d[0, 1 << 29], d[0, -1] = 1, 2, 4
    dy, dw = moe.combine_backward(d, y, plan, torch.full((1, 1), 0.5, device="cuda"))
    assert float(dw) == 7.0                                         # (sums of small whole numbers are exact)
    assert torch.equal(dy, d.mul_(0.5))
    assert torch.equal(moe.combine(y, plan, torch.full((1, 1), 0.5, device="cuda")), y.mul_(0.5))


# more choices than the two rows that are taken at a time, and the longest pitch that 32 bits hold
@pytest.mark.parametrize("dtype,pitch,k", [(F32, (1 << 30) + 4, 5), (F16, (1 << 31) + 1, 5), (F32, (1 << 30) - 4, 3), (BF16, (1 << 31) - 1, 3)])
def test_choices_of_one_token_far_apart(dtype, pitch, k):
    from eval_test_b200 import moe
    H = 600
    plan = moe.plan(choices(1, 7, k, 0.3, seed=3), 7)
    g = torch.Generator().manual_seed(4)
    near = torch.randn((k, H), generator=g).to(dtype).cuda()
    far = torch.empty((k - 1) * pitch + H, dtype=dtype, device="cuda").as_strided((k, H), (pitch, 1))
    far.copy_(near)
    w, d = torch.randn((1, k), generator=g).cuda(), torch.randn((1, H), generator=g).cuda()
    assert torch.equal(moe.combine(far, plan, w, dtype=F32), moe.combine(near, plan, w, dtype=F32))
    got, want = moe.combine_backward(d, far, plan, w), moe.combine_backward(d, near, plan, w)
    assert torch.equal(got[0], want[0])
    rows = plan.rows.long()
    size = torch.where(rows >= 0, (d.double()[:, None, :] * near.double()[rows.clamp(min=0)]).abs().sum(2), 0.0)
    assert torch.all((got[1].double() - want[1].double()).abs() <= 2 * H * EPS32 * size)
