"""The router's results inside a user's autograd function."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_weights_scaled_in_place_leave_the_choices_and_the_plan_as_they_were():
    """The results share memory of one allocation, but not the counter by which autograd sees changes."""
    from eval_test_b200 import moe

    class Route(torch.autograd.Function):
        @staticmethod
        def forward(ctx, logits):
            r = moe.route(logits, 2)
            ctx.save_for_backward(logits, r.weights.clone(), r.experts, r.plan.rows)
            ctx.mark_non_differentiable(r.experts)
            return r.weights, r.experts

        @staticmethod
        def backward(ctx, dw, _):
            logits, weights, experts, rows = ctx.saved_tensors
            assert int(rows.min()) == 0
            return moe.route_backward(dw.contiguous(), logits, weights, experts)

    logits = torch.randn((7, 9), generator=torch.Generator().manual_seed(1)).cuda().requires_grad_()
    weights, experts = Route.apply(logits)
    weights *= 2.5                                                  # a scaling factor of the routed part
    dw = torch.randn((7, 2), generator=torch.Generator().manual_seed(2)).cuda()
    weights.backward(dw)
    r = moe.route(logits.detach(), 2)
    assert torch.equal(experts, r.experts) and torch.equal(weights.detach(), r.weights * 2.5)
    assert torch.equal(logits.grad, moe.route_backward(dw * 2.5, logits.detach(), r.weights, r.experts))


def test_versions_are_apart():
    from eval_test_b200 import moe
    r = moe.route(torch.randn((5, 8), device="cuda"), 3)
    before = r.experts._version, r.plan.rows._version, r.plan.buffer._version
    r.weights.mul_(2.0)
    assert (r.experts._version, r.plan.rows._version, r.plan.buffer._version) == before
    r.experts.fill_(-1)
    assert r.plan.rows._version == before[1] and r.weights._version == 1
