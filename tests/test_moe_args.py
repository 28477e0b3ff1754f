"""What the mixture-of-experts entry points refuse, before any CUDA call is made (no GPU needed)."""
import pytest
import torch


def test_c_entries_reject_bad_arguments(lib):
    P = 32                                                # stands for an aligned pointer; nothing is read
    plan = (P,) * 7                                       # six tables and the scratch
    assert lib.nvfp4_moe_plan(None, 4, 4, 2, *plan, None) == -1
    assert lib.nvfp4_moe_plan(P, 0, 4, 2, *plan, None) == -2
    assert lib.nvfp4_moe_plan(P, 4, 0, 2, *plan, None) == -2
    assert lib.nvfp4_moe_plan(P, 4, 1025, 2, *plan, None) == -6
    assert lib.nvfp4_moe_plan(P, 4, 64, 33, *plan, None) == -6
    assert lib.nvfp4_moe_plan(P, 1 << 30, 4, 2, *plan, None) == -6       # copies are counted in 32 bits
    assert lib.nvfp4_moe_plan_scratch(2048, 64, 8) == 0 and lib.nvfp4_moe_plan_scratch(2049, 64, 8) > 0
    assert lib.nvfp4_moe_plan(P, 2049, 64, 8, *plan[:6], None, None) == -1
    route = lambda kind=0, ld=8, T=4, E=8, k=2, logits=P: lib.nvfp4_moe_route(  # noqa: E731
        logits, kind, ld, None, T, E, k, 1, P, P, *plan, None)
    assert route(logits=None) == -1
    assert route(kind=3) == -6
    assert route(T=0) == -2 and route(E=0) == -2 and route(k=0) == -2 and route(k=9) == -2 and route(ld=-1) == -2
    assert route(E=1025) == -6 and route(E=64, k=33) == -6
    back = lambda kind=0, k=2, dw=P, out=P: lib.nvfp4_moe_route_backward(dw, P, kind, 8, P, P, 4, 8, k, 1, out, None)  # noqa: E731
    assert back(dw=None) == -1 and back(out=8) == -5 and back(kind=-1) == -6 and back(k=9) == -2
    disp = lambda x=P, kind=0, T=4, H=8, xs=P, ld=8: lib.nvfp4_moe_dispatch(x, kind, ld, P, P, T, 8, 2, H, xs, None)  # noqa: E731
    assert disp(x=None) == -1 and disp(kind=9) == -6 and disp(T=0) == -2 and disp(H=0) == -2 and disp(T=1 << 30) == -6
    comb = lambda y=P, kind=0, ok=0, k=2: lib.nvfp4_moe_combine(y, kind, 8, None, P, 4, k, 8, P, ok, None)  # noqa: E731
    assert comb(y=None) == -1 and comb(kind=5) == -6 and comb(ok=5) == -6 and comb(k=0) == -2
    cb = lambda d=P, kind=0, w=P: lib.nvfp4_moe_combine_backward(d, 0, 8, P, kind, 8, w, P, P, 4, 8, 2, 8, P, P, None)  # noqa: E731
    assert cb(d=None) == -1 and cb(w=None) == -1 and cb(kind=7) == -6
    dq = lambda x=P, K=64, ld=64, kind=2, codes=P, T=4, scratch=None: lib.nvfp4_moe_dispatch_nvfp4(  # noqa: E731
        x, kind, ld, P, P, P, P, P, T, 8, 2, K, codes, P, scratch, None)
    assert dq(x=None) == -1 and dq(K=96, ld=96) == -3 and dq(x=8) == -5 and dq(ld=65) == -5 and dq(codes=8) == -5
    assert dq(kind=3) == -6
    assert lib.nvfp4_moe_dispatch_scratch(1 << 18, 2, 256) == 0 and lib.nvfp4_moe_dispatch_scratch(1 << 20, 2, 256) == 1 << 24
    assert lib.nvfp4_moe_dispatch_scratch(1 << 20, 2, 320) == 0
    assert dq(T=1 << 20, K=256, ld=256) == -1 and dq(T=1 << 20, K=256, ld=256, scratch=8) == -5
    gemm = lambda a=P, N=128, K=256, R=8, E=4, c=P, off=P, al=None, wide=P: lib.nvfp4_moe_gemm(  # noqa: E731
        a, P, P, P, off, P, wide, al, c, R, E, N, K, 1.0, None)
    assert gemm(a=None) == -1 and gemm(off=None) == -1 and gemm(wide=None) == -1
    assert gemm(N=64) == -4 and gemm(K=128) == -3 and gemm(R=0) == -2 and gemm(E=0) == -2
    assert gemm(a=8) == -5 and gemm(c=16) == -5 and gemm(al=2) == -5
    assert lib.nvfp4_moe_dual_gemm(P, P, P, P, None, P, P, P, P, None, P, 8, 4, 128, 256, 1.0, None) == -1
    assert lib.nvfp4_moe_dual_gemm_nvfp4(P, P, P, P, P, P, P, P, P, None, P, None, 8, 4, 128, 256, 1.0, None) == -1


def test_sizes_that_an_index_and_a_loop_s_stride_could_carry_past_31_bits_are_refused(lib):
    from eval_test_b200 import moe
    P, plan, most = 32, (32,) * 7, (1 << 31) - (1 << 20)
    assert moe.MAX_COPIES == most
    for T, E, k in ((most + 1, 1, 1), ((1 << 31) - 129, 1, 1), (most // 2 + 1, 8, 2)):
        assert lib.nvfp4_moe_plan(P, T, E, k, *plan, None) == -6
        assert lib.nvfp4_moe_route(P, 2, 8, None, T, E, k, 1, P, P, *plan, None) == -6
        assert lib.nvfp4_moe_route_backward(P, P, 2, 8, P, P, T, E, k, 1, P, None) == -6
        assert lib.nvfp4_moe_dispatch(P, 2, 8, P, P, T, E, k, 8, P, None) == -6
        assert lib.nvfp4_moe_combine(P, 2, 8, None, P, T, k, 8, P, 2, None) == -6
    H = most + 1
    assert lib.nvfp4_moe_dispatch(P, 2, H, P, P, 1, 8, 1, H, P, None) == -6
    assert lib.nvfp4_moe_combine(P, 2, H, None, P, 1, 1, H, P, 2, None) == -6
    assert lib.nvfp4_moe_combine_backward(P, 2, H, P, 2, H, P, P, P, 1, 8, 1, H, P, P, None) == -6
    with pytest.raises(ValueError, match="choices"):          # (past 32 bits the entry would see the low word)
        moe.Plan(1 << 32, 1, 8, torch.device("cpu"))


def test_python_entries_take_cuda_tensors_of_the_documented_types():
    from eval_test_b200 import moe
    x = torch.zeros((4, 64))
    with pytest.raises(ValueError, match="CUDA"):
        moe.route(x, 2)
    with pytest.raises(ValueError, match="CUDA"):
        moe.plan(torch.zeros((4, 2), dtype=torch.int32), 8)
    p = moe.Plan(4, 2, 8, torch.device("cpu"))
    for f in (moe.dispatch, moe.dispatch_nvfp4, moe.combine, moe.dispatch_backward):
        with pytest.raises(ValueError, match="CUDA"):
            f(x, p)
    with pytest.raises(ValueError, match="CUDA"):
        moe.combine_backward(x, x, p, torch.zeros((4, 2)))
    with pytest.raises(ValueError, match="CUDA"):
        moe.expert_gemm(torch.zeros((8, 128, 1), dtype=torch.uint8), None, torch.zeros((128, 128, 8)), None, p)


def test_most_tiles_bounds_every_distribution():
    """The buffers of the scales are sized by it: no way to spread the copies over the experts fills more tiles, and
    one way fills as many."""
    from itertools import product
    from eval_test_b200 import moe

    def tiles(counts):
        return sum((c + 127) // 128 for c in counts)

    for copies, E in ((0, 3), (1, 3), (2, 3), (130, 1), (256, 2), (257, 2), (400, 3), (513, 3)):
        p = moe.Plan(copies, 1, E, torch.device("cpu"))
        reached = max(tiles((*c, copies - sum(c))) for c in product(range(copies + 1), repeat=E - 1) if sum(c) <= copies)
        assert p.most_tiles == reached, (copies, E)


def test_a_plan_is_not_copied():
    import copy
    import pickle
    from eval_test_b200 import moe
    p = moe.Plan(4, 2, 8, torch.device("cpu"))
    for f in (copy.copy, copy.deepcopy, pickle.dumps):
        with pytest.raises(TypeError, match="Plan"):
            f(p)
