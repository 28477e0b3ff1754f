"""The experts' NVFP4 products of sorted tokens against 64-bit products of the same operands, and a whole layer."""
import pytest
import torch

from _moe import choices, dequant

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
# T, E, k, N, K, share of dropped choices: one row; short last boxes; several tiles of one expert; both tile widths, with
# more tiles than the machine takes at once
SIZES = [(1, 4, 2, 128, 256, 0.0), (5, 3, 1, 256, 512, 0.0), (40, 5, 3, 640, 768, 0.3), (300, 2, 2, 384, 256, 0.1),
         (129, 1, 1, 128, 512, 0.0), (700, 9, 1, 256, 1024, 0.0), (256, 64, 2, 1024, 512, 0.05), (2, 300, 2, 128, 256, 0.0),
         (1, 64, 8, 2048, 4096, 0.0), (1600, 4, 2, 1024, 512, 0.02), (3000, 8, 2, 2176, 512, 0.0),
         (40, 1024, 3, 128, 256, 0.1)]


def _operands(T, E, k, N, K, drop, weights=1, seed=0):
    from eval_test_b200 import formats as F, moe, quantize
    g = torch.Generator(device="cuda").manual_seed(seed + N + K)
    plan = moe.plan(choices(T, E, k, drop, seed=seed + T), E)
    x = torch.randn((T, K), generator=g, device="cuda").to(BF16)
    a, sfa = moe.dispatch_nvfp4(x, plan)
    codes, scales = F.quantize_nvfp4(x.float())
    src = plan.source.clamp(min=0).long() // k
    a64 = dequant(codes, scales.view(torch.float8_e4m3fn))[src]
    ops, w64 = [], []
    for _ in range(weights):
        b, sf, sf_p = quantize.quantize_operand(torch.randn((E, N, K), generator=g, device="cuda"))
        ops += [b, sf_p]
        w64.append(dequant(b.view(torch.uint8).permute(2, 0, 1), sf.permute(2, 0, 1)))
    return plan, a, sfa, ops, a64, w64


def _exact(plan, a64, w64):
    """(products, sums of absolute products) of every live row, 0 behind them."""
    out = torch.zeros((a64.shape[0], w64.shape[1]), dtype=torch.float64, device="cuda")
    size = torch.zeros_like(out)
    off = plan.offsets.tolist()
    for e in range(plan.num_experts):
        r = slice(off[e], off[e + 1])
        out[r] = a64[r] @ w64[e].T
        size[r] = a64[r].abs() @ w64[e].abs().T
    return out, size


def _alphas(E):
    return (torch.rand((E,), generator=torch.Generator().manual_seed(E)) * 0.05 + 0.01).cuda()


def _per_row(plan, alphas):
    e = torch.searchsorted(plan.offsets[1:].contiguous(), torch.arange(plan.source.numel(), device="cuda", dtype=torch.int32), right=True)
    return alphas.double()[e.clamp(max=plan.num_experts - 1)][:, None]


def _ok_status():
    from eval_test_b200 import _lib
    torch.cuda.synchronize()
    assert _lib.device_status(torch.cuda.current_device()) == 0


@pytest.mark.parametrize("T,E,k,N,K,drop", SIZES)
def test_expert_gemm(T, E, k, N, K, drop):
    from eval_test_b200 import moe
    plan, a, sfa, (b, sfb), a64, (w64,) = _operands(T, E, k, N, K, drop)
    exact, size = _exact(plan, a64, w64)
    al = _alphas(E)
    for alpha, by in ((0.125, 0.125), (al, _per_row(plan, al))):
        y = moe.expert_gemm(a, sfa, b, sfb, plan, alpha=alpha)
        _ok_status()
        assert y.shape == (T * k, N) and y.dtype == torch.float16
        # one fp32 rounding (of up to a step: the unit may cut) for each 64 elements of K, alpha's product, fp16
        room = (K / 64 + 4) * 2.0 ** -23 * size * by + 2.0 ** -11 * (exact * by).abs() * (1 + 2 ** -8) + 2.0 ** -25
        assert torch.all((y.double() - exact * by).abs() <= room)
        assert not y[int(plan.offsets[-1]):].any()


@pytest.mark.parametrize("T,E,k,N,K,drop", SIZES)
def test_expert_dual_gemm_and_its_nvfp4_form(T, E, k, N, K, drop):
    from eval_test_b200 import formats as F, moe
    plan, a, sfa, ops, a64, (w1, w2) = _operands(T, E, k, N, K, drop, weights=2)
    al = _alphas(E)
    by = _per_row(plan, al)
    (x, sx), (y, sy) = _exact(plan, a64, w1), _exact(plan, a64, w2)
    x, y, sx, sy = x * by, y * by, sx * by, sy * by
    c = moe.expert_dual_gemm(a, sfa, *ops, plan, alpha=al)
    _ok_status()
    silu = x * torch.sigmoid(x)
    exact = silu * y
    # the products' own errors through silu (slope at most 1.1) and through the product; the fast exponential's steps
    # grow with its argument (2 + 1.16 |x|), its division has 2, then the product and fp16
    ex, ey = ((K / 64 + 4) * 2.0 ** -23 * s for s in (sx, sy))
    room = 1.1 * ex * (y.abs() + ey) + silu.abs() * ey + exact.abs() * ((8 + 1.2 * x.abs()) * 2.0 ** -23 + 2.0 ** -11 * (1 + 2 ** -8)) + 2.0 ** -25
    assert torch.all((c.double() - exact).abs() <= room)
    live = int(plan.offsets[-1])
    assert not c[live:].any()

    h, sfh = moe.expert_dual_gemm_nvfp4(a, sfa, *ops, plan, alpha=al)
    _ok_status()
    codes, scales = F.quantize_nvfp4(c.float())
    got = h.view(torch.uint8)[:, :, 0]
    assert torch.equal(got[:live], codes[:live]) and not got[live:].any()
    flat = F.unswizzle_scales(sfh.view(torch.uint8).permute(5, 2, 4, 0, 1, 3).reshape(-1), plan.most_tiles * 128, N, 1)[0]
    copies = plan.source[:live].long()
    assert torch.equal(flat[plan.slots.reshape(-1)[copies].long()], scales[:live])


@pytest.mark.parametrize("N", [128, 512])
def test_nothing_routed_and_everything_to_one_expert(N):
    from eval_test_b200 import moe
    plan, a, sfa, (b, sfb), a64, (w64,) = _operands(70, 6, 2, N, 256, 0.0)
    ids = torch.full((70, 2), -1, dtype=torch.int32, device="cuda")
    none = moe.plan(ids, 6)
    assert not moe.expert_gemm(a, sfa, b, sfb, none).any()
    x = torch.randn((70, 256), generator=torch.Generator().manual_seed(1)).cuda()
    one = moe.plan(torch.full_like(ids, 5), 6)
    a, sfa = moe.dispatch_nvfp4(x, one)
    y = moe.expert_gemm(a, sfa, b, sfb, one)
    _ok_status()
    assert torch.equal(y[0::2], y[1::2])                            # both copies of a token
    empty = moe.plan(torch.empty((0, 2), dtype=torch.int32, device="cuda"), 6)
    a, sfa = moe.dispatch_nvfp4(x[:0], empty)
    assert moe.expert_gemm(a, sfa, b, sfb, empty).shape == (0, N)


def test_a_row_does_not_depend_on_its_neighbours():
    """The same token alone and among others: a tile may hold rows of other experts and what was left in memory."""
    from eval_test_b200 import moe
    T, E, k, N, K = 64, 8, 2, 256, 512
    plan, a, sfa, (b, sfb), _, _ = _operands(T, E, k, N, K, 0.0, seed=3)
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn((T, K), generator=g, device="cuda").to(BF16)
    ids = choices(T, E, k, seed=4)
    whole = moe.plan(ids, E)
    y = moe.expert_gemm(*moe.dispatch_nvfp4(x, whole), b, sfb, whole)
    for t in (0, 31, 63):
        alone = moe.plan(ids[t:t + 1].contiguous(), E)
        z = moe.expert_gemm(*moe.dispatch_nvfp4(x[t:t + 1], alone), b, sfb, alone)
        assert torch.equal(z[alone.rows[0].long()], y[whole.rows[t].long()])
    _ok_status()


def _layer(moe, x, logits, k, ops, mask=None):
    r = moe.route(logits, k, mask=mask)
    a, sfa = moe.dispatch_nvfp4(x, r.plan)
    h, sfh = moe.expert_dual_gemm_nvfp4(a, sfa, *ops[:4], r.plan, alpha=0.02)
    return moe.combine(moe.expert_gemm(h, sfh, *ops[4:], r.plan, alpha=0.05), r.plan, r.weights, dtype=x.dtype)


def _layer_weights(E, N, K):
    from eval_test_b200 import quantize
    g = torch.Generator(device="cuda").manual_seed(2)
    ops = []
    for shape in ((E, N, K), (E, N, K), (E, K, N)):
        b, _, sf_p = quantize.quantize_operand(torch.randn(shape, generator=g, device="cuda"), ref_scales=False)
        ops += [b, sf_p]
    return ops


def test_layer_against_the_entries_with_host_sizes():
    """The whole layer gives, bit for bit, what the dual GEMM and the GEMM give expert by expert on gathered tokens."""
    from eval_test_b200 import moe, nvfp4_dual_gemm, nvfp4_gemm, quantize
    T, E, k, N, K = 90, 5, 2, 256, 512
    ops = _layer_weights(E, N, K)
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((T, K), generator=g, device="cuda").to(BF16)
    logits = torch.randn((T, E), generator=g, device="cuda")
    out = _layer(moe, x, logits, k, ops)
    _ok_status()
    r = moe.route(logits, k)
    y = torch.zeros((T * k, K), dtype=torch.float16, device="cuda")
    off = r.plan.offsets.tolist()
    one = lambda t, e: t[..., e:e + 1]  # noqa: E731
    for e in range(E):
        tokens = r.plan.source[off[e]:off[e + 1]].long() // k
        m = tokens.numel()
        a, sfa, sfa_p = quantize.quantize_operand(x[tokens][None].contiguous())
        c = torch.empty((1, m, N), dtype=torch.float16, device="cuda").permute(1, 2, 0)
        h, _, h_p = nvfp4_dual_gemm.custom_kernel_nvfp4(
            (a, one(ops[0], e), one(ops[2], e), None, None, None, sfa_p, one(ops[1], e), one(ops[3], e), c), alpha=0.02)
        c = torch.empty((1, m, K), dtype=torch.float16, device="cuda").permute(1, 2, 0)
        nvfp4_gemm.custom_kernel((h, one(ops[4], e), None, None, h_p, one(ops[5], e), c), alpha=0.05)
        y[off[e]:off[e + 1]] = c[:, :, 0]
    assert torch.equal(moe.combine(y, r.plan, r.weights, dtype=BF16), out)


def test_layer_in_a_graph_follows_its_inputs():
    """Captured once and replayed on other tokens, whose experts and group sizes are others; two graphs in turn."""
    from eval_test_b200 import moe
    E, N, K, k = 12, 256, 512, 3
    ops = _layer_weights(E, N, K)
    g = torch.Generator(device="cuda").manual_seed(5)
    made = []
    for T in (1, 150, 6000):                                        # the last: a sort of several launches
        x, logits = torch.zeros((T, K), device="cuda", dtype=BF16), torch.zeros((T, E), device="cuda")
        mask = torch.ones((T,), dtype=torch.bool, device="cuda")
        _layer(moe, x, logits, k, ops, mask)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _layer(moe, x, logits, k, ops, mask)
        made.append((T, x, logits, mask, graph, out))
    for _ in range(3):
        for T, x, logits, mask, graph, out in made:
            x.copy_(torch.randn((T, K), generator=g, device="cuda"))
            logits.copy_(torch.randn((T, E), generator=g, device="cuda") * 3)
            mask.copy_(torch.rand((T,), generator=g, device="cuda") < 0.8)
        for m in made:
            m[4].replay()
        for T, x, logits, mask, graph, out in made:
            assert torch.equal(out, _layer(moe, x, logits, k, ops, mask))
    _ok_status()


def test_first_calls_of_a_process_can_be_captured():
    """Nothing has to have run before: what the first calls set up (the status word, kernel attributes) is no part of
    the graph and does not break the capture."""
    import subprocess
    import sys
    from pathlib import Path
    code = """
import sys; sys.path.insert(0, 'tests')
import torch
from test_moe_experts_gpu import _layer, _layer_weights, BF16
from eval_test_b200 import moe, _lib
ops = _layer_weights(6, 256, 512)
x, logits = torch.randn((40, 512), device='cuda').to(BF16), torch.randn((40, 6), device='cuda')
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = _layer(moe, x, logits, 2, ops)
graph.replay()
torch.cuda.synchronize()
assert torch.equal(out, _layer(moe, x, logits, 2, ops)) and out.any()
torch.cuda.synchronize()
assert _lib.device_status(0) == 0
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=str(Path(__file__).resolve().parent.parent), capture_output=True, text=True,
                          timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_outputs_behind_two_to_the_31_elements():
    """Rows whose offsets pass 32 bits, in elements and in bytes."""
    from eval_test_b200 import moe, quantize
    T, E, k, N, K = 34000, 4, 8, 8192, 256                          # 272000 rows of 8192: 2.2e9 outputs
    g = torch.Generator(device="cuda").manual_seed(4)
    ids = torch.randint(0, E, (T, k), generator=g, device="cuda", dtype=torch.int32)
    plan = moe.plan(ids, E)
    x = torch.randn((T, K), generator=g, device="cuda").to(BF16)
    b, sf, sf_p = quantize.quantize_operand(torch.randn((E, N, K), generator=g, device="cuda"))
    a, sfa = moe.dispatch_nvfp4(x, plan)
    y = moe.expert_gemm(a, sfa, b, sf_p, plan)
    _ok_status()
    from eval_test_b200 import formats as F
    codes, scales = F.quantize_nvfp4(x.float())
    a64 = dequant(codes, scales.view(torch.float8_e4m3fn))
    w64 = dequant(b.view(torch.uint8).permute(2, 0, 1), sf.permute(2, 0, 1))
    rows = torch.tensor([0, 131071, 262143, 262144, 262145, T * k - 1], device="cuda")
    copies = plan.source[rows].long()
    e = ids.reshape(-1)[copies].long()
    exact = torch.einsum("rk,rnk->rn", a64[copies // k], w64[e])
    size = torch.einsum("rk,rnk->rn", a64[copies // k].abs(), w64[e].abs())
    room = (K / 64 + 4) * 2.0 ** -23 * size + 2.0 ** -11 * exact.abs() * (1 + 2 ** -8) + 2.0 ** -25
    assert torch.all((y[rows].double() - exact).abs() <= room)
    # the same buffer back, and out again
    w = torch.rand((T, k), generator=g, device="cuda")
    out = moe.combine(y, plan, w, dtype=BF16)
    t = torch.tensor([0, 16000, T - 1], device="cuda")
    parts = w[t].double()[..., None] * y[plan.rows[t].long()].double()
    assert torch.all((out[t].double() - parts.sum(1)).abs() <= k * 2.0 ** -24 * parts.abs().sum(1) + 2.0 ** -8 * parts.sum(1).abs() * (1 + 2 ** -10))
    dy, dw = moe.combine_backward(out, y, plan, w)
    want = (w.reshape(-1)[copies][:, None] * out[copies // k].float()).half()
    assert torch.equal(dy[rows], want)
    xs = moe.dispatch(out, plan)
    assert torch.equal(xs[rows], out[copies // k])


def test_layer_on_two_streams_at_once():
    from eval_test_b200 import moe
    E, N, K, k = 12, 256, 512, 3
    ops = _layer_weights(E, N, K)
    g = torch.Generator(device="cuda").manual_seed(6)
    data = [(torch.randn((T, K), generator=g, device="cuda").to(BF16), torch.randn((T, E), generator=g, device="cuda")) for T in (200, 64)]
    want = [_layer(moe, x, l, k, ops) for x, l in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(_layer(moe, *data[i], k, ops))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(x, want[i]) for x in got[i])
    _ok_status()


def test_an_event_between_two_calls_is_waited_for():
    """The kernels may start before the one in front of them has ended, but not before an event of another stream."""
    from eval_test_b200 import moe
    T, E, k, H = 500, 8, 2, 512
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.zeros((T, H), device="cuda")
    new = torch.randn((T, H), generator=g, device="cuda")
    ids = choices(T, E, k, seed=1)
    plan = moe.plan(ids, E)
    want = moe.dispatch(new, plan)
    moe.dispatch_nvfp4(x, plan)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        x.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(a):
            torch.cuda._sleep(2_000_000)                            # a millisecond, then the copy
            x.copy_(new)
            ready = a.record_event()
        with torch.cuda.stream(b):
            plan = moe.plan(ids, E)
            b.wait_event(ready)
            xs = moe.dispatch(x, plan)
            back = moe.combine(xs, plan)
        torch.cuda.synchronize()
        assert torch.equal(xs, want) and torch.equal(back, new + new)


def test_refusals():
    from eval_test_b200 import moe
    plan, a, sfa, (b, sfb), _, _ = _operands(6, 4, 2, 256, 512, 0.0)
    for bad in (lambda: moe.expert_gemm(a[:5], sfa, b, sfb, plan), lambda: moe.expert_gemm(a, sfa, b[..., :3], sfb, plan),
                lambda: moe.expert_gemm(a, sfa, b, sfb[..., :3], plan), lambda: moe.expert_gemm(a, sfb, b, sfb, plan),
                lambda: moe.expert_gemm(a, sfa, b[:100], sfb, plan), lambda: moe.expert_gemm(a[:, :64], sfa, b, sfb, plan),
                lambda: moe.expert_gemm(a, sfa, b, sfb, plan, alpha=torch.ones(3, device="cuda")),
                lambda: moe.expert_gemm(a, sfa, b, sfb, plan, alpha=torch.ones(4)),
                lambda: moe.expert_dual_gemm(a, sfa, b, sfb, b[:128], sfb, plan)):
        with pytest.raises(ValueError):
            bad()
