"""A product that outlasts the limit of its epilogue's wait ends with a status, and the device goes on as before."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

CODE = """
import sys; sys.path.insert(0, 'tests')
import torch
from eval_test_b200 import _lib, moe, quantize
from test_moe_experts_gpu import _layer, _layer_weights, BF16
g = torch.Generator().manual_seed(1)
ops = _layer_weights(6, 256, 512)
x, logits = torch.randn((40, 512), generator=g).to(BF16).cuda(), torch.randn((40, 6), generator=g).cuda()
want = _layer(moe, x, logits, 2, ops)
torch.cuda.synchronize()
assert _lib.device_status(0) == 0
# one tile of 2^25 elements of K: each of its 131072 steps brings 21 KB to an SM, which takes in about 120 GB/s at most, so
# the product lasts more than 20 ms; the epilogue's limit of 4 runs out, while every other role waits for single steps
K = 1 << 25
plan = moe.plan(torch.zeros((1, 1), dtype=torch.int32, device='cuda'), 1)
a, sfa = moe.dispatch_nvfp4(torch.ones((1, K), dtype=BF16, device='cuda'), plan)
b = torch.zeros((128, K // 2, 1), dtype=torch.uint8, device='cuda').view(torch.float4_e2m1fn_x2)
sfb = torch.zeros((1, 1, K // 64, 512), dtype=torch.uint8, device='cuda').view(torch.float8_e4m3fn)
sfb = sfb.view(1, 1, K // 64, 32, 4, 4).permute(3, 4, 1, 5, 2, 0)
for product in (lambda: moe.expert_gemm(a, sfa, b, sfb, plan), lambda: moe.expert_dual_gemm(a, sfa, b, sfb, b, sfb, plan)):
    product()
    torch.cuda.synchronize()
    assert _lib.device_status(0) == 103, 'the epilogue gave up'
    for _ in range(3):
        assert torch.equal(_layer(moe, x, logits, 2, ops), want)
    torch.cuda.synchronize()
    assert _lib.device_status(0) == 0
"""


def test_a_wait_that_runs_out():
    done = subprocess.run([sys.executable, "-c", CODE], cwd=str(Path(__file__).resolve().parent.parent), capture_output=True, text=True,
                          timeout=300, env={**os.environ, "NVFP4_WAIT_BUDGET_MS": "4"})
    assert done.returncode == 0, done.stderr[-2000:]
