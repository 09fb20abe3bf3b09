"""What the fine-tuning losses on the lm_head make of logits far from zero."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EX2 = 1.44e-7  # the most that ex2.approx is off by, relative


@pytest.mark.parametrize("mathname,where", [("bf16", 5), ("bf16", 37), ("tf32", 37)])
def test_far_logits_keep_their_sums(cuda_dev, mathname, where):
    """One live token in each of 16 slots of 64 columns, all of one value in a row, all others 10^4 below: lp = -log 16 in
    every row, whatever the value. Each slot's term is 1 but for ex2.approx at an argument next to 0; its correction rounds
    three times, 32 sums of at most one slot each are added in 64 bits, and lp is rounded once. The value's product by
    log2 e, which the terms are formed with, is rounded by up to 5e-6 here and may not show."""
    import llmk
    rows, C, V, live = 4096, 64, 1024, 16
    dt, mode = (torch.bfloat16, llmk.MATH_BF16) if mathname == "bf16" else (torch.float32, llmk.MATH_TF32)
    a = (torch.linspace(-100, 100, rows, device=cuda_dev)).bfloat16()
    inp, W = torch.zeros(rows, C, dtype=dt, device=cuda_dev), torch.zeros(V, C, dtype=dt, device=cuda_dev)
    cols = torch.arange(live, device=cuda_dev) * 64 + where
    inp[:, 0], W[cols, 0] = a.to(dt), 1.0
    bias = torch.full((V,), -1e4, device=cuda_dev)
    bias[cols] = 0.0
    t = cols[torch.arange(rows, device=cuda_dev) % live].int()
    logits = torch.empty(rows, V, dtype=dt, device=cuda_dev)
    A, losses, logps = torch.ones(rows, device=cuda_dev), torch.empty(rows, device=cuda_dev), torch.empty(rows, device=cuda_dev)
    ws = torch.empty(llmk.lib().llmk_matmul_finetune_workspace(rows, V), dtype=torch.uint8, device=cuda_dev)
    P = llmk.ptr
    llmk.call("llmk_matmul_policy_forward", P(losses), None, P(logps), P(logits), llmk.dtype_code(logits), P(inp), P(W), P(bias),
              P(t), None, P(A), None, None, rows, C, V, V, 0.2, 0.2, 0.0, 1.0, 0, mode, P(ws), ws.numel(), llmk.stream_ptr())
    assert torch.equal(logits[:, cols], a.to(dt)[:, None].expand(rows, live))
    want = -math.log(live)
    assert (logps.double() - want).abs().max().item() <= EX2 + 4 * U + U * abs(want)
