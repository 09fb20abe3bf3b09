"""Calls of the fine-tuning operators that fail or are refused, without a GPU."""
import os
import subprocess
import sys

from test_finetune_cpu import UNSUPPORTED, matmul_policy, matmul_preference, policy, preference

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm.cpp_b200")
CUDA = 3

NO_DEVICE = """
import sys
sys.path.insert(0, {pkg!r})
import llmk
L, A = llmk.lib(), 1 << 20
tensors = (llmk.Tensor * 1)(llmk.Tensor(None, None, 0, 0, 0))
for f in (L.llmk_grad_norm, L.llmk_clip_grad_norm):
    assert f(A, tensors, 1, 1.0, A, 1 << 30, None) == {cuda}
    print(L.llmk_last_error().decode(), L.llmk_launch_count())
"""


def test_a_refused_launch_ends_the_norm(llmk_lib):
    """Where the kernel of the squares cannot be launched (here: no device), nothing is launched behind it, and the error
    names it: its partial sums are not there to scale by."""
    out = subprocess.run([sys.executable, "-c", NO_DEVICE.format(pkg=PKG, cuda=CUDA)], capture_output=True, text=True,
                         env={**os.environ, "CUDA_VISIBLE_DEVICES": ""}, timeout=300)
    assert out.returncode == 0, out.stderr
    lines = out.stdout.splitlines()
    assert len(lines) == 2
    for line in lines:
        assert line.startswith("grad_squares_kernel: ") and line.endswith(" 0"), line


def test_more_rows_than_the_losses_take(llmk_lib):
    """Up to 2^30 rows, in every form."""
    L, most = llmk_lib, 1 << 30
    for f, args in ((L.llmk_policy_loss, policy(rows=most + 1)), (L.llmk_matmul_policy_forward, matmul_policy(BT=most + 1)),
                    (L.llmk_preference_loss, preference(pairs=1, T=most // 2 + 1)),
                    (L.llmk_matmul_preference_forward, matmul_preference(pairs=1, T=most // 2 + 1))):
        assert f(*args) == UNSUPPORTED
        assert b"more than 2^30 rows" in L.llmk_last_error()
