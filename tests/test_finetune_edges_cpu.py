"""Calls of the fine-tuning operators that fail or are refused, without a GPU."""
import os
import subprocess
import sys

import pytest

from test_finetune_cpu import BF16, F32, INVALID, UNSUPPORTED, A, matmul_policy, matmul_preference, policy, preference, tensors

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm.cpp_b200")
CUDA = 3

NO_DEVICE = """
import sys
sys.path.insert(0, {pkg!r})
import llmk
L, A = llmk.lib(), 1 << 20
tensors = (llmk.Tensor * 1)(llmk.Tensor(None, None, 0, 0, 0))
for f in (L.llmk_grad_norm, L.llmk_clip_grad_norm):
    assert f(A, tensors, 1, 1.0, A + 64, 1 << 30, None) == {cuda}
    print(L.llmk_last_error().decode(), L.llmk_launch_count())
"""

FAR = A + (1 << 24)


@pytest.mark.parametrize("norm,ws,clip_only", [
    (A, FAR, True), (A + 396, FAR, True), (A + 8192, FAR, True), (A + 8192 + 196, FAR, True),  # the norm in a tensor, in an output
    (FAR, A + 384, False), (FAR, A, False), (FAR, A + 4096, False),  # the workspace across one
    (FAR, A + 8192 + 128, True),  # across an output only
])
def test_norm_and_workspace_inside_a_tensor(llmk_lib, norm, ws, clip_only):
    L, t = llmk_lib, tensors((A, A, 100, F32, F32), (A + 4096, A + 8192, 100, BF16, BF16), (None, None, 0, F32, F32))
    assert L.llmk_clip_grad_norm(norm, t, 3, 1.0, ws, 1 << 20, None) == INVALID
    assert b"clip_grad_norm: norm or workspace overlaps" in L.llmk_last_error()
    if not clip_only:  # the norm alone writes no tensor, and its result last
        assert L.llmk_grad_norm(norm, t, 3, 1.0, ws, 1 << 20, None) == INVALID


def test_norm_inside_the_workspace(llmk_lib):
    L, t = llmk_lib, tensors((A, A, 20000, F32, F32))  # three units: three partial sums of 8 bytes
    for norm in (FAR, FAR + 12, FAR + 20):
        assert L.llmk_clip_grad_norm(norm, t, 1, 1.0, FAR, 1 << 20, None) == INVALID
        assert b"clip_grad_norm: norm overlaps the workspace" in L.llmk_last_error()


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
