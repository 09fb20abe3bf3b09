"""Calls of the fine-tuning operators that fail or are refused, without a GPU."""
import os
import subprocess
import sys

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
