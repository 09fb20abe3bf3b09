"""A clipped fine-tuning step that the caller captures into a CUDA graph of its own."""
import numpy as np
import pytest
import torch

import oracle as O
from test_finetune_model_gpu import B, CFG, T

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["policy", "preference"])
def test_a_clipped_step_captured_by_the_caller(cuda_dev, which):
    """Replays do what the eager calls do, with the hyperparameters of the captured call: they are the graph's own, and not
    what a later call left where this one kept them."""
    import llmk
    cfg = O.config(**CFG)
    params, toks = O.init_params(cfg, 5), torch.from_numpy(O.tokens(B * T + 1, CFG["vocab_size"], 6)).to(cuda_dev)
    inp, tgt = toks[:-1].contiguous(), toks[1:].contiguous()
    w = (torch.rand(B * T, device=cuda_dev) < 0.6).float()
    A = torch.randn(B * T, device=cuda_dev)
    torch.cuda.synchronize()

    def step(m, lr):
        if which == "policy":
            m.forward_policy(inp.data_ptr(), tgt.data_ptr(), A.data_ptr(), weights=w.data_ptr())
        else:
            m.forward_preference(inp.data_ptr(), tgt.data_ptr(), weights=w.data_ptr(), beta=0.5)
        m.backward()
        m.update(lr, 1)

    models = [llmk.GPT2(B, T, math=llmk.MATH_BF16, **CFG) for _ in range(2)]
    eager, own = models
    try:
        for m in models:
            m.set_grad_clip(0.01)
            step(m, 1e-3)  # everything that a first call sets up
            m.synchronize()
        stream = torch.cuda.ExternalStream(own.stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
            step(own, 2e-3)
        for m in models:
            m.load_parameters(params)
            m.load_optimizer_state(np.zeros(m.n, np.float32), np.zeros(m.n, np.float32))
        for _ in range(3):
            step(eager, 2e-3)
            eager.synchronize()
            step_elsewhere = llmk.GPT2(B, T, math=llmk.MATH_BF16, **CFG)  # other calls in between, with other values
            step_elsewhere.set_grad_clip(0.5)
            step(step_elsewhere, 0.7)
            step_elsewhere.close()
            with torch.cuda.stream(stream):
                graph.replay()
            own.synchronize()
        assert np.array_equal(eager.read_parameters(), own.read_parameters())
        assert eager.grad_norm() == own.grad_norm() > 0
        del graph
    finally:
        for m in models:
            m.close()
