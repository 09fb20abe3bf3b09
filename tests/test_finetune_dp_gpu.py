"""Clipped updates under data parallelism: the norm is that of the mean of the ranks' gradients, taken once the last of them
is reduced, and every rank applies the same update.

One process per rank, as in test_dp_gpu; with one rank only the harness and the plain path run, two ranks need 2 GPUs."""
import datetime
import os

import numpy as np
import pytest

from test_dp_gpu import SMALL, B, T, _paths

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
CLIPS = [0.0, 0.3, 0.3, 1e3, 0.0, 0.05]  # off, on, on, on without an effect, off, on


def _worker(rank, world, port, params, toks, q, graph):
    _paths()
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), NCCL_NVLS_ENABLE="0")
    import torch
    import torch.distributed as dist
    import llmk
    torch.cuda.set_device(rank)
    dist.init_process_group("gloo", rank=rank, world_size=world, timeout=datetime.timedelta(seconds=60))
    m = llmk.GPT2(B, T, math=llmk.MATH_TF32, **SMALL)
    m.load_parameters(params)
    obj = [llmk.nccl_unique_id() if rank == 0 else None]
    dist.broadcast_object_list(obj, src=0)
    m.enable_dp(obj[0], rank, world)
    m.use_graph(graph)
    out = []
    for s, clip in enumerate(CLIPS):
        m.set_grad_clip(clip)
        chunk = toks[s][rank * B * T:(rank + 1) * B * T + 1]
        m.train_step(chunk[:-1], chunk[1:], 1e-3, t=s + 1)
        m.synchronize(timeout_ms=60000)
        g = m.read_gradients().astype(np.float64) / world  # the buffer holds the sum over ranks
        out.append((m.grad_norm(), float(np.sqrt((g * g).sum())), m.read_parameters()))
    q.put((rank, out))
    dist.barrier()
    m.close()
    dist.destroy_process_group()


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("world", [1, 2])
def test_clipped_steps_over_ranks(world, graph):
    import socket
    import torch
    import torch.multiprocessing as mp
    if torch.cuda.device_count() < world:
        pytest.skip(f"needs {world} GPUs")
    _paths()
    import llmk
    import oracle as O
    cfg = O.config(**SMALL)
    params = O.init_params(cfg, 31)
    toks = [O.tokens(world * B * T + 1, cfg.vocab_size, 31 + s) for s in range(len(CLIPS))]
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_worker, args=(r, world, port, params, toks, q, graph)) for r in range(world)]
    for p in procs:
        p.start()
    res = dict(q.get(timeout=300) for _ in range(world))
    for p in procs:
        p.join(timeout=120)
        assert p.exitcode == 0
    # one GPU, the ranks' micro-batches side by side
    m = llmk.GPT2(world * B, T, math=llmk.MATH_TF32, **SMALL)
    m.load_parameters(params)
    last = 0.0
    for s, clip in enumerate(CLIPS):
        m.set_grad_clip(clip)
        c = toks[s]
        m.train_step(np.concatenate([c[r * B * T:(r + 1) * B * T] for r in range(world)]),
                     np.concatenate([c[r * B * T + 1:(r + 1) * B * T + 1] for r in range(world)]), 1e-3, t=s + 1)
        one, whole = m.read_parameters(), m.grad_norm()
        for r in range(world):
            norm, of_buffer, p = res[r][s]
            if clip:  # the sum of squares rounds up to 40 times in fp32, half of it reaches the root
                assert abs(norm - of_buffer) <= 22 * U * of_buffer, (s, r)
                assert abs(norm - whole) <= 1e-2 * whole, (s, r)  # tf32 gradients of the same batch, parts of it summed apart
                last = norm
            else:
                assert norm == last, (s, r)  # no clipped update, no new norm
            assert np.array_equal(p, res[0][s][2]), f"ranks diverged at step {s}"
            assert np.abs(p.astype(np.float64) - one).mean() < 1e-5, (s, r)
    m.close()
