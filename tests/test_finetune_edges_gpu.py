"""Calls of the fine-tuning operators at the edges of what their documentation
allows, on the GPU."""
import math

import numpy as np
import pytest
import torch

from test_finetune_gpu import Policy, Preference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pairs", [1, 40, 700])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_log_probabilities_over_the_reference_of_one_row_sequences(cuda_dev, pairs, dt):
    """Sequences of one row: logps and ref_logps have one size, so the one may take the other's place, and every warp of
    the pair has to have read the reference before it is written."""
    q = Preference(pairs, 1, 1001, 1008, dt, cuda_dev, seed=41, masked=0.0)
    q.call()
    q.check()
    want = [t.clone() for t in (q.losses, q.rewards, q.logps, q.dx)]
    ref = q.ref.clone()
    for _ in range(20):
        q.ref.copy_(ref)
        q.call(logps=q.ref)
        assert all(torch.equal(a, b) for a, b in zip(want, (q.losses, q.rewards, q.ref, q.dx)))
        w = q.w.clone()  # the rewards in the weights' place at the same time
        q.ref.copy_(ref)
        q.call(logps=q.ref, weights=w, rewards=w)
        assert all(torch.equal(a, b) for a, b in zip(want, (q.losses, w, q.ref, q.dx)))


U = 2.0 ** -24
LEAN = 1.2e-8  # what the sum of a long row may be off by in the mean (its correction by expf's own), relative
ROWS = [(5, 1001, 1008), (300, 1001, 1008), (5000, 40, 40), (40, 50257, 50304), (200, 50257, 50304), (90, 131072, 131080),
        (3, 131072, 131080)]


def two_tokens(shape, dt, dev, **kw):
    """Rows whose whole mass lies on the target and on one other token, in equal parts: lp = -log 2 exactly, and the
    gradient is c / 2 at the one and -c / 2 at the other."""
    rows, V, Vp = shape
    p = Policy(rows, V, Vp, dt, dev, seed=rows + V, masked=0.0, **kw)
    p.x[:, :V] = -math.inf
    at = torch.arange(rows, device=dev)
    p.t[:] = (at * 37 % V).int()
    other = (at * 37 + 1 + at % (V - 1)) % V
    p.x[at, p.t.long()], p.x[at, other] = 0.0, 0.0
    return p, at, other


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", ROWS)
def test_policy_gradient_next_to_the_reference(cuda_dev, shape, dt):
    """Where the KL term is the whole gradient (advantage 0, or a clipped ratio) and the policy is next to its reference,
    that gradient is 1 - exp(d): no error of exp(d) itself may reach it. c is off by what the row's sum is (LEAN for
    d), and the results by three roundings of c or c / sum, against half of c, and by one to their type; 16-bit ones also by a
    step of log2 (c / sum), 32 u at 16 to 32, in the exponent, and by 4 u of the exponential."""
    p, at, other = two_tokens(shape, dt, cuda_dev, kl=0.5)
    rows = shape[0]
    size = torch.tensor([1e-5, -1e-5, 1e-4, -1e-4, 1e-3, -1e-3], device=cuda_dev, dtype=torch.float64)[at % 6]
    p.ref = (size * (1 + torch.rand(rows, device=cuda_dev, dtype=torch.float64)) - math.log(2)).float()
    # no policy term: advantage 0; a ratio of e^0.5 for a positive advantage, of e^-0.5 for a negative one
    p.A = torch.tensor([0.0, 1.0, -1.0], device=cuda_dev)[(at // 6) % 3]
    p.old = (-math.log(2) - 0.5 * p.A.double()).float()
    p.call()
    d = p.ref.double() + math.log(2)
    k = p.w.double() * p.kl * float(np.float32(p.dscale))
    want = -k * torch.expm1(d) / 2
    tol = want.abs() * ((8 if dt == torch.float32 else 40) * U + torch.finfo(dt).eps / 2) + k * LEAN
    for got, sign in ((p.dx[at, p.t.long()], 1), (p.dx[at, other], -1)):
        assert ((sign * got.double() - want).abs() <= tol).all()
    p.dx[at, p.t.long()], p.dx[at, other] = 0.0, 0.0
    assert (p.dx == 0).all()


@pytest.mark.parametrize("shape", ROWS)
def test_policy_loss_and_gradient_take_the_same_branch(cuda_dev, shape):
    """Ratios within a few steps of fp32 of a clipping bound: whether the gradient vanishes and whether the loss is the
    clipped one go by the ratio in 64 bits."""
    p, at, other = two_tokens(shape, torch.float32, cuda_dev, ref=False, kl=0.0)
    lo, hi = 1 - float(np.float32(p.lo)), 1 + float(np.float32(p.hi))
    p.A = torch.where(at % 2 == 0, 1.0, -1.0)
    limit = torch.tensor([hi, lo], dtype=torch.float64, device=cuda_dev)[at % 2]
    bound = -math.log(2) - torch.log(limit)
    p.old = bound.float() + (at // 2 % 17 - 8) * 2.0 ** -24  # a step of fp32 at 0.5 to 1
    past = torch.where(at % 2 == 0, 1.0, -1.0).double() * (bound - p.old.double())  # > 0: outside
    near = past.abs() < 2 * LEAN  # what the row's sum may decide
    p.call()
    rho = torch.exp(-math.log(2) - p.old.double())
    zero = (p.dx[at, p.t.long()] == 0) & (p.dx[at, other] == 0)
    assert torch.equal(zero[~near], (past > 0)[~near])
    loss = -p.w.double() * p.A.double() * torch.where(past > 0, limit, rho)
    assert ((p.losses.double() - loss).abs() <= loss.abs() * (U + 2 * LEAN)).all()


# The mean error of a long row's log-probability: expf's own mean of 6e-9 in the terms that correct the sum, and again in
# the factors that join it.
MEAN = 1.2e-8
# The other part of it, which differs from row to row: the roundings of a warp's and of a group's joins, 10 of them of
# u / sqrt(3) each (those of the lanes' sums average out over 32 lanes and more).
SPREAD = 10 ** 0.5 * U / 3 ** 0.5


def long_rows(rows, V, dt, dev, spread=0.0, peak=0.0, target_is_peak=False):
    """Normal logits of a spread, or even ones with one token in each row that stands `peak` above them; targets, and
    their log-probabilities in 64 bits."""
    g = torch.Generator(device=dev)
    g.manual_seed(rows + V)
    x = torch.empty(rows, -(-V // 8) * 8, device=dev, dtype=dt)
    t = torch.randint(0, V, (rows,), generator=g, device=dev, dtype=torch.int32)
    lp = torch.empty(rows, dtype=torch.float64, device=dev)
    for i in range(0, rows, 2048):
        part, pt = x[i:i + 2048], t[i:i + 2048].long()[:, None]
        if peak:
            v = torch.rand(part.shape, generator=g, device=dev)
            at = pt if target_is_peak else torch.randint(0, V, pt.shape, generator=g, device=dev)
            v.scatter_(1, at, peak + torch.rand(pt.shape, generator=g, device=dev))
        else:
            v = torch.randn(part.shape, generator=g, device=dev) * spread
        part.copy_(v)
        v = part[:, :V].double()
        lp[i:i + 2048] = v.gather(-1, pt)[:, 0] - torch.logsumexp(v, -1)
    return x, t, lp


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,V,kw", [(16384, 1000, dict(spread=1.0)), (16384, 20000, dict(spread=1.0)), (16384, 4097, dict(spread=4.0)),
                                    (16384, 20000, dict(peak=2.0)), (16384, 1000, dict(peak=10.0)), (8192, 4097, dict(peak=10.0)),
                                    (4096, 50257, dict(peak=8.0))])
def test_rewards_of_long_sequences_do_not_lean(cuda_dev, T, V, kw, dt):
    """A reward adds its sequence's log-probabilities: the mean error counts T times, the others' sum grows by sqrt(T).
    A row whose greatest logit stands out is off no more: that term is exactly 1, wherever it is met."""
    import llmk
    x, t, lp = long_rows(2 * T, V, dt, cuda_dev, **kw)
    L = lp.view(2, T).sum(-1)
    ref, rewards, loss = L.float(), torch.empty(2, device=cuda_dev), torch.empty(1, device=cuda_dev)
    ws = torch.empty(llmk.preference_loss_workspace(1, T, x.shape[1]), dtype=torch.uint8, device=cuda_dev)
    llmk.preference_loss(loss, x, t, V=V, ref_logps=ref, rewards=rewards, beta=1.0, workspace=ws)
    want = L - ref.double()  # what rounding the reference leaves
    assert ((rewards.double() - want).abs() <= T * MEAN + 6 * SPREAD * math.sqrt(T) + U * want.abs()).all()


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V,peak", [(16384, 1000, 8.0), (16384, 4097, 10.0), (8192, 50257, 10.0)])
def test_log_probabilities_of_confident_rows_do_not_lean(cuda_dev, rows, V, peak, dt, grad):
    """The mean error of the policy loss's log-probabilities where the target stands out, to 5 standard deviations, the
    results' own roundings (uniform in a step) among them."""
    import llmk
    x, t, lp = long_rows(rows, V, dt, cuda_dev, peak=peak, target_is_peak=True)
    A, losses, logps = torch.ones(rows, device=cuda_dev), torch.empty(rows, device=cuda_dev), torch.empty(rows, device=cuda_dev)
    ws = torch.empty(llmk.policy_loss_workspace(rows, x.shape[1]), dtype=torch.uint8, device=cuda_dev)
    llmk.policy_loss(losses, x, t, A, V=V, logps=logps, dlogits=x if grad else None, workspace=ws)
    step = 2.0 ** (torch.floor(torch.log2(lp.abs())) - 23)
    var = (step.square() / 12).mean().item() + SPREAD ** 2
    assert abs((logps.double() - lp).mean().item()) <= MEAN + 5 * math.sqrt(var / rows)
