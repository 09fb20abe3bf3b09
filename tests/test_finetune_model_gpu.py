"""The fine-tuning losses on top of the lm_head (llmk_matmul_policy_forward,
llmk_matmul_preference_forward) and in the native trainer, with gradient
clipping: a step on preferences or samples as a program makes it.

The fused operators are held to the unfused ones on the logits that the device
stores. Their row statistics come from the GEMM's epilogue, where a row's
log-probability is off by at most 2 LP (LP as in test_finetune_gpu: here 24 u
more for the rounding of the reference point, and 64-term sums); so the two
differ by at most 3 LP.
"""
import math

import numpy as np
import pytest
import torch

import oracle as O
from test_finetune_gpu import HALF, LP, U, Policy, Preference, within

pytestmark = pytest.mark.gpu


def operands(BT, C, V, Vp, mathname, dev, seed, bias):
    dt = torch.bfloat16 if mathname == "bf16" else torch.float32
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    x = torch.randn(BT, C, generator=g, device=dev).to(dt)
    W = (torch.randn(Vp, C, generator=g, device=dev) * (2.5 / math.sqrt(C))).to(dt)
    return x, W, torch.randn(Vp, generator=g, device=dev) if bias else None


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("mathname", ["bf16", "tf32"])
@pytest.mark.parametrize("which", ["policy", "preference"])
@pytest.mark.parametrize("shape", [(66, 128, 1001, 1008), (256, 256, 50257, 50304), (2, 64, 9, 16)])
def test_fused_with_the_lm_head(cuda_dev, shape, which, mathname, bias):
    import llmk
    BT, C, V, Vp = shape
    x, W, b = operands(BT, C, V, Vp, mathname, cuda_dev, 31, bias)
    math_mode = llmk.MATH_BF16 if mathname == "bf16" else llmk.MATH_TF32
    logits = torch.empty(BT, Vp, dtype=x.dtype, device=cuda_dev)
    llmk.gemm(logits, x, W, math=math_mode, bias=b)
    if which == "policy":
        p = Policy(BT, V, Vp, x.dtype, cuda_dev, seed=32)
        lp = torch.log_softmax(logits[:, :V].double(), -1).gather(-1, p.t.long()[:, None])[:, 0]
        p.old = (lp - torch.tensor([-0.5, 0.0, 0.1, 0.5], device=cuda_dev)[torch.arange(BT, device=cuda_dev) % 4]).float()
        p.ref = (lp + 0.3 * torch.sin(torch.arange(BT, device=cuda_dev))).float()
    else:
        p = Preference(BT // 2, 1, V, Vp, x.dtype, cuda_dev, seed=33) if BT < 10 else Preference(2, BT // 4, V, Vp, x.dtype, cuda_dev, seed=33)
        if BT % 4 and BT > 10:
            p = Preference(BT // 2, 1, V, Vp, x.dtype, cuda_dev, seed=33)
    p.x = logits
    p.call()  # the unfused form
    want = [v.clone() for v in (p.losses, p.logps, p.dx)] + [(p.kls if which == "policy" else p.rewards).clone()]
    out = torch.full_like(logits, 5.0)
    losses, logps, extra = torch.empty_like(p.losses), torch.empty_like(p.logps), torch.empty_like(want[3])
    ws = torch.empty(llmk.lib().llmk_matmul_finetune_workspace(BT, Vp), dtype=torch.uint8, device=cuda_dev)
    P, code, s = llmk.ptr, llmk.dtype_code(out), llmk.stream_ptr()
    for backward in (0, 1):
        if which == "policy":
            llmk.call("llmk_matmul_policy_forward", P(losses), P(extra), P(logps), P(out), code, P(x), P(W), P(b), P(p.t), P(p.w),
                      P(p.A), P(p.old), P(p.ref), BT, C, Vp, V, p.lo, p.hi, p.kl, p.dscale, backward, math_mode, P(ws), ws.numel(), s)
        else:
            llmk.call("llmk_matmul_preference_forward", P(losses), P(extra), P(logps), P(out), code, P(x), P(W), P(b), P(p.t), P(p.w),
                      P(p.ref), p.pairs, p.T, C, Vp, V, p.beta, p.smooth, p.dscale, backward, math_mode, P(ws), ws.numel(), s)
        if not backward:
            assert torch.equal(out, logits)
    tol = 3 * LP
    within(logps, want[1], tol + 2 * U * want[1].double().abs(), "logps")
    live = (p.w != 0)[:, None]
    if which == "policy":
        w, A = p.w.double(), p.A.double().abs()
        r = torch.exp(want[1].double() - p.old.double())
        e = torch.exp(p.ref.double() - want[1].double())
        within(losses, want[0], w * (r * A + p.kl * (1 + e)) * tol + 2 * U * want[0].double().abs(), "losses")
        within(extra, want[3], (1 + e) * tol + 2 * U * want[3].double().abs(), "kls")
        mag = (w * p.dscale * (r * A + p.kl * (1 + e)))[:, None]
    else:
        err = p.beta * tol * p.w.double().view(2 * p.pairs, -1).sum(-1)
        within(extra, want[3], err + 2 * U * want[3].double().abs(), "rewards")
        herr = err[:p.pairs] + err[p.pairs:]
        within(losses, want[0], herr + 2 * U * want[0].double().abs(), "losses")
        mag = (p.w.double() * p.beta * p.dscale)[:, None] * (1 + herr.max() / tol)
    prob = torch.softmax(logits[:, :V].double(), -1)
    hot = torch.zeros_like(prob).scatter_(-1, p.t.long()[:, None], 1.0)
    d = want[2][:, :V].double()
    # each side rounds the gradient by half a step of the logits' type
    within(out[:, :V], d, torch.where(live, 2 * HALF[out.dtype] * d.abs() + 2 * tol * mag * (prob + hot) + 1e-37, 0.0), "dlogits")
    assert (out[:, V:] == 0).all() and (out[~live[:, 0]] == 0).all()


CFG = dict(max_seq_len=64, vocab_size=1000, padded_vocab_size=1024, num_layers=2, num_heads=2, channels=128)
B, T = 4, 48


@pytest.fixture
def setup(cuda_dev):
    import llmk
    cfg = O.config(**CFG)
    params = O.init_params(cfg, 5)
    toks = torch.from_numpy(O.tokens(B * T + 1, cfg.vocab_size, 6)).to(cuda_dev)
    made = []

    def model(mathname="bf16"):
        m = llmk.GPT2(B, T, math=llmk.MATH_BF16 if mathname == "bf16" else llmk.MATH_TF32, **CFG)
        m.load_parameters(params)
        made.append(m)
        return m
    yield model, params, toks[:-1].contiguous(), toks[1:].contiguous()
    for m in made:
        m.close()


def ready():
    torch.cuda.synchronize()  # the model runs on its own stream


@pytest.mark.parametrize("mathname", ["bf16", "tf32"])
def test_policy_step_is_cross_entropy_where_they_coincide(cuda_dev, setup, mathname):
    """Without old log-probabilities, advantages 1 and weights 1 / (B T), the policy loss's gradient is the mean
    cross-entropy's; the log-probabilities' mean is minus its loss."""
    model, _, inp, tgt = setup
    n = B * T
    a = model(mathname)
    a.forward(inp.data_ptr(), tgt.data_ptr())
    a.backward()
    ce, g = a.loss(), a.read_gradients()
    lp = torch.empty(n, device=cuda_dev)
    a.logprobs(inp.data_ptr(), tgt.data_ptr(), lp.data_ptr())
    with pytest.raises(Exception):
        a.backward()  # log-probabilities leave no gradient
    w, A, got = torch.full((n,), 1.0 / n, device=cuda_dev), torch.ones(n, device=cuda_dev), torch.empty(n, device=cuda_dev)
    ready()
    assert abs(-lp.double().mean().item() - ce) < 2 * LP + 64 * U * ce  # the cross-entropy's own sum runs in fp32
    a.forward_policy(inp.data_ptr(), tgt.data_ptr(), A.data_ptr(), weights=w.data_ptr(), logps=got.data_ptr())
    loss = a.loss()
    assert torch.equal(got, lp)
    assert abs(loss + 1.0) < 1e-5  # -sum w A
    a.backward()
    h = a.read_gradients()
    # the two gradients of the logits differ by a step of their type (2 half steps) where their statistics round
    # apart, and everything after is linear in them
    step = 2 * (2.0 ** -8 if mathname == "bf16" else 2 ** -11)
    assert np.linalg.norm(h - g) <= step * np.linalg.norm(g)


@pytest.mark.parametrize("mathname", ["bf16", "tf32"])
def test_preference_step_is_a_weighted_policy_step(cuda_dev, setup, mathname):
    """The gradient of the preference loss is the policy gradient with advantages -+dloss/dL of each sequence."""
    model, _, inp, tgt = setup
    m = model(mathname)
    w = (torch.rand(B, T, device=cuda_dev) < 0.7).float()
    w[3, 20:] = 0  # padding
    ref = torch.tensor([-200.0, -210.0, -205.0, -90.0], device=cuda_dev)
    rewards, lp = torch.empty(B, device=cuda_dev), torch.empty(B * T, device=cuda_dev)
    ready()
    beta = 0.05
    m.forward_preference(inp.data_ptr(), tgt.data_ptr(), weights=w.data_ptr(), ref_logps=ref.data_ptr(), beta=beta,
                         label_smoothing=0.1, rewards=rewards.data_ptr(), logps=lp.data_ptr())
    loss = m.loss()
    m.backward()
    g = m.read_gradients()
    r = beta * ((lp.view(B, T).double() * w.double()).sum(-1) - ref.double())
    within(rewards, r, 1e-6 * r.abs() + beta * T * U * 20, "rewards")
    h = rewards[:2].double() - rewards[2:].double()
    want = (-0.9 * torch.nn.functional.logsigmoid(h) - 0.1 * torch.nn.functional.logsigmoid(-h)).mean().item()
    assert abs(loss - want) < 8 * U * max(1.0, want)
    slope = beta * (0.1 * torch.sigmoid(h) - 0.9 * torch.sigmoid(-h)) / 2
    A = torch.cat([-slope, slope])[:, None].expand(B, T).float().contiguous()
    ready()
    m.forward_policy(inp.data_ptr(), tgt.data_ptr(), A.data_ptr(), weights=w.data_ptr())
    m.backward()
    q = m.read_gradients()
    step = 2 * (2.0 ** -8 if mathname == "bf16" else 2 ** -11)
    assert np.linalg.norm(q - g) <= step * np.linalg.norm(g)


def test_preference_gradient_by_differences(cuda_dev, setup):
    """Along the gradient, the loss falls by the gradient's squared norm per unit step."""
    model, params, inp, tgt = setup
    m = model("tf32")
    args = dict(beta=0.1)

    def loss_at(p):
        m.load_parameters(p)
        m.forward_preference(inp.data_ptr(), tgt.data_ptr(), **args)
        return m.loss()
    loss_at(params)
    m.backward()
    g = m.read_gradients().astype(np.float64)
    n2 = float((g * g).sum())
    eps = 0.02 / math.sqrt(n2)  # a change of parameters of norm 0.02
    d = (loss_at((params + eps * g).astype(np.float32)) - loss_at((params - eps * g).astype(np.float32))) / (2 * eps)
    # tf32 products round by 2^-11, and the attention's 16-bit operands by 2^-11 too; a dozen of them on any path
    assert abs(d / n2 - 1) < 24 * 2.0 ** -11


@pytest.mark.parametrize("graph", [False, True])
def test_clipped_training(cuda_dev, setup, graph):
    """A clipped step is the plain step on gradients of the clipped norm; clipping can change between steps, with a
    captured graph too."""
    model, params, inp, tgt = setup
    plain, m = model(), model()
    m.use_graph(graph)
    h = [t.cpu().numpy() for t in (inp, tgt)]
    plain.train_step(*h, 1e-3, t=1)
    g = plain.read_gradients().astype(np.float64)
    norm = math.sqrt(float((g * g).sum()))
    clip = norm / 3
    m.set_grad_clip(clip)
    assert m.grad_norm() == 0.0
    m.train_step(*h, 1e-3, t=1)
    assert np.array_equal(m.read_gradients(), plain.read_gradients())  # the gradients stay as they are
    assert abs(m.grad_norm() - norm) < 25 * U * norm
    mom, var = m.read_optimizer_state()
    k = clip / (norm + 1e-6)
    assert np.allclose(mom, 0.1 * k * g, rtol=40 * U, atol=1e-30)
    assert np.allclose(var, 0.001 * (k * g) ** 2, rtol=1e-4, atol=1e-30)  # 1 - 0.999f itself is off by 6e-5
    m.set_grad_clip(0.0)
    m.load_parameters(params)
    m.train_step(*h, 1e-3, t=1)
    assert np.array_equal(m.read_parameters(), plain.read_parameters())
    m.set_grad_clip(math.inf)
    m.load_parameters(params)
    m.train_step(*h, 1e-3, t=1)
    assert np.array_equal(m.read_parameters(), plain.read_parameters())
    with pytest.raises(Exception):
        m.set_grad_clip(-1.0)
    with pytest.raises(Exception):
        m.set_grad_clip(math.nan)


def test_a_fine_tuning_run(cuda_dev, setup):
    """Reference log-probabilities, preference steps, policy steps on samples, all clipped: the operators as a program
    uses them, on finite numbers throughout and with the losses' signs."""
    model, _, inp, tgt = setup
    ref_model, m = model(), model()
    m.set_grad_clip(0.5)
    n = B * T
    w = torch.ones(B, T, device=cuda_dev)
    w[:, :10] = 0
    w[2, 30:] = 0
    lp, rewards, kls = torch.empty(n, device=cuda_dev), torch.empty(B, device=cuda_dev), torch.empty(n, device=cuda_dev)
    ready()
    ref_model.logprobs(inp.data_ptr(), tgt.data_ptr(), lp.data_ptr())
    ref_model.synchronize()
    ref = (lp.view(B, T) * w).sum(-1).contiguous()
    ready()
    first = None
    for t in range(1, 6):
        m.forward_preference(inp.data_ptr(), tgt.data_ptr(), weights=w.data_ptr(), ref_logps=ref.data_ptr(), beta=0.5,
                             rewards=rewards.data_ptr())
        loss = m.loss()
        first = loss if first is None else first
        m.backward()
        m.update(1e-3, t)
        assert math.isfinite(loss) and m.grad_norm() > 0
    assert abs(first - math.log(2)) < 1e-3  # the model is its own reference at first
    margin = rewards[:2] - rewards[2:]
    assert (margin > 0).all()
    wn = (w / w.sum()).contiguous()
    A = torch.randn(n, device=cuda_dev)
    ready()
    m.forward_policy(inp.data_ptr(), tgt.data_ptr(), A.data_ptr(), weights=wn.data_ptr(), old_logps=lp.data_ptr(),
                     ref_logps=lp.data_ptr(), kl_coef=0.1, kls=kls.data_ptr())
    loss = m.loss()
    m.backward()
    m.update(1e-3, 6)
    m.synchronize()
    assert math.isfinite(loss) and math.isfinite(m.grad_norm())
    assert (kls.view(B, T)[w == 0] == 0).all() and (kls >= 0).all() and kls.sum() > 0
    assert np.isfinite(m.read_parameters()).all()
    import llmk
    assert llmk.device_status() == 0


def test_odd_batch_is_refused(cuda_dev):
    import llmk
    m = llmk.GPT2(3, 16, **CFG)
    with pytest.raises(llmk.LlmkError) as e:
        m.forward_preference(m.buffers()[0], m.buffers()[1])
    assert e.value.code == 1
    m.close()
