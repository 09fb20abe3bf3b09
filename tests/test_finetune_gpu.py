"""The fine-tuning operators on the GPU against their formulas in 64 bits:
clipped policy loss with KL term, preference loss, gradient norm, clipping and
AdamW on clipped gradients.

Tolerances count roundings. u = 2^-24 is half a step of fp32. A row's
log-probability is off by at most LP = 256 u: a sum of exponentials takes at
most 200 roundings on any path (a thread's partial sum of up to 128 terms, the
tree over a block, the slices), each exponential is off by 2 steps (4 u) and
its argument, a difference of logits up to 24 apart, by 24 u; all of them
relative errors of the sum, so absolute ones of its logarithm. Everything after
that is computed in 64 bits and rounded once, by half a step of its type.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
LP = 256 * U
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
TINY = 1e-37  # results this small may be flushed to zero


def within(got, want, tol, what=""):
    got, want, tol = got.double(), want.double(), torch.as_tensor(tol, dtype=torch.float64, device=got.device)
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what + ": NaN elsewhere"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), what
    bad = ((got - want).abs() > tol) & torch.isfinite(want)
    if bad.any():
        i = int(bad.flatten().nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {i}: {got.flatten()[i]} is not "
                             f"{want.flatten()[i]} within {tol.expand_as(got).flatten()[i]}")


def make_logits(rows, V, Vp, dt, seed, dev):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    x = (torch.randn(rows, Vp, generator=g, device=dev) * 2.5).to(dt)
    x[:, V:] = float("nan")  # padding columns hold anything
    t = torch.randint(0, V, (rows,), generator=g, device=dev, dtype=torch.int32)
    return x, t, g


def logps_of(x, t, V):
    """Softmax and target log-probabilities in 64 bits."""
    x = x[:, :V].double()
    lse = torch.logsumexp(x, -1)
    return torch.exp(x - lse[:, None]), x.gather(-1, t.long().clamp(0, V - 1)[:, None])[:, 0] - lse


def check_dlogits(got, p, t, c, c_err, live, V, dt):
    """got against c ([j = target] - p); c_err bounds what c itself may be off by (absolute)."""
    rows, Vp = got.shape
    onehot = torch.zeros_like(p).scatter_(-1, t.long().clamp(0, V - 1)[:, None], 1.0)
    want = torch.where(live[:, None], c[:, None] * (onehot - p), torch.zeros_like(p))
    tol = HALF[dt] * want.abs() + c_err[:, None] * (onehot + p) + 2 * LP * c.abs()[:, None] * p + 4 * U * c.abs()[:, None] * onehot + TINY
    within(got[:, :V], want, torch.where(live[:, None], tol, torch.zeros_like(tol)), "dlogits")
    assert (got[:, V:] == 0).all()  # an exact zero, no NaN
    assert (got[~live] == 0).all()


class Policy:
    """Inputs of one policy-loss call, its 64-bit results and their tolerances."""

    def __init__(self, rows, V, Vp, dt, dev, seed=0, masked=0.3, old=True, ref=True, lo=0.2, hi=0.2, kl=0.05, dscale=0.7):
        import llmk
        self.V, self.Vp, self.dt, self.kl, self.lo, self.hi, self.dscale = V, Vp, dt, kl, lo, hi, dscale
        self.x, self.t, g = make_logits(rows, V, Vp, dt, seed, dev)
        _, lp = logps_of(self.x, self.t, V)
        n = lambda s: torch.randn(rows, generator=g, device=dev) * s  # noqa: E731
        self.w = torch.rand(rows, generator=g, device=dev) + 0.5
        if masked:
            self.w[torch.rand(rows, generator=g, device=dev) < masked] = 0.0
        self.A = n(1.0)
        drift = n(0.2)
        for b in (math.log1p(hi), math.log(1 - lo) if lo < 1 else 9.0):  # no ratio on a bound, where rounding decides
            drift[(drift - b).abs() < 1e-4] += 1e-3
        self.old = (lp - drift).float() if old else None
        self.ref = (lp + n(0.3)).float() if ref else None
        mk = lambda *s, d=torch.float32: torch.full(s, 7.0, device=dev, dtype=d)  # noqa: E731
        self.losses, self.logps = mk(rows), mk(rows)
        self.kls = mk(rows) if ref else None
        self.dx = mk(rows, Vp, d=dt)
        self.ws = torch.empty(llmk.policy_loss_workspace(rows, Vp), dtype=torch.uint8, device=dev)

    def call(self, **kw):
        import llmk
        a = dict(V=self.V, weights=self.w, old_logps=self.old, ref_logps=self.ref, kls=self.kls, logps=self.logps,
                 dlogits=self.dx, clip_low=self.lo, clip_high=self.hi, kl_coef=self.kl, dscale=self.dscale,
                 workspace=self.ws)
        a.update(kw)
        llmk.policy_loss(self.losses, a.pop("logits", self.x), self.t, self.A, **a)

    def check(self, dx=None):
        w = torch.ones_like(self.A) if self.w is None else self.w
        live = w != 0
        p, lp = logps_of(self.x, self.t, self.V)
        w, A, zero = w.double(), self.A.double(), torch.zeros_like(lp)
        rho = torch.exp(lp - self.old.double()) if self.old is not None else torch.ones_like(lp)
        s1, s2 = rho * A, rho.clamp(1 - float(np.float32(self.lo)), 1 + float(np.float32(self.hi))) * A
        loss, c = -torch.minimum(s1, s2), torch.where(s1 > s2, zero, -s1)
        # rho is off by rho LP; the clamped product by no more
        mag = (rho * A.abs()) * LP
        if self.ref is not None:
            d = self.ref.double() - lp
            e, kl = torch.expm1(d), torch.expm1(d) - d
            kerr = e.abs() * LP + (1 + e) * LP * LP
            within(self.kls, torch.where(live, kl, zero), torch.where(live, kerr + U * kl + TINY, zero), "kls")
            beta = float(np.float32(self.kl))
            loss, c, mag = loss + beta * kl, c - beta * e, mag + beta * ((1 + e) * LP + kerr)
        within(self.losses, torch.where(live, w * loss, zero), torch.where(live, w * mag + U * (w * loss).abs() + TINY, zero), "losses")
        within(self.logps, torch.where(live, lp, zero), torch.where(live, LP + U * lp.abs(), zero), "logps")
        k = w * float(np.float32(self.dscale))
        dx = self.dx if dx is None else dx
        if dx is not None:
            check_dlogits(dx, p, self.t, c * k, (mag + 2 * U * c.abs()) * k, live, self.V, self.dt)


SHAPES = [(1, 1, 8), (1, 5, 8), (3, 7, 16), (5, 1001, 1008), (37, 4097, 4104), (2, 8192, 8192), (4, 8193, 8200),
          (9, 50257, 50304), (150, 12345, 12352), (3, 131072, 131080)]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_policy_loss(cuda_dev, shape, dt):
    p = Policy(*shape, dt, cuda_dev, seed=sum(shape))
    p.call()
    p.check()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,V,Vp", [(1, 7, 8), (2, 1555, 1696), (3, 501, 504), (8, 2000, 2000), (100, 5000, 5000)])
def test_few_rows_of_small_vocabularies(cuda_dev, rows, V, Vp, dt, monkeypatch):
    """Here a log-probability is off by at most 40 u: expf 2 u, the difference it is of 8 u (in the mean over the terms,
    8 apart), 8 additions in a lane, 5 in a warp and 5 over warps, and two factors expf(m - max) of 3 u; in all 34 u."""
    import sys
    monkeypatch.setattr(sys.modules[__name__], "LP", 40 * U)
    for grad in (True, False):
        p = Policy(rows, V, Vp, dt, cuda_dev, seed=V + rows, masked=0.0)
        if not grad:
            p.dx = None
        p.call()
        p.check()


@pytest.mark.parametrize("rows,V,Vp,dt", [(90, 131072, 131080, torch.bfloat16), (301, 110593, 110600, torch.bfloat16),
                                          (80, 400001, 400008, torch.bfloat16), (160, 55297, 55304, torch.float32),
                                          (75, 200003, 200008, torch.float32), (74, 131072, 131072, torch.bfloat16)])
def test_policy_loss_long_rows(cuda_dev, rows, V, Vp, dt):
    """Rows that do not fit an SM's shared memory, by one kernel and (few of them) by three."""
    p = Policy(rows, V, Vp, dt, cuda_dev, seed=rows)
    n = V // 7
    for i in range(0, rows, 3):  # targets in every stretch of a row, its ends included
        p.t[i] = min(V - 1, (i // 3) % 8 * n) if i % 2 else V - 1 - min(V - 1, (i // 3) % 8 * n)
    _, lp = logps_of(p.x, p.t, V)
    p.old, p.ref = (lp + 0.05).float(), (lp - 0.1).float()
    p.call()
    p.check()
    p.kl, p.A[1::2] = 0.0, 0.0  # every other live row without a gradient
    p.call()
    p.check()
    assert (p.dx[1::2] == 0).all()
    y = p.x.clone()
    p.call(logits=y, dlogits=y)
    assert torch.equal(y, p.dx)


@pytest.mark.parametrize("kw", [dict(old=False), dict(ref=False, kl=0.0), dict(kl=0.0), dict(masked=0.0),
                                dict(lo=0.0, hi=0.0), dict(lo=1.0, hi=5.0), dict(old=False, ref=False, kl=0.0)])
def test_policy_loss_forms(cuda_dev, kw):
    p = Policy(200, 1001, 1008, torch.float32, cuda_dev, seed=5, **kw)
    p.call()
    p.check()


def test_policy_loss_without_weights_in_place_and_without_gradient(cuda_dev):
    p = Policy(300, 2000, 2048, torch.bfloat16, cuda_dev, seed=6, masked=0.0)
    p.w = None
    p.call()
    p.check()
    first = p.dx.clone()
    buf = p.x.clone()
    p.call(logits=buf, dlogits=buf)  # the gradient over the logits
    assert torch.equal(buf, first)
    p.losses.fill_(7.0), p.logps.fill_(7.0)
    keep = p.dx.fill_(3.0)
    p.call(dlogits=None)
    assert (keep == 3.0).all()
    p.check(dx=first)


@pytest.mark.parametrize("rows", [1, 147, 148, 149, 296, 1000])
def test_policy_loss_row_counts(cuda_dev, rows):
    """Row counts around the number of SMs: every way of sharing rows out."""
    for V, Vp, dt in ((50257, 50304, torch.bfloat16), (20000, 20000, torch.float32)):
        p = Policy(rows, V, Vp, dt, cuda_dev, seed=rows)
        p.call()
        p.check()


def test_policy_loss_masked_rows_are_not_read(cuda_dev):
    p = Policy(64, 1000, 1000, torch.bfloat16, cuda_dev, seed=8, masked=0.5)
    dead = p.w == 0
    assert dead.any()
    p.x[dead] = float("nan")
    p.t[dead] = -100
    for v in (p.A, p.old, p.ref):
        v[dead] = float("nan")
    p.call()
    assert all((v[dead] == 0).all() for v in (p.losses, p.kls, p.logps, p.dx))
    for v, fill in ((p.A, 0.0), (p.old, 0.0), (p.ref, 0.0), (p.x, 0.0)):
        v[dead] = fill
    p.t[dead] = 0
    p.check()
    p.w.zero_()  # nothing left
    p.call()
    assert all((v == 0).all() for v in (p.losses, p.kls, p.logps, p.dx))


def test_policy_loss_special_values(cuda_dev):
    """-inf logits are probability 0; the type's lowest value too; NaN, +inf, a row of -inf and a bad target give NaN in
    their own row only; advantage 0 has no policy term, whatever the ratio."""
    rows, V, Vp = 10, 9000, 9000
    for dt in (torch.float32, torch.bfloat16):
        p = Policy(rows, V, Vp, dt, cuda_dev, seed=9, masked=0.0, ref=False, kl=0.0)
        nan_rows = [3, 4, 5, 6, 7]
        p.x[0, 1::2], p.t[0] = -math.inf, 4
        p.x[1, 100:], p.t[1] = torch.finfo(dt).min, 5
        p.x[2, :], p.t[2] = -math.inf, 8500
        p.x[2, 8500] = 1.0  # all mass on the target: lp = 0, zero gradient
        p.x[3, 17] = math.nan
        p.x[4, 8999] = math.inf
        p.x[5, :] = -math.inf
        p.t[6], p.t[7] = -1, V
        _, lp = logps_of(p.x, p.t, V)
        p.old = torch.where(torch.isfinite(lp), lp, torch.zeros_like(lp)).float() - 0.05
        p.A[8], p.old[8] = 0.0, -1e30  # rho = inf
        p.call()
        for v in (p.losses, p.logps):
            assert torch.isnan(v[nan_rows]).all() and torch.isfinite(v[[0, 1, 2, 8, 9]]).all()
        assert torch.isnan(p.dx[nan_rows][:, :V]).all()
        assert p.losses[8] == 0 and (p.dx[8] == 0).all()
        assert (p.dx[0, 1::2] == 0).all() and (p.dx[1, 100:] == 0).all()
        assert p.logps[2] == 0 and (p.dx[2] == 0).all()
        p.w = torch.ones(rows, device=cuda_dev)
        for r in nan_rows + [8]:
            p.w[r] = 0
            p.x[r], p.t[r], p.old[r] = 0.0, 0, 0.0
        p.call()
        p.check()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_policy_loss_terms_next_to_nothing(cuda_dev, dt):
    """Two tokens share the mass, all others are where an exponential leaves fp32's normal range: the row's
    log-probability is -log 2."""
    for rows, V in ((3, 1000), (2, 20000)):
        p = Policy(rows, V, V, dt, cuda_dev, seed=21, masked=0.0, ref=False, kl=0.0)
        far = torch.arange(V, device=cuda_dev) % 9
        p.x[:] = (-85.0 - 0.5 * far).to(dt)
        for at in ((5, 13), (V - 3, 21), (11, V // 2 + 5)):
            p.x[:, at[0]], p.x[:, at[1]] = 0.0, 0.0
            p.t[:] = at[0]
            p.old = torch.full((rows,), -0.7, device=cuda_dev)
            p.call()
            p.check()
            p.x[:, at[0]], p.x[:, at[1]] = -86.0, -86.0


def test_policy_loss_unreachable_target(cuda_dev):
    """A target of probability 0: the KL estimate is infinite, not NaN; without a KL term the gradient vanishes."""
    p = Policy(4, 500, 504, torch.float32, cuda_dev, seed=22, masked=0.0)
    p.t[1] = 77
    p.x[1, 77] = -math.inf
    p.old[1], p.ref[1] = -3.0, -3.0
    p.call()
    assert p.logps[1] == -math.inf and p.kls[1] == math.inf and p.losses[1] == math.inf
    p.call(kl_coef=0.0)
    # rho = 0: -min(0 A, 0.8 A) is 0 for A > 0 and -0.8 A for A < 0, without a gradient either way
    want = p.w[1].item() * max(0.0, -(1 - float(np.float32(p.lo))) * p.A[1].item())
    assert abs(p.losses[1].item() - want) <= 2 * U * want
    assert (p.dx[1] == 0).all() and p.kls[1] == math.inf


@pytest.mark.parametrize("grad", [True, False])
def test_losses_of_very_many_rows(cuda_dev, grad):
    """More rows than one launch takes on."""
    p = Policy(350001, 7, 8, torch.bfloat16, cuda_dev, seed=23)
    p.call(**({} if grad else dict(dlogits=None)))
    if not grad:
        p.dx = None
        p.check()
        return
    p.check()
    q = Preference(1, 175001, 5, 8, torch.float32, cuda_dev, seed=24, beta=1e-4)
    q.call()
    q.check()


def test_losses_at_once_on_two_streams(cuda_dev):
    """Two calls in flight, each with a workspace of its own, and masked rows all over."""
    a, b = (Policy(700, 9001, 9008, torch.bfloat16, cuda_dev, seed=s, masked=0.6) for s in (25, 26))
    c = Preference(3, 200, 9001, 9008, torch.float32, cuda_dev, seed=27, masked=0.6)
    torch.cuda.synchronize()
    s = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(5):
        for p, st in zip((a, b, c), s):
            p.call(stream=st)
    torch.cuda.synchronize()
    for p in (a, b, c):
        p.check()


def test_policy_gradient_by_differences(cuda_dev):
    """dlogits against the difference quotient of the summed losses, in a random direction."""
    p = Policy(40, 500, 504, torch.float32, cuda_dev, seed=10, dscale=1.0)
    p.x[:, p.V:] = 0
    # ratios inside the bounds and well outside them: no step crosses a bound
    _, lp = logps_of(p.x, p.t, p.V)
    p.old = (lp - torch.tensor([-0.5, 0.0, 0.5, 0.05], device=cuda_dev).repeat(10)).float()
    p.call()
    base, g = p.x.clone(), p.dx.double()
    torch.manual_seed(1)
    step = 1e-2
    for _ in range(3):
        d = torch.randn_like(base)
        d[:, p.V:] = 0
        total = []
        for sign in (1, -1):
            p.x = base + sign * step * d
            p.call()
            total.append(p.losses.double().sum())
        # central differences: the third derivative's term (under 2 a row at these sizes) times step^2, and the rounding
        # of the losses, 40 rows of LP each, over the step
        tol = 40 * 2 * step ** 2 + 40 * 3 * LP / step
        assert abs(((total[0] - total[1]) / (2 * step) - (g * d.double()).sum()).item()) < tol


class Preference:
    def __init__(self, pairs, T, V, Vp, dt, dev, seed=0, masked=0.4, ref=True, beta=0.1, smooth=0.0, dscale=0.7):
        import llmk
        self.pairs, self.T, self.V, self.Vp, self.dt = pairs, T, V, Vp, dt
        self.beta, self.smooth, self.dscale = beta, smooth, dscale
        rows = 2 * pairs * T
        self.x, self.t, g = make_logits(rows, V, Vp, dt, seed, dev)
        self.w = torch.rand(rows, generator=g, device=dev) + 0.5
        if masked:
            self.w[torch.rand(rows, generator=g, device=dev) < masked] = 0.0
        _, lp = logps_of(self.x, self.t, V)
        L = (lp * self.w.double()).view(2 * pairs, T).sum(-1)
        self.ref = (L + torch.randn(2 * pairs, generator=g, device=dev) * 5).float() if ref else None
        mk = lambda *s, d=torch.float32: torch.full(s, 7.0, device=dev, dtype=d)  # noqa: E731
        self.losses, self.rewards, self.logps, self.dx = mk(pairs), mk(2 * pairs), mk(rows), mk(rows, Vp, d=dt)
        self.ws = torch.empty(llmk.preference_loss_workspace(pairs, T, Vp), dtype=torch.uint8, device=dev)

    def call(self, **kw):
        import llmk
        a = dict(V=self.V, weights=self.w, ref_logps=self.ref, rewards=self.rewards, logps=self.logps, dlogits=self.dx,
                 beta=self.beta, label_smoothing=self.smooth, dscale=self.dscale, workspace=self.ws)
        a.update(kw)
        llmk.preference_loss(self.losses, a.pop("logits", self.x), self.t, **a)

    def check(self, dx=None):
        w = torch.ones(self.x.shape[0], device=self.x.device) if self.w is None else self.w
        live = w != 0
        p, lp = logps_of(self.x, self.t, self.V)
        w, n = w.double(), self.pairs
        lp = torch.where(live, lp, torch.zeros_like(lp))
        within(self.logps, lp, torch.where(live, LP + U * lp.abs(), torch.zeros_like(lp)), "logps")
        beta, sm, ds = (float(np.float32(v)) for v in (self.beta, self.smooth, self.dscale))
        L = (w * lp).view(2 * n, -1).sum(-1)
        Lerr = beta * (LP * w.abs()).view(2 * n, -1).sum(-1)
        r = beta * (L - (self.ref.double() if self.ref is not None else 0.0))
        within(self.rewards, r, Lerr + U * r.abs() + TINY, "rewards")
        h, herr = r[:n] - r[n:], Lerr[:n] + Lerr[n:]
        f = torch.nn.functional.logsigmoid
        loss = -(1 - sm) * f(h) - sm * f(-h)
        within(self.losses, loss, herr + U * loss.abs() + TINY, "losses")  # |dloss/dh| <= 1
        slope = beta * ds * (sm * torch.sigmoid(h) - (1 - sm) * torch.sigmoid(-h))
        c = torch.stack([slope, -slope])[:, :, None].expand(2, n, self.T).reshape(-1) * w
        cerr = (beta * ds * herr / 4).repeat(2)[:, None].expand(2 * n, self.T).reshape(-1) * w.abs() + 2 * U * c.abs()
        dx = self.dx if dx is None else dx
        check_dlogits(dx, p, self.t, c, cerr, live, self.V, self.dt)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1, 1, 8), (1, 1, 9, 16), (2, 3, 1001, 1008), (5, 33, 4097, 4104), (1, 1025, 520, 520),
                                   (3, 40, 50257, 50304), (2, 1, 131072, 131080), (300, 2, 700, 704)])
def test_preference_loss(cuda_dev, shape, dt):
    p = Preference(*shape, dt, cuda_dev, seed=sum(shape))
    p.call()
    p.check()


@pytest.mark.parametrize("kw", [dict(ref=False, beta=0.01), dict(smooth=0.2), dict(smooth=1.0), dict(masked=0.0), dict(beta=2.0)])
def test_preference_loss_forms(cuda_dev, kw):
    p = Preference(7, 20, 1001, 1008, torch.float32, cuda_dev, seed=3, **kw)
    p.call()
    p.check()


def test_preference_loss_without_weights_in_place_and_without_gradient(cuda_dev):
    p = Preference(4, 50, 2000, 2048, torch.bfloat16, cuda_dev, seed=4, masked=0.0)
    p.w = None
    p.ref = None
    p.beta = 0.01
    p.call()
    p.check()
    first, buf = p.dx.clone(), p.x.clone()
    p.call(logits=buf, dlogits=buf)
    assert torch.equal(buf, first)
    for v in (p.losses, p.rewards, p.logps):
        v.fill_(7.0)
    keep = p.dx.fill_(3.0)
    p.call(dlogits=None)
    assert (keep == 3.0).all()
    p.check(dx=first)


def test_preference_loss_masks(cuda_dev):
    """A sequence without live rows, a pair without any, masked rows that hold NaN, and a NaN that stays in its pair."""
    p = Preference(4, 30, 1000, 1000, torch.float32, cuda_dev, seed=5, masked=0.3)
    w = p.w.view(8, 30)
    w[0] = 0  # the preferred sequence of pair 0
    w[1], w[5] = 0, 0  # pair 1
    dead = p.w == 0
    p.x[dead], p.t[dead] = math.nan, -100
    p.call()
    losses, dx = p.losses.clone(), p.dx.clone()
    assert torch.isfinite(losses).all() and (dx[dead] == 0).all() and (p.logps[dead] == 0).all()
    p.x[dead], p.t[dead] = 0.0, 0
    p.check()
    row = int((p.w.view(8, 30)[2] != 0).nonzero()[0]) + 60  # pair 2
    p.t[row] = 1000
    p.call()
    assert torch.isnan(p.losses[2]) and torch.equal(p.losses[[0, 1, 3]], losses[[0, 1, 3]])
    bad = torch.zeros(8, 30, dtype=torch.bool, device=cuda_dev)
    bad[2], bad[6] = True, True
    bad = bad.view(-1)
    assert torch.isnan(p.dx[bad & ~dead]).all() and torch.equal(p.dx[~bad], dx[~bad]) and (p.dx[dead] == 0).all()


def test_preference_loss_far_apart(cuda_dev):
    """Rewards far apart: the loss neither overflows nor vanishes where it should not."""
    p = Preference(2, 4, 64, 64, torch.float32, cuda_dev, seed=6, masked=0.0, beta=1.0)
    p.ref[:] = torch.tensor([-3000.0, 3000.0, 3000.0, -3000.0], device=cuda_dev)
    p.call()
    p.check()
    assert p.losses[0] == 0 and p.losses[1] > 5000


@pytest.mark.parametrize("which", ["policy", "preference"])
def test_losses_repeat_bit_for_bit_on_another_stream_and_in_a_graph(cuda_dev, which):
    mk = (lambda s: Policy(333, 5000, 5000, torch.bfloat16, cuda_dev, seed=s)) if which == "policy" else (
        lambda s: Preference(3, 111, 5000, 5000, torch.bfloat16, cuda_dev, seed=s))
    a, b = mk(11), mk(12)
    a.call()
    a.check()
    first = [a.losses.clone(), a.dx.clone()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    a.dx.fill_(1.0)
    torch.cuda.synchronize()
    a.call(stream=s)
    s.synchronize()
    assert torch.equal(a.losses, first[0]) and torch.equal(a.dx, first[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.call()
    for v in ("x", "t", "w", "A", "old", "ref"):
        if hasattr(a, v):
            getattr(a, v).copy_(getattr(b, v))
    for _ in range(2):
        a.dx.fill_(1.0)
        graph.replay()
        torch.cuda.synchronize()
        a.check()
    del graph


@pytest.mark.parametrize("V,Vp", [(101, 104), (50257, 50304), (131072, 131080)])
def test_per_row_outputs_over_inputs(cuda_dev, V, Vp):
    """An output may take the place of an input of its size: every row and pair reads its own before it writes."""
    p = Policy(70, V, Vp, torch.bfloat16, cuda_dev, seed=21)
    p.call()
    want = [t.clone() for t in (p.losses, p.kls, p.logps, p.dx)]
    p.losses, kls, logps = p.w, p.ref, p.old
    p.call(kls=kls, logps=logps)
    assert all(torch.equal(a, b) for a, b in zip(want, (p.losses, kls, logps, p.dx)))
    q = Preference(40, 3, V, Vp, torch.bfloat16, cuda_dev, seed=22)
    q.call()
    want = [t.clone() for t in (q.losses, q.rewards, q.logps, q.dx)]
    rewards, logps = q.ref, q.w
    q.call(rewards=rewards, logps=logps)
    assert all(torch.equal(a, b) for a, b in zip(want, (q.losses, rewards, logps, q.dx)))


def test_two_graphs_share_a_workspace(cuda_dev):
    a, b = Policy(50, 3001, 3008, torch.float32, cuda_dev, seed=13), Preference(2, 20, 3001, 3008, torch.float32, cuda_dev, seed=14)
    ws = a.ws if a.ws.numel() > b.ws.numel() else b.ws
    a.ws = b.ws = ws
    a.call(), b.call()
    torch.cuda.synchronize()
    graphs = []
    for p in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            p.call()
        graphs.append(g)
    for g in graphs + graphs[::-1]:
        g.replay()
    torch.cuda.synchronize()
    a.check(), b.check()
    del graphs


# ------------------------------------------------------ norm, clip, AdamW
# A norm's sum of squares: at most 40 fp32 roundings before the 64-bit sums (a
# thread's 34 terms), half of which reach the square root, and one at the end.
NORM = 22 * U


def norm_workspace(tl, dev):
    import llmk
    return torch.empty(llmk.grad_norm_workspace(tl), dtype=torch.uint8, device=dev)


def norm64(tensors):
    return math.sqrt(sum(float(t.double().square().sum()) for t in tensors))


def pieces(sizes, dt, dev, seed, scale=0.1, offset=0):
    """Tensors one behind another in one buffer, so most start off the 16-byte grid."""
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    flat = (torch.randn(sum(sizes) + offset, generator=g, device=dev) * scale).to(dt)
    return list(flat[offset:].split(sizes))


SIZES = [[1], [7], [8], [0, 5, 0], [4096], [8191, 1, 8193], [3, 100000, 17, 0, 1, 65536, 12345], [1] * 300, [13] * 1001 + [40000]]


@pytest.mark.parametrize("dt,out", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                    (torch.bfloat16, torch.float32), (torch.float16, torch.float32)])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{sum(s)}")
def test_clip_grad_norm(cuda_dev, sizes, dt, out):
    import llmk
    for offset, scale, max_norm in ((0, 1.0, 0.5), (3, 1e-4, 1e6)):  # clipped; left as it is
        ts = pieces(sizes, dt, cuda_dev, len(sizes), scale, offset)
        want = norm64(ts)
        outs = [torch.full_like(t, 9.0, dtype=out) for t in ts]
        tl, norm = llmk.TensorList(ts, outs), torch.zeros(1, device=cuda_dev)
        ws = norm_workspace(tl, cuda_dev)
        llmk.grad_norm(norm, tl, scale=-2.0, workspace=ws)
        assert abs(norm.item() - 2 * want) <= 2 * want * NORM + TINY
        llmk.clip_grad_norm(norm, tl, max_norm, workspace=ws)
        assert abs(norm.item() - want) <= want * NORM + TINY
        k = min(1.0, max_norm / (want + 1e-6))
        for t, o in zip(ts, outs):
            w = t.double() * k
            tiny = {torch.float32: TINY, torch.bfloat16: TINY, torch.float16: 2.0 ** -25}[out]  # half of the least step
            within(o, w, w.abs() * (NORM + 4 * U + HALF[out]) + tiny, "clipped")
        llmk.clip_grad_norm(norm, llmk.TensorList(ts), max_norm, workspace=ws)  # in place
        if dt is out:
            assert all(torch.equal(t, o) for t, o in zip(ts, outs))


def test_clip_mixed_types_and_untouched_neighbours(cuda_dev):
    import llmk
    flat = torch.full((1000,), 5.0, device=cuda_dev)
    a, b = flat[1:500], torch.randn(333, device=cuda_dev).bfloat16()[1:]
    c = torch.randn(77, device=cuda_dev).half()
    out_b = torch.full((340,), 5.0, device=cuda_dev)
    ts, outs = [a, b, c], [a, out_b[2:334], c]
    want = norm64(ts)
    ref = [t.double() / (want + 1e-6) for t in ts]
    tl, norm = llmk.TensorList(ts, outs), torch.zeros(1, device=cuda_dev)
    llmk.clip_grad_norm(norm, tl, 1.0, workspace=norm_workspace(tl, cuda_dev))
    for o, w in zip(outs, ref):
        within(o, w, w.abs() * (NORM + 4 * U + HALF[o.dtype]) + 2.0 ** -25, "mixed")
    assert flat[0] == 5 and (flat[500:] == 5).all() and (out_b[:2] == 5).all() and (out_b[334:] == 5).all()


@pytest.mark.parametrize("value", [0.0, 1e-30, 1e-42, 1e25, 3e38])
def test_norm_range(cuda_dev, value):
    """Squares that leave the range of fp32."""
    import llmk
    x = torch.full((20001,), value, device=cuda_dev)
    x[::2] *= 0.5
    tl, norm = llmk.TensorList([x[1:]]), torch.full((1,), 9.0, device=cuda_dev)
    llmk.grad_norm(norm, tl, workspace=norm_workspace(tl, cuda_dev))
    want = norm64([x[1:]])
    if want > torch.finfo(torch.float32).max:
        assert norm.item() == math.inf
    else:
        assert abs(norm.item() - want) <= want * NORM + 2.0 ** -149


def test_norm_of_nothing(cuda_dev):
    import llmk
    t = (llmk.Tensor * 2)(llmk.Tensor(None, None, 0, 0, 0), llmk.Tensor(None, None, 0, 1, 1))
    norm, ws = torch.full((1,), 9.0, device=cuda_dev), torch.empty(1 << 16, dtype=torch.uint8, device=cuda_dev)
    for name, x in (("llmk_grad_norm", 1.0), ("llmk_clip_grad_norm", 2.0)):
        norm.fill_(9.0)
        llmk.call(name, norm.data_ptr(), t, 2, x, ws.data_ptr(), ws.numel(), llmk.stream_ptr())
        assert norm.item() == 0.0


def test_clip_many_units(cuda_dev):
    """Enough elements for a block per unit: odd sizes, an empty tensor, a start off the 16-byte grid."""
    import llmk
    ts = pieces([9_000_001, 0, 7, 8_191_999, 3], torch.float32, cuda_dev, 5, 1.0, 1)
    outs = [torch.full_like(t, 9.0) for t in ts]
    tl, norm = llmk.TensorList(ts, outs), torch.zeros(1, device=cuda_dev)
    llmk.clip_grad_norm(norm, tl, 1.0, workspace=norm_workspace(tl, cuda_dev))
    want = norm64(ts)
    assert abs(norm.item() - want) <= want * NORM
    for t, o in zip(ts, outs):
        w = t.double() / (want + 1e-6)
        within(o, w, w.abs() * (NORM + 5 * U) + TINY, "clipped")


def test_norm_not_finite(cuda_dev):
    import llmk
    for bad in (math.nan, math.inf, -math.inf):
        x = torch.ones(5000, device=cuda_dev)
        x[4321] = bad
        tl, norm = llmk.TensorList([x]), torch.zeros(1, device=cuda_dev)
        llmk.clip_grad_norm(norm, tl, 1.0, workspace=norm_workspace(tl, cuda_dev))
        if math.isnan(bad):
            assert torch.isnan(norm).all() and torch.isnan(x).all()
        else:
            assert norm.item() == math.inf and torch.isnan(x[4321]) and (x[:4321] == 0).all()


def test_clip_repeats_bit_for_bit_and_in_a_graph(cuda_dev):
    import llmk
    ts = pieces([100003, 5, 70000, 1 << 20], torch.float32, cuda_dev, 3, 1.0, 1)
    outs = [torch.empty_like(t) for t in ts]
    tl, norm = llmk.TensorList(ts, outs), torch.zeros(1, device=cuda_dev)
    ws = norm_workspace(tl, cuda_dev)
    call = lambda: llmk.clip_grad_norm(norm, tl, 1.0, workspace=ws)  # noqa: E731
    call()
    first = [norm.clone()] + [o.clone() for o in outs]
    for _ in range(3):
        call()
        assert all(torch.equal(a, b) for a, b in zip(first, [norm] + outs))
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        call()
    for t in ts:
        t.mul_(2.0)
    ws.fill_(255)  # nothing may be left in the workspace from one call for the next
    g.replay()
    torch.cuda.synchronize()
    assert norm.item() == 2 * first[0].item()
    del g


@pytest.mark.parametrize("n", [4, 1000, 40004, 1 << 20])
@pytest.mark.parametrize("scale", [1e-6, 10.0])
def test_adamw_clipped(cuda_dev, n, scale):
    """Against the formula in 64 bits, and against llmk_adamw on the gradients that llmk_clip_grad_norm writes."""
    import ctypes
    import llmk
    g = torch.Generator(device=cuda_dev)
    g.manual_seed(n)
    r = lambda s: torch.randn(n, generator=g, device=cuda_dev) * s  # noqa: E731
    p, grad, m, v = r(0.1), r(scale), r(scale * 0.1), r(scale).square()
    lr, b1, b2, eps, wd, t, gs = 1e-3, 0.9, 0.99, 1e-8, 0.1, 7, 0.5
    hp = (ctypes.c_float * 8)()
    llmk.lib().llmk_adamw_hparams(hp, lr, b1, b2, eps, wd, t, gs)
    h = torch.tensor(list(hp), device=cuda_dev)
    tl, norm = llmk.TensorList([grad]), torch.zeros(1, device=cuda_dev)
    llmk.grad_norm(norm, tl, scale=gs, workspace=norm_workspace(tl, cuda_dev))
    want = norm64([grad]) * gs
    assert abs(norm.item() - want) <= want * NORM
    lr, b1, b2, eps, wd, c1, c2, gs = h.double().tolist()
    G = grad.double() * gs * min(1.0, 1.0 / (want + 1e-6))
    M, V = b1 * m.double() + (1 - b1) * G, b2 * v.double() + (1 - b2) * G * G
    # the clipped gradient is off by the norm's error and 6 roundings; m and v add 3 roundings of each term
    R = NORM + 6 * U
    Merr = (R + 3 * U) * (b1 * m.double().abs() + (1 - b1) * G.abs())
    Verr = (2 * R + 4 * U) * V
    P = p.double()
    den = torch.sqrt(V * c2) + eps
    step = lr * (M * c1 / den + wd * P)
    P2 = P - step
    Perr = lr * (Merr * c1 / den + (M * c1 / den).abs() * (Verr / V.clamp(min=1e-60) + 6 * U) + 3 * U * wd * P.abs()) + 3 * U * step.abs() + U * P2.abs()
    pb = torch.empty(n, dtype=torch.bfloat16, device=cuda_dev)
    p1, m1, v1 = p.clone(), m.clone(), v.clone()
    llmk.adamw_clipped(p1, grad, m1, v1, h, norm, 1.0, params_bf16=pb)
    within(m1, M, Merr + U * M.abs() + TINY, "m")
    within(v1, V, Verr + U * V + TINY, "v")
    within(p1, P2, Perr + TINY, "p")
    assert torch.equal(pb, p1.bfloat16())
    p2, m2, v2 = p.clone(), m.clone(), v.clone()
    llmk.adamw_clipped(p2, grad, m2, v2, h, norm, math.inf)  # no clipping: llmk_adamw's own bits
    p3, m3, v3 = p.clone(), m.clone(), v.clone()
    llmk.call("llmk_adamw_device_hparams", p3.data_ptr(), None, grad.data_ptr(), m3.data_ptr(), v3.data_ptr(), n,
              h.data_ptr(), llmk.stream_ptr())
    assert torch.equal(p2, p3) and torch.equal(m2, m3) and torch.equal(v2, v3)


def test_wrappers_refuse_wrong_tensors(cuda_dev):
    import llmk
    p = Policy(4, 10, 16, torch.float32, cuda_dev)
    for kw in (dict(weights=p.w[:3]), dict(old_logps=p.old.double()), dict(dlogits=p.dx.bfloat16()), dict(logps=p.w.cpu()),
               dict(logits=p.x.t())):
        with pytest.raises((TypeError, ValueError)):
            p.call(**kw)
    q = Preference(2, 3, 10, 16, torch.float32, cuda_dev)
    for kw in (dict(ref_logps=q.ref[:3]), dict(rewards=q.losses), dict(logits=q.x[:11])):
        with pytest.raises((TypeError, ValueError)):
            q.call(**kw)
    for c in (p, q):  # a workspace that the GPU cannot reach, or does not own whole
        for ws in (c.ws.cpu(), c.ws.repeat(2)[::2]):
            with pytest.raises(ValueError):
                c.call(workspace=ws)
    tl, norm = llmk.TensorList([p.w]), torch.zeros(1, device=cuda_dev)
    for call in (lambda ws: llmk.grad_norm(norm, tl, workspace=ws), lambda ws: llmk.clip_grad_norm(norm, tl, 1.0, workspace=ws)):
        with pytest.raises(ValueError):
            call(norm_workspace(tl, "cpu"))
    with pytest.raises(llmk.LlmkError):
        p.call(logits=p.x[:, :0], dlogits=None, V=None)  # no vocabulary
    with pytest.raises(llmk.LlmkError) as e:
        p.call(workspace=p.ws[:16])
    assert e.value.code == 5
