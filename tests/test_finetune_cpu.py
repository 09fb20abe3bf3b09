"""Refusals of the fine-tuning operators (policy and preference loss, gradient
norm, clipping, clipped AdamW): every bad call is turned down on the host, so
none of these needs a GPU; the addresses passed are never dereferenced."""
import ctypes as C

import pytest

INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 5
A = 1 << 20  # a stand-in for a device address, 16-byte aligned
BIG = 1 << 40


def policy(**kw):
    a = dict(losses=A, kls=None, logps=None, dlogits=A + (1 << 30), logits=A, dtype=1, targets=A, weights=None,
             advantages=A, old=None, ref=None, rows=8, V=100, Vp=104, lo=0.2, hi=0.2, kl=0.0, dscale=1.0, ws=A,
             ws_bytes=BIG, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return tuple(a.values())


def preference(**kw):
    a = dict(losses=A, rewards=None, logps=None, dlogits=A + (1 << 30), logits=A, dtype=1, targets=A, weights=None,
             ref=None, pairs=2, T=4, V=100, Vp=104, beta=0.1, smooth=0.0, dscale=1.0, ws=A, ws_bytes=BIG, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return tuple(a.values())


COMMON = [
    (dict(losses=None), INVALID), (dict(logits=None), INVALID), (dict(targets=None), INVALID),
    (dict(V=0), INVALID), (dict(V=105), INVALID), (dict(Vp=100), UNSUPPORTED),
    (dict(dtype=2), UNSUPPORTED), (dict(dtype=7), UNSUPPORTED),
    (dict(logits=A + 8), UNSUPPORTED), (dict(dlogits=A + (1 << 30) + 2), UNSUPPORTED),
    (dict(dlogits=A + 16), INVALID), (dict(dlogits=A - 16), INVALID),  # overlapping, but not the same buffer
    (dict(ws=None), WORKSPACE), (dict(ws=A + 4), WORKSPACE), (dict(ws_bytes=64), WORKSPACE),
    (dict(dscale=float("inf")), INVALID), (dict(dscale=float("nan")), INVALID),
]


@pytest.mark.parametrize("kw,code", COMMON + [
    (dict(advantages=None), INVALID), (dict(rows=0), INVALID), (dict(rows=-1), INVALID),
    (dict(lo=-0.1), INVALID), (dict(lo=1.5), INVALID), (dict(hi=-0.1), INVALID), (dict(hi=float("nan")), INVALID),
    (dict(hi=float("inf")), INVALID), (dict(kl=0.1), INVALID), (dict(kl=float("nan"), ref=A), INVALID),
    (dict(kls=A), INVALID),  # no reference to estimate from
])
def test_policy_loss_refuses(llmk_lib, kw, code):
    assert llmk_lib.llmk_policy_loss(*policy(**kw)) == code
    assert b"policy_loss" in llmk_lib.llmk_last_error()


@pytest.mark.parametrize("kw,code", COMMON + [
    (dict(pairs=0), INVALID), (dict(T=0), INVALID), (dict(beta=0.0), INVALID), (dict(beta=-1.0), INVALID),
    (dict(beta=float("nan")), INVALID), (dict(smooth=-0.1), INVALID), (dict(smooth=1.1), INVALID),
    (dict(pairs=1 << 20, T=1 << 20), UNSUPPORTED),  # more than 2^31 - 1 rows
])
def test_preference_loss_refuses(llmk_lib, kw, code):
    assert llmk_lib.llmk_preference_loss(*preference(**kw)) == code
    assert b"preference_loss" in llmk_lib.llmk_last_error()


def test_loss_workspaces(llmk_lib):
    L = llmk_lib
    assert L.llmk_policy_loss_workspace(0, 104) == 0 and L.llmk_preference_loss_workspace(1, 0, 104) == 0
    assert L.llmk_policy_loss_workspace(8, 104) > 0
    assert L.llmk_preference_loss_workspace(2, 4, 50304) == L.llmk_policy_loss_workspace(16, 50304)
    need = L.llmk_policy_loss_workspace(8, 104)
    assert L.llmk_policy_loss(*policy(ws_bytes=need - 1)) == WORKSPACE


def tensors(*rows):
    import llmk
    return (llmk.Tensor * len(rows))(*[llmk.Tensor(*r) for r in rows])


F32, BF16, F16 = 0, 1, 2
GOOD = (A, A, 100, F32, F32)
BAD = [
    ([(None, A, 4, F32, F32)], INVALID), ([(A, A, -1, F32, F32)], INVALID), ([(A, A, 4, 7, F32)], UNSUPPORTED),
    ([(A + 2, A + 2, 4, F32, F32)], UNSUPPORTED), ([(A + 1, A + 1, 4, BF16, BF16)], UNSUPPORTED),
    ([(A, A, 1 << 62, F32, F32)], UNSUPPORTED),
]
BAD_OUT = [
    ([(A, None, 4, F32, F32)], INVALID), ([(A, A + 4096, 4, F32, BF16)], UNSUPPORTED),
    ([(A, A + 4096, 4, BF16, F16)], UNSUPPORTED), ([(A, A + 4098, 4, BF16, F32)], UNSUPPORTED),
    ([(A, A, 100, BF16, F32)], INVALID),  # widened in place
    ([(A, A + 8, 100, F32, F32)], INVALID), ([GOOD, GOOD], INVALID),  # the same tensor twice
    ([GOOD, (A + 4096, A + 396, 1, F32, F32)], INVALID),  # written into the last element of another one
    ([(A + 8192, A + 4096, 100, F32, F32), (A + 4000, A + 16384, 100, F32, F32)], INVALID),
]


@pytest.mark.parametrize("rows,code", BAD)
def test_grad_norm_refuses(llmk_lib, rows, code):
    t = tensors(*rows)
    assert llmk_lib.llmk_grad_norm(A, t, len(rows), 1.0, A, BIG, None) == code
    assert llmk_lib.llmk_clip_grad_norm(A, t, len(rows), 1.0, A, BIG, None) == code
    assert b"tensor 0" in llmk_lib.llmk_last_error()


@pytest.mark.parametrize("rows,code", BAD_OUT)
def test_clip_grad_norm_refuses(llmk_lib, rows, code):
    t = tensors(*rows)
    assert llmk_lib.llmk_clip_grad_norm(A, t, len(rows), 1.0, A, BIG, None) == code
    assert b"clip_grad_norm" in llmk_lib.llmk_last_error()


def test_norm_arguments(llmk_lib):
    L, t, nan, inf = llmk_lib, tensors(GOOD), float("nan"), float("inf")
    need = L.llmk_grad_norm_workspace(t, 1)
    assert need > 0 and L.llmk_grad_norm_workspace(None, 1) == 0 and L.llmk_grad_norm_workspace(t, 0) == 0
    for args in ((None, t, 1, 1.0, A, BIG), (A, None, 1, 1.0, A, BIG), (A, t, 0, 1.0, A, BIG), (A, t, 1, nan, A, BIG),
                 (A, t, 1, inf, A, BIG)):
        assert L.llmk_grad_norm(*args, None) == INVALID
    for args in ((None, t, 1, 1.0, A, BIG), (A, t, 1, 0.0, A, BIG), (A, t, 1, -1.0, A, BIG), (A, t, 1, nan, A, BIG)):
        assert L.llmk_clip_grad_norm(*args, None) == INVALID
    for ws, n in ((None, BIG), (A + 8, BIG), (A, need - 1)):
        assert L.llmk_grad_norm(A, t, 1, 1.0, ws, n, None) == WORKSPACE
        assert L.llmk_clip_grad_norm(A, t, 1, 1.0, ws, n, None) == WORKSPACE


def test_adamw_clipped_refuses(llmk_lib):
    f = llmk_lib.llmk_adamw_clipped
    good = [A, None, A, A, A, 8, A, A, 1.0, None]
    for at, value, code in ((0, None, 1), (2, None, 1), (3, None, 1), (4, None, 1), (5, -4, 1), (6, None, 1),
                            (7, None, 1), (8, 0.0, 1), (8, float("nan"), 1), (5, 6, 2), (0, A + 4, 2), (1, A + 8, 2),
                            (6, A + 4, 2)):
        bad = list(good)
        bad[at] = value
        assert f(*bad) == code, (at, value)


def test_wrappers_check_their_tensors(llmk_lib):
    """The Python helpers refuse host tensors, and lists that do not match, before the library sees an address."""
    import llmk
    import torch
    x = torch.zeros(4, 104)
    with pytest.raises(ValueError):
        llmk.policy_loss(torch.zeros(4), x, torch.zeros(4, dtype=torch.int32), torch.zeros(4))
    with pytest.raises(ValueError):
        llmk.preference_loss(torch.zeros(3), x, torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError):
        llmk.TensorList([torch.zeros(4)], [torch.zeros(5)])
    with pytest.raises(ValueError):
        llmk.TensorList([torch.zeros(4, 4).t()])
    assert C.sizeof(llmk.Tensor) == 32


def matmul_policy(**kw):
    a = dict(losses=A, kls=None, logps=None, logits=A, dtype=1, inp=A, W=A, bias=None, targets=A, weights=None,
             advantages=A, old=None, ref=None, BT=8, C=64, Vp=104, V=100, lo=0.2, hi=0.2, kl=0.0, dscale=1.0, backward=1,
             math=1, ws=A, ws_bytes=BIG, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return tuple(a.values())


def matmul_preference(**kw):
    a = dict(losses=A, rewards=None, logps=None, logits=A, dtype=1, inp=A, W=A, bias=None, targets=A, weights=None,
             ref=None, pairs=2, T=4, C=64, Vp=104, V=100, beta=0.1, smooth=0.0, dscale=1.0, backward=1, math=1, ws=A,
             ws_bytes=BIG, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return tuple(a.values())


MATMUL = [(dict(losses=None), INVALID), (dict(targets=None), INVALID), (dict(logits=None), INVALID), (dict(inp=None), INVALID),
          (dict(W=None), INVALID), (dict(C=0), INVALID), (dict(V=105), INVALID), (dict(dtype=2), INVALID),
          (dict(math=3), INVALID), (dict(Vp=102), UNSUPPORTED), (dict(ws=None), WORKSPACE), (dict(ws_bytes=200), WORKSPACE),
          (dict(dscale=float("nan")), INVALID)]


@pytest.mark.parametrize("kw,code", MATMUL + [(dict(BT=0), INVALID), (dict(advantages=None), INVALID), (dict(kl=0.1), INVALID),
                                              (dict(lo=2.0), INVALID)])
def test_matmul_policy_refuses(llmk_lib, kw, code):
    assert llmk_lib.llmk_matmul_policy_forward(*matmul_policy(**kw)) == code
    assert b"matmul_policy" in llmk_lib.llmk_last_error()


@pytest.mark.parametrize("kw,code", MATMUL + [(dict(pairs=0), INVALID), (dict(T=0), INVALID), (dict(beta=0.0), INVALID),
                                              (dict(smooth=2.0), INVALID), (dict(pairs=1 << 20, T=1 << 20), UNSUPPORTED)])
def test_matmul_preference_refuses(llmk_lib, kw, code):
    assert llmk_lib.llmk_matmul_preference_forward(*matmul_preference(**kw)) == code
    assert b"matmul_preference" in llmk_lib.llmk_last_error()


def test_finetune_workspace(llmk_lib):
    L = llmk_lib
    assert L.llmk_matmul_finetune_workspace(0, 104) == 0
    need = L.llmk_matmul_finetune_workspace(8, 104)
    assert need >= L.llmk_matmul_softmax_workspace(8, 104) + 8 * 32
    assert L.llmk_matmul_policy_forward(*matmul_policy(ws_bytes=need - 1)) == WORKSPACE


def test_model_entry_points_refuse(llmk_lib):
    L = llmk_lib
    assert L.llmk_gpt2_logprobs(None, A, A, A) == INVALID
    assert L.llmk_gpt2_forward_policy(None, A, A, None, A, None, None, 0.2, 0.2, 0.0, None, None) == INVALID
    assert L.llmk_gpt2_forward_preference(None, A, A, None, None, 0.1, 0.0, None, None) == INVALID
    assert L.llmk_gpt2_set_grad_clip(None, 1.0) == INVALID
    assert L.llmk_gpt2_grad_norm(None, None) == INVALID
