"""Token log probabilities and top-k distillation without a GPU: the float64 forms against other routes to the same numbers,
the ops' shapes and refusals, and a graph of both on the oracle device."""
import numpy as np
import pytest
from scipy.special import log_softmax

from autograd_amd import capi
from autograd_amd.op import MAX_TOP, TokenLogprobsOp, TopKDistillOp
from autograd_amd.optimizer import AdamW
from autograd_amd.runtime import Runtime
from autograd_amd.tensor import Tensor
from autograd_amd.utils import BF16
from oracle import closed_form as cf
from oracle import cpu_device

cpu_device.register()


def T(shape, dtype=np.float32, grad=True, val=None):
    return Tensor(shape=shape, dtype=dtype, device="cpu", requires_grad=grad, init_val=val)


# ---- the float64 forms ---------------------------------------------------------------------------
def test_token_logprobs_form():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((4, 31))
    x[1, rng.random(31) < 0.5] = -np.inf
    x[1, 3] = 0.5
    t = np.array([0, 3, 30, -1])
    logp, ent, lse, ids, top = cf.token_logprobs(x, t, 0.5, 31)
    want = log_softmax(0.5 * x, axis=-1)
    np.testing.assert_allclose(logp[:3], want[np.arange(3), t[:3]], rtol=1e-13)
    assert logp[3] == 0
    p = np.exp(want)
    np.testing.assert_allclose(ent, -(p * np.where(p > 0, want, 0)).sum(-1), rtol=1e-12)
    np.testing.assert_allclose(np.exp(0.5 * x - lse[:, None]).sum(-1), 1, rtol=1e-13)
    for r in range(4):
        n = np.isfinite(x[r]).sum()
        assert (np.diff(x[r, ids[r, :n]]) <= 0).all() and (ids[r, n:] == -1).all()
    equal = cf.token_logprobs(np.zeros((1, 9)), [2], 1.0, 9)
    np.testing.assert_array_equal(equal[3][0], np.arange(9))
    np.testing.assert_allclose([equal[0][0], equal[1][0]], [-np.log(9), np.log(9)], rtol=1e-14)


@pytest.mark.parametrize("tail", [False, True])
def test_gradients_of_the_forms_against_differences(tail):
    rng = np.random.default_rng(1)
    rows, V, K, step = 4, 23, 6, 1e-5
    x = rng.standard_normal((rows, V))
    x[1, 5] = -np.inf
    t = np.array([1, 2, 22, -1])
    g, h = rng.standard_normal(rows), rng.standard_normal(rows)
    ids = np.stack([rng.choice(V, K, replace=False) for _ in range(rows)])
    ids[0, 2], ids[2, 1], ids[3] = -1, ids[2, 4], [0, 1, 2, 3, 4, 6]
    ids[1] = np.where(ids[1] == 5, 7, ids[1])
    u = rng.standard_normal((rows, K + 1))
    u = (u - np.log(np.exp(u).sum(-1, keepdims=True)))[:, :K] - (0.5 if tail else 0.0)
    kw = dict(scale=0.75, teacher_scale=1.0 if tail else 1.5, tail=tail)

    def total(y):
        logp, ent, *_ = cf.token_logprobs(y, t, 0.75)
        return (g * logp + h * ent).sum(), (g * cf.topk_distill(y, ids, u, **kw)[0]).sum()

    got = cf.token_logprobs_grad(x, t, g, h, 0.75), cf.topk_distill(x, ids, u, **kw)[1] * g[:, None]
    for r in range(rows):
        for v in range(V):
            if not np.isfinite(x[r, v]):
                assert got[0][r, v] == 0 and got[1][r, v] == 0
                continue
            hi, lo = x.copy(), x.copy()
            hi[r, v] += step
            lo[r, v] -= step
            for k, (a, b) in enumerate(zip(total(hi), total(lo))):
                assert abs((a - b) / (2 * step) - got[k][r, v]) <= 1e-8, (k, r, v)


def test_distill_form_is_cross_entropy_at_its_ends():
    """one sure class: the cross-entropy; all classes, renormalised or with an empty tail: the whole divergence"""
    rng = np.random.default_rng(2)
    x, t = rng.standard_normal((3, 11)), np.array([[4], [0], [10]])
    loss, grad = cf.topk_distill(x, t, np.zeros((3, 1)), tail=False)
    np.testing.assert_allclose(loss, cf.cross_entropy(x, t[:, 0]), rtol=1e-13)
    np.testing.assert_allclose(grad, cf.cross_entropy_grad(x, t[:, 0], np.ones(3)), atol=1e-14)
    ids = np.tile(rng.permutation(11), (3, 1))
    u = log_softmax(rng.standard_normal((3, 11)), axis=-1)
    want = (np.exp(u) * (u - np.take_along_axis(log_softmax(x, axis=-1), ids, 1))).sum(-1)
    for tail in (False, True):
        np.testing.assert_allclose(cf.topk_distill(x, ids, u, tail=tail)[0], want, rtol=1e-12)
    # a teacher that is the student: nothing to learn
    logp, _, _, ids, top = cf.token_logprobs(x, t[:, 0], 1.0, 4)
    loss, grad = cf.topk_distill(x, ids, top, tail=True)
    assert np.abs(loss).max() < 1e-14 and np.abs(grad).max() < 1e-15


def test_distill_form_of_a_student_at_a_masks_lowest_value():
    """a gradient's row adds up to 0, whatever the offset between the ids and the other classes"""
    x = np.full((2, 40), float(np.finfo(np.float32).min))
    x[:, :5] = np.arange(5)
    x[1, 20:] /= 2
    loss, grad = cf.topk_distill(x, np.tile(np.arange(5), (2, 1)), np.full((2, 5), np.log(0.15)), tail=True)
    np.testing.assert_allclose(grad.sum(-1), 0, atol=1e-12)
    np.testing.assert_allclose(grad[0, 5:], -0.25 / 35, rtol=1e-12)
    np.testing.assert_allclose(grad[1, 20:], -0.25 / 20, rtol=1e-12)
    assert not grad[1, 5:20].any()


# ---- ops -----------------------------------------------------------------------------------------
def test_ops_refuse_what_the_kernels_do_not_take():
    assert MAX_TOP == capi.MAX_TOP
    x, t = T((2, 3, 9)), T((2, 3), np.int32, False)
    for bad in (dict(top=-1), dict(top=MAX_TOP + 1), dict(scale=0.0), dict(scale=-1), dict(scale=float("nan")), dict(scale=float("inf"))):
        with pytest.raises(ValueError):
            x.token_logprobs(t, **bad)
    for tokens in (T((2, 2), np.int32, False), T((2, 3), np.float32, False), T((2, 3), BF16, False), T((2, 3), np.int64, False)):
        with pytest.raises(ValueError):
            x.token_logprobs(tokens)
    with pytest.raises(RuntimeError):
        x.transpose(0, 1).token_logprobs(T((3, 2), np.int32, False))
    ids, u = T((2, 3, 4), np.int32, False), T((2, 3, 4), np.float32, False)
    for bad in (dict(scale=0), dict(teacher_scale=-1), dict(tail=True, teacher_scale=0.5)):
        with pytest.raises(ValueError):
            x.distill_topk(ids, u, **bad)
    for i, v in ((T((2, 3, 5), np.int32, False), u), (T((2, 2, 4), np.int32, False), T((2, 2, 4), np.float32, False)),
                 (T((2, 3, 4), np.int64, False), u), (ids, T((2, 3, 4), BF16, False)), (ids, T((2, 3, 4))),
                 (T((2, 3, 0), np.int32, False), T((2, 3, 0), np.float32, False)),
                 (T((2, 3, 129), np.int32, False), T((2, 3, 129), np.float32, False))):
        with pytest.raises(ValueError):
            x.distill_topk(i, v)


def test_ops_give_what_was_asked_for():
    x, t = T((2, 3, 9)), T((2, 3), np.int32, False)
    r = x.token_logprobs(t)
    assert r.logp.shape == (2, 3) and r.entropy is None and r.top_ids is None and r.top_logp is None
    assert isinstance(r.logp.op.op, TokenLogprobsOp) and len(r.logp.op.outputs) == 2
    r = x.token_logprobs(t, top=4, entropy=True)
    assert r.top_ids.shape == (2, 3, 4) and np.dtype(r.top_ids.dtype) == np.int32 and not r.top_logp.requires_grad
    assert r.entropy.requires_grad and r.logp.op.op.split(r.logp.op.outputs)[2:] == (r.entropy, r.top_ids, r.top_logp)
    loss = x.distill_topk(r.top_ids, r.top_logp, tail=True)
    assert loss.shape == (2, 3) and isinstance(loss.op.op, TopKDistillOp)


def test_a_student_learns_its_teachers_alternatives_on_the_oracle_device():
    """teacher logits -> alternatives -> the student's loss, in one graph; the student's table is what a step changes"""
    rng = np.random.default_rng(3)
    B, N, V, K = 2, 4, 17, 5
    teacher = T((B, N, V), grad=False, val=(2 * rng.standard_normal((B, N, V))).astype(np.float32))
    tokens = T((B, N), np.int32, False, rng.integers(0, V, (B, N)).astype(np.int32))
    ids = T((B, N), np.int32, False, rng.integers(0, 6, (B, N)).astype(np.int32))
    table = T((6, V), val=(0.1 * rng.standard_normal((6, V))).astype(np.float32))
    said = teacher.token_logprobs(tokens, top=K)
    loss = ids.gather(table).distill_topk(said.top_ids, said.top_logp, tail=True)
    rt = Runtime(device="cpu")
    rt.loss = loss
    rt.build_topo(loss)
    rt.bind_memory()
    rt.is_compiled = True
    opt = AdamW([table], lr=1e-2, runtime=rt)
    before = None
    for _ in range(2):
        rt.backward(loss, grad_scale=1.0 / (B * N))
        value, grad = rt.backend.copy_to_host(loss).copy(), rt.backend.copy_to_host(table.grad).copy()
        x = rt.backend.copy_to_host(table)[ids.storage.data.reshape(-1)]
        flat = teacher.storage.data.reshape(-1, V)
        _, _, _, top_ids, top = cf.token_logprobs(flat, tokens.storage.data.reshape(-1), 1.0, K)
        want, dz = cf.topk_distill(x, top_ids, top.astype(np.float32), tail=True)
        np.testing.assert_allclose(value.reshape(-1), want, rtol=1e-5, atol=1e-6)
        dw = np.zeros((6, V))
        np.add.at(dw, ids.storage.data.reshape(-1), dz / (B * N))
        np.testing.assert_allclose(grad, dw, rtol=1e-5, atol=1e-6)
        assert before is None or not np.array_equal(value, before)
        before = value
        opt.step()


def test_a_tail_takes_so_many_classes():
    from autograd_amd.op import MAX_TAIL_CLASSES
    assert MAX_TAIL_CLASSES == capi.MAX_TAIL_CLASSES
    ids, u = T((1, 2), np.int32, False), T((1, 2), np.float32, False)
    x, long = (T((1, MAX_TAIL_CLASSES + more), grad=False) for more in (0, 1))
    assert x.distill_topk(ids, u, tail=True).shape == (1,) and long.distill_topk(ids, u).shape == (1,)
    with pytest.raises(ValueError):
        long.distill_topk(ids, u, tail=True)


def test_ops_refuse_scales_that_a_call_would_refuse():
    x, t = T((2, 9)), T((2,), np.int32, False)
    ids, u = T((2, 4), np.int32, False), T((2, 4), np.float32, False)
    for bad in (1e-46, 2.1e38, 1e39):
        for make in (lambda: x.token_logprobs(t, scale=bad), lambda: x.distill_topk(ids, u, scale=bad), lambda: x.distill_topk(ids, u, teacher_scale=bad)):
            with pytest.raises(ValueError):
                make()
    for good in (1e-45, 2e38):
        x.token_logprobs(t, scale=good), x.distill_topk(ids, u, scale=good, teacher_scale=good)
