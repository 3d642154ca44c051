"""Token log probabilities and top-k distillation through Runtime(device="hip"), beside the oracle device, recorded into
graphs and from two contexts at once."""
import ctypes as C
import threading

import numpy as np
import pytest

from autograd_amd import capi
from autograd_amd.optimizer import AdamW
from autograd_amd.runtime import Runtime
from autograd_amd.tensor import Tensor
from autograd_amd.utils import BF16
from oracle import closed_form as cf
from oracle import cpu_device
from tests import logits_ops as L

pytestmark = pytest.mark.gpu
cpu_device.register()


def leaf(device, shape, dtype, grad, val):
    return Tensor(shape=shape, dtype=dtype, device=device, requires_grad=grad, init_val=val)


def compiled(device, loss, **kw):
    rt = Runtime(device=device, **kw)
    rt.loss = loss
    rt.build_topo(loss)
    rt.bind_memory()
    rt.is_compiled = True
    return rt


def test_policy_gradient_graph():
    """loss = logp * advantage + entropy * bonus, where both come from one node; against the oracle device"""
    rng = np.random.default_rng(1)
    B, N, V = 3, 5, 301
    x_np = (2 * rng.standard_normal((B, N, V))).astype(np.float32)
    t_np = rng.integers(0, V, (B, N)).astype(np.int32)
    t_np[0, 0] = -1
    adv, bonus = rng.standard_normal((B, N)).astype(np.float32), np.full((B, N), 0.05, np.float32)
    got = {}
    for device in ("cpu", "hip"):
        for fuse in (True, False):
            x, t = leaf(device, x_np.shape, np.float32, True, x_np), leaf(device, t_np.shape, np.int32, False, t_np)
            a, b = leaf(device, adv.shape, np.float32, False, adv), leaf(device, adv.shape, np.float32, False, bonus)
            r = x.token_logprobs(t, entropy=True, scale=0.8)
            loss = r.logp * a + r.entropy * b
            rt = compiled(device, loss, fuse_grad_zeroing=fuse)
            rt.backward(loss)
            got[device, fuse] = rt.backend.copy_to_host(loss).copy(), rt.backend.copy_to_host(x.grad).copy()
            rt.release()
    want = cf.token_logprobs_grad(x_np.reshape(-1, V), t_np.reshape(-1), adv.reshape(-1), bonus.reshape(-1), 0.8).reshape(x_np.shape)
    for key, (value, grad) in got.items():
        # kernel bounds: 2e-5 of values up to 8 in the loss; p (|g| + |h| (|log p| + entropy)) <= 4 with 1e-5 in the gradient
        np.testing.assert_allclose(value, got["cpu", True][0], rtol=0, atol=2e-5, err_msg=str(key))
        np.testing.assert_allclose(grad, want, rtol=1e-5, atol=1e-5, err_msg=str(key))


def test_alternatives_alone_leave_a_zero_gradient():
    """logits that need a gradient but whose node gives none: the first writer writes zeros"""
    rng = np.random.default_rng(2)
    x_np = rng.standard_normal((1, 4, 50)).astype(np.float32)
    x = leaf("hip", x_np.shape, np.float32, True, x_np)
    t = leaf("hip", (1, 4), np.int32, False, np.zeros((1, 4), np.int32))
    s_np = rng.standard_normal((1, 4, 50)).astype(np.float32)
    s = leaf("hip", s_np.shape, np.float32, True, s_np)
    r = x.token_logprobs(t, top=3)
    loss = s.distill_topk(r.top_ids, r.top_logp, tail=True)
    rt = compiled("hip", loss)
    rt.backend.copy_from_host(x.grad, np.full_like(x_np, 5.0))
    rt.backward(loss)
    assert not rt.backend.copy_to_host(x.grad).any()
    ids, top = cf.token_logprobs(x_np[0], np.zeros(4, int), 1.0, 3)[3:]
    want = cf.topk_distill(s_np[0], ids, top.astype(np.float32), tail=True)[1]
    np.testing.assert_allclose(rt.backend.copy_to_host(s.grad)[0], want, rtol=1e-5, atol=1e-5)
    rt.release()


def distillation(device, dtype, seed=3, B=4, N=16, V=500, K=12):
    """an embedding student -> norm -> logits table, its teacher's logits as an input; returns what a step needs"""
    rng = np.random.default_rng(seed)
    cast = (lambda a: L.rounded(a, "bf16")) if dtype == BF16 else (lambda a: a.astype(np.float32))
    table = leaf(device, (40, V), dtype, True, cast(0.5 * rng.standard_normal((40, V))))
    gamma = leaf(device, (V,), np.float32, True, np.ones(V, np.float32))
    ids = leaf(device, (B, N), np.int32, False, np.zeros((B, N), np.int32))
    teacher = leaf(device, (B, N, V), dtype, False, cast(rng.standard_normal((B, N, V))))
    tokens = leaf(device, (B, N), np.int32, False, np.zeros((B, N), np.int32))
    said = teacher.token_logprobs(tokens, top=K, entropy=True, scale=0.9)
    loss = ids.gather(table).rms_norm(gamma).distill_topk(said.top_ids, said.top_logp, tail=True, scale=1.1)
    return compiled(device, loss), loss, (ids, tokens, teacher), (table, gamma)


def batch(rng, V, cast):
    return (rng.integers(0, 40, (4, 16)).astype(np.int32), rng.integers(0, V, (4, 16)).astype(np.int32),
            cast(2 * rng.standard_normal((4, 16, V))))


@pytest.mark.parametrize("dtype", [np.float32, BF16])
def test_teacher_and_student_train_together_on_both_devices(dtype):
    """Four optimizer steps of teacher -> alternatives -> student loss -> gradient -> AdamW on "hip" and on the oracle device.
    Every step starts from the oracle's parameters, so that each comparison is of one step."""
    cast = (lambda a: L.rounded(a, "bf16")) if dtype == BF16 else (lambda a: a.astype(np.float32))
    steps = {}
    for device in ("cpu", "hip"):
        steps[device] = distillation(device, dtype)
    rng = np.random.default_rng(4)
    opts = {d: AdamW([s[3][1]], lr=1e-2, runtime=s[0]) for d, s in steps.items()}
    for step in range(4):
        data = batch(rng, 500, cast)
        out = {}
        for device, (rt, loss, feeds, params) in steps.items():
            for t, v in zip(feeds, data):
                rt.backend.copy_from_host(t, v)
            if device == "hip":
                for mine, theirs in zip(params, steps["cpu"][3]):
                    rt.backend.copy_from_host(mine, before[id(theirs)])
            before = {id(p): rt.backend.copy_to_host(p).copy() for p in params} if device == "cpu" else before
            rt.backward(loss, grad_scale=1.0 / 64)
            out[device] = [rt.backend.copy_to_host(loss).copy()] + [rt.backend.copy_to_host(p.grad).copy() for p in params]
            opts[device].step()
            out[device].append(rt.backend.copy_to_host(params[1]).copy())
        a, b = out["hip"], out["cpu"]
        if dtype == BF16:
            # The student's logits are rounded to bf16 on both devices from fp32 values that differ by 1e-6: where that falls on
            # two sides of a rounding, a logit of size <= 8 differs by a step, 2^-5, in rare places; p <= 1 of it reaches the loss.
            np.testing.assert_allclose(a[0], b[0], rtol=0, atol=2 ** -5)
            scale = np.abs(b[1]).max()
            assert np.abs(a[1] - b[1]).max() <= 4 * 2 ** -8 * scale + 2 ** -5 * scale     # (three roundings on the way, and that step)
        else:
            np.testing.assert_allclose(a[0], b[0], rtol=1e-5, atol=5e-5)     # sum_error(500) on logarithms up to 12
            for g, w in zip(a[1:3], b[1:3]):
                assert np.abs(g - w).max() <= 5e-5 * max(1e-3, np.abs(w).max())
        assert np.isfinite(a[3]).all() and not np.array_equal(a[3], before[id(steps["cpu"][3][1])])
    for rt, *_ in steps.values():
        if rt.allocator.device == "hip":
            rt.release()


def test_recorded_step_replays_like_the_eager_one():
    """the whole step in a graph, replayed with other data and eager work of the same leaves between the replays"""
    rt, loss, feeds, params = distillation("hip", np.float32)
    rng = np.random.default_rng(5)
    datas = [batch(rng, 500, lambda a: a.astype(np.float32)) for _ in range(4)]

    def feed(d):
        for t, v in zip(feeds, d):
            rt.backend.copy_from_host(t, v)

    def results():
        rt.backend.synchronize()
        return [rt.backend.copy_to_host(t).copy() for t in [loss] + [p.grad for p in params]]

    eager = []
    for d in datas:
        feed(d)
        rt.backward(loss)
        eager.append(results())
    feed(datas[0])
    g = rt.capture(rt.execute)
    # (the table's gradient is cleared by the rows of the pass before: every replay follows another replay)
    feed(datas[3])
    rt.backend.fill(params[0].grad, 0)
    for again in range(2):
        for d, want in zip(datas, eager):
            feed(d)
            rt.backend.fill(params[0].grad, 0)
            g.launch()
            for a, b in zip(results(), want):
                np.testing.assert_array_equal(a, b)
    g.destroy()
    rt.release()


def single_rows(ctx, seed):
    """what two graphs of one context share is its own scratch: a few long rows of both operators"""
    rng = np.random.default_rng(seed)
    x = L.store(L.logits(rng, 2, 60000, "bf16"), "bf16")
    t = rng.integers(0, 60000, 2).astype(np.int32)
    ids, u = L.teacher(rng, 2, 60000, 9, True)
    return x, t, ids, u


def enqueue(ctx, dev, data):
    x, t, ids, u = data
    rows, V = x.shape
    d = dict(x=dev.up(x), t=dev.up(t), i=dev.up(ids), u=dev.up(u), logp=dev.up(np.zeros(rows, np.float32)), ent=dev.up(np.zeros(rows, np.float32)),
             top=dev.up(np.zeros((rows, 7), np.int32)), tl=dev.up(np.zeros((rows, 7), np.float32)), loss=dev.up(np.zeros(rows, np.float32)),
             dx=dev.up(np.zeros_like(x)))

    def launch():
        ctx.call("agrad_token_logprobs_forward", capi.BF16, L.p(d["x"]), L.p(d["t"]), L.p(d["logp"]), L.p(d["ent"]), None, L.p(d["top"]),
                 L.p(d["tl"]), rows, V, V, 7, 1.0)
        ctx.call("agrad_topk_distill_fused", capi.BF16, L.p(d["x"]), L.p(d["i"]), L.p(d["u"]), L.p(d["loss"]), None, L.p(d["dx"]), rows, V, V,
                 9, 1.0, 1.0, 1.0, 1)

    def results():
        ctx.synchronize()
        return {k: d[k].download() for k in ("logp", "ent", "top", "tl", "loss", "dx")}

    return launch, results


def test_two_recorded_graphs_and_eager_calls_in_turn(ctx):
    with L.Device(ctx) as dev:
        calls = [enqueue(ctx, dev, single_rows(ctx, s)) for s in (1, 2, 3)]
        want = []
        for launch, results in calls:
            launch()
            want.append(results())
        graphs = []
        for launch, _ in calls[:2]:
            ctx.call("agrad_graph_begin")
            launch()
            g = C.c_uint64()
            ctx.call("agrad_graph_end", C.byref(g))
            graphs.append(g.value)
        for _ in range(4):
            ctx.call("agrad_graph_launch", graphs[0])
            calls[2][0]()
            ctx.call("agrad_graph_launch", graphs[1])
            ctx.call("agrad_graph_launch", graphs[0])
            for (_, results), w in zip(calls, want):
                for k, v in results().items():
                    np.testing.assert_array_equal(v, w[k], err_msg=k)
        for g in graphs:
            ctx.call("agrad_graph_destroy", g)


def test_two_contexts_at_once(ctx):
    """calls of two contexts run on two streams: neither reads what the other leaves in its scratch"""
    other = capi.Context(0)
    try:
        data = [single_rows(ctx, s) for s in (11, 12)]
        with L.Device(ctx) as a, L.Device(other) as b:
            calls = [enqueue(ctx, a, data[0]), enqueue(other, b, data[1])]
            want = []
            for launch, results in calls:
                launch()
                want.append(results())
            errors = []

            def work(c, w):
                try:
                    for _ in range(30):
                        c[0]()
                    for k, v in c[1]().items():
                        np.testing.assert_array_equal(v, w[k], err_msg=k)
                except Exception as e:      # noqa: BLE001
                    errors.append(e)

            threads = [threading.Thread(target=work, args=(c, w)) for c, w in zip(calls, want)]
            for t in threads:
                t.start()
            for t in threads:
                t.join()
            assert not errors, errors
    finally:
        other.close()


def test_buffers_of_another_context_or_too_small_are_refused():
    from autograd_amd import hip_ext
    one, two = hip_ext.HipContext(0), hip_ext.HipContext(0)
    x, t, o = one.alloc(4 * 64), one.alloc(4 * 8), one.alloc(4 * 8)
    foreign = two.alloc(4 * 64)
    one.fill_scalar("", [x], [0], 0.0, 64)
    one.fill_scalar("", [t], [0], 0.0, 8)
    offs = [0] * 7

    def call(ids, rows=8, V=8, ld=8, top=0, offs=offs):
        one.token_logprobs_forward(hip_ext.F32, ids, offs, rows, V, ld, top, 1.0)

    call([x, t, o, 0, 0, 0, 0])
    one.synchronize()
    for bad in (dict(ids=[foreign, t, o, 0, 0, 0, 0]), dict(ids=[x, t, o, 0, 0, 0, 0], rows=9), dict(ids=[x, t, o, 0, 0, 0, 0], ld=9),
                dict(ids=[x, t, o, 0, 0, 0, 0], offs=[4] + [0] * 6), dict(ids=[x, t, o]), dict(ids=[0, t, o, 0, 0, 0, 0]),
                dict(ids=[x, t, o, 0, 0, o, o], top=2)):
        with pytest.raises(ValueError):
            call(**bad)
    one.synchronize()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tail", [False, True])
def test_step_by_buffer_ids(ctx, dtype, tail):
    """HipContext.topk_distill_fused: loss and gradient of the C ABI's call, at offsets, in place, without a loss or row scales; operands that
    are not the context's, or too small, are refused before anything is written"""
    from autograd_amd import hip_ext
    rng = np.random.default_rng(21)
    rows, V, ld, K, lead = 6, 1003, 1024, 9, 32
    x = L.store(L.logits(rng, rows, V, dtype), dtype)
    ids, values = L.teacher(rng, rows, V, K, tail)
    w = rng.standard_normal(rows).astype(np.float32)
    kw = dict(scale=0.75, teacher_scale=1.0 if tail else 0.5, tail=tail, ld=ld, offset=lead // x.itemsize)
    want_loss, want = L.distill_fused(ctx, x, ids, values, row_scale=w, **kw)
    _, flat = L.distill_fused(ctx, x, ids, values, grad_scale=-0.25, **kw)
    one, other = hip_ext.HipContext(0), hip_ext.HipContext(0)
    kind, item = (hip_ext.BF16, 2) if dtype == "bf16" else (hip_ext.F32, 4)
    padded = np.full((rows, ld), L.PAD, x.dtype)
    padded[:, :V] = x

    def up(context, a):
        buf = context.alloc(lead + a.nbytes)
        context.copy_from_host(buf, lead, a)
        return buf

    def down(buf, like):
        return one.copy_to_host(buf, lead, list(like.shape), like.dtype.name)

    bx, bi, bv, bw = up(one, padded), up(one, ids), up(one, values), up(one, w)
    loss0, dx0 = np.full(rows, -7.0, np.float32), np.full((rows, ld), 3, x.dtype)
    bl, bd = up(one, loss0), up(one, dx0)
    good = dict(ids=[bx, bi, bv, bl, bw, bd], offs=[lead] * 6, rows=rows, V=V, ld=ld, top=K)

    def call(grad_scale=1.0, **over):
        a = {**good, **over}
        one.topk_distill_fused(kind, a["ids"], a["offs"], a["rows"], a["V"], a["ld"], a["top"], kw["scale"], kw["teacher_scale"], grad_scale, int(tail))

    foreign = up(other, padded)
    for at in range(6):
        for bad in (foreign, 1):
            with pytest.raises(ValueError):
                call(ids=[bad if i == at else b for i, b in enumerate(good["ids"])])
        with pytest.raises(ValueError):
            call(offs=[lead + item * (ld - V) + 4 if i == at else lead for i in range(6)])     # (the last row would end behind its buffer)
    for over in (dict(ids=good["ids"][:5]), dict(offs=[lead] * 5), dict(rows=rows + 1), dict(top=K + 1), dict(ld=ld + 8), dict(ld=V - 1), dict(top=0),
                 dict(ids=[0, bi, bv, bl, bw, bd]), dict(ids=[bx, 0, bv, bl, bw, bd]), dict(ids=[bx, bi, 0, bl, bw, bd]), dict(ids=[bx, bi, bv, bl, bw, 0])):
        with pytest.raises(ValueError):
            call(**over)
    one.synchronize()
    np.testing.assert_array_equal(down(bl, loss0), loss0)
    np.testing.assert_array_equal(down(bd, dx0), dx0)
    np.testing.assert_array_equal(down(bx, padded), padded)

    call()
    one.synchronize()
    np.testing.assert_array_equal(down(bl, loss0), want_loss)
    np.testing.assert_array_equal(down(bd, dx0)[:, :V], want)
    assert (down(bd, dx0)[:, V:] == 3).all()
    call(grad_scale=-0.25, ids=[bx, bi, bv, 0, 0, bx])                 # (no loss, one scale, in place)
    one.synchronize()
    np.testing.assert_array_equal(down(bx, padded)[:, :V], flat)
    np.testing.assert_array_equal(down(bl, loss0), want_loss)


@pytest.mark.parametrize("dtype", [np.float32, BF16])
@pytest.mark.parametrize("order", [(0, 1, 2), (2, 0, 1), (1, 2, 0), (2, 1, 0)])
def test_logits_that_several_operators_read(order, dtype):
    """cross-entropy, distillation and a policy term of the same logits, whichever writes the gradient first and whichever adds to it"""
    U = L.U
    rng = np.random.default_rng(31)
    B, N, V, K = 2, 7, 259, 5
    cast = (lambda a: L.rounded(a, "bf16")) if dtype == BF16 else (lambda a: a.astype(np.float32))
    x_np = cast(2 * rng.standard_normal((B, N, V)))
    t_np = rng.integers(0, V, (B, N)).astype(np.int32)
    ids_np, u_np = L.teacher(rng, B * N, V, K, True)
    adv = rng.standard_normal((B, N)).astype(np.float32)
    x, t = leaf("hip", x_np.shape, dtype, True, x_np), leaf("hip", t_np.shape, np.int32, False, t_np)
    ids, u = leaf("hip", (B, N, K), np.int32, False, ids_np.reshape(B, N, K)), leaf("hip", (B, N, K), np.float32, False, u_np.reshape(B, N, K))
    a = leaf("hip", adv.shape, np.float32, False, adv)

    def policy():
        said = x.token_logprobs(t, entropy=True, top=3, scale=0.8)
        return said.logp * a + said.entropy * a

    terms = [lambda: x.cross_entropy(t), lambda: x.distill_topk(ids, u, tail=True, scale=1.25), policy]
    loss = None
    for i in order:
        term = terms[i]()
        loss = term if loss is None else loss + term
    rt = compiled("hip", loss)
    flat, tf = x_np.reshape(-1, V), t_np.reshape(-1)
    parts = [cf.cross_entropy_grad(flat, tf, np.ones(B * N)), cf.topk_distill(flat, ids_np, u_np, 1.25, tail=True)[1],
             cf.token_logprobs_grad(flat, tf, adv.reshape(-1), adv.reshape(-1), 0.8)]
    want = sum(parts)
    # sizes of what the gradients add up, and relative errors of tests/logits_ops.py (logarithms up to 20 here); bf16: a rounding of each
    # part and of each sum on the way
    p1, p2, (p3, l3, _) = cf._softmax_rows(flat)[0], cf._softmax_rows(1.25 * flat)[0], cf._softmax_rows(0.8 * flat)
    at = (np.arange(V) == tf[:, None]) * 1.0
    q = np.zeros_like(p1)
    for r in range(B * N):
        np.add.at(q[r], ids_np[r][ids_np[r] >= 0], np.exp(u_np[r][ids_np[r] >= 0]))
    rest = np.where(q == 0, p2, 0.0)
    size = p1 + at + 2 * p2 + q + rest / rest.sum(-1, keepdims=True) + np.abs(adv).reshape(-1, 1) * (at + p3 * (1 - l3 - (p3 * l3).sum(-1, keepdims=True)))
    off = L.sum_error(V) + 2 * U * 100
    bound = (8 * off + (4 * 2.0 ** -8 if dtype == BF16 else 0.0)) * size
    # (loss: three logarithms, an entropy of up to log V with an error of 2 + 2 log V such, and terms of the ids)
    b_value = off * (20 + np.abs(adv).reshape(-1) * (3 + 2 * np.log(V)))
    value = (cf.cross_entropy(flat, tf) + cf.topk_distill(flat, ids_np, u_np, 1.25, tail=True)[0]
             + sum(cf.token_logprobs(flat, tf, 0.8)[:2]) * adv.reshape(-1))
    for _ in range(2):
        rt.backward(loss)
        L.assert_within(rt.backend.copy_to_host(x.grad), want.reshape(x_np.shape), bound.reshape(x_np.shape), "gradient")
        L.assert_within(rt.backend.copy_to_host(loss).reshape(-1), value, b_value, "loss")
    rt.release()


def test_two_threads_of_one_context(ctx):
    """the launches of one call follow one another on the stream, whichever thread enqueues in between: a few long rows take two, and the
    second reads what the first left in the context's memory"""
    with L.Device(ctx) as dev:
        calls = [enqueue(ctx, dev, single_rows(ctx, s)) for s in (41, 42, 43)]
        want = []
        for launch, results in calls:
            launch()
            want.append(results())
        errors = []

        def work(launch):
            try:
                for _ in range(200):
                    launch()
            except Exception as e:      # noqa: BLE001
                errors.append(e)

        threads = [threading.Thread(target=work, args=(c[0],)) for c in calls]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not errors, errors
        for (_, results), w in zip(calls, want):
            for k, v in results().items():
                np.testing.assert_array_equal(v, w[k], err_msg=k)


@pytest.mark.parametrize("fuse", [True, False])
@pytest.mark.parametrize("read", ["entropy", "logp"])
def test_outputs_that_nothing_reads(read, fuse):
    """an output with a gradient of its own that no loss comes from adds nothing, whatever its memory held"""
    rng = np.random.default_rng(51)
    B, N, V = 2, 5, 130
    x_np, t_np = rng.standard_normal((B, N, V)).astype(np.float32), rng.integers(0, V, (B, N)).astype(np.int32)
    a_np = rng.standard_normal((B, N)).astype(np.float32)
    x, t, a = leaf("hip", x_np.shape, np.float32, True, x_np), leaf("hip", t_np.shape, np.int32, False, t_np), leaf("hip", a_np.shape, np.float32, False, a_np)
    said = x.token_logprobs(t, entropy=True, top=4)
    loss = getattr(said, read) * a
    rt = compiled("hip", loss, fuse_grad_zeroing=fuse)
    other = said.logp if read == "entropy" else said.entropy
    if other.grad is not None:
        rt.backend.copy_from_host(other.grad, np.full((B, N), 7.0, np.float32))
    g = a_np.reshape(-1)
    want = cf.token_logprobs_grad(x_np.reshape(-1, V), t_np.reshape(-1), g if read == "logp" else None, g if read == "entropy" else None)
    for _ in range(2):
        rt.backward(loss)
        # (as above: p (|g| + |h| (|log p| + entropy)) <= 4, with 1e-5)
        np.testing.assert_allclose(rt.backend.copy_to_host(x.grad).reshape(-1, V), want, rtol=1e-5, atol=1e-5)
    rt.release()
