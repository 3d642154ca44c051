"""agrad_topk_distill_forward / _backward / _fused against the float64 form, through the C ABI.  The bounds are derived in
tests/logits_ops.py and below."""
import ctypes as C

import numpy as np
import pytest

from autograd_amd import capi
from oracle import closed_form as cf
from tests import logits_ops as L
from tests.logits_ops import U

pytestmark = pytest.mark.gpu


def parts(x, ids, values, scale, teacher_scale, tail):
    """per row: sizes of what the loss adds up, and per element the sizes of what the gradient adds up"""
    p, logp, lse = cf._softmax_rows(cf.f64(x) * float(np.float32(scale)))
    rows, V = p.shape
    size, q_at, rest = np.ones(rows), np.zeros((rows, V)), np.zeros((rows, V))
    for r in range(rows):
        used = ids[r] >= 0
        if not used.any() or np.isneginf(lse[r]):
            continue
        u = cf.f64(values[r, used]) * (1.0 if tail else teacher_scale)
        log_q = u if tail else cf._softmax_rows(u[None])[1][0]
        q = np.exp(log_q)
        lp = logp[r, ids[r, used]]
        fine = (q > 0) & np.isfinite(lp)
        size[r] += np.abs(u[np.isfinite(u)]).max(initial=0.0) + (q[fine] * (np.abs(log_q[fine]) + np.abs(lp[fine]))).sum()
        np.add.at(q_at[r], ids[r, used], q)
        if tail:
            out = np.ones(V, bool)
            out[ids[r, used]] = False
            if out.any() and np.isfinite(logp[r, out]).any():
                m = logp[r, out].max()
                e = np.exp(logp[r, out] - m)
                log_rest = m + np.log(e.sum())
                left = max(1.0 - q.sum(), 1e-9)
                size[r] += np.abs(np.log(left)) + np.abs(log_rest)
                rest[r, out] = e / e.sum()
    return p, logp, lse, size, q_at, rest


def bounds(x, ids, values, scale, teacher_scale, tail, dtype, upstream, want_grad):
    """loss: every term's relative errors, (K + 64) roundings of the teacher's side and sum_error(V) of the student's, on the
    size of the logarithms that are added; a gradient element: the same on p W, q and r (W p_rest - q_rest)"""
    rows, V = x.shape
    K = ids.shape[1]
    p, logp, lse, size, q_at, rest = parts(x, ids, values, scale, teacher_scale, tail)
    z = np.abs(np.where(np.isfinite(x), x, 0.0)).max() * scale
    one = L.sum_error(V) + 2 * U * (K + 64) + 2 * U * 2 * z
    loss = 2 * one * size
    l = np.abs(np.where(p > 0, logp, 0.0))
    per = one + U * (4 * np.abs(np.where(np.isfinite(lse), lse, 0.0))[:, None] + 4 * l + 16)
    grad = np.abs(upstream)[:, None] * scale * (2 * per * (p + q_at + rest)) + 1e-37
    # (q = exp(log q) is off by the error of its argument)
    grad = grad + np.abs(upstream)[:, None] * scale * q_at * 4 * U * size[:, None]
    if dtype == "bf16":
        grad = grad + (np.abs(want_grad) + grad) * 2.0 ** -8
    return loss, grad


def check(ctx, x, ids, values, dtype, scale=1.0, teacher_scale=1.0, tail=False, ld=None, offset=0, what="", fused=True):
    rng = np.random.default_rng(3)
    rows = len(x)
    w = rng.standard_normal(rows).astype(np.float32)
    bits = L.store(x, dtype)
    loss, dz = cf.topk_distill(x, ids, values, scale, teacher_scale, tail)
    want = dz * w.astype(np.float64)[:, None]
    b_loss, b_grad = bounds(x, ids, values, scale, teacher_scale, tail, dtype, w, want)
    kw = dict(scale=scale, teacher_scale=teacher_scale, tail=tail, ld=ld, offset=offset)
    got, stats = L.distill_forward(ctx, bits, ids, values, **kw)
    L.assert_within(got, loss, b_loss, what + " loss")
    dx = L.distill_backward(ctx, bits, ids, values, w, stats, **kw)
    L.assert_within(L.value(dx), want, b_grad, what + " gradient")
    f_loss, f_dx = L.distill_fused(ctx, bits, ids, values, row_scale=w, **kw)
    L.assert_within(f_loss, loss, b_loss, what + " loss of the step")
    L.assert_within(L.value(f_dx), want, b_grad, what + " gradient of the step")
    return got, L.value(dx), f_loss, L.value(f_dx)


SHAPES = [(1, 1, 1), (3, 7, 3), (4, 129, 128), (5, 1000, 20), (6, 4099, 64), (200, 517, 9), (3, 32768, 100), (2, 50257, 32),
          (2, 90000, 16), (1, 128256, 128), (2, 151936, 64)]


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,V,K", SHAPES)
def test_loss_and_gradient(ctx, rows, V, K, dtype, tail):
    rng = np.random.default_rng(rows + V + K)
    x = L.logits(rng, rows, V, dtype)
    ids, values = L.teacher(rng, rows, V, K, tail)
    check(ctx, x, ids, values, dtype, scale=0.8, teacher_scale=1.0 if tail else 0.5, tail=tail)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,V,K", [(70, 40, 33), (70, 257, 64), (70, 600, 65), (9, 1030, 64), (9, 2049, 128), (9, 4100, 7), (9, 8200, 64), (5, 17000, 128)])
def test_short_rows_and_many_slots(ctx, rows, V, K, dtype, tail):
    """every size of a workgroup, with a thread a slot"""
    rng = np.random.default_rng(rows + V + K)
    x = L.logits(rng, rows, V, dtype)
    ids, values = L.teacher(rng, rows, V, K, tail)
    check(ctx, x, ids, values, dtype, scale=1.1, tail=tail)
    check(ctx, x, ids, values, dtype, tail=tail, ld=V + 9, offset=3)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [45001, 60000, 80003, 90001, 162000, 170000])
def test_more_rows_than_are_shared(ctx, V, dtype, tail):
    """a workgroup a row, in registers or read twice; copies of three rows, which have to be copies afterwards where they start
    at the same place within 128 bytes (elsewhere threads take other classes, and the sums other orders)"""
    rng = np.random.default_rng(V)
    x = L.logits(rng, 3, V, dtype)
    ids, values = L.teacher(rng, 3, V, 70, tail)
    ids[0, :2] = [0, V - 1]
    x[2, :V // 2] = -np.inf
    x[2, ids[2]] = 1.0
    bits = L.store(x, dtype)
    loss, dz = cf.topk_distill(x, ids, values, 0.8, tail=tail)
    w = np.array([1.0, -0.5, 2.0], np.float32)
    b_loss, b_grad = bounds(x, ids, values, 0.8, 1.0, tail, dtype, w, dz * w[:, None])
    n = 65
    got, dx = L.distill_fused(ctx, np.tile(bits, (n, 1)), np.tile(ids, (n, 1)), np.tile(values, (n, 1)), scale=0.8, tail=tail,
                              row_scale=np.tile(w, n))
    for r in range(3 * n):
        if r >= 192:
            assert got[r] == got[r - 192] and (dx[r] == dx[r - 192]).all(), r
        else:
            L.assert_within(got[r], loss[r % 3], b_loss[r % 3], f"loss of row {r}")
            L.assert_within(L.value(dx[r]), dz[r % 3] * w[r % 3], b_grad[r % 3], f"gradient of row {r}")
    again, same = L.distill_fused(ctx, np.tile(bits, (n, 1)), np.tile(ids, (n, 1)), np.tile(values, (n, 1)), scale=0.8, tail=tail,
                                  row_scale=np.tile(w, n), in_place=True)
    np.testing.assert_array_equal(again, got)
    np.testing.assert_array_equal(same, dx)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [20, 300, 5003])
def test_classes_that_are_named_many_times(ctx, V, dtype, tail):
    rng = np.random.default_rng(V)
    rows, K = 6, 128
    x = L.logits(rng, rows, V, dtype)
    ids, values = L.teacher(rng, rows, V, K, tail, ragged=False)
    ids[0, :] = 17                                   # one class, 128 times
    ids[1, :] = rng.integers(0, V, K)
    ids[2, :] = rng.integers(0, 10, K)
    ids[3, 64:] = ids[3, :64]
    ids[4, :] = np.where(np.arange(K) % 2, V - 1, 0)
    ids[5, ::3] = -1
    check(ctx, x, ids, values, dtype, tail=tail)
    check(ctx, x, ids, values, dtype, tail=tail, ld=V + 3, offset=1)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V,ld,offset", [(1003, 1003, 1), (1003, 1088, 3), (50257, 50304, 0), (37, 40, 5), (4096, 4100, 7), (16385, 16400, 2)])
def test_strides_and_offsets(ctx, V, ld, offset, dtype, tail):
    rng = np.random.default_rng(V + offset)
    x = L.logits(rng, 5, V, dtype)
    ids, values = L.teacher(rng, 5, V, 12, tail)
    ids[0, :4] = [0, 1, V - 1, V - 2]                # classes before and behind the aligned vectors
    ids[0, 4:] = [v for v in range(2, 10)]
    check(ctx, x, ids, values, dtype, tail=tail, ld=ld, offset=offset)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("V", [60, 5003, 100000])
def test_masks_duplicates_and_rows_without_anything(ctx, V, tail):
    rng = np.random.default_rng(V)
    K = 8
    x = L.logits(rng, 9, V, "f32")
    ids, values = L.teacher(rng, 9, V, K, tail, ragged=False)
    values = values - 1.0 if tail else values        # (room for values that are given twice)
    ids[0, 3] = ids[0, 5]                            # the same class twice
    ids[1, :] = ids[1, 0]
    x[2, :] = -np.inf                                # no class is left
    ids[3, :] = -1                                   # no slot
    x[3, 7] = np.nan                                 # (and what it holds does not matter)
    values[4, 2:5] = -np.inf                         # slots of probability 0
    x[5, ids[5, 0]] = -np.inf                        # mass on a masked class
    keep = np.zeros(V, bool)
    keep[ids[6]] = True
    x[6, ~keep] = -np.inf                            # nothing outside the ids
    x[7, rng.random(V) < 0.5] = -np.inf
    x[7, ids[7]] = 1.0
    x[8, ids[8, 0]] = 200.0                          # the student is sure: what it leaves is below the smallest number
    loss, dx, f_loss, f_dx = check(ctx, np.where(np.isnan(x), 0.0, x), ids, values, "f32", tail=tail)
    for a, g in ((loss, dx), (f_loss, f_dx)):
        assert a[2] == 0 and a[3] == 0 and not g[2].any() and not g[3].any()
        assert a[5] == np.inf and np.isfinite(g[5]).all()
        assert np.isfinite(a[[0, 1, 4, 6, 7, 8]]).all()
    # NaN in a row without slots
    w = np.ones(9, np.float32)
    some, stats = L.distill_forward(ctx, x, ids, values, tail=tail)
    g = L.distill_backward(ctx, x, ids, values, w, stats, tail=tail)
    f_some, f_g = L.distill_fused(ctx, x, ids, values, tail=tail)
    assert some[3] == 0 and not g[3].any() and f_some[3] == 0 and not f_g[3].any()
    if not tail:
        values[4, :] = -np.inf                       # a teacher that says nothing
        none, stats = L.distill_forward(ctx, x, ids, values)
        assert none[4] == 0 and not L.distill_backward(ctx, x, ids, values, w, stats)[4].any()


@pytest.mark.parametrize("tail", [False, True])
def test_nan_and_infinity(ctx, tail):
    V = 3000
    rng = np.random.default_rng(4)
    x = L.logits(rng, 4, V, "f32")
    ids, values = L.teacher(rng, 4, V, 6, tail, ragged=False)
    x[0, (ids[0].max() + 1) % V] = np.nan
    x[1, ids[1, 2]] = np.inf
    values[2, 1] = np.nan
    loss, stats = L.distill_forward(ctx, x, ids, values, tail=tail)
    dx = L.distill_backward(ctx, x, ids, values, np.ones(4, np.float32), stats, tail=tail)
    f_loss, f_dx = L.distill_fused(ctx, x, ids, values, tail=tail)
    for a, g in ((loss, dx), (f_loss, f_dx)):
        assert np.isnan(a[:3]).all() and np.isfinite(a[3]) and np.isfinite(g[3]).all()
        assert np.isnan(g[0]).all() and np.isnan(g[1]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_in_place_accumulate_and_scales(ctx, dtype):
    for V in (519, 20000, 100000):
        rng = np.random.default_rng(V)
        rows = 4
        x = L.logits(rng, rows, V, dtype)
        bits = L.store(x, dtype)
        for tail in (False, True):
            ids, values = L.teacher(rng, rows, V, 17, tail)
            w = rng.standard_normal(rows).astype(np.float32)
            loss, dx = L.distill_fused(ctx, bits, ids, values, tail=tail, row_scale=w)
            again, same = L.distill_fused(ctx, bits, ids, values, tail=tail, row_scale=w, in_place=True)
            np.testing.assert_array_equal(same, dx)
            np.testing.assert_array_equal(again, loss)
            _, flat = L.distill_fused(ctx, bits, ids, values, tail=tail, grad_scale=0.25, want_loss=False)
            _, ones = L.distill_fused(ctx, bits, ids, values, tail=tail)
            np.testing.assert_array_equal(L.value(flat), L.value(ones) * 0.25)     # (a power of two: exact)
            _, stats = L.distill_forward(ctx, bits, ids, values, tail=tail)
            dx = L.distill_backward(ctx, bits, ids, values, w, stats, tail=tail)
            same = L.distill_backward(ctx, bits, ids, values, w, stats, tail=tail, in_place=True)
            np.testing.assert_array_equal(same, dx)
            base = L.rounded(rng.standard_normal((rows, V)), dtype)
            acc = L.distill_backward(ctx, bits, ids, values, w, stats, tail=tail, flags=capi.ACC_INPUT_GRAD, init=L.store(base, dtype))
            want = base + cf.topk_distill(x, ids, values, tail=tail)[1] * w.astype(np.float64)[:, None]
            _, bound = bounds(x, ids, values, 1.0, 1.0, tail, dtype, w, want)
            L.assert_within(L.value(acc), want, bound + 4 * U * np.abs(want) + (2.0 ** -8 * np.abs(want) if dtype == "bf16" else 0.0), "accumulated")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [300, 5003, 70000])
def test_tail_far_below_the_ids(ctx, V, dtype):
    """what the student gives to all other classes is below the smallest number: masks of the lowest value, large offsets"""
    rng = np.random.default_rng(V)
    rows, K, far = 6, 70, float(np.finfo(np.float32).min) if dtype == "f32" else -3.3895313892515355e38
    x = L.logits(rng, rows, V, dtype)
    ids, values = L.teacher(rng, rows, V, K, True, ragged=False)
    values = (values - 0.5).astype(np.float32)
    ids[1, 3] = ids[1, 66]
    out = np.ones((rows, V), bool)
    for r in range(rows):
        out[r, ids[r]] = False
    x[0, out[0]] = far
    for r, by in ((1, 60000.0), (2, 150.0), (3, 101.0), (4, 90.0)):
        x[r, out[r]] -= by
    x[5, out[5]] = np.where(np.arange(out[5].sum()) % 2, far, far / 2)
    x = L.rounded(x, dtype)
    w = np.array([1, -0.5, 2, 1, 0.25, -1], np.float32)
    for scale in (1.0, 0.75):
        loss, dz = cf.topk_distill(x, ids, values, scale, tail=True)
        p, logp, lse, size, q_at, rest = parts(x, ids, values, scale, 1.0, True)
        want = dz * w[:, None]
        # Distances are taken from the largest of their own kind, so that l is what an exponential's argument is off by in units of U;
        # log p_rest enters it where it is above -100 (4 roundings); q = exp(u) is off by |u| U.
        with np.errstate(divide="ignore"):
            l = np.where(out, np.abs(np.where(rest > 0, np.log(np.where(rest > 0, rest, 1.0)), 0.0)), np.abs(np.where(p > 0, logp, 0.0)))
        per = L.sum_error(V) + 2 * U * (K + 64) + U * (4 * l + 16 + 400)
        u_max = np.abs(values).max()
        bound = np.abs(w)[:, None] * scale * 2 * (per + 2 * U * u_max) * (p + q_at + rest) + 1e-37
        if dtype == "bf16":
            bound = bound + (np.abs(want) + bound) * 2.0 ** -8
        bits = L.store(x, dtype)
        got, stats = L.distill_forward(ctx, bits, ids, values, scale=scale, tail=True)
        # (its terms are as large as the largest, with relative errors as above and of q_rest, a difference from 1)
        b_loss = 2 * (L.sum_error(V) + 2 * U * (K + 64)) * size / np.minimum(1.0, 1.0 - q_at.sum(1))
        L.assert_within(got, loss, b_loss, "loss")
        dx = L.distill_backward(ctx, bits, ids, values, w, stats, scale=scale, tail=True)
        f_loss, f_dx = L.distill_fused(ctx, bits, ids, values, scale=scale, tail=True, row_scale=w)
        L.assert_within(f_loss, loss, b_loss, "loss of the step")
        rel_q = (2 * U * (K + 64) / (1.0 - q_at.sum(1)))[:, None] * np.abs(w)[:, None] * scale * (rest + p)      # (q_rest is a difference)
        L.assert_within(L.value(f_dx), want, bound + rel_q, f"gradient of the step, scale {scale}")
        L.assert_within(L.value(dx), want, bound + rel_q, f"gradient, scale {scale}")


def test_gradient_against_differences(ctx):
    rng = np.random.default_rng(5)
    rows, V, K, step = 3, 60, 5, 1e-5
    x = rng.standard_normal((rows, V)).astype(np.float32)
    for tail in (False, True):
        ids, values = L.teacher(rng, rows, V, K, tail, ragged=False)
        kw = dict(scale=0.8, teacher_scale=1.0 if tail else 1.5, tail=tail)
        _, dx = L.distill_fused(ctx, x, ids, values, **kw)
        for r in range(rows):
            for v in list(ids[r, :2]) + [0, 31, 59]:
                hi, lo = cf.f64(x).copy(), cf.f64(x).copy()
                hi[r, v] += step
                lo[r, v] -= step
                want = (cf.topk_distill(hi, ids, values, **kw)[0] - cf.topk_distill(lo, ids, values, **kw)[0])[r] / (2 * step)
                assert abs(dx[r, v] - want) <= 1e-5, (tail, r, v)     # (fp32 arithmetic on terms below 1)


def test_rows_far_apart(ctx):
    """row offsets past 32 bits"""
    rng = np.random.default_rng(6)
    rows, V, ld, K = 3, 1200, 2_200_000_000, 7
    x = L.logits(rng, rows, V, "bf16")
    bits = L.store(x, "bf16")
    ids, values = L.teacher(rng, rows, V, K, True)
    loss_want, dz = cf.topk_distill(x, ids, values, tail=True)
    w = np.ones(rows, np.float32)
    b_loss, b_grad = bounds(x, ids, values, 1.0, 1.0, True, "bf16", w, dz)
    buf, grad = ctx.alloc((2 * ld + V) * 2), ctx.alloc((2 * ld + V) * 2)
    with L.Device(ctx) as dev:
        for r in range(rows):
            ctx.call("agrad_copy_from_host", buf, r * ld * 2, bits[r].ctypes.data_as(C.c_void_p), V * 2)
        i, v, g, loss, stats = dev.up(ids), dev.up(values), dev.up(w), dev.up(w), dev.up(np.zeros((rows, 4), np.float32))
        for fused in (False, True):
            if fused:
                ctx.call("agrad_topk_distill_fused", capi.BF16, C.c_void_p(buf), L.p(i), L.p(v), L.p(loss), None, C.c_void_p(grad),
                         rows, V, ld, K, 1.0, 1.0, 1.0, 1)
            else:
                ctx.call("agrad_topk_distill_forward", capi.BF16, C.c_void_p(buf), L.p(i), L.p(v), L.p(loss), L.p(stats), rows, V, ld, K,
                         1.0, 1.0, 1)
                ctx.call("agrad_topk_distill_backward", capi.BF16, C.c_void_p(buf), L.p(i), L.p(v), L.p(g), L.p(stats), C.c_void_p(grad),
                         rows, V, ld, K, 1.0, 1.0, 1, 0)
            ctx.synchronize()
            L.assert_within(loss.download(), loss_want, b_loss, "loss")
            row = np.empty(V, np.uint16)
            for r in range(rows):
                ctx.call("agrad_copy_to_host", grad, r * ld * 2, row.ctypes.data_as(C.c_void_p), V * 2)
                L.assert_within(L.value(row), dz[r], b_grad[r], f"row {r}")
    ctx.free(buf)
    ctx.free(grad)


def test_ids_out_of_range(ctx):
    x = np.random.default_rng(7).standard_normal((2, 50)).astype(np.float32)
    ids, values = np.array([[3, 50, 5], [-2, 7, 9]], np.int32), np.zeros((2, 3), np.float32)
    safe = np.where((ids < 0) | (ids >= 50), -1, ids).astype(np.int32)
    want, stats = L.distill_forward(ctx, x, safe, values)
    with L.Device(ctx) as dev:
        d_x, i, v, loss, st, dx = dev.up(x), dev.up(ids), dev.up(values), dev.up(np.zeros(2, np.float32)), dev.up(stats), dev.up(x)
        for _ in range(2):
            ctx.call("agrad_topk_distill_forward", capi.F32, L.p(d_x), L.p(i), L.p(v), L.p(loss), None, 2, 50, 50, 3, 1.0, 1.0, 0)
            with pytest.raises(IndexError):
                ctx.synchronize()
            np.testing.assert_array_equal(loss.download(), want)
        ctx.call("agrad_topk_distill_backward", capi.F32, L.p(d_x), L.p(i), L.p(v), L.p(loss), L.p(st), L.p(dx), 2, 50, 50, 3, 1.0, 1.0, 0, 0)
        with pytest.raises(IndexError):
            ctx.synchronize()
        ctx.call("agrad_topk_distill_fused", capi.F32, L.p(d_x), L.p(i), L.p(v), None, None, L.p(dx), 2, 50, 50, 3, 1.0, 1.0, 1.0, 0)
        with pytest.raises(IndexError):
            ctx.synchronize()


def test_refusals_and_no_rows(ctx):
    with L.Device(ctx) as dev:
        x, i, o = dev.up(np.zeros(64, np.float32)), dev.up(np.zeros(256, np.int32)), dev.up(np.zeros(256, np.float32))
        fwd = dict(dtype=capi.F32, x=L.p(x), ids=L.p(i), values=L.p(o), loss=L.p(o), stats=L.p(o), rows=2, V=8, ld=8, top=2, scale=1.0,
                   teacher=1.0, mode=0)
        bwd = dict(dtype=capi.F32, x=L.p(x), ids=L.p(i), values=L.p(o), dloss=L.p(o), stats=L.p(o), dx=L.p(x), rows=2, V=8, ld=8, top=2,
                   scale=1.0, teacher=1.0, mode=0, flags=0)
        fused = dict(dtype=capi.F32, x=L.p(x), ids=L.p(i), values=L.p(o), loss=L.p(o), w=None, dx=L.p(x), rows=2, V=8, ld=8, top=2,
                     scale=1.0, teacher=1.0, grad_scale=1.0, mode=0)
        both = [dict(dtype=5), dict(x=None), dict(ids=None), dict(values=None), dict(top=0), dict(top=129), dict(ld=7), dict(V=0),
                dict(scale=0.0), dict(scale=float("nan")), dict(teacher=0.0), dict(teacher=float("inf")), dict(mode=2), dict(mode=-1),
                dict(mode=1, teacher=0.5), dict(x=C.c_void_p(x.ptr + 1)), dict(rows=1 << 22)]
        for name, good, own in (("forward", fwd, [dict(loss=None)]),
                                ("backward", bwd, [dict(dloss=None), dict(stats=None), dict(dx=None), dict(flags=2)]),
                                ("fused", fused, [dict(dx=None), dict(dx=C.c_void_p(x.ptr + 2))])):
            for over in both + own:
                with pytest.raises(capi.AgradError) as e:
                    ctx.call("agrad_topk_distill_" + name, *{**good, **over}.values())
                assert e.value.code == capi.EINVAL, (name, over)
            none = {k: (None if isinstance(v, C.c_void_p) else v) for k, v in good.items()}
            ctx.call("agrad_topk_distill_" + name, *{**none, "rows": 0}.values())
    ctx.synchronize()


def three_ways(ctx, bits, ids, values, w, **kw):
    """(name, loss, gradient) of forward and backward, of the step, and of a backward call that accumulates"""
    loss, stats = L.distill_forward(ctx, bits, ids, values, **kw)
    yield "two calls", loss, L.value(L.distill_backward(ctx, bits, ids, values, w, stats, **kw))
    f_loss, f_dx = L.distill_fused(ctx, bits, ids, values, row_scale=w, **kw)
    yield "step", f_loss, L.value(f_dx)
    acc = L.distill_backward(ctx, bits, ids, values, w, stats, flags=capi.ACC_INPUT_GRAD, init=np.zeros_like(bits), **kw)
    yield "accumulated", loss, L.value(acc)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V,copies", [(20, 1), (300, 1), (5003, 1), (90000, 1), (90000, 8)])
def test_rows_with_nan_or_infinity_are_nan(ctx, V, copies, dtype, tail):
    """loss and whole gradient, also where no class of the row is a number; what is left of other rows is as it was"""
    rng = np.random.default_rng(V)
    rows, K = 12, 6
    x = L.logits(rng, rows, V, dtype)
    ids, values = L.teacher(rng, rows, V, K, tail, ragged=False)
    other = [next(v for v in range(V // 2, V) if v not in ids[r]) for r in range(rows)]
    x[0, :] = np.nan
    x[1, :] = -np.inf
    x[1, other[1]] = np.nan
    x[2, :] = -np.inf
    x[2, ids[2, 0]] = np.nan
    x[3, :] = -np.inf
    x[3, other[3]] = np.inf
    x[4, ids[4, 3]] = np.nan
    x[5, other[5]] = np.nan
    values[6, 1] = np.nan
    values[7, 2] = np.inf
    for r, low in ((8, -200.0), (9, -np.inf)):           # the teacher's NaN where the student gives next to nothing, or nothing, to the rest
        out = np.ones(V, bool)
        out[ids[r]] = False
        x[r, out] = low
        values[r, 0] = np.nan
    bad = np.arange(rows) < 10
    bits, at = L.store(x, dtype), np.tile(np.arange(rows), copies)
    w = np.where(np.arange(rows) % 2, -0.5, 2.0).astype(np.float32)
    ok = ~bad
    want_loss, dz = cf.topk_distill(x[ok], ids[ok], values[ok], tail=tail)
    want = dz * w[ok, None]
    b_loss, b_grad = bounds(x[ok], ids[ok], values[ok], 1.0, 1.0, tail, dtype, w[ok], want)
    for name, loss, dx in three_ways(ctx, bits[at], ids[at], values[at], w[at], tail=tail):
        for r in np.flatnonzero(bad[at]):
            assert np.isnan(loss[r]) and np.isnan(dx[r]).all(), (name, at[r], loss[r], np.isnan(dx[r]).mean())
        for r in np.flatnonzero(ok[at]):
            i = at[r] - 10
            L.assert_within(loss[r], want_loss[i], b_loss[i], f"{name}: loss of row {r}")
            L.assert_within(dx[r], want[i], b_grad[i], f"{name}: gradient of row {r}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V,copies", [(300, 1), (5003, 1), (60000, 1), (60000, 10)])
def test_teachers_far_from_zero(ctx, V, copies, dtype):
    """Renormalised values with a common offset, of which q is free.  Their distances to the largest are exact (numbers of one
    size) and take at most two roundings more with the scale, so that the bound is that of values without the offset."""
    rng = np.random.default_rng(V)
    rows, K, low = 8, 64, np.finfo(np.float32).min
    x = L.logits(rng, rows, V, dtype)
    ids, values = L.teacher(rng, rows, V, K, False)
    values[0] += np.float32(1e6)
    values[1] -= np.float32(1e6)
    values[2] = 1e6                                  # all equal: q = 1 / 64
    values[3] = low
    values[4] = -low
    values[5, 1:] = low                              # one class and a mask of the lowest value
    values[6] += np.float32(300.0)
    values[7] = np.where(np.arange(K) % 2, low, -np.inf)
    bits, at = L.store(x, dtype), np.tile(np.arange(rows), copies)
    w = np.where(np.arange(rows) % 2, -0.5, 2.0).astype(np.float32)
    for teacher_scale in (1.0, 0.5, 1.75):
        loss_want, dz = cf.topk_distill(x, ids, values, 0.8, teacher_scale)
        want = dz * w[:, None]
        top = np.where(ids >= 0, values, -np.inf).max(1, keepdims=True).astype(np.float64)
        about = np.where(np.isfinite(values), values - top, -np.inf)
        about = np.where(about < -1e30, -np.inf, about)                    # (q = 0)
        b_loss, b_grad = bounds(x, ids, about, 0.8, teacher_scale, False, dtype, w, want)
        for name, loss, dx in three_ways(ctx, bits[at], ids[at], values[at], w[at], scale=0.8, teacher_scale=teacher_scale):
            L.assert_within(loss, loss_want[at], b_loss[at], f"{name}: loss, {teacher_scale}")
            L.assert_within(dx, want[at], b_grad[at], f"{name}: gradient, {teacher_scale}")


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V,copies", [(20, 1), (300, 1), (5003, 1), (60000, 1), (60000, 40)])
def test_masked_ids_among_classes_at_the_lowest_value(ctx, V, copies, dtype, tail):
    """mass on classes at -inf alone: the loss is +inf, whatever the others' offset times the scale is; the gradient is that of
    equal classes (p = 1 / n, a sum of ones: exact but for sum_error and a few roundings)"""
    rng = np.random.default_rng(V)
    rows, K = 2, 5
    low = float(np.finfo(np.float32).min) if dtype == "f32" else -3.3895313892515355e38
    ids, values = L.teacher(rng, rows, V, K, tail, ragged=False)
    x = np.full((rows, V), low, np.float32)
    np.put_along_axis(x, ids, -np.inf, 1)
    at = np.tile(np.arange(rows), copies)
    w = np.array([1.0, -0.5], np.float32)
    for scale in (1.0, 1.5):
        loss_want, dz = cf.topk_distill(x, ids, values, scale, tail=tail)
        assert np.isposinf(loss_want).all()
        want = dz * w[:, None]
        # W <= 1 plus roundings; among the others p W - r q_rest, r = p: terms of 1 / n
        bound = scale * np.abs(w)[:, None] * (L.sum_error(V) + 2 * U * (K + 64)) * np.where(np.isneginf(x), 1.0, 2.0 / (V - K))
        bound = bound + (2.0 ** -8 * (np.abs(want) + bound) if dtype == "bf16" else 0.0)
        for name, loss, dx in three_ways(ctx, L.store(x, dtype)[at], ids[at], values[at], w[at], scale=scale, tail=tail):
            assert np.isposinf(loss).all(), (name, scale, loss)
            L.assert_within(dx, want[at], bound[at], f"{name}: gradient, scale {scale}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [capi.MAX_TAIL_CLASSES, capi.MAX_TAIL_CLASSES - 1, 163840, 163841, 2 * 163840 + 3])
def test_most_classes_with_a_tail(ctx, V, dtype):
    """rows in as many parts as their bit maps need; the largest fill every part's map"""
    rng = np.random.default_rng(V)
    rows = 2 if V > 1000000 else 3
    x = L.logits(rng, rows, V, dtype)
    ids, values = L.teacher(rng, rows, V, 40, True)
    ids[0, :4] = [0, 1, V - 2, V - 1]                # (the first and the last bits)
    ids[1, :6] = [v for k in (1, 2, 4) for v in (k * (V // 8), k * (V // 8) + 1)]
    check(ctx, x, ids, values, dtype, tail=True)
    if V < 1000000:
        n = 12
        check(ctx, np.tile(x, (n, 1)), np.tile(ids, (n, 1)), np.tile(values, (n, 1)), dtype, tail=True, ld=V + 3, offset=1)


@pytest.mark.parametrize("V", [163840, 163847])
def test_loss_of_many_rows_as_long_as_a_bit_map(ctx, V):
    """a workgroup a row, or two where its bits are one map more"""
    rng = np.random.default_rng(V)
    rows, n = 3, 344
    x = L.logits(rng, rows, V, "bf16")
    ids, values = L.teacher(rng, rows, V, 40, True)
    ids[0, :4] = [0, 1, V - 2, V - 1]
    want, dz = cf.topk_distill(x, ids, values, tail=True)
    bound, _ = bounds(x, ids, values, 1.0, 1.0, True, "bf16", np.ones(rows), dz)
    got, _ = L.distill_forward(ctx, np.tile(L.store(x, "bf16"), (n, 1)), np.tile(ids, (n, 1)), np.tile(values, (n, 1)), tail=True)
    L.assert_within(got, np.tile(want, n), np.tile(bound, n), "loss")


def test_more_classes_than_a_tail_takes_are_refused(ctx):
    V = capi.MAX_TAIL_CLASSES + 1
    with L.Device(ctx) as dev:
        x, dx = dev.up(np.zeros(V, np.float32)), dev.up(np.zeros(V, np.float32))
        i, o = dev.up(np.zeros(2, np.int32)), dev.up(np.zeros(16, np.float32))
        for dtype in (capi.F32, capi.BF16):
            for name, args in (("forward", (L.p(o), L.p(o), 1, V, V, 2, 1.0, 1.0, 1)), ("backward", (L.p(o), L.p(o), L.p(dx), 1, V, V, 2, 1.0, 1.0, 1, 0)),
                               ("fused", (L.p(o), None, L.p(dx), 1, V, V, 2, 1.0, 1.0, 1.0, 1))):
                with pytest.raises(capi.AgradError) as e:
                    ctx.call("agrad_topk_distill_" + name, dtype, L.p(x), L.p(i), L.p(o), *args)
                assert e.value.code == capi.EINVAL, name
        assert not dx.download().any()
    ctx.synchronize()
