"""agrad_token_logprobs_forward / _backward against the float64 forms, through the C ABI.  The bounds are derived in
tests/logits_ops.py."""
import ctypes as C

import numpy as np
import pytest

from autograd_amd import capi
from oracle import closed_form as cf
from tests import logits_ops as L
from tests.logits_ops import U

pytestmark = pytest.mark.gpu


def check_forward(got, x, tokens, scale=1.0, top=0, what=""):
    V = x.shape[1]
    logp, entropy, lse, ids, top_logp = cf.token_logprobs(x, tokens if tokens is not None else np.full(len(x), -1), scale, top)
    z = np.abs(np.where(np.isfinite(x), x, 0.0)).max() * scale
    far = L.sum_error(V) + 2 * U * (2 * z + 16)
    with np.errstate(invalid="ignore"):
        if tokens is not None:
            L.assert_within(got["logp"], logp, far, what + " logp")
        if got["lse"] is not None:
            L.assert_within(got["lse"], lse, far, what + " lse")
        if got["entropy"] is not None:
            L.assert_within(got["entropy"], entropy, far * (2 + 2 * np.log(V + 1)), what + " entropy")
        if top:
            np.testing.assert_array_equal(got["top_ids"], ids, err_msg=what)
            L.assert_within(got["top_logp"], top_logp, far, what + " top_logp")


def backward_bound(x, tokens, dlogp, dentropy, scale, dtype, want):
    p, logp, lse = cf._softmax_rows(cf.f64(x) * float(np.float32(scale)))
    l = np.abs(np.where(p > 0, logp, 0.0))
    z = np.abs(np.where(np.isfinite(x), x, 0.0)) * scale
    lse = np.abs(np.where(np.isfinite(lse), lse, 0.0))[:, None]
    h_row = (p * l).sum(-1, keepdims=True)
    g = np.abs(dlogp if dlogp is not None else np.zeros(len(x)))[:, None]
    h = np.abs(dentropy if dentropy is not None else np.zeros(len(x)))[:, None]
    delta = U * (2 * lse + z + 3 * l + 12) + L.sum_error(x.shape[1])
    bound = scale * (p * (g + h * (l + h_row)) * (2 * delta) + 8 * U * g * (np.arange(x.shape[1])[None] == np.asarray(tokens)[:, None]))
    # (the entropy that is handed over is itself off by its own bound)
    bound = bound + scale * p * h * L.sum_error(x.shape[1]) * (2 + 2 * np.log(x.shape[1] + 1)) + 1e-37
    return bound + (np.abs(want) + bound) * 2.0 ** -8 if dtype == "bf16" else bound


SHAPES = [(1, 1), (3, 7), (5, 64), (4, 129), (2, 1000), (6, 4099), (300, 517), (3, 32768), (2, 50257), (1, 128256), (2, 151936)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,V", SHAPES)
def test_forward(ctx, rows, V, dtype):
    rng = np.random.default_rng(1000 + V + rows)
    x = L.logits(rng, rows, V, dtype)
    tokens = rng.integers(0, V, rows).astype(np.int32)
    if rows > 2:
        tokens[1] = -1
    for top, scale in ((0, 1.0), (1, 0.5), (20, 1.25), (128, 1.0)):
        got = L.forward(ctx, L.store(x, dtype), tokens, top, scale)
        check_forward(got, x, tokens, scale, top, f"top {top}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,V", [(70, 40), (70, 257), (70, 600), (9, 1030), (9, 2049), (9, 3001), (9, 7001), (9, 9001), (3, 16003), (3, 30011), (40, 50257)])
def test_forward_of_rows_that_are_kept(ctx, rows, V, dtype):
    """rows and parts of every length that stays in registers, in every size of a workgroup"""
    rng = np.random.default_rng(V + rows)
    few = L.logits(rng, min(rows, 9), V, dtype)
    few[0, rng.random(V) < 0.7] = -np.inf
    few[0, 5] = 1.0
    x, tokens = np.tile(few, (-(-rows // len(few)), 1))[:rows], rng.integers(0, V, rows).astype(np.int32)
    x[np.arange(rows), tokens] = 2.0
    for top in (0, 3, 16, 32, 100):
        got = L.forward(ctx, L.store(x, dtype), tokens, top, 0.9)
        check_forward(got, x, tokens, 0.9, top, f"top {top}")


def test_forward_outputs_on_their_own_and_together_have_the_same_bits(ctx):
    rng = np.random.default_rng(1)
    for V, dtype in ((777, "f32"), (50257, "bf16")):
        x = L.store(L.logits(rng, 5, V, dtype), dtype)
        t = rng.integers(0, V, 5).astype(np.int32)
        full = L.forward(ctx, x, t, 16)
        again = L.forward(ctx, x, t, 16)
        for k in full:
            np.testing.assert_array_equal(full[k], again[k], err_msg=k)
        top = L.forward(ctx, x, None, 16, entropy=False, lse=False)
        np.testing.assert_array_equal(top["top_ids"], full["top_ids"])
        logp = L.forward(ctx, x, t, 0, entropy=False, lse=False)
        np.testing.assert_allclose(logp["logp"], full["logp"], rtol=0, atol=2 * L.sum_error(V))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V,ld,offset", [(1003, 1003, 1), (1003, 1088, 3), (50257, 50304, 0), (37, 40, 5), (4096, 4100, 7)])
def test_forward_strides_and_offsets(ctx, V, ld, offset, dtype):
    rng = np.random.default_rng(V + offset)
    rows = 6
    x = L.logits(rng, rows, V, dtype)
    t = rng.integers(0, V, rows).astype(np.int32)
    t[0], t[1] = 0, V - 1
    got = L.forward(ctx, L.store(x, dtype), t, 8, 0.8, ld=ld, offset=offset)
    check_forward(got, x, t, 0.8, 8)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [90, 3001, 40000])
def test_forward_masks(ctx, V, dtype):
    rng = np.random.default_rng(V)
    x = np.tile(L.logits(rng, 1, V, dtype), (9, 1))
    low = float(np.finfo(np.float32).min) if dtype == "f32" else -3.3895313892515355e38
    x[1, rng.random(V) < 0.95] = -np.inf
    x[2, :] = -np.inf                                # nothing is left
    x[3, :] = -np.inf
    x[3, V // 3] = 2.0                               # one class is left
    x[4, rng.random(V) < 0.9] = low                  # a mask of the lowest value
    x[5, :] = low                                    # all of them: uniform
    x[6, V // 2:] = -np.inf
    x[7, :V - 2] = -np.inf
    x[8, ::2] = -np.inf
    x[4, 5], x[8, 1] = 3.0, 90.0
    t = np.array([3, 5, 4, V // 3, 5, 6, 0, V - 1, 2], np.int32)
    got = L.forward(ctx, L.store(x, dtype), t, 24)
    w = cf.token_logprobs(x, t, 1.0, 24)
    # (a lse of -3.4e38 + log V, and distances to it, in fp32: the lowest values have their own row below)
    keep = np.arange(9) != 5
    keep[4] = False
    check_forward({k: v[keep] for k, v in got.items()}, x[keep], t[keep], 1.0, 24)
    assert got["logp"][2] == 0 and got["entropy"][2] == 0 and got["lse"][2] == -np.inf
    assert (got["top_ids"][2] == -1).all() and (got["top_logp"][2] == -np.inf).all()
    assert got["top_ids"][3, 0] == V // 3 and got["top_ids"][3, 1] == -1
    for r in (4, 5):
        np.testing.assert_array_equal(got["top_ids"][r], w[3][r])
        assert abs(got["logp"][r] - w[0][r]) <= L.sum_error(V) + 64 * U
        assert abs(got["entropy"][r] - w[1][r]) <= 26 * L.sum_error(V) + 64 * U
    assert abs(got["logp"][5] + np.log(V)) <= L.sum_error(V) + 64 * U


def test_forward_nan_and_infinity(ctx):
    for V in (70, 5000):
        x = np.random.default_rng(V).standard_normal((5, V)).astype(np.float32)
        x[0, 11] = np.nan
        x[1, 11] = np.inf
        x[2, :] = -np.inf
        x[2, 3] = np.nan
        x[3, :] = np.nan
        t = np.array([1, 11, 5, 5, 5], np.int32)
        got = L.forward(ctx, x, t, 4)
        for r in range(4):
            assert np.isnan(got["logp"][r]) and np.isnan(got["entropy"][r]) and np.isnan(got["lse"][r]), r
        np.testing.assert_array_equal(got["top_ids"][0], [i for i in np.argsort(-x[0], kind="stable") if i != 11][:4])
        assert got["top_ids"][1, 0] == 11 and np.isnan(got["top_logp"][1]).all()
        assert (got["top_ids"][2:4] == -1).all() and (got["top_logp"][2:4] == -np.inf).all()
        check_forward({k: v[4:] for k, v in got.items()}, x[4:], t[4:], 1.0, 4)


def order_cases(V):
    """rows whose largest classes lie where a selection by parts can go wrong"""
    rng = np.random.default_rng(V)
    i = np.arange(V)
    yield "equal", np.zeros(V)
    yield "zeros of both signs", np.where(i % 3 == 0, -0.0, 0.0)
    yield "ascending", i / 16.0
    yield "descending", -i / 16.0
    yield "two values", np.where(rng.random(V) < 0.5, 1.0, 2.0)
    yield "few values", rng.integers(0, 5, V).astype(float)
    yield "a block in front", np.where(i < 300, 9.0 + rng.random(V), rng.random(V))
    yield "a block behind", np.where(i >= V - 300, 9.0 + rng.random(V), rng.random(V))
    for period in (1024, 2048, 4096, 8192):
        yield f"every {period}th vector", np.where(i % period < 8, 9.0 + rng.random(V), rng.random(V))
    yield "equal among masked", np.where(rng.random(V) < 0.01, 1.0, -np.inf)
    yield "negative", -100.0 - rng.random(V)
    yield "tiny", rng.standard_normal(V) * 1e-30
    yield "huge", rng.standard_normal(V) * 1e30


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [130, 2049, 40001, 151936])
def test_alternatives_come_in_order(ctx, V, dtype):
    names, xs = zip(*order_cases(V))
    x = L.rounded(np.stack(xs), dtype)
    want = {k: cf.token_logprobs(x, np.full(len(x), -1), 1.0, k)[3] for k in (128,)}[128]
    for top in (1, 5, 64, 128):
        got = L.forward(ctx, L.store(x, dtype), None, top, entropy=False)
        for r, name in enumerate(names):
            np.testing.assert_array_equal(got["top_ids"][r], want[r][:top], err_msg=f"{name}, top {top}")
    many = L.forward(ctx, L.store(np.tile(x, (40, 1)), dtype), None, 64, entropy=False)     # (many rows: another split)
    np.testing.assert_array_equal(many["top_ids"], np.tile(want[:, :64], (40, 1)))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [300, 700, 1500, 7001, 15001, 30011])
def test_alternatives_of_rows_that_are_kept_come_in_order(ctx, V, dtype):
    names, xs = zip(*order_cases(V))
    x = L.rounded(np.stack(xs), dtype)
    want = cf.token_logprobs(x, np.full(len(x), -1), 1.0, 128)[3]
    for top in (1, 16, 17, 32, 128):
        got = L.forward(ctx, L.store(x, dtype), None, top, entropy=False)
        for r, name in enumerate(names):
            np.testing.assert_array_equal(got["top_ids"][r], want[r][:top], err_msg=f"{name}, top {top}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [40, 257, 601, 1000, 2001, 4000])
def test_alternatives_of_many_short_rows_come_in_order(ctx, V, dtype):
    xs = [x for _, x in order_cases(V)]
    x = L.rounded(np.stack(xs), dtype)
    want = cf.token_logprobs(x, np.full(len(x), -1), 1.0, 128)[3]
    n = -(-1030 // len(x))
    for top in (5, 20, 32, 33, 50, 64, 65, 100, 128):
        got = L.forward(ctx, L.store(np.tile(x, (n, 1)), dtype), None, top, entropy=False)
        np.testing.assert_array_equal(got["top_ids"], np.tile(want[:, :top], (n, 1)), err_msg=f"top {top}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,V", [(1, 1), (3, 7), (4, 129), (5, 1000), (3, 4099), (40, 517), (2, 50257), (2, 151936)])
def test_backward(ctx, rows, V, dtype):
    rng = np.random.default_rng(2000 + V)
    x = L.logits(rng, rows, V, dtype)
    if V > 100:
        x[0, rng.random(V) < 0.3] = -np.inf
    t = rng.integers(0, V, rows).astype(np.int32)
    x[np.arange(rows), t] = 1.0
    if rows > 2:
        t[1] = -1
        x[2, :] = -np.inf
    g, h = rng.standard_normal(rows).astype(np.float32), rng.standard_normal(rows).astype(np.float32)
    bits = L.store(x, dtype)
    scale = 0.7
    f = L.forward(ctx, bits, t, 0, scale)
    for dg, dh in ((g, None), (None, h), (g, h)):
        want = cf.token_logprobs_grad(x, t, dg, dh, scale)
        got = L.backward(ctx, bits, t, f["lse"], f["entropy"], dg, dh, scale)
        L.assert_within(L.value(got), want, backward_bound(x, t, dg, dh, scale, dtype, want), "dlogits")
        if rows > 2:
            assert not L.value(got)[2].any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V,ld,offset,dx_offset", [(1003, 1003, 1, 1), (1003, 1088, 3, 2), (4096, 4100, 0, 0), (37, 40, 5, 5), (4096, 4096, 0, 1)])
def test_backward_strides_offsets_accumulate_and_in_place(ctx, V, ld, offset, dx_offset, dtype):
    rng = np.random.default_rng(V + ld)
    rows = 5
    x = L.logits(rng, rows, V, dtype)
    bits = L.store(x, dtype)
    t = rng.integers(0, V, rows).astype(np.int32)
    t[0], t[1] = 0, V - 1
    g, h = rng.standard_normal(rows).astype(np.float32), rng.standard_normal(rows).astype(np.float32)
    f = L.forward(ctx, bits, t, 0, 1.0)
    want = cf.token_logprobs_grad(x, t, g, h)
    bound = backward_bound(x, t, g, h, 1.0, dtype, want)
    got = L.backward(ctx, bits, t, f["lse"], f["entropy"], g, h, ld=ld, offset=offset, dx_offset=dx_offset)
    L.assert_within(L.value(got), want, bound, "strided")
    base = L.rounded(rng.standard_normal((rows, V)), dtype)
    acc = L.backward(ctx, bits, t, f["lse"], f["entropy"], g, h, ld=ld, offset=offset, dx_offset=dx_offset, flags=capi.ACC_INPUT_GRAD,
                     init=L.store(base, dtype))
    bound = bound + 2 * U * np.abs(base + want) + (2.0 ** -8 * np.abs(base + want) if dtype == "bf16" else 0.0)
    L.assert_within(L.value(acc), base + want, bound, "accumulated")
    if offset == dx_offset:
        same = L.backward(ctx, bits, t, f["lse"], f["entropy"], g, h, ld=ld, offset=offset, in_place=True)
        np.testing.assert_array_equal(same, got)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [70, 5003, 70000])
def test_backward_of_rows_far_from_zero(ctx, V, dtype):
    """rows of which fp32 holds no lse: all at a mask's lowest value, or shifted as a whole"""
    rng = np.random.default_rng(V)
    low = float(np.finfo(np.float32).min) if dtype == "f32" else -3.3895313892515355e38
    x = np.tile(L.logits(rng, 1, V, dtype), (7, 1))
    x[0, :] = low
    x[1, V // 2:] = low
    x[2] = L.rounded(x[2] + 60000.0, dtype)
    x[3] = L.rounded(x[3] - 60000.0, dtype)
    x[4, :] = -np.inf
    x[5, :] = -np.inf
    x[5, 3] = low
    t = np.array([2, 3, int(x[2].argmax()), int(x[3].argmin()), 1, 3, -1], np.int32)
    g, h = rng.standard_normal(7).astype(np.float32), rng.standard_normal(7).astype(np.float32)
    bits = L.store(x, dtype)
    for scale in (1.0, 1.5):
        f = L.forward(ctx, bits, t, 0, scale)
        p, logp, _ = cf._softmax_rows(cf.f64(x) * scale)
        l = np.abs(np.where(p > 0, logp, 0.0))
        want = cf.token_logprobs_grad(x, t, g, h, scale)
        # distances to the largest logit, which is taken off exactly or with half a step, and their product with the scale
        delta = U * (6 * l + 16) + 2 * L.sum_error(V)
        size = p * (np.abs(g)[:, None] + np.abs(h)[:, None] * (l + (p * l).sum(-1, keepdims=True) + 1))
        bound = scale * (size * 2 * delta + np.abs(h)[:, None] * p * L.sum_error(V) * (2 + 2 * np.log(V + 1)))
        bound = bound + scale * 8 * U * np.abs(g)[:, None] * (np.arange(V) == t[:, None]) + 1e-37
        for r in (1, 6):                                   # (ordinary ones, whose lse is rounded)
            one = slice(r, r + 1)
            bound[r] = backward_bound(cf.f64(x[one]), t[one], g[one], h[one], scale, "f32", want[one])[0]
        bound = bound + (np.abs(want) + bound) * 2.0 ** -8 if dtype == "bf16" else bound
        got = L.backward(ctx, bits, t, f["lse"], f["entropy"], g, h, scale)
        L.assert_within(L.value(got), want, bound, f"scale {scale}")
        assert not L.value(got)[4].any()
        same = L.backward(ctx, bits, t, f["lse"], f["entropy"], g, h, scale, in_place=True)
        np.testing.assert_array_equal(same, got)
        base = L.rounded(rng.standard_normal((7, V)), dtype)
        acc = L.value(L.backward(ctx, bits, t, f["lse"], f["entropy"], g, h, scale, flags=capi.ACC_INPUT_GRAD, init=L.store(base, dtype)))
        half = 2.0 ** -8 if dtype == "bf16" else U
        L.assert_within(acc, base + want, bound + 2 * half * (np.abs(base + want) + bound), f"accumulated, scale {scale}")
        np.testing.assert_array_equal(acc[4], base[4])


def test_backward_against_differences(ctx):
    """d(dlogp . logp + dentropy . entropy) along single logits, central differences of the float64 form"""
    rng = np.random.default_rng(5)
    rows, V, scale, step = 3, 50, 0.8, 1e-5
    x = rng.standard_normal((rows, V)).astype(np.float32)
    t = np.array([4, 9, 49], np.int32)
    g, h = rng.standard_normal(rows).astype(np.float32), rng.standard_normal(rows).astype(np.float32)
    f = L.forward(ctx, x, t, 0, scale)
    got = L.backward(ctx, x, t, f["lse"], f["entropy"], g, h, scale)

    def total(y):
        logp, ent, *_ = cf.token_logprobs(y, t, scale)
        return (g * logp + h * ent).sum()

    for r in range(rows):
        for v in (0, 4, 9, 30, 49):
            hi, lo = cf.f64(x).copy(), cf.f64(x).copy()
            hi[r, v] += step
            lo[r, v] -= step
            want = (total(hi) - total(lo)) / (2 * step)
            assert abs(got[r, v] - want) <= 1e-5, (r, v)     # (step^2 and 1e-16 / step both below 1e-9; fp32 arithmetic below 1e-5)


def test_rows_far_apart(ctx):
    """row offsets past 32 bits"""
    rng = np.random.default_rng(6)
    rows, V, ld = 3, 1200, 2_200_000_000
    x = L.logits(rng, rows, V, "bf16")
    bits = L.store(x, "bf16")
    t = rng.integers(0, V, rows).astype(np.int32)
    buf, grad = ctx.alloc((2 * ld + V) * 2), ctx.alloc((2 * ld + V) * 2)
    with L.Device(ctx) as dev:
        for r in range(rows):
            ctx.call("agrad_copy_from_host", buf, r * ld * 2, bits[r].ctypes.data_as(C.c_void_p), V * 2)
        out = [dev.up(np.zeros(rows, np.float32)) for _ in range(3)]
        ids, tl = dev.up(np.zeros((rows, 5), np.int32)), dev.up(np.zeros((rows, 5), np.float32))
        tok, g = dev.up(t), dev.up(np.ones(rows, np.float32))
        ctx.call("agrad_token_logprobs_forward", capi.BF16, C.c_void_p(buf), L.p(tok), *map(L.p, out), L.p(ids), L.p(tl), rows, V, ld, 5, 1.0)
        ctx.call("agrad_token_logprobs_backward", capi.BF16, C.c_void_p(buf), L.p(tok), L.p(out[2]), L.p(out[1]), L.p(g), None,
                 C.c_void_p(grad), rows, V, ld, 1.0, 0)
        ctx.synchronize()
        got = dict(zip(("logp", "entropy", "lse"), (d.download() for d in out)), top_ids=ids.download(), top_logp=tl.download())
        check_forward(got, x, t, 1.0, 5)
        want = cf.token_logprobs_grad(x, t, np.ones(rows), None)
        bound = backward_bound(x, t, np.ones(rows), None, 1.0, "bf16", want)
        row = np.empty(V, np.uint16)
        for r in range(rows):
            ctx.call("agrad_copy_to_host", grad, r * ld * 2, row.ctypes.data_as(C.c_void_p), V * 2)
            L.assert_within(L.value(row), want[r], bound[r], f"row {r}")
    ctx.free(buf)
    ctx.free(grad)


def test_many_classes(ctx):
    rng = np.random.default_rng(8)
    V = 3_000_001
    x = L.logits(rng, 2, V, "f32")
    t = np.array([V - 1, 5], np.int32)
    check_forward(L.forward(ctx, x, t, 100), x, t, 1.0, 100)


def test_tokens_out_of_range_and_no_rows(ctx):
    x = np.zeros((3, 8), np.float32)
    with L.Device(ctx) as dev:
        d_x, t, logp, dx = dev.up(x), dev.up(np.array([3, 8, -2], np.int32)), dev.up(np.full(3, -7.0, np.float32)), dev.up(x)
        lse = dev.up(np.full(3, np.log(8.0), np.float32))
        ctx.call("agrad_token_logprobs_forward", capi.F32, L.p(d_x), L.p(t), L.p(logp), None, None, None, None, 3, 8, 8, 0, 1.0)
        with pytest.raises(IndexError):
            ctx.synchronize()
        np.testing.assert_allclose(logp.download(), [-np.log(8.0), 0, 0], rtol=1e-6)
        ctx.call("agrad_token_logprobs_backward", capi.F32, L.p(d_x), L.p(t), L.p(lse), None, L.p(lse), None, L.p(dx), 3, 8, 8, 1.0, 0)
        with pytest.raises(IndexError):
            ctx.synchronize()
        assert not dx.download()[1:].any()
        ctx.call("agrad_token_logprobs_forward", capi.F32, None, None, None, None, None, None, None, 0, 8, 8, 0, 1.0)
        ctx.call("agrad_token_logprobs_backward", capi.F32, None, None, None, None, None, None, None, 0, 8, 8, 1.0, 0)
        ctx.synchronize()


def test_refusals(ctx):
    with L.Device(ctx) as dev:
        x, t, o = dev.up(np.zeros(64, np.float32)), dev.up(np.zeros(8, np.int32)), dev.up(np.zeros(64, np.float32))
        good = dict(dtype=capi.F32, x=L.p(x), tokens=L.p(t), logp=L.p(o), entropy=None, lse=None, ids=None, tl=None, rows=2, V=8, ld=8,
                    top=0, scale=1.0)

        def refused(**over):
            a = {**good, **over}
            with pytest.raises(capi.AgradError) as e:
                ctx.call("agrad_token_logprobs_forward", *a.values())
            assert e.value.code == capi.EINVAL

        for over in (dict(dtype=2), dict(V=0), dict(ld=7), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                     dict(scale=float("inf")), dict(x=None), dict(tokens=None), dict(logp=None), dict(tokens=None, logp=None),
                     dict(top=129, ids=L.p(t), tl=L.p(o)), dict(top=1), dict(top=1, ids=L.p(t)), dict(ids=L.p(t), tl=L.p(o)),
                     dict(x=C.c_void_p(x.ptr + 2)), dict(rows=1 << 22), dict(V=0x7fffffff, ld=0x7fffffff)):
            refused(**over)
        back = dict(dtype=capi.F32, x=L.p(x), tokens=L.p(t), lse=L.p(o), entropy=L.p(o), dlogp=L.p(o), dentropy=L.p(o), dx=L.p(x),
                    rows=2, V=8, ld=8, scale=1.0, flags=0)
        for over in (dict(x=None), dict(dx=None), dict(lse=None), dict(tokens=None), dict(entropy=None), dict(dlogp=None, dentropy=None),
                     dict(scale=0.0), dict(ld=3), dict(dtype=9), dict(dx=C.c_void_p(x.ptr + 1)), dict(flags=2)):
            with pytest.raises(capi.AgradError) as e:
                ctx.call("agrad_token_logprobs_backward", *{**back, **over}.values())
            assert e.value.code == capi.EINVAL
    ctx.synchronize()


def crowded_cases(V):
    """order_cases, and rows in which a workgroup's threads find all that they hold among the candidates, or none"""
    yield from order_cases(V)
    rng = np.random.default_rng(V + 1)
    i = np.arange(V)
    for period in (1024, 2048):
        yield f"masked but for every {period}th vector", np.where(i % period < 8, 1.0 + i / V, -np.inf)
    yield "far from zero", 1000.0 + rng.standard_normal(V)               # (few steps of 16 bits)
    yield "far below zero", -60000.0 + rng.standard_normal(V)
    yield "one class", np.where(i == V - 3, 1.0, -np.inf)


def assert_order(ctx, dtype, V, rows):
    names, xs = zip(*crowded_cases(V))
    x = L.rounded(np.stack(xs), dtype)
    want = cf.token_logprobs(x, np.full(len(x), -1), 1.0, 128)[3]
    n = -(-rows // len(x)) if rows else 1
    at = np.arange(n * len(x))[:rows or None] % len(x)
    bits = L.store(x, dtype)[at]
    for top in (1, 5, 20, 64, 128):
        got = L.forward(ctx, bits, None, top, entropy=False)["top_ids"]
        for r, i in enumerate(at):
            np.testing.assert_array_equal(got[r], want[i, :top], err_msg=f"row {r}, {names[i]}, top {top}")


@pytest.mark.parametrize("dtype,V", [("f32", 4096), ("f32", 8192), ("f32", 15364), ("f32", 16384), ("f32", 16387),
                                     ("bf16", 8192), ("bf16", 16384), ("bf16", 30736), ("bf16", 32000), ("bf16", 32768), ("bf16", 32775)])
def test_alternatives_of_rows_that_fill_their_threads(ctx, dtype, V):
    """rows of 4, 8 and 16 vectors a thread, and next to that: up to all of a thread's vectors are candidates"""
    assert_order(ctx, dtype, V, 0)


@pytest.mark.parametrize("dtype,V,rows", [("f32", 32768, 400), ("f32", 65536, 220), ("bf16", 65536, 200), ("bf16", 65536, 256),
                                          ("bf16", 131072, 110), ("bf16", 128256, 128)])
def test_alternatives_of_parts_that_fill_their_threads(ctx, dtype, V, rows):
    """the same for rows that two or four workgroups share, of 16 vectors a thread each"""
    assert_order(ctx, dtype, V, rows)


@pytest.mark.parametrize("dtype,V", [("f32", 16384), ("bf16", 32768)])
def test_equal_logits_have_their_alternatives(ctx, dtype, V):
    """an output head of zeros: every class as likely as another, the lowest ids first"""
    x = np.zeros((3, V), np.float32)
    got = L.forward(ctx, L.store(x, dtype), np.array([0, V - 1, -1], np.int32), 9)
    check_forward(got, x, np.array([0, V - 1, -1]), 1.0, 9)
    np.testing.assert_array_equal(got["top_ids"], np.tile(np.arange(9), (3, 1)))


def test_scales_at_their_ends(ctx):
    """the largest scale takes the largest logits for the whole distribution, the smallest none; beyond them a call is refused"""
    x = np.array([[0.0, 1.0, 1.0, -np.inf, 0.5], [-3.0, -2.0, -2.0, -2.0, -np.inf]], np.float32)
    t = np.array([1, 2], np.int32)
    for scale, n in ((2e38, (2, 3)), (1e-45, (4, 4))):
        got = L.forward(ctx, x, t, 2, scale)
        for r in range(2):
            assert abs(got["logp"][r] + np.log(n[r])) <= 16 * U and abs(got["entropy"][r] - np.log(n[r])) <= 16 * U
            assert np.abs(got["top_logp"][r] + np.log(n[r])).max() <= 16 * U
        loss, stats = L.distill_forward(ctx, x, np.array([[1, 2], [1, 2]], np.int32), np.zeros((2, 2), np.float32), scale=scale)
        assert np.abs(loss - np.log(np.array(n) / 2.0)).max() <= 32 * U
    with L.Device(ctx) as dev:
        d, i, o = dev.up(x), dev.up(np.zeros(16, np.int32)), dev.up(np.zeros(16, np.float32))
        for bad in (2.1e38, 3.4e38, 1e39):
            for name, args in (("token_logprobs_forward", (L.p(i), L.p(o), None, None, None, None, 2, 5, 5, 0, bad)),
                               ("token_logprobs_backward", (L.p(i), L.p(o), None, L.p(o), None, L.p(d), 2, 5, 5, bad, 0)),
                               ("topk_distill_forward", (L.p(i), L.p(o), L.p(o), None, 2, 5, 5, 1, bad, 1.0, 0)),
                               ("topk_distill_backward", (L.p(i), L.p(o), L.p(o), L.p(o), L.p(d), 2, 5, 5, 1, bad, 1.0, 0, 0)),
                               ("topk_distill_fused", (L.p(i), L.p(o), L.p(o), None, L.p(d), 2, 5, 5, 1, bad, 1.0, 1.0, 0))):
                with pytest.raises(capi.AgradError) as e:
                    ctx.call("agrad_" + name, capi.F32, L.p(d), *args)
                assert e.value.code == capi.EINVAL, name
    ctx.synchronize()
