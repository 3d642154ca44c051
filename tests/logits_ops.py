"""numpy-in / numpy-out wrappers over the C-ABI operators on logits, and their error bounds, for tests.

bf16 logits are passed and returned as uint16 bit arrays.  `ld` gives the rows a stride, `offset` shifts the tensor by
elements; the padding is filled with a pattern that has to be there afterwards.

Error bounds.  u = 2^-24 is half a step of fp32.  A sum of exponentials of V positive terms is added up by threads one
after the other, at most V / 256 + 64 additions deep, so its relative error, and the absolute error of its logarithm, is
at most sum_error(V) = (V / 256 + 64) u.  A probability exp(z - lse) from rounded z, lse and argument is off by
delta = u (|lse| + |z| + 3 |z - lse| + 8) relative, plus the error of lse.  A bf16 output is off by half a step more,
2^-8 relative.
"""
import ctypes as C

import numpy as np

from autograd_amd import capi
from tests.helpers import from_bf16_bits, to_bf16_bits

U = 2.0 ** -24
PAD = 77           # what the columns behind the classes hold


def sum_error(V):
    return (V / 256 + 64) * U


def store(x, dtype):
    return to_bf16_bits(x) if dtype == "bf16" else np.asarray(x, np.float32)


def value(bits):
    return from_bf16_bits(bits) if bits.dtype == np.uint16 else bits


def rounded(x, dtype):
    """x as a tensor of that type holds it"""
    return value(store(np.asarray(x, np.float32), dtype))


def kind(a):
    return capi.BF16 if a.dtype == np.uint16 else capi.F32


class Matrix:
    """[rows, V] on the device with a row stride and an offset"""

    def __init__(self, ctx, bits, ld=None, offset=0):
        self.shape, self.ld, self.offset = bits.shape, ld or bits.shape[1], offset
        rows, V = bits.shape
        full = np.full(offset + rows * self.ld + 5, PAD, bits.dtype)
        body = full[offset:offset + rows * self.ld].reshape(rows, self.ld)
        body[:, :V] = bits
        self.d = ctx.upload(full)
        self.item = bits.dtype.itemsize

    def ptr(self):
        return C.c_void_p(self.d.ptr + self.offset * self.item)

    def get(self):
        full = self.d.download()
        rows, V = self.shape
        body = full[self.offset:self.offset + rows * self.ld].reshape(rows, self.ld)
        assert (body[:, V:] == PAD).all() and (full[:self.offset] == PAD).all() and (full[self.offset + rows * self.ld:] == PAD).all(), \
            "something outside the classes was written"
        return body[:, :V].copy()

    def free(self):
        self.d.free()


def p(d):
    return C.c_void_p(d.ptr) if d is not None else None


class Device:
    """uploads that are freed together"""

    def __init__(self, ctx):
        self.ctx, self.all = ctx, []

    def up(self, a):
        if a is None:
            return None
        d = self.ctx.upload(np.ascontiguousarray(a))
        self.all.append(d)
        return d

    def matrix(self, bits, ld=None, offset=0):
        m = Matrix(self.ctx, bits, ld, offset)
        self.all.append(m)
        return m

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        for d in self.all:
            d.free()


def forward(ctx, bits, tokens=None, top=0, scale=1.0, entropy=True, lse=True, ld=None, offset=0):
    """{"logp", "entropy", "lse", "top_ids", "top_logp"} of one call"""
    rows, V = bits.shape
    with Device(ctx) as dev:
        x = dev.matrix(bits, ld, offset)
        t = dev.up(None if tokens is None else np.asarray(tokens, np.int32))
        f = lambda on: dev.up(np.full(rows, -7.0, np.float32)) if on else None  # noqa: E731
        logp, ent, ls = f(tokens is not None), f(entropy), f(lse)
        ids = dev.up(np.full((rows, top), -7, np.int32)) if top else None
        tl = dev.up(np.full((rows, top), -7.0, np.float32)) if top else None
        ctx.call("agrad_token_logprobs_forward", kind(bits), x.ptr(), p(t), p(logp), p(ent), p(ls), p(ids), p(tl), rows, V,
                 x.ld, top, scale)
        ctx.synchronize()
        np.testing.assert_array_equal(x.get(), bits)
        return {k: None if d is None else d.download() for k, d in
                (("logp", logp), ("entropy", ent), ("lse", ls), ("top_ids", ids), ("top_logp", tl))}


def backward(ctx, bits, tokens, lse, entropy, dlogp, dentropy, scale=1.0, flags=0, init=None, ld=None, offset=0, dx_offset=None,
             in_place=False):
    rows, V = bits.shape
    with Device(ctx) as dev:
        x = dev.matrix(bits, ld, offset)
        dx = x if in_place else dev.matrix(np.full_like(bits, 3) if init is None else init, ld, offset if dx_offset is None else dx_offset)
        f = lambda a, t=np.float32: dev.up(None if a is None else np.asarray(a, t))  # noqa: E731
        ctx.call("agrad_token_logprobs_backward", kind(bits), x.ptr(), p(f(tokens, np.int32)), p(f(lse)), p(f(entropy)), p(f(dlogp)),
                 p(f(dentropy)), dx.ptr(), rows, V, x.ld, scale, flags)
        ctx.synchronize()
        return dx.get()


def distill_forward(ctx, bits, ids, values, scale=1.0, teacher_scale=1.0, tail=False, ld=None, offset=0):
    rows, V = bits.shape
    with Device(ctx) as dev:
        x, i, v = dev.matrix(bits, ld, offset), dev.up(ids), dev.up(values)
        loss, stats = dev.up(np.full(rows, -7.0, np.float32)), dev.up(np.full((rows, 4), -7.0, np.float32))
        ctx.call("agrad_topk_distill_forward", kind(bits), x.ptr(), p(i), p(v), p(loss), p(stats), rows, V, x.ld, ids.shape[1], scale,
                 teacher_scale, int(tail))
        ctx.synchronize()
        np.testing.assert_array_equal(x.get(), bits)
        return loss.download(), stats.download()


def distill_backward(ctx, bits, ids, values, dloss, stats, scale=1.0, teacher_scale=1.0, tail=False, flags=0, init=None, ld=None,
                     offset=0, dx_offset=None, in_place=False):
    rows, V = bits.shape
    with Device(ctx) as dev:
        x, i, v, g, st = dev.matrix(bits, ld, offset), dev.up(ids), dev.up(values), dev.up(dloss), dev.up(stats)
        dx = x if in_place else dev.matrix(np.full_like(bits, 3) if init is None else init, ld, offset if dx_offset is None else dx_offset)
        ctx.call("agrad_topk_distill_backward", kind(bits), x.ptr(), p(i), p(v), p(g), p(st), dx.ptr(), rows, V, x.ld, ids.shape[1],
                 scale, teacher_scale, int(tail), flags)
        ctx.synchronize()
        return dx.get()


def distill_fused(ctx, bits, ids, values, scale=1.0, teacher_scale=1.0, tail=False, row_scale=None, grad_scale=1.0, ld=None, offset=0,
                  dx_offset=None, in_place=False, want_loss=True):
    rows, V = bits.shape
    with Device(ctx) as dev:
        x, i, v, w = dev.matrix(bits, ld, offset), dev.up(ids), dev.up(values), dev.up(row_scale)
        dx = x if in_place else dev.matrix(np.full_like(bits, 3), ld, offset if dx_offset is None else dx_offset)
        loss = dev.up(np.full(rows, -7.0, np.float32))
        ctx.call("agrad_topk_distill_fused", kind(bits), x.ptr(), p(i), p(v), p(loss) if want_loss else None, p(w), dx.ptr(), rows, V,
                 x.ld, ids.shape[1], scale, teacher_scale, grad_scale, int(tail))
        ctx.synchronize()
        return loss.download(), dx.get()


def assert_within(got, want, bound, what):
    """|got - want| <= bound where want is finite, the same infinities and NaN elsewhere"""
    got, want, bound = (np.asarray(a, np.float64) for a in (got, want, bound))
    assert got.shape == want.shape, f"{what}: {got.shape} {want.shape}"
    fine = np.isfinite(want)
    np.testing.assert_array_equal(got[~fine], want[~fine], err_msg=what)
    assert np.isfinite(got[fine]).all(), f"{what}: not finite where it should be"
    off = np.where(fine, np.abs(np.where(fine, got, 0.0) - np.where(fine, want, 0.0)), 0.0)
    bound = np.broadcast_to(bound, off.shape)
    if (off > bound).any():
        i = np.unravel_index(np.argmax(np.where(fine, off - bound, -np.inf)), off.shape)
        raise AssertionError(f"{what}: {int((off > bound).sum())} of {off.size} outside; worst at {i}: got {got[i]!r}, want "
                             f"{want[i]!r}, off by {off[i]:.3e}, allowed {bound[i]:.3e}")


def logits(rng, rows, V, dtype, spread=3.0):
    x = spread * rng.standard_normal((rows, V)) + rng.standard_normal((rows, 1))
    x[np.arange(rows), rng.integers(0, V, rows)] += 8.0
    return rounded(x, dtype)


def teacher(rng, rows, V, K, tail, ragged=True):
    """distinct ids a row in no order; some rows have unused slots in between"""
    ids = np.full((rows, K), -1, np.int32)
    n = min(K, V)
    for r in range(rows):
        ids[r, :n] = rng.choice(V, n, replace=False) if V < 5000 else rng.permutation(np.unique(rng.integers(0, V, 4 * n + 64))).astype(np.int32)[:n]
        if ragged and r % 3 == 1:
            ids[r, rng.random(K) < 0.4] = -1
    u = 2.5 * rng.standard_normal((rows, K + 1))
    if tail:
        u = u - np.log(np.exp(u).sum(-1, keepdims=True))
    return ids, u[:, :K].astype(np.float32)
