"""The operators of a recurrent model's serving step on the GPU through the C ABI, each against its definition in 64
bits: norms with 8-bit rows, 8-bit products, the gated delta rule, beam search's selection and reordering.

Tolerances count roundings: u = 2^-24 is half a step of fp32, and an output held in bf16 adds its own half step 2^-8
relative.
"""
import ctypes as C

import numpy as np
import pytest

from pssa_amd import HipDevice, ModelWeights, PSSAConfig, PSSALayer, _abi
from test_gpu_operators import Held, from_bf16, to_bf16, typed

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
U16 = 2.0 ** -8
NONE = _abi.NO_TOKEN


def say(*a):
    print("[step]", *a, flush=True)


def back(buf, dtype, shape=None):
    """A device array's values."""
    a = buf.to_host()
    a = from_bf16(a) if dtype == "bf16" else a
    return a if shape is None else a.reshape(shape)


def within(got, want, tol, what=""):
    """Equal where the tolerance has nothing to say (infinities, NaN), near elsewhere."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want), err_msg=what)
    fine = np.isfinite(want)
    np.testing.assert_array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)], err_msg=what)
    tol = np.broadcast_to(np.asarray(tol, np.float64), want.shape)
    off = np.abs(got[fine] - want[fine]) / np.maximum(tol[fine], 1e-300)
    assert not off.size or off.max() <= 1, f"{what}: {off.max():.3g} of the tolerance"


# ---------------------------------------------------------------------------
# Norms


def wide_rows(values, ld, dtype, offset, fill=1e30):
    """Rows at stride ld behind `offset` elements, as stored, and their values."""
    rows, width = values.shape
    w = np.full((rows, ld), fill, np.float32)
    w[:, :width] = values
    stored, held = typed(w, dtype)
    return np.concatenate([np.zeros(offset, stored.dtype), stored.ravel()]), held[:, :width]


def codes32(t):
    """The codes' formula in 32 bits, and max |t|; rows that are not finite have codes 0."""
    most = np.abs(t).max(1, keepdims=True)
    fine = np.isfinite(t).all(1, keepdims=True)
    with np.errstate(all="ignore"):
        # Maxima whose 127 / max overflows: the same with the row scaled up by a power of two.
        up = np.where(most < 1e-30, np.float32(2.0 ** 64), np.float32(1.0)).astype(np.float32)
        q = np.rint((t * up) * (np.float32(127.0) / (most * up)).astype(np.float32))
    return np.where(fine & (most > 0), q, 0).astype(np.int8), most[:, 0], fine[:, 0]


def check_norm(hip, x, res, gamma, dtype, pad=0, offset=0, eps=1e-5, codes=True, out=True, total=True, where="apart"):
    rows, width = x.shape
    ld, size = width + pad, 4 if dtype == "f32" else 2
    sx, hx = wide_rows(x, ld, dtype, offset)
    sr, hr = (None, None) if res is None else wide_rows(res, ld, dtype, offset)
    g = gamma.astype(np.float32)
    with Held(hip) as h, np.errstate(all="ignore"):
        dx, dr, dg = h.up(sx), None if res is None else h.up(sr), h.up(g)
        do = h.new(offset + rows * ld, sx.dtype, 7)
        ds = {"apart": None, "x": dx, "residual": dr}[where] or h.new(offset + rows * ld, sx.dtype, 7)
        dq, dc = h.new((rows, width + 3), np.int8, 77), h.new(rows, np.float32, 7.0)
        at = offset * size
        hip.rms_norm_resident(dx.ptr + at, dtype, rows, width, dg.ptr, None if res is None else dr.ptr + at,
                              ds.ptr + at if total else None, do.ptr + at if out else None, dq.ptr if codes else None,
                              dc.ptr if codes else None, eps=eps, ld_x=ld, ld_residual=ld, ld_sum=ld, ld_out=ld,
                              ld_codes=width + 3)
        hip.synchronize()
        gs, go = (back(b, dtype)[offset:].reshape(rows, ld) for b in (ds, do))
        gq, gc = dq.to_host(), dc.to_host()
        assert (gq[:, width:] == 77).all()  # what lies between the rows is left
        u16 = U16 if dtype == "bf16" else 0.0
        h64 = hx.astype(np.float64) + (0 if hr is None else hr.astype(np.float64))
        h32 = hx if hr is None else (hx + hr).astype(np.float32)
        h64 = np.where(np.isfinite(h32), h64, h32)
        if total:
            within(gs[:, :width], h64, np.abs(h64) * (U32 + u16), "sum")
            if where == "apart":
                assert (gs[:, width:] == back(h.new(1, sx.dtype, 7), dtype)[0]).all()
        ok = np.isfinite(h64).all(1)
        inv = 1.0 / np.sqrt((h64 ** 2).mean(1, keepdims=True) + eps)
        # A square's sum has at most 64 terms in a thread and 10 steps across threads, half of which reaches its root;
        # the mean, root, quotient and two products add five, h its own.
        rel = (37 + 5 + 3) * U32
        if out:
            want = h64 * inv * g
            within(go[ok, :width], want[ok], np.abs(want[ok]) * (rel + u16) + 1e-44, "out")
            for r in np.flatnonzero(~ok):  # as the formula leaves them
                if np.isnan(h64[r]).any():
                    assert np.isnan(go[r, :width]).all()
                else:
                    assert np.isnan(go[r, :width][np.isinf(h64[r])]).all() and not go[r, :width][np.isfinite(h64[r])].any()
        if codes:
            q, most, fine = codes32((h32 * g).astype(np.float32))
            np.testing.assert_array_equal(gq[:, :width], q)
            want = np.where(fine, most.astype(np.float64) * inv[:, 0] / 127.0, np.nan)
            within(gc, want, np.abs(want) * (rel + 2 * U32) + 1e-44, "scales")


def stream(rng, rows, width):
    """Rows of different size with some wide channels."""
    return rng.normal(0, 1, (rows, width)) * np.where(rng.random(width) < 0.05, 8.0, 1.0) * rng.uniform(0.3, 3.0, (rows, 1))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,width", [(1, 1), (5, 3), (3, 16), (7, 255), (4, 256), (9, 257), (2, 768), (6, 1021), (3, 1025),
                                        (2, 2049), (2, 4099), (2, 8192), (1, 16385), (2, 32771), (1, 65536), (300, 64)])
def test_norm(hip, dtype, rows, width):
    say("norm", dtype, rows, width)
    rng = np.random.default_rng(rows * 1000 + width)
    x, res, g = stream(rng, rows, width), rng.normal(0, 1, (rows, width)), rng.normal(1, 0.3, width)
    check_norm(hip, x, res, g, dtype)
    check_norm(hip, x, None, g, dtype, pad=5, offset=1)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_norm_outputs_one_by_one_and_in_place(hip, dtype):
    rng = np.random.default_rng(5)
    x, res, g = stream(rng, 5, 700), rng.normal(0, 1, (5, 700)), rng.normal(1, 0.3, 700)
    for codes, out, total in ((True, False, False), (False, True, False), (False, False, True), (True, False, True)):
        check_norm(hip, x, res, g, dtype, pad=2, offset=3, codes=codes, out=out, total=total)
    check_norm(hip, x, res, g, dtype, pad=2, offset=1, where="x")
    check_norm(hip, x, res, g, dtype, pad=2, offset=1, where="residual")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_norm_rows_of_zeros_extremes_and_values_that_are_not_finite(hip, dtype):
    rng = np.random.default_rng(6)
    x, g = rng.normal(0, 1, (12, 300)), rng.normal(1, 0.2, 300)
    x[0] = 0
    x[1] *= 1e25  # squares past fp32's range
    x[2] *= 1e-35  # nothing beside eps, 127 / max past fp32's range
    x[3, 7] = np.nan
    x[4, 299] = np.inf
    x[5, 0], x[5, 1] = np.inf, -np.inf
    x[6], x[6, 5] = 0, -3.0
    x[7] = 2.5
    x[8, ::2] = 0
    check_norm(hip, x, None, g, dtype)
    res = np.zeros_like(x)
    res[9, 3] = -np.inf
    check_norm(hip, x, res, g, dtype, codes=True)
    g[4] = 0.0
    check_norm(hip, x[:3], None, g, dtype, eps=1e-12)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,width,pad,offset", [(1, 1, 0, 0), (3, 65, 1, 1), (5, 4096, 0, 0), (2, 8193, 3, 2)])
def test_quantize_i8(hip, dtype, rows, width, pad, offset):
    rng = np.random.default_rng(width)
    x = stream(rng, rows, width)
    x[0] = 0
    stored, held = wide_rows(x, width + pad, dtype, offset)
    with Held(hip) as h:
        dx, dq, dc = h.up(stored), h.new((rows, width), np.int8, 77), h.new(rows, np.float32, 7.0)
        hip.quantize_i8_resident(dx.ptr + offset * stored.itemsize, dtype, rows, width, dq.ptr, dc.ptr, ld_x=width + pad)
        hip.synchronize()
        q, most, _ = codes32(held)
        np.testing.assert_array_equal(dq.to_host(), q)
        within(dc.to_host(), most.astype(np.float64) / 127.0, most * U32, "scales")


# ---------------------------------------------------------------------------
# 8-bit products


def check_i8(hip, m, n, k, y_dtype="f32", pads=(0, 0, 0), offset=0, codes=None, scales=None, reserve=False):
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    lo, hi = codes or (-127, 128)
    x, w = (rng.integers(lo, hi, (r, k + p)).astype(np.int8) for r, p in ((m, pads[0]), (n, pads[1])))
    sx, sw = rng.uniform(0.01, 0.1, m).astype(np.float32), rng.uniform(0.001, 0.01, n).astype(np.float32)
    if scales is not None:
        sx[::2] = scales
    with Held(hip) as h, np.errstate(all="ignore"):
        dx, dw = h.up(np.concatenate([np.zeros(offset, np.int8), x.ravel()])), h.up(np.concatenate([np.zeros(offset, np.int8), w.ravel()]))
        dsx, dsw = h.up(sx), h.up(sw)
        ld_y = n + pads[2]
        dy = h.new((m, ld_y), np.float32 if y_dtype == "f32" else np.uint16, 7)
        if reserve:
            hip.matmul_i8_reserve(m, n, k)
        hip.matmul_i8_resident(dx.ptr + offset, dsx.ptr, dw.ptr + offset, dsw.ptr, m, n, k, dy.ptr, y_dtype,
                               ld_x=k + pads[0], ld_w=k + pads[1], ld_y=ld_y)
        hip.synchronize()
        y = back(dy, y_dtype)
        assert (dy.to_host()[:, n:] == 7).all()
        # Whole numbers below 2^31: exact in 64 bits.
        want = (x[:, :k].astype(np.float64) @ w[:, :k].astype(np.float64).T) * sx[:, None].astype(np.float64) * sw.astype(np.float64)
        tol = np.abs(want) * (3.01 * U32 + (U16 if y_dtype == "bf16" else 0)) + 1e-44
        within(y[:, :n], want, tol, f"{m} x {n} x {k}")


I8_SHAPES = [(1, 1, 1), (1, 16384, 768), (3, 5, 17), (16, 64, 64), (17, 65, 63), (5, 256, 128), (24, 300, 1000), (33, 129, 257),
             (64, 64, 4096), (100, 1000, 515), (128, 128, 128), (129, 257, 384), (200, 512, 2048), (256, 256, 256),
             (257, 300, 640), (1, 7, 131071), (40, 40, 20000), (513, 1025, 192), (300, 2000, 100)]


@pytest.mark.parametrize("m,n,k", I8_SHAPES)
def test_matmul_i8(hip, m, n, k):
    say("i8", m, n, k)
    check_i8(hip, m, n, k, reserve=True)
    check_i8(hip, m, n, k, "bf16", pads=(3, 1, 5), offset=1)
    check_i8(hip, m, n, k, "f32", pads=(16, 32, 2))
    check_i8(hip, m, n, k, "bf16", pads=(-k % 4, -k % 4, 1), offset=4)


@pytest.mark.parametrize("m,n,k", [(3300, 4200, 272), (2000, 2500, 528), (1150, 4300, 1040), (1025, 2100, 1000), (70, 16400, 16)])
def test_matmul_i8_of_many_tiles(hip, m, n, k):
    """Each size of tiles, and k that ends in a slab's first and later units."""
    say("i8 tiles", m, n, k)
    check_i8(hip, m, n, k)
    check_i8(hip, m, n, k, "bf16", pads=(16, 0, 3))
    check_i8(hip, m, n, k, "bf16", pads=(3, 1, 5), offset=1)


@pytest.mark.parametrize("m,n,k", [(1, 64, 131071), (2, 2, 131071), (130, 130, 2048)])
def test_matmul_i8_of_the_largest_codes(hip, m, n, k):
    """Sums of -128 squared: the largest that 32 bits hold."""
    check_i8(hip, m, n, k, codes=(-128, -127))
    check_i8(hip, m, n, k, "bf16", codes=(127, 128))


def test_matmul_i8_scales_that_are_zero_or_not_finite(hip):
    """A row's scale reaches its own row alone."""
    for scale in (0.0, np.nan, np.inf):
        rng = np.random.default_rng(3)
        m, n, k = 21, 70, 130
        x, w = rng.integers(1, 128, (m, k)).astype(np.int8), rng.integers(1, 128, (n, k)).astype(np.int8)
        sx, sw = np.ones(m, np.float32), np.ones(n, np.float32)
        sx[4] = scale
        with Held(hip) as h:
            d = [h.up(a) for a in (x, sx, w, sw)]
            y = h.new((m, n), np.float32, 7.0)
            hip.matmul_i8_resident(d[0].ptr, d[1].ptr, d[2].ptr, d[3].ptr, m, n, k, y.ptr)
            hip.synchronize()
            got = y.to_host()
            want = x.astype(np.float64) @ w.astype(np.float64).T
            np.testing.assert_array_equal(np.delete(got, 4, 0), np.delete(want, 4, 0))  # below 2^24: exact
            np.testing.assert_array_equal(got[4], np.full(n, np.float32(scale)))


# ---------------------------------------------------------------------------
# The gated delta rule


def delta64(q, k, v, g, beta, scale, lens, state, heads, key_heads):
    """The recurrence in 64 bits; with it, for every output and state a bound of the error that steps with relative
    error 1 would make: what is added to a column at a token carries a step's error, and an error moves on as the column
    does (times a <= 1, and 1 - beta k k^T <= 1 for keys up to length one and beta in 0..2)."""
    dk, dv = k.shape[2], v.shape[2]
    out, oerr = np.zeros(v.shape), np.zeros(v.shape)
    S = np.zeros((len(lens), heads, dk, dv)) if state is None else state.astype(np.float64).copy()
    serr = np.zeros((len(lens), heads, dv))
    rep = heads // key_heads
    t = 0
    for s, n in enumerate(lens):
        recent = np.zeros((heads, dv))  # |u| of a chunk's tokens
        err = np.zeros((heads, dv))
        for i in range(n):
            kk, qq = np.repeat(k[t], rep, 0), np.repeat(q[t], rep, 0)
            a = np.exp(g[t])[:, None, None]
            before = np.where(np.isneginf(g[t])[:, None, None], 0.0, a * S[s])
            seen = np.einsum("hk,hkv->hv", kk, before)
            u = beta[t][:, None] * (v[t] - seen)
            S[s] = before + kk[:, :, None] * u[:, None, :]
            out[t] = np.einsum("hk,hkv->hv", qq, S[s]) * scale
            recent += np.abs(u)
            norm = np.sqrt((before ** 2).sum(1)) + np.sqrt((S[s] ** 2).sum(1))
            step = norm + beta[t][:, None] * np.abs(v[t]) + recent
            err = err * np.exp(g[t])[:, None] + step
            oerr[t] = abs(scale) * np.sqrt((qq ** 2).sum(1))[:, None] * (err + norm + recent)
            serr[s] = err
            if i % 64 == 63:
                recent[:] = 0
            t += 1
    return out, S, oerr, serr


def delta_case(rng, lens, heads, key_heads, dk, dv, state, pace=0.2):
    n = sum(lens)
    q, k = rng.normal(0, 1, (n, key_heads, dk)), rng.normal(0, 1, (n, key_heads, dk)) + 0.4 * rng.normal(0, 1, (1, key_heads, dk))
    q, k = (t / np.maximum(np.sqrt((t ** 2).sum(2, keepdims=True)), 1e-9) for t in (q, k))
    return dict(q=q, k=k * 0.99, v=rng.normal(0, 1, (n, heads, dv)), g=-pace * rng.exponential(1.0, (n, heads)),
                beta=rng.uniform(0, 1, (n, heads)),
                state=rng.normal(0, 0.5, (len(lens), heads, dk, dv)).astype(np.float32) if state else None)


def run_delta(hip, c, lens, heads, key_heads, dk, dv, dtype, scale, layout="packed", reserve=False, in_place=False):
    """One call; the arrays' values as held, the outputs and the states."""
    n, es = sum(lens), 4 if dtype == "f32" else 2
    wk, wv = key_heads * dk, heads * dv
    sq, hq = typed(c["q"].reshape(n, wk), dtype)
    sk, hk = typed(c["k"].reshape(n, wk), dtype)
    sv, hv = typed(c["v"].reshape(n, wv), dtype)
    gates = np.concatenate([c["g"], c["beta"]], 1).astype(np.float32)
    uniform = len(set(lens)) == 1
    with Held(hip) as h:
        if layout == "row":  # one projection's rows, the outputs behind them
            buf = h.up(np.concatenate([sq, sk, sv, np.full((n, wv), 7, sv.dtype)], 1))
            ld = 2 * wk + 2 * wv
            ptrs, lds = [buf.ptr + es * o for o in (0, wk, 2 * wk)], [ld] * 3
            out_ptr, ld_out, out = buf.ptr + es * (2 * wk + wv), ld, buf
        else:
            off = {"packed": 0, "odd": 1}[layout]
            ups = [h.up(np.concatenate([np.zeros(off, a.dtype), a.ravel()])) for a in (sq, sk, sv)]
            ptrs, lds = [u.ptr + es * off for u in ups], [wk, wk, wv]
            out = h.new((n, wv + 3), sv.dtype, 7)
            out_ptr, ld_out = out.ptr, wv + 3
        dg = h.up(gates)
        state = None if c["state"] is None else h.up(c["state"])
        last = state if in_place and state else h.new((len(lens), heads, dk, dv), np.float32, 7.0)
        kw = dict(n_seqs=len(lens), seq_len=lens[0]) if uniform else dict(lens=lens)
        if reserve:
            hip.delta_rule_reserve(dtype, heads, dk, dv, **kw)
        hip.delta_rule_resident(*ptrs, dg.ptr, dg.ptr + 4 * heads, dtype, heads, dk, dv, out_ptr, key_heads=key_heads,
                                scale=scale, state_in_ptr=state.ptr if state else None, state_out_ptr=last.ptr, ld_q=lds[0],
                                ld_k=lds[1], ld_v=lds[2], ld_gates=2 * heads, ld_out=ld_out, **kw)
        hip.synchronize()
        o = back(out, dtype)
        if layout == "row":
            np.testing.assert_array_equal(o[:, :2 * wk + wv], np.concatenate([hq, hk, hv], 1))
            o = o[:, 2 * wk + wv:]
        elif n:
            assert (out.to_host()[:, wv:] == 7).all()
            o = o[:, :wv]
        return (hq.reshape(n, key_heads, dk), hk.reshape(n, key_heads, dk), hv.reshape(n, heads, dv),
                o.reshape(n, heads, dv), last.to_host())


def delta_steps(dk, dtype):
    """Roundings of a step, in u: sums over d_key and a chunk's 64 tokens with some across lanes, the exponentials, the
    factors; in bf16 three products in a row of operands held in two bf16 parts, 2^-17 of each (outputs; states have
    none)."""
    return 2 * (dk + 64) + 32 + (3 * 2 * 2.0 ** -17 / U32 if dtype == "bf16" else 0)


def check_delta(hip, c, lens, heads, key_heads, dk, dv, dtype, scale=0.5, **kw):
    q, k, v, out, S = run_delta(hip, c, lens, heads, key_heads, dk, dv, dtype, scale, **kw)
    g, beta = c["g"].astype(np.float32).astype(np.float64), c["beta"].astype(np.float32).astype(np.float64)
    want, state, oerr, serr = delta64(q.astype(np.float64), k.astype(np.float64), v.astype(np.float64), g, beta, scale, lens,
                                      c["state"], heads, key_heads)
    steps = delta_steps(dk, dtype) * U32
    within(out, want, steps * oerr + (U16 if dtype == "bf16" else U32) * np.abs(want), "outputs")
    within(S, state, delta_steps(dk, "f32") * U32 * serr[:, :, None, :] + U32 * np.abs(state), "states")


DELTA_SHAPES = [  # lens, heads, key heads, d_key, d_val
    ([1], 1, 1, 1, 1), ([1, 1, 1], 2, 1, 16, 32), ([1] * 5, 4, 4, 64, 64), ([2, 3, 1, 4], 2, 2, 20, 9), ([5], 3, 1, 64, 64),
    ([0, 7, 0, 1], 2, 1, 32, 40), ([63], 1, 1, 64, 64), ([64], 2, 1, 64, 64), ([65], 2, 2, 128, 128), ([128, 128], 2, 2, 32, 64),
    ([200, 31, 64, 1, 129], 3, 3, 64, 72), ([300], 2, 1, 100, 72), ([33, 96, 70], 2, 1, 128, 192), ([17, 18], 1, 1, 30, 130),
    ([700], 1, 1, 128, 64), ([40, 41], 2, 2, 7, 5), ([90, 130], 4, 2, 48, 16), ([1500], 1, 1, 64, 64)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens,heads,key_heads,dk,dv", DELTA_SHAPES)
def test_delta_rule(hip, dtype, lens, heads, key_heads, dk, dv):
    say("delta", dtype, lens, heads, key_heads, dk, dv)
    rng = np.random.default_rng(sum(lens) + dk)
    check_delta(hip, delta_case(rng, lens, heads, key_heads, dk, dv, True), lens, heads, key_heads, dk, dv, dtype, reserve=True)
    check_delta(hip, delta_case(rng, lens, heads, key_heads, dk, dv, False, pace=0.01), lens, heads, key_heads, dk, dv, dtype,
                layout="odd")
    check_delta(hip, delta_case(rng, lens, heads, key_heads, dk, dv, True, pace=2.0), lens, heads, key_heads, dk, dv, dtype,
                layout="row", in_place=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_delta_rule_of_many_ragged_sequences(hip, dtype):
    """More lengths than a kernel's arguments hold."""
    rng = np.random.default_rng(9)
    lens = [int(n) for n in rng.integers(0, 12, 300)]
    check_delta(hip, delta_case(rng, lens, 2, 1, 16, 24, True), lens, 2, 1, 16, 24, dtype, reserve=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [3, 150])
def test_delta_rule_extreme_gates_and_keys(hip, dtype, n):
    """Tokens that forget all before them, that do not decay, that do not update, whose update replaces; keys of zero;
    keys that are all alike."""
    rng = np.random.default_rng(11)
    c = delta_case(rng, [n], 2, 1, 32, 48, True)
    c["g"][1::7] = -np.inf
    c["g"][2::5] = 0.0
    c["g"][4::9] = -150.0
    c["beta"][0::4] = 0.0
    c["beta"][2::4] = 1.0
    c["beta"][3::8] = 2.0
    c["k"][5::6] = 0.0
    check_delta(hip, c, [n], 2, 1, 32, 48, dtype)
    c = delta_case(rng, [n], 1, 1, 64, 64, False, pace=0.001)
    c["k"][:] = c["k"][0]
    c["beta"][:] = 1.0
    check_delta(hip, c, [n], 1, 1, 64, 64, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("what", ["v", "k", "q", "g", "beta", "state"])
@pytest.mark.parametrize("n,at", [(4, 2), (200, 100), (70, 0)])
def test_delta_rule_values_that_are_not_finite(hip, dtype, what, n, at):
    """A NaN reaches the outputs from its own token on and no earlier one, its own sequence, and for v its own column; a
    query's its own token."""
    rng = np.random.default_rng(12)
    lens = [n, 66]
    c = delta_case(rng, lens, 2, 1, 32, 40, True)
    if what == "state":
        c["state"][0, 1, 3, 5] = np.nan
        at = 0
    else:
        index = {"v": (at, 1, 7), "k": (at, 0, 3), "q": (at, 0, 3), "g": (at, 1), "beta": (at, 1)}[what]
        c[what][index] = np.nan
    q, k, v, out, S = run_delta(hip, c, lens, 2, 1, 32, 40, dtype, 1.0)
    clean = {x: (None if y is None else np.where(np.isnan(y), 0, y).astype(y.dtype)) for x, y in c.items()}
    _, _, _, plain, S0 = run_delta(hip, clean, lens, 2, 1, 32, 40, dtype, 1.0)
    heads = {"v": [1], "k": [0, 1], "q": [0, 1], "g": [1], "beta": [1], "state": [1]}[what]
    col = {"v": [7], "state": [5]}.get(what, list(range(40)))
    bad = np.zeros(out.shape, bool)
    last = at + 1 if what == "q" else n
    for h in heads:
        bad[at:last, h, col] = True
    np.testing.assert_array_equal(np.isnan(out), bad)
    # What it does not reach is as near the sound call's as another order of sums leaves it.
    scale = np.abs(plain).max()
    assert np.abs(out - plain)[~bad].max() <= scale * ((U16 * 2 if dtype == "bf16" else 0) + delta_steps(32, dtype) * 64 * U32)
    if what == "q":
        assert np.isfinite(S).all()
    else:
        assert np.isnan(S[0, heads][:, :, col]).all()
        assert np.isfinite(S[1]).all() and np.isfinite(np.delete(S[0, 1], col, 1)).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens,heads,key_heads,dk,dv", [([3000], 1, 1, 64, 64), ([2177], 2, 1, 128, 72), ([1300, 1300], 1, 1, 32, 40),
                                                        ([1700, 3, 0, 900, 64], 2, 2, 64, 64), ([1601], 1, 1, 100, 130)])
def test_delta_rule_in_segments(hip, dtype, lens, heads, key_heads, dk, dv):
    """Few long walks are split; a forgotten state is forgotten across segments, and a NaN stays behind its token."""
    say("segments", dtype, lens, heads, dk, dv)
    rng = np.random.default_rng(sum(lens))
    c = delta_case(rng, lens, heads, key_heads, dk, dv, True, pace=0.01)
    c["g"][lens[0] // 2] = -np.inf
    check_delta(hip, c, lens, heads, key_heads, dk, dv, dtype, reserve=True)
    check_delta(hip, delta_case(rng, lens, heads, key_heads, dk, dv, False, pace=0.1), lens, heads, key_heads, dk, dv, dtype,
                layout="row")
    clean = run_delta(hip, c, lens, heads, key_heads, dk, dv, dtype, 1.0)
    at, again = lens[0] // 3, lens[0] // 2
    c["v"][at, 0, 1] = np.nan
    c["state"][0, 0, 0, 0] = np.nan
    out = run_delta(hip, c, lens, heads, key_heads, dk, dv, dtype, 1.0)
    bad = np.zeros(clean[3].shape, bool)
    bad[at:again, 0, 1] = bad[:again, 0, 0] = True  # what is forgotten is no more
    np.testing.assert_array_equal(np.isnan(out[3]), bad)
    assert np.isfinite(out[4]).all()
    scale = np.abs(clean[3]).max()
    assert np.abs(out[3] - clean[3])[~bad].max() <= scale * ((U16 * 2 if dtype == "bf16" else 0) + delta_steps(dk, dtype) * 64 * U32)


def test_delta_rule_single_tokens_continue_a_prompt(hip):
    """A prompt, then single tokens from its state, equal the whole sequence."""
    rng = np.random.default_rng(13)
    heads, dk, dv, n = 2, 64, 64, 133
    c = delta_case(rng, [n], heads, 1, dk, dv, False)
    whole = run_delta(hip, c, [n], heads, 1, dk, dv, "f32", 1.0)
    cut = 130
    part = {x: (y if y is None else y[:cut]) for x, y in c.items()}
    first = run_delta(hip, part, [cut], heads, 1, dk, dv, "f32", 1.0)
    state, outs = first[4], [first[3]]
    for t in range(cut, n):
        part = {x: (y if y is None else y[t:t + 1]) for x, y in c.items()}
        part["state"] = state
        r = run_delta(hip, part, [1], heads, 1, dk, dv, "f32", 1.0)
        outs.append(r[3])
        state = r[4]
    tol = delta_steps(dk, "f32") * U32 * 64  # both within a step's roundings over the memory of some 64 tokens
    np.testing.assert_allclose(np.concatenate(outs), whole[3], rtol=0, atol=tol * np.abs(whole[3]).max())
    np.testing.assert_allclose(state, whole[4], rtol=0, atol=tol * np.abs(whole[4]).max())


# ---------------------------------------------------------------------------
# Beam search


def candidates64(z, scores, last, eos):
    """[beams, vocab] values of a group in 64 bits, -inf where there is no candidate."""
    z = z.astype(np.float64)
    val = np.full(z.shape, -np.inf)
    for b in range(len(z)):
        if not np.isfinite(scores[b]):
            continue
        if last is not None and last[b] == eos:
            val[b, eos] = scores[b]
        elif not (np.isnan(z[b]).any() or (z[b] == np.inf).any() or (z[b] == -np.inf).all()):
            m = z[b].max()
            val[b] = np.float64(scores[b]) + (z[b] - (np.log(np.exp(z[b] - m).sum()) + m))
    return val


def check_beams(hip, z, scores, last, eos, keep, dtype, pad=0, offset=0, in_place=False):
    """z [groups, beams, vocab]."""
    groups, beams, vocab = z.shape
    stored, held = wide_rows(z.reshape(-1, vocab), vocab + pad, dtype, offset, fill=3e30)
    scores = scores.astype(np.float32)
    with Held(hip) as h:
        dz, ds = h.up(stored), h.up(scores)
        dl = None if last is None else h.up(last.astype(np.uint32))
        par = h.new((groups, keep), np.uint32, 7)
        tok = dl if in_place and dl else h.new((groups, keep), np.uint32, 7)
        out = ds if in_place else h.new((groups, keep), np.float32, 7.0)
        hip.beam_select_resident(dz.ptr + offset * stored.itemsize, dtype, groups, beams, vocab, ds.ptr, keep, par.ptr,
                                 tok.ptr, out.ptr, last_ptr=dl.ptr if dl else None, eos=eos, ld=vocab + pad)
        hip.synchronize()
        par, tok, out = (x.to_host().reshape(groups, keep) for x in (par, tok, out))
    held = held.reshape(z.shape)
    for g in range(groups):
        val = candidates64(held[g], scores[g], None if last is None else last[g], eos)
        flat = val.ravel()
        order = np.argsort(-flat, kind="stable")[:keep]
        order = order[flat[order] > -np.inf]
        n = len(order)
        assert (par[g, n:] == NONE).all() and (tok[g, n:] == NONE).all() and (out[g, n:] == -np.inf).all()
        # The sums' terms are fp32 exponentials, two roundings of an argument d with weight e^-d and one of their own.
        near = 4 * U32
        want = flat[order]
        within(out[g, :n], want, U32 * np.abs(want) + near, "scores")
        got = par[g, :n].astype(np.int64) * vocab + tok[g, :n]
        for i in range(n):  # another candidate only where the two are as near as that
            assert got[i] == order[i] or abs(flat[got[i]] - want[i]) <= 2 * near, (g, i, got[i], order[i], flat[got[i]], want[i])
        assert len(set(got.tolist())) == n
        same = np.diff(want) == 0
        np.testing.assert_array_equal(got[1:][same], order[1:][same])  # equal values by beam, then by token


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("groups,beams,vocab,keep", [(1, 1, 1, 1), (1, 1, 5, 8), (2, 4, 100, 4), (3, 5, 1023, 10), (1, 4, 16384, 4),
                                                    (2, 2, 50001, 5), (1, 64, 300, 64), (1, 1, 131072, 64), (70, 8, 2049, 8),
                                                    (600, 4, 513, 4), (5, 3, 8193, 17)])
def test_beam_select(hip, dtype, groups, beams, vocab, keep):
    say("beam", dtype, groups, beams, vocab, keep)
    rng = np.random.default_rng(groups + beams + vocab + keep)
    z = rng.normal(0, 2.5, (groups, beams, vocab))
    scores = rng.normal(-20, 2, (groups, beams))
    check_beams(hip, z, scores, None, NONE, keep, dtype, pad=3, offset=1)
    last = rng.integers(0, min(vocab, 4), (groups, beams))
    z[rng.random(z.shape) < 0.3] = -np.inf
    check_beams(hip, z, scores, last, 0, keep, dtype, in_place=keep == beams)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_beam_select_ties_masks_and_beams_without_candidates(hip, dtype):
    rng = np.random.default_rng(21)
    z = np.round(rng.normal(0, 1, (6, 4, 700)) * 4) / 4  # many equal logits
    scores = np.full((6, 4), -3.0)
    z[0] = z[0, 0]  # equal beams: ties across them
    z[1] = 1.25  # all tokens equal
    z[2, 0] = -np.inf
    z[2, 1, 5] = np.nan
    z[2, 2, 6] = np.inf
    z[3], z[3, :, 9] = -np.inf, 2.0  # one token left in each beam
    scores[4] = [-np.inf, np.nan, np.inf, -7.0]
    scores[5] = -np.inf
    check_beams(hip, z, scores, None, NONE, 8, dtype)
    z[z < 0] = np.finfo(np.float32).min if dtype == "f32" else -3.3895e38  # masks of the type's lowest value
    check_beams(hip, z, scores, None, NONE, 64, dtype)
    last = np.full((6, 4), 3)
    last[0, 1] = last[4, 3] = last[5, 0] = 1
    last[3] = 1
    check_beams(hip, z, scores, last, 1, 4, dtype, in_place=True)


def test_beam_select_takes_a_tokens_id_as_its_sign_of_the_end(hip):
    """The end may lie outside the vocabulary; -0 and 0 are equal logits."""
    z = np.zeros((1, 2, 40))
    z[0, :, ::2] = -0.0
    check_beams(hip, z, np.array([[-1.0, -1.0]]), np.array([[7, 8]]), 7, 40, "f32")


@pytest.mark.parametrize("row_bytes,n_in,n_out,pad", [(16, 4, 4, 0), (4096, 1, 8, 0), (1000, 8, 8, 0), (37, 5, 3, 2), (160, 17, 33, 16),
                                                      (64, 64, 64, 0), (20, 40, 40, 4), (196608, 3, 3, 0)])
def test_beam_gather(hip, row_bytes, n_in, n_out, pad):
    rng = np.random.default_rng(row_bytes)
    groups, ld = 5, row_bytes + pad
    src = rng.integers(0, 256, (groups, n_in, ld)).astype(np.uint8)
    par = rng.integers(0, n_in, (groups, n_out)).astype(np.uint32)
    par[1, 0], par[2, n_out - 1] = NONE, n_in
    with Held(hip) as h:
        ds, dp, dd = h.up(src), h.up(par), h.new((groups, n_out, ld), np.uint8, 7)
        hip.beam_gather_resident(ds.ptr, dd.ptr, row_bytes, groups, n_in, dp.ptr, n_out, ld_src=ld, ld_dst=ld)
        hip.synchronize()
        want = np.full((groups, n_out, ld), 7, np.uint8)
        for g in range(groups):
            for j in range(n_out):
                if par[g, j] < n_in:
                    want[g, j, :row_bytes] = src[g, par[g, j], :row_bytes]
        np.testing.assert_array_equal(dd.to_host(), want)
        np.testing.assert_array_equal(ds.to_host(), src)
        if n_in != n_out:
            return
        hip.beam_gather_resident(ds.ptr, ds.ptr, row_bytes, groups, n_in, dp.ptr, n_out, ld_src=ld, ld_dst=ld)
        hip.synchronize()
        want = src.copy()
        for g in range(groups):
            for j in range(n_out):
                if par[g, j] < n_in:
                    want[g, j, :row_bytes] = src[g, par[g, j], :row_bytes]
        np.testing.assert_array_equal(ds.to_host(), want)


# ---------------------------------------------------------------------------
# Beam search on a model's lanes


def small_layer(hip, lanes, loops=1, dtype="f32"):
    cfg = PSSAConfig(depth=2, d_vocab=97, d_latent=64, d_state=16, d_mem_key=16, mem_capacity=32)
    w = ModelWeights.init(cfg, 5, "baseline")
    w.unembed *= 40.0  # logits apart enough to rank
    w.populate_banks(2, count=24)
    layer = PSSALayer(hip, w, lanes=lanes, max_tokens=lanes * 16, weight_dtype=dtype)
    if loops > 1:
        layer.set_loops(loops)
    return layer


def search64(layer, prompts, beams, steps, eos):
    """Beam search by whole forward passes of every beam's tokens, one at a time."""
    n = len(prompts)
    ids, scores = np.zeros((n, beams, steps), np.uint32), np.full((n, beams), -np.inf)

    def next_logits(tokens):
        layer.reset_recurrent_state()
        return layer.prefill_inference(np.array([tokens]))[0]

    for g, prompt in enumerate(prompts):
        live = [([], 0.0)]
        for _ in range(steps):
            z = np.stack([next_logits(list(prompt) + t) for t, _ in live])
            last = np.array([t[-1] for t, _ in live]) - 1 if live[0][0] and eos != NONE else None
            val = candidates64(z[:, 1:], np.array([s for _, s in live]), last, eos - 1)
            order = np.argsort(-val.ravel(), kind="stable")[:beams]
            live = [(live[i // val.shape[1]][0] + [int(i % val.shape[1]) + 1], val.ravel()[i]) for i in order]
        for b, (t, s) in enumerate(live):
            ids[g, b], scores[g, b] = t, s
    return ids, scores


@pytest.mark.parametrize("loops", [1, 2])
@pytest.mark.parametrize("groups,beams,steps", [(1, 1, 4), (1, 4, 6), (3, 3, 5), (2, 5, 1)])
def test_beam_search_equals_one_by_one(hip, groups, beams, steps, loops):
    say("search", groups, beams, steps, loops)
    rng = np.random.default_rng(groups * 10 + beams)
    prompts = rng.integers(1, 97, (groups, 7))
    layer = small_layer(hip, groups * beams, loops)
    eos = NONE
    for _ in range(2):
        layer.reset_recurrent_state()
        layer.prefill_inference(prompts)
        ids, scores = layer.beam_search(steps, beams, eos=eos)
        # The next tokens of the best beams continue from the lanes' states.
        follow = layer.forward_inference(ids[:, :, -1].ravel())
        want, ws = search64(layer, prompts, beams, steps, eos)
        np.testing.assert_array_equal(ids, want)
        np.testing.assert_allclose(scores, ws, rtol=0, atol=1e-4 * steps * np.abs(follow).max())  # the forward's gate
        for g in range(groups):
            for b in range(beams):
                layer.reset_recurrent_state()
                z = layer.prefill_inference(np.array([list(prompts[g]) + ids[g, b].tolist()]))[0]
                np.testing.assert_allclose(follow[g * beams + b], z, rtol=0, atol=1e-4 * np.abs(z).max())
        eos = int(want[0, 0, 0])  # now with a token that ends the first beam at once
    layer.close()


def test_beam_search_greedy_is_one_beam(hip):
    """One beam is the greedy decode, and searching it leaves the model as decoding does."""
    rng = np.random.default_rng(31)
    prompts = rng.integers(1, 97, (3, 6))
    layer = small_layer(hip, 3)
    layer.prefill_inference(prompts)
    ids, _ = layer.beam_search(8, 1)
    carry = layer.get_carry()
    layer.reset_recurrent_state()
    layer.prefill_inference(prompts)
    greedy = layer.decode(8)
    np.testing.assert_array_equal(ids[:, 0, :], greedy.T)
    np.testing.assert_allclose(carry, layer.get_carry(), rtol=0, atol=1e-4 * np.abs(carry).max())
    layer.close()


def test_beam_search_refuses(hip):
    layer = small_layer(hip, 4)
    layer.prefill_inference(np.ones((2, 3), np.uint32))
    with pytest.raises(_abi.HipError, match="lanes"):
        layer.beam_search(2, 3)
    with pytest.raises(_abi.HipError, match="last prefill"):
        layer.beam_search(2, 2, n_groups=1)
    layer.set_repetition_penalty(1.25)
    with pytest.raises(_abi.HipError, match="repetition"):
        layer.beam_search(2, 2)
    layer.set_repetition_penalty(1.0)
    layer.set_sampling(0.7)
    with pytest.raises(_abi.HipError, match="sampling"):
        layer.beam_search(2, 2)
    layer.set_sampling(0.0)
    layer.beam_search(2, 2)
    with pytest.raises(_abi.HipError, match="last prefill"):
        layer.beam_search(2, 2, n_groups=2)
    layer.close()


# ---------------------------------------------------------------------------
# Together


def test_a_serving_step(hip):
    """Norm and 8-bit rows, the projection, the delta rule, its norm, the head, the selection, the states reordered: every
    stage against its definition on what the stage before it left."""
    rng = np.random.default_rng(41)
    groups, beams, d, heads, dk, dv, vocab = 3, 4, 256, 4, 64, 64, 1000
    n, width = groups * beams, 2 * heads * dk + heads * dv
    x, res, gamma = stream(rng, n, d), rng.normal(0, 1, (n, d)), rng.normal(1, 0.2, d)
    w_in = rng.normal(0, d ** -0.5, (width, d)).astype(np.float32)
    w_head = rng.normal(0, 2 * (heads * dv) ** -0.5, (vocab, heads * dv)).astype(np.float32)
    gates = np.concatenate([-rng.exponential(0.1, (n, heads)), rng.uniform(0, 1, (n, heads))], 1).astype(np.float32)
    state = rng.normal(0, 0.3, (n, heads, dk, dv)).astype(np.float32)
    scores = rng.normal(-9, 1, (groups, beams)).astype(np.float32)
    with Held(hip) as h:
        up, new = h.up, h.new
        bx, hx = to_bf16(x)
        br, hr = to_bf16(res)
        dx, dr, dg = up(bx), up(br), up(gamma.astype(np.float32))
        wq, wc, hq, hc = new((width, d), np.int8, 0), new(width, np.float32, 0), new((vocab, heads * dv), np.int8, 0), new(vocab, np.float32, 0)
        dw, dh = up(w_in), up(w_head)
        hip.quantize_i8_resident(dw.ptr, "f32", width, d, wq.ptr, wc.ptr)
        hip.quantize_i8_resident(dh.ptr, "f32", vocab, heads * dv, hq.ptr, hc.ptr)
        ds, q1, c1 = new((n, d), np.uint16, 0), new((n, d), np.int8, 0), new(n, np.float32, 0)
        row, o = new((n, width), np.uint16, 0), new((n, heads * dv), np.uint16, 0)
        dgate, dstate, moved = up(gates), up(state), new((n, heads, dk, dv), np.float32, 0)
        q2, c2, ones, logits = new((n, heads * dv), np.int8, 0), new(n, np.float32, 0), up(np.ones(heads * dv, np.float32)), new((n, vocab), np.float32, 0)
        dsc, par, tok = up(scores), new((groups, beams), np.uint32, 0), new((groups, beams), np.uint32, 0)
        hip.rms_norm_resident(dx.ptr, "bf16", n, d, dg.ptr, dr.ptr, sum_ptr=ds.ptr, codes_ptr=q1.ptr, scales_ptr=c1.ptr)
        hip.matmul_i8_resident(q1.ptr, c1.ptr, wq.ptr, wc.ptr, n, width, d, row.ptr, "bf16")
        hip.delta_rule_resident(row.ptr, row.ptr + 2 * heads * dk, row.ptr + 4 * heads * dk, dgate.ptr, dgate.ptr + 4 * heads,
                                "bf16", heads, dk, dv, o.ptr, n_seqs=n, seq_len=1, scale=0.125, state_in_ptr=dstate.ptr,
                                state_out_ptr=dstate.ptr, ld_q=width, ld_k=width, ld_v=width, ld_gates=2 * heads)
        hip.rms_norm_resident(o.ptr, "bf16", n, heads * dv, ones.ptr, codes_ptr=q2.ptr, scales_ptr=c2.ptr)
        hip.matmul_i8_resident(q2.ptr, c2.ptr, hq.ptr, hc.ptr, n, vocab, heads * dv, logits.ptr)
        hip.beam_select_resident(logits.ptr, "f32", groups, beams, vocab, dsc.ptr, beams, par.ptr, tok.ptr, dsc.ptr)
        hip.beam_gather_resident(dstate.ptr, moved.ptr, heads * dk * dv * 4, groups, beams, par.ptr, beams)
        hip.synchronize()
        h32 = (hx + hr).astype(np.float32)
        np.testing.assert_array_equal(q1.to_host(), codes32(h32 * gamma.astype(np.float32))[0])
        np.testing.assert_array_equal(ds.to_host(), to_bf16(h32)[0])
        y = (q1.to_host().astype(np.float64) @ wq.to_host().astype(np.float64).T) * c1.to_host()[:, None].astype(np.float64) * wc.to_host().astype(np.float64)
        got = from_bf16(row.to_host())
        within(got, y, np.abs(y) * (U16 + 3.01 * U32) + 1e-44, "projection")
        q, k, v = (got[:, i * heads * dk:(i + 1) * heads * dk].reshape(n, heads, dk).astype(np.float64) for i in range(3))
        before = np.exp(gates[:, :heads].astype(np.float64))[..., None, None] * state
        u = gates[:, heads:, None].astype(np.float64) * (v - np.einsum("nhk,nhkv->nhv", k, before))
        after = before + k[..., None] * u[:, :, None, :]
        mass = np.abs(before) + np.abs(k)[..., None] * (np.abs(gates[:, heads:, None]) * (np.abs(v) + np.einsum("nhk,nhkv->nhv", np.abs(k), np.abs(before))))[:, :, None, :]
        within(dstate.to_host(), after, (dk + 40) * U32 * mass, "states")
        want = np.einsum("nhk,nhkv->nhv", q, after) * 0.125
        lim = np.einsum("nhk,nhkv->nhv", np.abs(q), mass) * 0.125
        within(from_bf16(o.to_host()).reshape(n, heads, dv), want, U16 * np.abs(want) + 2 * (dk + 40) * U32 * lim, "outputs")
        np.testing.assert_array_equal(q2.to_host(), codes32(from_bf16(o.to_host()))[0])
        z = logits.to_host()
        y = (q2.to_host().astype(np.float64) @ hq.to_host().astype(np.float64).T) * c2.to_host()[:, None].astype(np.float64) * hc.to_host().astype(np.float64)
        within(z, y, np.abs(y) * 3.01 * U32 + 1e-44, "logits")
        par, tok = par.to_host(), tok.to_host()
        for g in range(groups):
            val = candidates64(z[g * beams:(g + 1) * beams], scores[g], None, NONE).ravel()
            np.testing.assert_array_equal(par[g].astype(np.int64) * vocab + tok[g], np.argsort(-val, kind="stable")[:beams])
        rows = (np.arange(groups)[:, None] * beams + par).ravel()
        np.testing.assert_array_equal(moved.to_host(), dstate.to_host()[rows])


def test_two_contexts_at_once(hip):
    """Each context has its stream and scratch."""
    other = HipDevice(0)
    try:
        rng = np.random.default_rng(51)
        lens = [150, 3, 70]
        c = delta_case(rng, lens, 2, 1, 64, 64, True)
        want = run_delta(hip, c, lens, 2, 1, 64, 64, "bf16", 0.5)
        for _ in range(3):
            got = run_delta(other, c, lens, 2, 1, 64, 64, "bf16", 0.5)
            np.testing.assert_array_equal(got[3], want[3])
            np.testing.assert_array_equal(got[4], want[4])
            check_i8(hip, 40, 40, 20000)
    finally:
        other.close()


# ---------------------------------------------------------------------------
# Offsets past 31 and 32 bits


class Far(Held):
    """Arrays of rows far apart, of which only the rows are written and read."""

    def rows(self, values, ld):
        b = self.dev.empty(((len(values) - 1) * ld + values.shape[1],), values.dtype)
        self.bufs.append(b)
        for i, row in enumerate(values):
            b.write(row, i * ld * values.itemsize)
        return b

    def back(self, buf, n, width, ld):
        out = np.empty((n, width), buf.dtype)
        for i in range(n):
            _abi.call(self.dev._lib.pssa_hip_memcpy, self.dev.handle, out[i].ctypes.data, buf.ptr + i * ld * out.itemsize,
                      out[i].nbytes, _abi.D2H)
        return out


def test_norm_rows_far_apart(hip):
    rng = np.random.default_rng(61)
    rows, width, ld = 3, 100, 2 ** 31 - 1
    stored, held = to_bf16(stream(rng, rows, width))
    g = rng.normal(1, 0.2, width).astype(np.float32)
    with Far(hip) as h:
        x, codes = h.rows(stored, ld), h.rows(np.zeros((rows, width), np.int8), ld)
        dg, sc, out = h.up(g), h.new(rows, np.float32, 0), h.new((rows, width), np.uint16, 0)
        hip.rms_norm_resident(x.ptr, "bf16", rows, width, dg.ptr, sum_ptr=x.ptr, out_ptr=out.ptr, codes_ptr=codes.ptr,
                              scales_ptr=sc.ptr, ld_x=ld, ld_sum=ld, ld_codes=ld)
        hip.synchronize()
        np.testing.assert_array_equal(h.back(x, rows, width, ld), stored)  # no residual: the sum is x
        np.testing.assert_array_equal(h.back(codes, rows, width, ld), codes32((held * g).astype(np.float32))[0])
        h64 = held.astype(np.float64)
        want = h64 / np.sqrt((h64 ** 2).mean(1, keepdims=True) + 1e-5) * g
        within(from_bf16(out.to_host()), want, np.abs(want) * (45 * U32 + U16), "out")


@pytest.mark.parametrize("m,ld", [(3, 2 ** 24), (70, 2 ** 24), (70, 2 ** 24 + 16)])
def test_matmul_i8_rows_far_apart(hip, m, ld):
    rng = np.random.default_rng(62)
    n, k = 300, 80
    x, w = rng.integers(-128, 128, (m, k)).astype(np.int8), rng.integers(-128, 128, (n, k)).astype(np.int8)
    with Far(hip) as h:
        dx, dw, ones, y = h.rows(x, ld), h.rows(w, ld), h.up(np.ones(max(m, n), np.float32)), h.new((m, n), np.float32, 0)
        hip.matmul_i8_resident(dx.ptr, ones.ptr, dw.ptr, ones.ptr, m, n, k, y.ptr, ld_x=ld, ld_w=ld)
        hip.synchronize()
        np.testing.assert_array_equal(y.to_host(), x.astype(np.float64) @ w.astype(np.float64).T)  # below 2^24: exact


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_delta_rule_rows_far_apart(hip, dtype):
    rng = np.random.default_rng(63)
    n, ld = 150, 2 ** 24 - 8
    c = delta_case(rng, [n], 1, 1, 64, 64, False)
    (sq, hq), (sk, hk), (sv, hv) = (typed(c[x].reshape(n, 64), dtype) for x in "qkv")
    gates = np.concatenate([c["g"], c["beta"]], 1).astype(np.float32)
    with Far(hip) as h:
        q, k, v, out = h.up(sq), h.rows(sk, ld), h.rows(sv, ld), h.rows(np.zeros((n, 64), sv.dtype), ld)
        dg = h.up(gates)
        hip.delta_rule_resident(q.ptr, k.ptr, v.ptr, dg.ptr, dg.ptr + 4, dtype, 1, 64, 64, out.ptr, n_seqs=1, seq_len=n,
                                scale=0.5, ld_k=ld, ld_v=ld, ld_gates=2, ld_out=ld)
        hip.synchronize()
        got = h.back(out, n, 64, ld)
    got = from_bf16(got) if dtype == "bf16" else got
    q, k, v = (a.astype(np.float64).reshape(n, 1, 64) for a in (hq, hk, hv))
    want, _, oerr, _ = delta64(q, k, v, gates[:, :1].astype(np.float64), gates[:, 1:].astype(np.float64), 0.5, [n], None, 1, 1)
    within(got.reshape(want.shape), want, delta_steps(64, dtype) * U32 * oerr + (U16 if dtype == "bf16" else U32) * np.abs(want), "outputs")


def test_beams_far_apart(hip):
    rng = np.random.default_rng(64)
    beams, vocab, ld = 9, 1000, 2 ** 28 + 1
    stored, held = to_bf16(rng.normal(0, 2.5, (beams, vocab)))
    scores = rng.normal(-20, 1, beams).astype(np.float32)
    with Far(hip) as h:
        z, sc = h.rows(stored, ld), h.up(scores)
        par, tok, out = h.new(beams, np.uint32, 7), h.new(beams, np.uint32, 7), h.new(beams, np.float32, 7)
        hip.beam_select_resident(z.ptr, "bf16", 1, beams, vocab, sc.ptr, beams, par.ptr, tok.ptr, out.ptr, ld=ld)
        hip.synchronize()
        val = candidates64(held, scores, None, NONE).ravel()
        order = np.argsort(-val, kind="stable")[:beams]
        np.testing.assert_array_equal(par.to_host().astype(np.int64) * vocab + tok.to_host(), order)
        within(out.to_host(), val[order], U32 * np.abs(val[order]) + 4 * U32, "scores")
        src, parents = rng.integers(0, 256, (3, 48)).astype(np.uint8), np.array([2, 2, 0], np.uint32)
        far = 2 ** 31 + 16
        a, dp, b = h.rows(src, far), h.up(parents), h.new((3, 48), np.uint8, 0)
        hip.beam_gather_resident(a.ptr, b.ptr, 48, 1, 3, dp.ptr, 3, ld_src=far, ld_dst=48)
        hip.beam_gather_resident(a.ptr, a.ptr, 48, 1, 3, dp.ptr, 3, ld_src=far, ld_dst=far)
        hip.synchronize()
        np.testing.assert_array_equal(b.to_host(), src[parents])
        np.testing.assert_array_equal(h.back(a, 3, 48, far), src[parents])


def test_calls_one_behind_another(hip):
    """Calls that share the scratch, in a row without a wait, two rounds of them: the second equals the first."""
    rng = np.random.default_rng(65)
    m, n, k, t, heads, vocab = 100, 500, 5000, 300, 2, 4000
    with Held(hip) as h:
        x, w, s = h.up(rng.integers(-128, 128, (m, k)).astype(np.int8)), h.up(rng.integers(-128, 128, (n, k)).astype(np.int8)), h.up(rng.uniform(0.1, 1, n).astype(np.float32))
        q, kk, v = (h.up(typed(rng.normal(0, 0.1, (t, heads * 64)), "bf16")[0]) for _ in range(3))
        g = h.up(np.concatenate([-rng.exponential(0.1, (t, heads)), rng.uniform(0, 1, (t, heads))], 1).astype(np.float32))
        z, sc = h.up(rng.normal(0, 2, (4, vocab)).astype(np.float32)), h.up(np.zeros(4, np.float32))
        outs = []
        for _ in range(2):
            y, o, S = h.new((m, n), np.float32, 0), h.new((t, heads * 64), np.uint16, 0), h.new((1, heads, 64, 64), np.float32, 0)
            par, tok, best = h.new(4, np.uint32, 0), h.new(4, np.uint32, 0), h.new(4, np.float32, 0)
            hip.matmul_i8_resident(x.ptr, s.ptr, w.ptr, s.ptr, m, n, k, y.ptr)
            hip.delta_rule_resident(q.ptr, kk.ptr, v.ptr, g.ptr, g.ptr + 4 * heads, "bf16", heads, 64, 64, o.ptr, n_seqs=1,
                                    seq_len=t, ld_gates=2 * heads, state_out_ptr=S.ptr)
            hip.beam_select_resident(z.ptr, "f32", 1, 4, vocab, sc.ptr, 4, par.ptr, tok.ptr, best.ptr)
            outs.append([y, o, S, par, tok, best])
        hip.synchronize()
        for a, b in zip(*outs):
            np.testing.assert_array_equal(a.to_host(), b.to_host())
        want = (x.to_host().astype(np.float64) @ w.to_host().astype(np.float64).T) * s.to_host()[:m, None].astype(np.float64) * s.to_host().astype(np.float64)
        within(outs[0][0].to_host(), want, np.abs(want) * 3.01 * U32, "product")


def test_beam_select_of_scores_that_round_the_logits_away(hip):
    """Values of a beam that are one in 64 bits: as many as there are, each once, in the places' order."""
    rng = np.random.default_rng(71)
    for vocab, beams, keep in [(40, 4, 16), (60, 64, 64)]:
        z = rng.normal(0, 1e-6, (2, beams, vocab)).astype(np.float32)
        with Held(hip) as h:
            dz, ds = h.up(z), h.up(np.full((2, beams), -1e14, np.float32))
            par, tok, out = h.new((2, keep), np.uint32, 7), h.new((2, keep), np.uint32, 7), h.new((2, keep), np.float32, 7.0)
            hip.beam_select_resident(dz.ptr, "f32", 2, beams, vocab, ds.ptr, keep, par.ptr, tok.ptr, out.ptr)
            hip.synchronize()
            got = par.to_host().astype(np.int64) * vocab + tok.to_host()
            assert (got < beams * vocab).all() and (out.to_host() == np.float32(-1e14)).all()
            assert (np.diff(got, axis=1) > 0).all()


def test_beam_search_of_more_beams_than_tokens(hip):
    """The first steps leave beams without a candidate, whose lanes run idle until there are enough."""
    cfg = PSSAConfig(depth=2, d_vocab=4, d_latent=64, d_state=16, d_mem_key=16, mem_capacity=32)
    w = ModelWeights.init(cfg, 5, "baseline")
    w.unembed *= 40.0
    layer = PSSALayer(hip, w, lanes=12, max_tokens=12 * 16)
    prompts = np.random.default_rng(72).integers(1, 4, (2, 5))
    for steps in (1, 2, 4):
        layer.reset_recurrent_state()
        layer.prefill_inference(prompts)
        ids, scores = layer.beam_search(steps, 6)
        want, ws = search64(layer, prompts, 6, steps, NONE)
        there = np.isfinite(ws)
        np.testing.assert_array_equal(np.isfinite(scores), there)
        np.testing.assert_array_equal(ids[there], want[there])
        assert (ids[~there] == NONE).all()
        np.testing.assert_allclose(scores[there], ws[there], rtol=0, atol=1e-4 * steps * np.abs(ws[there]).max())
    layer.close()


def test_beam_search_with_bf16_weights(hip):
    """The beams are different, best first, and have their tokens' summed log probabilities."""
    layer, steps, beams = small_layer(hip, 8, dtype="bf16"), 5, 4
    prompts = np.random.default_rng(73).integers(1, 97, (2, 7))
    layer.prefill_inference(prompts)
    ids, scores = layer.beam_search(steps, beams)
    assert (np.diff(scores, axis=1) <= 0).all()
    for g in range(2):
        assert len({tuple(t) for t in ids[g].tolist()}) == beams
        for b in range(beams):
            total, gate = 0.0, 0.0
            for t in range(steps):
                layer.reset_recurrent_state()
                z = layer.prefill_inference(np.array([list(prompts[g]) + ids[g, b, :t].tolist()]))[0].astype(np.float64)[1:]
                total += z[ids[g, b, t] - 1] - (np.log(np.exp(z - z.max()).sum()) + z.max())
                gate += 2 * 2e-2 * np.abs(z).max()  # the bf16 forward's gate, of the logit and of the sum's
            assert abs(scores[g, b] - total) <= gate
    layer.close()


def test_beam_search_behind_prompts_of_different_lengths(hip):
    rng = np.random.default_rng(74)
    prompts = [rng.integers(1, 97, n) for n in (9, 2, 5)]
    layer = small_layer(hip, 9)
    layer.prefill_ragged(prompts)
    ids, scores = layer.beam_search(4, 3)
    want, ws = search64(layer, prompts, 3, 4, NONE)
    np.testing.assert_array_equal(ids, want)
    np.testing.assert_allclose(scores, ws, rtol=0, atol=1e-4 * 4 * np.abs(ws).max())
    layer.close()


# ---------------------------------------------------------------------------
# What a call holds on its way to an output


def beside_ties(shape):
    """fp32 values a step above and a step below the middle of two bf16 neighbours: a value that was held in fewer bits
    on its way lies on the middle, and half of these are then rounded to the wrong side."""
    i = np.arange(np.prod(shape))
    tie = 1 + (2 * (i // 2 % 128) + 1) * 2.0 ** -8
    return ((tie + np.where(i % 2, 2.0 ** -23, -2.0 ** -23)) * 2.0 ** (i % 3 - 1) * np.where(i // 5 % 2, -1, 1)).reshape(shape).astype(np.float32)


@pytest.mark.parametrize("dk", [32, 64, 128])
@pytest.mark.parametrize("what", ["state", "update", "scale"])
def test_delta_rule_rounds_bf16_outputs_once(hip, dk, what):
    """Queries and keys of a single one leave one term in every sum, factors of one and powers of two leave it as it is:
    what fp32 holds is exact, and the output is its rounding."""
    rng = np.random.default_rng(dk)
    n, dv = min(dk, 64), 64
    at = rng.integers(0, np.arange(n) + 1)  # a token's query meets one key, of a token before it or its own
    eye, two = np.eye(dk)[:n, None], 2.0 ** (np.arange(n * dv) % 5 - 2).reshape(n, 1, dv)
    zero, one = np.zeros((n, 1)), np.ones((n, 1))
    base = dict(g=zero, k=eye, q=np.eye(dk)[at, None], v=two, state=None, beta=one)
    if what == "state":  # nothing is added to it
        state = beside_ties((1, 1, dk, dv))
        cases = [(dict(base, state=state, beta=zero), 1.0, state[0, 0, at])]
    elif what == "update":
        beta = np.abs(beside_ties((n, 1)))
        cases = [(dict(base, beta=beta), 1.0, (beta[:, :, None] * two)[at, 0])]
    else:
        cases = [(base, float(s), s * two[at, 0]) for s in beside_ties(64)[7::9]]
    for c, scale, want in cases:
        out = run_delta(hip, c, [n], 1, 1, dk, dv, "bf16", scale)[3]
        np.testing.assert_array_equal(out[:, 0], to_bf16(want)[1])


# ---------------------------------------------------------------------------
# Values that are not finite, across segments


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens,heads,dk,dv", [([3000], 1, 64, 64), ([2177, 1300], 2, 32, 72), ([1601], 1, 100, 40), ([4100], 2, 128, 64)])
def test_delta_rule_segments_pass_on_what_is_not_finite(hip, dtype, lens, heads, dk, dv):
    """Decays of e^-0.5 a token take a segment's transition below what fp32 holds, but no token forgets: a NaN stays."""
    say("segments, not finite", dtype, lens, heads, dk, dv)
    rng = np.random.default_rng(sum(lens) + dk)
    c = delta_case(rng, lens, heads, 1, dk, dv, True)
    c["g"][:] = -0.5 - 0.2 * rng.random(c["g"].shape)
    clean = run_delta(hip, c, lens, heads, 1, dk, dv, dtype, 1.0)
    at, n = 150, lens[0]
    c["v"][at, 0, 1] = np.nan
    c["state"][0, 0, dk - 1, 0] = np.nan
    c["state"][0, heads - 1, 3, dv - 1] = np.inf
    _, _, _, out, S = run_delta(hip, c, lens, heads, 1, dk, dv, dtype, 1.0)
    bad, gone = np.zeros(out.shape, bool), np.zeros(S.shape, bool)
    bad[at:n, 0, 1] = bad[:n, 0, 0] = bad[:n, heads - 1, dv - 1] = True
    gone[0, 0, :, :2] = gone[0, heads - 1, :, dv - 1] = True
    np.testing.assert_array_equal(np.isfinite(out), ~bad)
    np.testing.assert_array_equal(np.isfinite(S), ~gone)
    # What it does not reach is as near the sound call's as another order of sums leaves it.
    for got, was, there, u in ((out, clean[3], ~bad, U16 * 2 if dtype == "bf16" else 0), (S, clean[4], ~gone, 0)):
        assert np.abs(got - was)[there].max() <= np.abs(was).max() * (u + delta_steps(dk, "f32") * 64 * U32)


# ---------------------------------------------------------------------------
# Norms at the ends of fp32's range


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("width", [4, 700, 9000])
def test_norm_of_rows_near_the_largest_value(hip, dtype, width):
    """Rows whose squares' mean is past fp32's range by far are normed all the same."""
    rng = np.random.default_rng(width)
    x = rng.choice([-1.0, 1.0], (4, width)) * rng.uniform(0.3, 1.0, (4, width)) * np.array([[3e38], [1.2e38], [2e30], [3e19]])
    check_norm(hip, x, None, rng.uniform(0.2, 0.9, width), dtype, pad=1)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("eps", [1e-12, 1e-5])
def test_norm_scales_of_rows_near_the_least_value(hip, dtype, eps):
    """max|t| / 127 would be held in a few bits where it is below fp32's normal range, the scale itself is not."""
    rng = np.random.default_rng(17)
    x = rng.normal(0, 1, (4, 300)) * np.array([[1e-38], [3e-39], [4e-37], [1e-35]])
    check_norm(hip, x, None, rng.normal(1, 0.2, 300), dtype, eps=eps)


# ---------------------------------------------------------------------------
# Scratch: what a call takes


def free_bytes(dev):
    dev.synchronize()
    free, total = C.c_size_t(), C.c_size_t()
    assert C.CDLL("libamdhip64.so").hipMemGetInfo(C.byref(free), C.byref(total)) == 0
    return free.value


def test_matmul_i8_in_units_takes_no_scratch_for_copies(hip):
    m, n, k = 65, 2 ** 20, 512
    dev = HipDevice(0)
    try:
        with Held(dev) as h:
            x, w, y = h.up(np.ones((m, k), np.int8)), h.up(np.ones((n, k), np.int8)), dev.empty((m, n), np.float32)
            h.bufs.append(y)
            s = h.up(np.ones(n, np.float32))
            before = free_bytes(dev)
            dev.matmul_i8_resident(x.ptr, s.ptr, w.ptr, s.ptr, m, n, k, y.ptr)
            assert before - free_bytes(dev) < 64 << 20
            assert (y.to_host() == k).all()
            # Weights that begin at an odd byte are copied, and the rows stay.
            dev.matmul_i8_resident(x.ptr, s.ptr, w.ptr + 1, s.ptr, m, n - 1, k, y.ptr)
            taken = before - free_bytes(dev)
            assert n * k - (64 << 20) < taken < n * k + (64 << 20)
            assert (y.to_host().ravel()[:m * (n - 1)] == k).all()
    finally:
        dev.close()


def test_delta_rule_takes_scratch_for_the_rows_it_copies(hip):
    n, heads, dk, dv = 2 ** 17, 8, 128, 128
    dev = HipDevice(0)
    try:
        with Held(dev) as h:
            q, k, v = h.up(np.zeros((n + 1, dk), np.uint16)), h.up(np.zeros((n + 1, dk), np.uint16)), h.up(np.zeros((n + 1, heads * dv), np.uint16))
            g, out = h.up(np.zeros((n, 2 * heads), np.float32)), dev.empty((n, heads * dv), np.uint16)
            h.bufs.append(out)

            def call(off):
                dev.delta_rule_resident(q.ptr + off, k.ptr + off, v.ptr + off, g.ptr, g.ptr + 4 * heads, "bf16", heads, dk, dv,
                                        out.ptr, n_seqs=1, seq_len=n, key_heads=1, ld_gates=2 * heads)

            before = free_bytes(dev)
            call(0)
            own = before - free_bytes(dev)
            # 11 KiB a chunk and head; the states and transitions of at most a segment for two chunks.
            assert own < n // 64 * heads * (11 << 10) + n // 128 * heads * 2 * (dk * dv * 4) + (64 << 20)
            call(2)
            copies = 2 * n * dk * 2 + n * heads * dv * 2
            assert copies - (32 << 20) < before - free_bytes(dev) - own < copies + (32 << 20)
    finally:
        dev.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens,heads,key_heads,dk,dv", [([300, 70], 4, 2, 64, 64), ([2000], 2, 1, 100, 72), ([65], 3, 1, 7, 5)])
def test_delta_rule_of_odd_rows_in_a_context_of_its_own(hip, dtype, lens, heads, key_heads, dk, dv):
    """The first call of a context: its scratch is what this call takes."""
    c = delta_case(np.random.default_rng(81), lens, heads, key_heads, dk, dv, True)
    want = run_delta(hip, c, lens, heads, key_heads, dk, dv, dtype, 0.5, reserve=True)
    for layout in ("odd", "row"):
        dev = HipDevice(0)
        try:
            got = run_delta(dev, c, lens, heads, key_heads, dk, dv, dtype, 0.5, layout=layout)
            for a, b in zip(got[3:], want[3:]):
                np.testing.assert_array_equal(a, b)
        finally:
            dev.close()


# ---------------------------------------------------------------------------
# Two contexts, and values that are one


def test_two_contexts_run_at_once(hip):
    """Calls that take scratch, enqueued in turn on two contexts without a wait between them: each as if it ran alone."""
    rng = np.random.default_rng(91)
    m, n, k, heads, vocab, steps = 100, 300, 5001, 2, 9000, 6
    lens = [2100, 40, 700]
    t = sum(lens)
    host = []
    for _ in range(2):  # other values for each
        c = delta_case(rng, lens, heads, 1, 64, 64, True)
        host.append(dict(x=rng.integers(-128, 128, (m, k)).astype(np.int8), w=rng.integers(-128, 128, (n, k)).astype(np.int8),
                         s=rng.uniform(0.1, 1, n).astype(np.float32), q=to_bf16(c["q"].reshape(t, 64))[0], kk=to_bf16(c["k"].reshape(t, 64))[0],
                         v=to_bf16(c["v"].reshape(t, heads * 64))[0], g=np.concatenate([c["g"], c["beta"]], 1).astype(np.float32),
                         state=c["state"], z=rng.normal(0, 2, (8, vocab)).astype(np.float32), score=rng.normal(-9, 1, 8).astype(np.float32)))
    dev = [HipDevice(0), HipDevice(0)]
    held = [Held(d) for d in dev]
    try:
        arrays = [{x: h.up(a) for x, a in of.items()} for h, of in zip(held, host)]

        def outputs(h):
            return dict(y=h.new((m, n), np.float32, 0), o=h.new((t, heads * 64), np.uint16, 0), S=h.new((len(lens), heads, 64, 64), np.float32, 0),
                        par=h.new((2, 4), np.uint32, 0), tok=h.new((2, 4), np.uint32, 0), best=h.new((2, 4), np.float32, 0))

        def calls(d, a, o):
            yield lambda: d.matmul_i8_resident(a["x"].ptr, a["s"].ptr, a["w"].ptr, a["s"].ptr, m, n, k, o["y"].ptr)
            yield lambda: d.delta_rule_resident(a["q"].ptr, a["kk"].ptr, a["v"].ptr, a["g"].ptr, a["g"].ptr + 4 * heads, "bf16", heads, 64,
                                                64, o["o"].ptr, lens, key_heads=1, ld_gates=2 * heads, state_in_ptr=a["state"].ptr,
                                                state_out_ptr=o["S"].ptr)
            yield lambda: d.beam_select_resident(a["z"].ptr, "f32", 2, 4, vocab, a["score"].ptr, 4, o["par"].ptr, o["tok"].ptr, o["best"].ptr)

        alone = []
        for d, h, a in zip(dev, held, arrays):
            d.matmul_i8_reserve(m, n, k)
            d.delta_rule_reserve("bf16", heads, 64, 64, lens)
            d.beam_select_reserve(2, 4, vocab, 4)
            o = outputs(h)
            for call in calls(d, a, o):
                call()
                d.synchronize()
            alone.append({x: b.to_host() for x, b in o.items()})
        together = [[outputs(h) for _ in range(steps)] for h in held]
        for d in dev:
            d.synchronize()
        for i in range(steps):
            for pair in zip(*(calls(d, a, o[i]) for d, a, o in zip(dev, arrays, together))):
                for call in pair:
                    call()
        for d in dev:
            d.synchronize()
        for want, outs in zip(alone, together):
            for o in outs:
                for x, b in o.items():
                    np.testing.assert_array_equal(b.to_host(), want[x], err_msg=x)
        want = (host[0]["x"].astype(np.float64) @ host[0]["w"].astype(np.float64).T) * host[0]["s"][:m, None].astype(np.float64) * host[0]["s"].astype(np.float64)
        within(alone[0]["y"], want, np.abs(want) * 3.01 * U32, "product")
    finally:
        for h in held:
            h.__exit__()
        for d in dev:
            d.close()


@pytest.mark.parametrize("beams,vocab,keep", [(4, 40, 16), (3, 1000, 64), (2, 10, 16)])
def test_beam_select_keeps_the_larger_of_logits_whose_values_are_one(hip, beams, vocab, keep):
    """A score that rounds the logits away: the first beams' places, of a beam its largest logits, in the tokens' order."""
    z = np.random.default_rng(vocab).permutation(beams * vocab).reshape(1, beams, vocab).astype(np.float32) * 2.0 ** -20
    with Held(hip) as h:
        dz, ds = h.up(z), h.up(np.full((1, beams), -1e14, np.float32))
        par, tok, out = h.new(keep, np.uint32, 7), h.new(keep, np.uint32, 7), h.new(keep, np.float32, 7.0)
        hip.beam_select_resident(dz.ptr, "f32", 1, beams, vocab, ds.ptr, keep, par.ptr, tok.ptr, out.ptr)
        hip.synchronize()
        want = [b * vocab + i for b in range(beams) for i in sorted(np.argsort(-z[0, b])[:keep])][:keep]
        np.testing.assert_array_equal(par.to_host().astype(np.int64) * vocab + tok.to_host(), want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pace", [0.01, 0.3, 0.9])
def test_delta_rule_decays_to_the_last_bits(hip, dtype, pace):
    """The decays themselves: of a state of ones that nothing is added to, and of ones that tokens add.  An exponential
    is within a step of fp32 and the rounding of a fraction, three half steps; a chunk's two products and what the chunks
    before it left are four of them."""
    rng = np.random.default_rng(int(pace * 100))
    n, dk, dv = 64, 64, 64  # two chunks in fp32
    g = -pace * rng.uniform(0.8, 1.2, (n, 1))
    total = np.cumsum(g.astype(np.float32).astype(np.float64))
    tol = 4 * 4 * U32 + (U16 if dtype == "bf16" else 0)
    # The state.
    q = np.zeros((n, 1, dk))
    q[:, 0, 5] = 1
    c = dict(q=q, k=np.zeros((n, 1, dk)), v=np.zeros((n, 1, dv)), g=g, beta=np.zeros((n, 1)), state=np.ones((1, 1, dk, dv), np.float32))
    _, _, _, out, S = run_delta(hip, c, [n], 1, 1, dk, dv, dtype, 1.0)
    within(out[:, 0], np.exp(total)[:, None] + 0 * out[:, 0], tol * np.exp(total)[:, None], "state")
    within(S[0, 0], np.exp(total[-1]) + 0 * S[0, 0], 16 * U32 * np.exp(total[-1]), "last state")
    # Updates: token j adds ones to its own row, token i reads that of one before it.
    at = rng.integers(0, np.arange(n) + 1)
    c = dict(q=np.eye(dk)[at, None], k=np.eye(dk)[:n, None], v=np.ones((n, 1, dv)), g=g, beta=np.ones((n, 1)), state=None)
    _, _, _, out, S = run_delta(hip, c, [n], 1, 1, dk, dv, dtype, 1.0)
    want = np.exp(total - total[at])
    within(out[:, 0], want[:, None] + 0 * out[:, 0], tol * want[:, None], "updates")
    want = np.exp(total[-1] - total)
    within(S[0, 0], want[:, None] + 0 * S[0, 0], 16 * U32 * want[:, None], "states of updates")
