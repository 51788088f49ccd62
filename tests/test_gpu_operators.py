"""Language-model operators on the GPU through the C ABI, each against its
definition in 64 bits.

Tolerances count roundings: u = 2^-24 is half a step of fp32, and an output
held in bf16 adds its own half step 2^-8 relative.
"""
import numpy as np
import pytest

from pssa_amd import _abi
from pssa_amd._abi import HipError

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
U16 = 2.0 ** -8  # bf16, relative to the value
NONE = _abi.NO_TOKEN


def say(*a):
    print("[operators]", *a, flush=True)


def to_bf16(x):
    """(bits, value) of an array rounded to bf16, ties to even; infinities and NaN kept."""
    x = np.ascontiguousarray(x, np.float32)
    u = x.view(np.uint32).astype(np.uint64)
    bits = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    bits = np.where(np.isfinite(x), bits, (u >> 16).astype(np.uint16) | np.where(np.isnan(x), 0x40, 0).astype(np.uint16))
    bits = bits.astype(np.uint16)
    return bits, from_bf16(bits)


def from_bf16(bits):
    return (np.ascontiguousarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32)


class Held:
    """Device arrays of one test, freed together."""

    def __init__(self, dev):
        self.dev, self.bufs = dev, []

    def up(self, a):
        self.bufs.append(self.dev.upload(a))
        return self.bufs[-1]

    def new(self, shape, dtype, fill):
        return self.up(np.full(shape, fill, dtype))

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.dev.synchronize()
        for b in self.bufs:
            b.close()


def typed(x, dtype):
    """The array in the operator's storage type, and the values it holds."""
    return (np.ascontiguousarray(x, np.float32),) * 2 if dtype == "f32" else to_bf16(x)


# ---------------------------------------------------------------------------
# Log probabilities


def log_softmax64(z, tau):
    """log softmax in 64 bits, the entropy, and each row's kind: 0 ordinary, 1 empty, 2 not a number."""
    z = z.astype(np.float64)
    kind = np.where(np.isnan(z).any(1) | (z == np.inf).any(1), 2, np.where((z == -np.inf).all(1), 1, 0))
    lp, ent = np.full(z.shape, -np.inf), np.zeros(len(z))
    for r in range(len(z)):
        if kind[r] == 2:
            lp[r], ent[r] = np.nan, np.nan
        elif kind[r] == 0:
            d = (z[r] - z[r].max()) / tau
            e = np.exp(d)
            i = int(np.argmax(d))
            lp[r] = d - np.log1p(np.delete(e, i).sum())
            p = np.exp(lp[r])
            ent[r] = -np.where(p > 0, p * np.where(p > 0, lp[r], 0.0), 0.0).sum()
            lp[r][lp[r] < -np.finfo(np.float32).max] = -np.inf  # past fp32's range
    return lp, ent, kind


def top64(z, k):
    """ids of the k largest logits, equal ones by id; NONE where a token cannot occur."""
    ids = np.full((len(z), k), NONE, np.uint32)
    for r, row in enumerate(z):
        if np.isnan(row).any() or (row == np.inf).any():
            continue
        live = np.flatnonzero(row > -np.inf)
        order = live[np.argsort(-row[live].astype(np.float64), kind="stable")][:k]
        ids[r, :len(order)] = order
    return ids


def run_logprobs(hip, stored, rows, vocab, ld, targets, tau, k, dtype, offset=0):
    """`offset`: elements before the first row in its buffer."""
    with Held(hip) as h:
        flat = np.concatenate([np.zeros(offset, stored.dtype), stored.ravel()])
        x, t = h.up(flat), h.up(targets.astype(np.uint32))
        lp, en = h.new(rows, np.float32, 7.0), h.new(rows, np.float32, 7.0)
        ids, tl = h.new((rows, max(k, 1)), np.uint32, 7), h.new((rows, max(k, 1)), np.float32, 7.0)
        hip.token_logprobs_resident(x.ptr + offset * stored.itemsize, dtype, rows, vocab, t.ptr, lp.ptr, en.ptr, k,
                                    ids.ptr if k else None, tl.ptr if k else None, temperature=tau, ld=ld)
        hip.synchronize()
        return lp.to_host(), en.to_host(), ids.to_host()[:, :k], tl.to_host()[:, :k]


def check_logprobs(hip, z, targets, tau, k, dtype, pad=0, offset=0):
    rows, vocab = z.shape
    wide = np.full((rows, vocab + pad), 1e30, np.float32)  # what lies between the rows is not read as tokens
    wide[:, :vocab] = z
    stored, held = typed(wide, dtype)
    held = held[:, :vocab]
    lp, en, ids, tl = run_logprobs(hip, stored, rows, vocab, vocab + pad, targets, tau, k, dtype, offset)
    ref, ent, kind = log_softmax64(held, tau)
    # A log probability d - log(1 + S): d has three roundings, S at most the sum's depth (64 in a thread, 10 across)
    # plus the exponential's argument (|d| u relative, weighed by e^-|d| <= 1) and its own last place.
    fin = np.where(np.isfinite(ref), ref, 0.0)
    tol = U32 * (4 * np.abs(fin) + 100)
    given = np.array([0.0 if t == NONE else np.nan if t >= vocab else ref[r, t] for r, t in enumerate(targets)])
    given = np.where((targets != NONE) & (kind == 2), np.nan, given)
    gtol = np.array([0.0 if t == NONE or t >= vocab else tol[r, t] for r, t in enumerate(targets)])
    np.testing.assert_array_equal(np.isnan(lp), np.isnan(given))
    assert np.all((np.abs(lp - given) <= gtol) | (lp == given) | np.isnan(given)), np.nanmax(np.abs(lp - given) / np.maximum(gtol, 1e-30))
    # Entropy: every term p log p carries the error of its log p, sum p = 1.
    span = np.array([(-row[np.isfinite(row)]).max() if np.isfinite(row).any() else 0.0 for row in ref])
    etol = U32 * (4 * np.minimum(span, 60.0) + 200) * (1 + np.nan_to_num(ent))
    np.testing.assert_array_equal(np.isnan(en), np.isnan(ent))
    assert np.all((np.abs(en - ent) <= etol) | np.isnan(ent)), np.nanmax(np.abs(en - ent) / etol)
    if k:
        want = top64(held, k)
        np.testing.assert_array_equal(ids, want)
        for r in range(rows):
            for j in range(k):
                if want[r, j] == NONE:
                    assert np.isnan(tl[r, j]) if kind[r] == 2 else tl[r, j] == -np.inf
                else:
                    assert tl[r, j] == ref[r, want[r, j]] or abs(tl[r, j] - ref[r, want[r, j]]) <= tol[r, want[r, j]]


def logits_like(rng, rows, vocab):
    z = rng.normal(0, 3, (rows, vocab))
    z[np.arange(rows), rng.integers(0, vocab, rows)] += rng.uniform(0, 25, rows)
    return z.astype(np.float32)


def some_targets(rng, rows, vocab):
    t = rng.integers(0, vocab, rows).astype(np.uint32)
    t[rng.random(rows) < 0.2] = NONE
    return t


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab,k,pad,tau", [
    (1, 1, 1, 0, 1.0), (5, 2, 2, 3, 1.0), (3, 3, 3, 0, 2.0), (2, 7, 4, 1, 1.0), (4, 9, 9, 0, 0.5), (7, 64, 64, 0, 1.0),
    (3, 255, 20, 2, 1.0), (2, 1024, 8, 0, 1.0), (2, 1025, 64, 1, 0.7), (2, 2049, 0, 5, 1.0), (3, 4099, 64, 0, 1.0),
    (2, 8192, 5, 0, 1.0), (2, 16384, 64, 0, 1.0), (2, 16387, 8, 3, 3.0), (1, 33000, 64, 0, 1.0), (1, 70001, 20, 0, 1.0),
    (2, 131075, 64, 1, 1.0), (1, 300007, 64, 0, 1.0)])
def test_logprobs_match_64_bits(hip, dtype, rows, vocab, k, pad, tau):
    """Every workgroup shape, its borders, and rows past the registers."""
    say(f"logprobs {rows} x {vocab} (+{pad}) {dtype} top {k} tau {tau}")
    rng = np.random.default_rng(vocab + k)
    check_logprobs(hip, logits_like(rng, rows, vocab), some_targets(rng, rows, vocab), tau, k, dtype, pad)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("offset", [1, 2, 3])
def test_logprobs_rows_at_any_element(hip, dtype, offset):
    say("logprobs, first row at element", offset, dtype)
    rng = np.random.default_rng(offset)
    check_logprobs(hip, logits_like(rng, 5, 1501), some_targets(rng, 5, 1501), 1.0, 8, dtype, pad=offset, offset=offset)


@pytest.mark.parametrize("vocab,k", [(50, 64), (3001, 64), (16384, 8), (140000, 64)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_logprobs_masks_ties_and_bad_rows(hip, dtype, vocab, k):
    """Rows with nothing left, with fewer tokens than alternatives, of one value, nearly certain, with signed zeros,
    with the type's lowest and highest values, and with NaN or +inf."""
    say("logprobs masks", vocab, k, dtype)
    rng = np.random.default_rng(vocab)
    z = logits_like(rng, 12, vocab)
    z[0] = -np.inf
    z[1] = -np.inf
    z[1, [vocab - 1, 3, 4]] = [1.0, 2.0, 2.0]
    z[2] = 0.25
    z[3] = np.where(np.arange(vocab) % 2, 0.0, -0.0)
    z[4, :] = -40.0
    z[4, vocab // 2] = 20.0
    low = 3.38e38  # finite in both types
    z[5, :] = -low
    z[5, 7] = low
    z[6, 9] = np.nan
    z[7, 1] = np.inf
    z[8] = np.sort(z[8])  # the largest all in one thread's reach or behind it
    z[9] = np.sort(z[9])[::-1]
    z[10, rng.random(vocab) < 0.5] = -np.inf
    z[11] = rng.integers(-2, 3, vocab)  # many equal
    t = some_targets(rng, 12, vocab)
    t[[0, 1, 6, 7]] = [0, 3, 9, 2]
    t[11] = vocab  # no such token
    check_logprobs(hip, z, t, 1.0, k, dtype)


@pytest.mark.parametrize("rows,k", [(300, 8), (520, 64), (513, 3), (257, 0)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_logprobs_of_many_rows(hip, dtype, rows, k):
    """Many rows take their tiles one by one: what the alternatives gather in each, with tiles that hold nothing, that
    hold more and more, and that hold too many."""
    vocab = 20011
    say("logprobs of many rows", rows, k, dtype)
    rng = np.random.default_rng(rows + k)
    z = logits_like(rng, rows, vocab)
    z[0] = -np.inf
    z[1, :18000] = -np.inf
    z[2] = -np.inf
    z[2, [5, 9000, 9001, vocab - 1]] = [1.0, 3.0, 3.0, 2.0]
    z[3] = np.sort(z[3])
    for i in range(vocab // 1000):
        z[4, 1000 * i:1000 * i + 150] = 40 + i
        z[5, 1000 * i:1000 * i + 75] = 40 + i
    z[6] = 0.25
    z[7, vocab - 1] = np.nan
    z[8, 12000] = np.inf
    z[9] = rng.integers(-2, 3, vocab)
    z[10, 16000:] = -np.inf
    z[11] = -40.0
    z[11, 19000] = 20.0
    t = some_targets(rng, rows, vocab)
    t[[0, 7, 8]] = [1, 2, 3]
    check_logprobs(hip, z, t, 1.0, k, dtype)


def test_logprobs_outputs_are_optional_and_the_rest_is_untouched(hip):
    rng = np.random.default_rng(5)
    z = logits_like(rng, 3, 500)
    ref, ent, _ = log_softmax64(z, 1.0)
    with Held(hip) as h:
        x, en = h.up(z), h.new(4, np.float32, 7.0)
        hip.token_logprobs_resident(x.ptr, "f32", 3, 500, entropy_ptr=en.ptr)
        hip.synchronize()
        got = en.to_host()
        assert np.all(np.abs(got[:3] - ent) <= U32 * 600 * (1 + ent)) and got[3] == 7.0


# ---------------------------------------------------------------------------
# Distillation


def distill64(z, ids, t, tau, w):
    """Loss and gradient in 64 bits (rows with ordinary values)."""
    z, t, w = z.astype(np.float64), t.astype(np.float64), w.astype(np.float64)
    loss, grad = np.zeros(len(z)), np.zeros(z.shape)
    for r in range(len(z)):
        live = (ids[r] != NONE) & (t[r] > -np.inf)
        if not live.any() or w[r] == 0:
            continue
        tr = t[r][live] / tau
        q = np.exp(tr - tr.max())
        q /= q.sum()
        with np.errstate(divide="ignore", invalid="ignore"):
            top = z[r].max()
            e = np.exp((z[r] - top) / tau) if top > -np.inf else np.zeros_like(z[r])
            p = e / e.sum() if e.sum() else e
            lp = (z[r] - top) / tau - np.log(e.sum()) if e.sum() else np.full_like(z[r], -np.inf)
        at = ids[r][live].astype(np.int64)
        use = q > 0
        loss[r] = w[r] * tau * tau * (q[use] * (np.log(q[use]) - lp[at[use]])).sum()
        np.subtract.at(p, at, q)
        grad[r] = w[r] * tau * p
    return loss, grad


def run_distill(hip, stored, rows, vocab, ld, ids, t, tau, w, dtype, in_place=False, want_grad=True, ld_grad=None):
    with Held(hip) as h:
        x, di, dt = h.up(stored), h.up(ids.astype(np.uint32)), h.up(t.astype(np.float32))
        dw = None if w is None else h.up(w.astype(np.float32))
        loss = h.new(rows, np.float32, 7.0)
        ld_grad = ld if in_place else ld_grad or vocab
        g = x if in_place else h.new((rows, ld_grad), stored.dtype, 7) if want_grad else None
        hip.distill_resident(x.ptr, dtype, rows, vocab, di.ptr, dt.ptr, ids.shape[1], loss.ptr, g.ptr if g else None,
                             temperature=tau, row_weights_ptr=dw.ptr if dw else None, ld=ld, ld_grad=ld_grad)
        hip.synchronize()
        grad = g.to_host().reshape(rows, ld_grad) if want_grad else None
        return loss.to_host(), grad


def check_distill(hip, z, ids, t, tau, w, dtype, pad=0, in_place=False, ld_grad=None):
    rows, vocab = z.shape
    wide = np.full((rows, vocab + pad), 1e30, np.float32)
    wide[:, :vocab] = z
    stored, held = typed(wide, dtype)
    loss, grad = run_distill(hip, stored, rows, vocab, vocab + pad, ids, t, tau, w, dtype, in_place, True, ld_grad)
    if in_place or ld_grad:  # what lies behind the rows stays
        behind = grad[:, vocab:]
        assert np.all(behind == (stored[:, vocab:] if in_place else 7))
    grad = grad[:, :vocab]
    ww = np.ones(rows, np.float32) if w is None else w
    ref, gref = distill64(held[:, :vocab], ids, t, tau, ww)
    got = grad if dtype == "f32" else from_bf16(grad)
    live = (ids != NONE) & (t > -np.inf)
    zr = np.where(np.isfinite(held[:, :vocab]), held[:, :vocab], 0)
    span = (zr.max(1) - zr.min(1)) / tau + np.where(live, np.abs(t), 0).max(1) / tau + np.log(vocab)
    scale = np.abs(ww) * tau
    # p and q: the exponential's argument (|d| u, against p e^..: at most u once weighed), the sum's depth, two divisions.
    gtol = (U32 * (100 + 4 * np.minimum(span, 90.0)))[:, None] * (np.abs(gref) + scale[:, None] * 2.0 / 3) + \
        (U16 * np.abs(gref) if dtype == "bf16" else 0) + 1e-37
    assert np.all(np.abs(got.astype(np.float64) - gref) <= gtol), np.max(np.abs(got - gref) / gtol)
    ltol = U32 * (200 + 8 * span) * scale * tau * (1 + span)
    ok = (np.abs(loss - ref) <= ltol) | (loss == ref)
    assert ok.all(), (loss[~ok], ref[~ok], ltol[~ok])
    return loss, got


def teacher(rng, rows, vocab, k, dead=0.1):
    ids = np.stack([rng.choice(vocab, k, replace=k > vocab) for _ in range(rows)]).astype(np.uint32)
    t = rng.normal(0, 3, (rows, k)).astype(np.float32)
    ids[rng.random((rows, k)) < dead] = NONE
    return ids, t


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab,k,pad,tau", [
    (1, 1, 1, 0, 1.0), (3, 2, 2, 1, 1.0), (4, 5, 3, 0, 2.0), (2, 9, 9, 0, 1.0), (7, 64, 8, 0, 1.0), (3, 255, 20, 2, 0.7),
    (2, 1025, 64, 0, 1.0), (3, 2048, 100, 0, 4.0), (3, 4099, 8, 1, 1.0), (2, 8193, 20, 0, 1.0), (2, 16384, 64, 0, 2.0),
    (2, 33001, 1024, 0, 1.0), (1, 65537, 64, 3, 1.5), (2, 140001, 20, 0, 1.0), (260, 33001, 20, 1, 1.0)])
def test_distill_matches_64_bits(hip, dtype, rows, vocab, k, pad, tau):
    say(f"distill {rows} x {vocab} (+{pad}) {dtype} teacher {k} tau {tau}")
    rng = np.random.default_rng(vocab + k)
    ids, t = teacher(rng, rows, vocab, k)
    w = rng.uniform(0.1, 1.0, rows).astype(np.float32)
    check_distill(hip, logits_like(rng, rows, vocab), ids, t, tau, w, dtype, pad)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [37, 5003, 140003])
def test_distill_in_place_equals_apart(hip, dtype, vocab):
    say("distill in place", vocab, dtype)
    rng = np.random.default_rng(vocab)
    z = logits_like(rng, 4, vocab)
    ids, t = teacher(rng, 4, vocab, 16)
    a = check_distill(hip, z, ids, t, 1.5, None, dtype, pad=3, in_place=True)
    b = check_distill(hip, z, ids, t, 1.5, None, dtype, pad=3, ld_grad=vocab + 5)
    np.testing.assert_array_equal(a[0], b[0])
    np.testing.assert_array_equal(a[1], b[1])
    stored, _ = typed(z, dtype)
    alone, _ = run_distill(hip, stored, 4, vocab, vocab, ids, t, 1.5, None, dtype, want_grad=False)
    np.testing.assert_array_equal(alone, a[0])


def test_distill_special_rows(hip):
    """Duplicate entries, frames without entries, rows without weight (whatever they hold), masked student tokens, one
    certain teacher token, and rows that are not numbers."""
    say("distill special rows")
    rng = np.random.default_rng(3)
    V, K = 3001, 12
    z = logits_like(rng, 10, V)
    ids, t = teacher(rng, 10, V, K, dead=0.0)
    w = rng.uniform(0.5, 1.0, 10).astype(np.float32)
    ids[0, [3, 7, 11]] = ids[0, 0]  # one token four times
    ids[1] = NONE
    t[1] = np.nan  # not read as entries
    w[2], z[2, 5] = 0.0, np.nan
    t[3, 1:] = -np.inf
    z[4, rng.random(V) < 0.5] = -np.inf
    z[4, ids[4]] = 1.0
    z[5] = -np.inf
    z[5, ids[5]] = 0.5
    good = [0, 1, 3, 4, 5]
    check_distill(hip, z[good], ids[good], t[good], 1.3, w[good], "f32")
    z[6, 17] = np.nan
    z[7, 18] = np.inf
    t[8, 2] = np.nan
    ids[9, 4] = V
    z2, i2, t2, w2 = z[[6, 7, 8, 9, 2]], ids[[6, 7, 8, 9, 2]], t[[6, 7, 8, 9, 2]], w[[6, 7, 8, 9, 2]]
    loss, grad = run_distill(hip, z2, 5, V, V, i2, t2, 1.0, w2, "f32")
    assert np.isnan(loss[:4]).all() and np.isnan(grad[:4]).all()
    assert loss[4] == 0 and not grad[4].any()
    # A taught token that the student masks: infinite loss, the gradient of what is left finite; a student without
    # any token likewise.
    z3 = logits_like(rng, 2, V)
    i3, t3 = teacher(rng, 2, V, K, dead=0.0)
    z3[0, i3[0, 0]] = -np.inf
    z3[1] = -np.inf
    loss, grad = run_distill(hip, z3, 2, V, V, i3, t3, 1.0, None, "f32")
    assert np.all(loss == np.inf) and np.isfinite(grad).all()
    _, gref = distill64(z3, i3, t3, 1.0, np.ones(2))
    assert np.max(np.abs(grad - gref)) <= U32 * 500


def test_distill_gradient_is_the_losses_slope(hip):
    """Central differences of the loss itself: step h, error h^2/6 |f'''| (third derivatives of a log-sum-exp are at
    most 1/tau of the row's weight) plus the loss's own rounding over 2h."""
    rng = np.random.default_rng(9)
    V, K, tau, h = 40, 6, 1.5, 2.0 ** -4
    z = rng.normal(0, 1, (1, V)).astype(np.float32)
    ids, t = teacher(rng, 1, V, K, dead=0.0)
    _, grad = run_distill(hip, z, 1, V, V, ids, t, tau, None, "f32")
    up, down = np.repeat(z, V, 0), np.repeat(z, V, 0)
    up[np.arange(V), np.arange(V)] += np.float32(h)
    down[np.arange(V), np.arange(V)] -= np.float32(h)
    step = (up - down).diagonal().astype(np.float64)
    rep = lambda a: np.repeat(a, V, 0)
    lu, _ = run_distill(hip, up, V, V, V, rep(ids), rep(t), tau, None, "f32", want_grad=False)
    ld, _ = run_distill(hip, down, V, V, V, rep(ids), rep(t), tau, None, "f32", want_grad=False)
    slope = (lu.astype(np.float64) - ld) / step
    tol = h * h / 6 / tau + U32 * 400 * tau * tau * 8 / h
    assert np.max(np.abs(slope - grad[0])) <= tol


# ---------------------------------------------------------------------------
# Both on a batch forward's logits


def test_batch_scores_and_distillation(hip):
    """A teacher model scores a ragged batch and keeps each token's top alternatives; a student of the same vocabulary
    is taught by them: losses and gradients of the packed tokens, in that order."""
    from pssa_amd import ModelWeights, PSSAConfig, PSSALayer, Sequence

    say("batch scores and distillation")
    cfg = PSSAConfig(depth=2, d_vocab=517, d_latent=48, d_state=24, d_mem_key=8, mem_capacity=30)
    rng = np.random.default_rng(4)
    seqs = [Sequence(lane, rng.integers(0, 517, n, dtype=np.uint32), rng.integers(0, 517, n, dtype=np.uint32), True)
            for lane, n in ((2, 9), (0, 30), (3, 1), (1, 17))]
    layers = []
    for seed in (1, 2):
        w = ModelWeights.init(cfg, seed, "baseline")
        w.unembed *= 40.0
        w.populate_banks(seed + 5, count=27)
        layers.append(PSSALayer(hip, w, lanes=4, max_tokens=64))
    teach, learn = layers
    with pytest.raises((HipError, ValueError)):
        teach.token_logprobs()
    K, tau = 10, 2.0
    loss, token_losses, lg = teach.batch_forward(seqs, want_token_losses=True, want_logits=True)
    got = teach.token_logprobs(top_k=K)
    ref, ent, _ = log_softmax64(lg, 1.0)
    targets = np.concatenate([s.targets for s in seqs])
    tol = U32 * (4 * np.abs(ref).max() + 200)
    assert np.max(np.abs(got["logprobs"] - ref[np.arange(len(targets)), targets])) <= tol
    assert np.max(np.abs(got["logprobs"] + token_losses)) <= 2 * tol + U32 * 400
    assert np.max(np.abs(got["entropy"] - ent)) <= tol * (1 + ent.max())
    np.testing.assert_array_equal(got["top_ids"], top64(lg, K))
    other = targets.copy()
    other[::3] = NONE
    again = teach.token_logprobs(targets=other)
    np.testing.assert_array_equal(again["logprobs"], np.where(other == NONE, 0, got["logprobs"]).astype(np.float32))

    _, slg = learn.batch_forward(seqs, want_logits=True)
    n = len(targets)
    weights = np.full(n, 1.0 / n, np.float32)
    losses, grad = learn.distill(got["top_ids"], got["top_logprobs"], tau, weights)
    lref, gref = distill64(slg, got["top_ids"], got["top_logprobs"], tau, weights)
    assert np.max(np.abs(losses - lref)) <= U32 * 2000 * tau * tau / n
    assert np.max(np.abs(grad - gref)) <= U32 * 400 * tau / n
    np.testing.assert_array_equal(learn.distill(got["top_ids"], got["top_logprobs"], tau, weights, want_grad=False), losses)
    # The head's adjoints take the gradient as it is: d logits . unembed and d logits^T . features.
    back = hip.gemm_nn(grad, w.unembed, n, cfg.d_vocab, cfg.d_latent).reshape(n, -1)
    want = gref @ w.unembed.astype(np.float64)
    assert np.max(np.abs(back - want)) <= 1e-4 * np.abs(want).max()
    with pytest.raises(HipError, match="outside model vocabulary"):
        bad = got["top_ids"].copy()
        bad[3, 2] = 517
        learn.distill(bad, got["top_logprobs"], tau)
    for layer in layers:
        layer.close()


# ---------------------------------------------------------------------------
# 4-bit weights


def w4_inputs(rng, n, k, group, zeros):
    codes = rng.integers(0, 16, (n, k), dtype=np.uint8)
    scales = (rng.uniform(0.5, 1.5, (n, -(-k // group))) * 0.1).astype(np.float32)
    zp = rng.integers(0, 16, scales.shape, dtype=np.uint8) if zeros else None
    at = np.arange(k) // group
    w = (codes - (zp[:, at].astype(np.float64) if zeros else 8.0)) * scales[:, at].astype(np.float64)
    return codes, scales, zp, w


def w4_tolerance(x, codes, scales, zp, group):
    """Exact products; sums of 32 in the matrix instruction, of a group's four, of the groups and of the waves: at most
    32 + 4 + k / group + 8 roundings of partial sums that sum |x| (|2q - 15| + |15 - 2z|) s / 2 bounds."""
    at = np.arange(codes.shape[1]) // group
    z = zp[:, at].astype(np.float64) if zp is not None else 8.0
    mag = (np.abs(2.0 * codes - 15) + np.abs(15 - 2 * z)) * scales[:, at] / 2
    return U32 * (44 + codes.shape[1] / group) * (np.abs(x.astype(np.float64)) @ mag.T) + 1e-37


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k,group,zeros", [
    (1, 1, 1, 32, False), (1, 16, 128, 32, True), (2, 17, 129, 64, False), (1, 100, 768, 64, False),
    (5, 33, 100, 32, True), (6, 48, 300, 128, True), (10, 64, 257, 64, True), (11, 20, 500, 32, False),
    (16, 31, 640, 128, False), (17, 40, 333, 32, True), (33, 70, 1030, 64, True), (3, 5000, 96, 32, True),
    (1, 40, 8192, 128, True), (4, 70000, 130, 64, False), (70, 24, 128, 128, True), (9, 8195, 700, 64, True),
    (11, 8209, 130, 32, False), (6, 8177, 260, 128, True)])
def test_matvec_w4_matches_64_bits(hip, dtype, m, n, k, group, zeros):
    say(f"w4 {m} x {n} x {k} group {group} {dtype} zeros {zeros}")
    rng = np.random.default_rng(n + k)
    codes, scales, zp, w = w4_inputs(rng, n, k, group, zeros)
    pad_x, pad_y = 3, 5
    stored, held = typed(rng.normal(0, 1, (m, k + pad_x)).astype(np.float32), dtype)
    mat = hip.w4_matrix(codes, scales, group, zp)
    with Held(hip) as h:
        x, y = h.up(stored), h.new((m, n + pad_y), np.float32, 7.0)
        hip.matvec_w4_resident(x.ptr, dtype, m, mat, y.ptr, ld_x=k + pad_x, ld_y=n + pad_y)
        hip.synchronize()
        got = y.to_host()
        assert np.all(got[:, n:] == 7.0)
        ref = held[:, :k].astype(np.float64) @ w.T
        tol = w4_tolerance(held[:, :k], codes, scales, zp, group)
        assert np.all(np.abs(got[:, :n] - ref) <= tol), np.max(np.abs(got[:, :n] - ref) / tol)
        # A row alone has the same bits.
        i = m // 2
        hip.matvec_w4_resident(x.ptr + i * (k + pad_x) * stored.itemsize, dtype, 1, mat, y.ptr)
        hip.synchronize()
        np.testing.assert_array_equal(y.to_host().ravel()[:n].view(np.uint32), got[i, :n].view(np.uint32))
    if dtype == "f32":
        np.testing.assert_array_equal(hip.matvec_w4(held[:, :k], mat), got[:, :n])
    mat.close()


def test_matvec_w4_takes_any_fp32_value(hip):
    """Rows of very large, very small and mixed values (nothing of x is rounded away), of one sign, of zeros, and rows
    that are not numbers, which leave the rows beside them alone."""
    say("w4 values")
    rng = np.random.default_rng(8)
    n, k, group = 50, 300, 64
    codes, scales, zp, w = w4_inputs(rng, n, k, group, True)
    x = rng.normal(0, 1, (8, k)).astype(np.float32)
    x[0] *= np.float32(1e35)
    x[1] *= np.float32(1e-30)
    x[2] *= np.exp2(rng.integers(-30, 30, k)).astype(np.float32)
    x[3] = np.abs(x[3])
    x[4] = 0
    x[5, 7] = np.inf
    x[6, 8] = np.nan
    x[7] = np.float32(1) + np.float32(2) ** -23
    mat = hip.w4_matrix(codes, scales, group, zp)
    got = hip.matvec_w4(x, mat)
    good = [0, 1, 2, 3, 4, 7]
    tol = w4_tolerance(x[good], codes, scales, zp, group)
    assert np.all(np.abs(got[good] - x[good].astype(np.float64) @ w.T) <= tol)
    assert not np.isfinite(got[[5, 6]]).any()
    mat.close()


def test_matvec_w4_refuses_on_a_handle(hip):
    codes, scales, _, _ = w4_inputs(np.random.default_rng(0), 16, 64, 32, False)
    with pytest.raises(HipError, match="codes must be"):
        hip.w4_matrix(codes, scales[:, :1], 32)
    mat = hip.w4_matrix(codes, scales, 32)
    buf = hip.empty((4096,), np.float32)
    for args, message in (((buf.ptr, "f32", 0, mat, buf.ptr + 8192), "positive"),
                          ((buf.ptr, "f32", 1, mat, buf.ptr + 128), "overlaps"),
                          ((buf.ptr, "f32", 70000, mat, buf.ptr + 8192), "65535"),
                          ((buf.ptr, "f32", 1, mat, buf.ptr + 8192, 63), "row stride"),
                          ((buf.ptr, "f32", 1, mat, buf.ptr + 8192, 64, 15), "row stride"),
                          ((buf.ptr + 2, "f32", 1, mat, buf.ptr + 8192), "misaligned"),
                          ((0, "f32", 1, mat, buf.ptr), "null")):
        with pytest.raises(HipError, match=message):
            hip.matvec_w4_resident(*args)
    with pytest.raises(ValueError, match="m, 64"):
        hip.matvec_w4(np.ones((2, 65), np.float32), mat)
    mat.close()
    with pytest.raises(HipError, match="null weights"):
        hip.matvec_w4_resident(buf.ptr, "f32", 1, mat, buf.ptr + 8192)
    buf.close()


# ---------------------------------------------------------------------------
# Linear attention


def linear64(q, k, v, log_decay, lens, scale, state):
    """The recurrence in 64 bits; q [tokens, h, dk], k and v [tokens, hk, .]."""
    h, dk, dv, rep = q.shape[1], q.shape[2], v.shape[2], q.shape[1] // k.shape[1]
    q, k, v = (a.astype(np.float64) for a in (q, np.repeat(k, rep, 1), np.repeat(v, rep, 1)))
    lam = np.exp(log_decay.astype(np.float64))[:, None, None]
    out, last, at = np.zeros((len(q), h, dv)), np.zeros((len(lens), h, dk, dv)), 0
    size = np.zeros_like(out), np.zeros_like(last)  # the same sums of magnitudes: what roundings are relative to
    for i, n in enumerate(lens):
        s = np.zeros((h, dk, dv)) if state is None else state[i].astype(np.float64)
        m = np.abs(s)
        for t in range(at, at + n):
            s = lam * s + k[t][:, :, None] * v[t][:, None, :]
            m = lam * m + np.abs(k[t][:, :, None] * v[t][:, None, :])
            out[t] = scale * np.einsum("hd,hdv->hv", q[t], s)
            size[0][t] = abs(scale) * np.einsum("hd,hdv->hv", np.abs(q[t]), m)
        last[i], size[1][i], at = s, m, at + n
    return out, last, size


def run_linear(hip, q, k, v, g, lens, scale, state, dtype, gap=0, out_gap=0, in_place=False, keep=True):
    """Through one row buffer of q | k | v with `gap` elements behind each row."""
    n, h, dk = q.shape
    hk, dv = v.shape[1], v.shape[2]
    row = np.concatenate([q.reshape(n, h * dk), k.reshape(n, hk * dk), v.reshape(n, hk * dv), np.full((n, gap), 1e30)], 1)
    stored, held = typed(row.astype(np.float32), dtype)
    wide = row.shape[1]
    with Held(hip) as b:
        x, d = b.up(stored if n else np.zeros(8, stored.dtype)), b.up(g)
        o = b.new((n + 1, h * dv + out_gap), stored.dtype, 7)
        s_in = None if state is None else b.up(state)
        s_out = s_in if in_place else b.new((len(lens), h, dk, dv), np.float32, 7.0) if keep else None
        size = stored.itemsize
        hip.linear_attention_resident(x.ptr, x.ptr + h * dk * size, x.ptr + (h + hk) * dk * size, d.ptr, dtype, h, dk, dv,
                                      o.ptr, lens, kv_heads=hk, scale=scale, state_in_ptr=s_in.ptr if s_in else None,
                                      state_out_ptr=s_out.ptr if s_out else None, ld_q=wide, ld_k=wide, ld_v=wide,
                                      ld_out=h * dv + out_gap)
        hip.synchronize()
        out = o.to_host()
        assert np.all(out[n] == 7) and np.all(out[:, h * dv:] == 7)  # behind the last token and between the rows
        out = out[:n, :h * dv].reshape(n, h, dv)
        out = out if dtype == "f32" else from_bf16(out)
        parts = np.split(held, [h * dk, (h + hk) * dk, (h + hk) * dk + hk * dv], 1)[:3]
        return out, s_out.to_host() if s_out else None, [p.reshape(n, c, d) for p, c, d in zip(parts, (h, hk, hk), (dk, dk, dv))]


def check_linear(hip, lens, h, hk, dk, dv, dtype, with_state, gap=0, out_gap=0, decays=None, in_place=False, seed=0):
    rng = np.random.default_rng([seed, sum(lens), dk, dv])
    n = sum(lens)
    q, k, v = (rng.normal(0, 1, s) for s in ((n, h, dk), (n, hk, dk), (n, hk, dv)))
    g = np.log(rng.uniform(0.5, 0.999, h)) if decays is None else np.asarray(decays)
    g = g.astype(np.float32)
    state = rng.normal(0, 1, (len(lens), h, dk, dv)).astype(np.float32) if with_state else None
    out, last, held = run_linear(hip, q, k, v, g, lens, 0.37, state, dtype, gap, out_gap, in_place)
    ref, rlast, (so, ss) = linear64(*held, g, lens, 0.37, state)
    # Roundings of a path through the sums: d_key + 64 terms in a product, one for each chunk's state, six for a decay's
    # power (its exponent's own, weighed by |x| e^-|x|) and the products; bf16 operands of two parts carry 2^-17 each.
    chunks = max(lens, default=0) // 64 + 1
    part = U32 * (dk + 64 + 2 * min(chunks, 40) + 12)
    low = 3 * 2.0 ** -17 if dtype == "bf16" else 0.0
    otol = (part + low) * so + (U16 * np.abs(ref) if dtype == "bf16" else 0)
    assert np.all(np.abs(out - ref) <= otol + 1e-30), np.max(np.abs(out - ref) / (otol + 1e-30))
    assert np.all(np.abs(last - rlast) <= part * ss + 1e-30), np.max(np.abs(last - rlast) / (part * ss + 1e-30))
    return out, last


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens,h,hk,dk,dv,with_state", [
    ([1], 1, 1, 1, 1, False), ([1], 2, 1, 16, 32, True), ([1] * 9, 3, 3, 64, 64, True), ([1, 0, 1], 2, 2, 128, 72, True),
    ([2, 4, 3], 2, 1, 100, 5, True), ([0], 1, 1, 8, 8, True), ([0, 0], 1, 1, 8, 8, False), ([5], 1, 1, 7, 9, False),
    ([63], 1, 1, 32, 64, False), ([64], 2, 2, 64, 64, True), ([65], 1, 1, 128, 128, True), ([127, 1, 0, 129], 2, 1, 33, 70, True),
    ([200], 3, 1, 100, 192, False), ([300, 17], 1, 1, 128, 64, True), ([7] * 300, 1, 1, 16, 16, True),
    (list(range(300)), 1, 1, 16, 24, False), ([1500], 2, 2, 64, 32, True),
    # Split into segments: ragged ends, sequences of one segment and of none, one end on a segment's border.
    ([900, 0, 3, 513, 256, 512], 2, 1, 24, 72, True), ([1029], 1, 1, 128, 130, True), ([640, 640], 3, 3, 40, 8, False),
    ([1500] + [3] * 299, 1, 1, 16, 16, True)])
def test_linear_attention_matches_the_recurrence(hip, dtype, lens, h, hk, dk, dv, with_state):
    say(f"linear {len(lens)} sequences, {sum(lens)} tokens, {h}/{hk} heads {dk} x {dv} {dtype}")
    check_linear(hip, lens, h, hk, dk, dv, dtype, with_state)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("gap,out_gap", [(1, 3), (2, 0), (3, 1), (8, 8)])
def test_linear_attention_strides_and_states_in_place(hip, dtype, gap, out_gap):
    say("linear strides", gap, out_gap, dtype)
    check_linear(hip, [70, 1, 130], 2, 1, 36, 40, dtype, True, gap, out_gap, in_place=True)
    check_linear(hip, [1] * 5, 2, 1, 36, 40, dtype, True, gap, out_gap, in_place=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens", [[1, 1], [3, 2], [64], [131, 70]])
def test_linear_attention_decays(hip, dtype, lens):
    """No decay, hardly any, one that leaves nothing within a chunk, and none of the past at all (-inf)."""
    say("linear decays", lens, dtype)
    check_linear(hip, lens, 5, 1, 32, 48, dtype, True, decays=[0.0, -1e-6, -3.0, -200.0, -np.inf])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_linear_attention_long_sums(hip, dtype):
    """Thousands of tokens without decay: the state only grows."""
    say("linear long", dtype)
    check_linear(hip, [4100], 1, 1, 16, 16, dtype, False, decays=[0.0])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("length,at", [(150, 100), (150, 64), (4, 2), (70, 69), (700, 300)])
def test_linear_attention_keeps_what_is_not_finite_to_later_tokens(hip, dtype, length, at):
    """A NaN, an infinity in v, k or q: earlier tokens and other sequences are as without it."""
    say("linear not finite", length, at, dtype)
    rng = np.random.default_rng(at)
    lens, h, dk, dv = [length, 20], 2, 32, 40
    n = sum(lens)
    q, k, v = (rng.normal(0, 1, s) for s in ((n, h, dk), (n, h, dk), (n, h, dv)))
    g = np.log(np.array([0.9, 0.99])).astype(np.float32)
    clean, _, _ = run_linear(hip, q, k, v, g, lens, 1.0, None, dtype)
    for which, value in (("v", np.nan), ("v", np.inf), ("k", np.inf), ("k", np.nan), ("q", np.nan)):
        x = {"q": q.copy(), "k": k.copy(), "v": v.copy()}
        x[which][at, 1, 3] = value
        out, _, held = run_linear(hip, x["q"], x["k"], x["v"], g, lens, 1.0, None, dtype)
        with np.errstate(invalid="ignore"):
            ref, _, (size, _) = linear64(*held, g, lens, 1.0, None)
        fine = np.isfinite(ref)
        assert fine[:at].all() and fine[length:].all() and not fine.all()
        assert np.isfinite(out[fine]).all() and not np.isfinite(out[~fine]).any(), which
        tol = (U32 * 200 + 3 * 2.0 ** -17) * size[fine] + U16 * np.abs(ref[fine])
        assert np.all(np.abs(out[fine] - ref[fine]) <= tol)
    assert np.isfinite(clean).all()


def test_linear_attention_prompt_then_tokens_equals_the_whole(hip):
    """A prompt's state carried on by single tokens gives the outputs of the longer prompt."""
    say("linear prompt then tokens")
    rng = np.random.default_rng(6)
    lens, h, dk, dv, more = [90, 33], 2, 64, 64, 6
    g = np.log(np.array([0.95, 0.999])).astype(np.float32)
    whole = [rng.normal(0, 1, (n + more, 3, h, 64)) for n in lens]
    cut = lambda f: [np.concatenate([f(w, n) for w, n in zip(whole, lens)])[:, i] for i in range(3)]
    full, fstate, _ = run_linear(hip, *cut(lambda w, n: w), g, [n + more for n in lens], 0.5, None, "f32")
    part, state, _ = run_linear(hip, *cut(lambda w, n: w[:n]), g, lens, 0.5, None, "f32")
    outs = [part]
    for t in range(more):
        out, state, _ = run_linear(hip, *cut(lambda w, n: w[n + t:n + t + 1]), g, [1, 1], 0.5, state, "f32")
        outs.append(out)
    ends = np.cumsum([n + more for n in lens])
    for i, n in enumerate(lens):
        start, first = ends[i] - n - more, sum(lens[:i])
        got = np.concatenate([part[first:first + n]] + [o[i:i + 1] for o in outs[1:]])
        scale = np.abs(full).max()
        assert np.max(np.abs(got - full[start:ends[i]])) <= U32 * 400 * scale * 8
    assert np.max(np.abs(state - fstate)) <= U32 * 400 * np.abs(fstate).max() * 8


def test_a_step_of_a_served_model_runs_through_the_operators(hip):
    """As they are used together: a token of each stream through linear attention, a 4-bit head, and the next token's
    log probabilities and alternatives, on the context's stream without a wait between."""
    say("served step")
    rng = np.random.default_rng(12)
    streams, h, d, V, K = 3, 2, 64, 997, 6
    codes, scales, zp, w = w4_inputs(rng, V, h * d, 64, True)
    mat = hip.w4_matrix(codes, scales, 64, zp)
    row = rng.normal(0, 1, (streams, 3 * h * d)).astype(np.float32)
    state = rng.normal(0, 1, (streams, h, d, d)).astype(np.float32)
    g = np.log(np.array([0.9, 0.99])).astype(np.float32)
    targets = rng.integers(0, V, streams).astype(np.uint32)
    with Held(hip) as b:
        x, s, dg, t = b.up(row), b.up(state), b.up(g), b.up(targets)
        o, logits = b.new((streams, h * d), np.float32, 0), b.new((streams, V), np.float32, 0)
        lp, en = b.new(streams, np.float32, 0), b.new(streams, np.float32, 0)
        ids, tl = b.new((streams, K), np.uint32, 0), b.new((streams, K), np.float32, 0)
        ld = 3 * h * d
        hip.linear_attention_resident(x.ptr, x.ptr + 4 * h * d, x.ptr + 8 * h * d, dg.ptr, "f32", h, d, d, o.ptr,
                                      n_seqs=streams, scale=0.125, state_in_ptr=s.ptr, state_out_ptr=s.ptr, ld_q=ld,
                                      ld_k=ld, ld_v=ld)
        hip.matvec_w4_resident(o.ptr, "f32", streams, mat, logits.ptr)
        hip.token_logprobs_resident(logits.ptr, "f32", streams, V, t.ptr, lp.ptr, en.ptr, K, ids.ptr, tl.ptr)
        hip.synchronize()
        got = [a.to_host() for a in (o, s, logits, lp, ids)]
    q, k, v = (row.reshape(streams, 3, h, d)[:, i] for i in range(3))
    ref, rs, (so, ss) = linear64(q, k, v, g, [1] * streams, 0.125, state)
    assert np.all(np.abs(got[0].reshape(ref.shape) - ref) <= U32 * 200 * so)
    assert np.all(np.abs(got[1] - rs) <= U32 * 20 * ss)
    # The later stages against 64 bits from what the stage before handed on.
    assert np.all(np.abs(got[2] - got[0].astype(np.float64) @ w.T) <= w4_tolerance(got[0], codes, scales, zp, 64))
    lref, _, _ = log_softmax64(got[2], 1.0)
    assert np.max(np.abs(got[3] - lref[np.arange(streams), targets])) <= U32 * (4 * np.abs(lref).max() + 100)
    np.testing.assert_array_equal(got[4], top64(got[2], K))
    mat.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens,h,hk,dk,dv", [([900, 0, 130], 2, 1, 36, 40), ([2000, 5], 1, 1, 64, 64), ([1100, 700], 2, 1, 128, 128)])
def test_linear_attention_in_segments_with_states_in_place(hip, dtype, lens, h, hk, dk, dv):
    """Few long walks are split; their states may be written where they were read."""
    say("linear segments in place", lens, dtype)
    a = check_linear(hip, lens, h, hk, dk, dv, dtype, True, in_place=True)
    b = check_linear(hip, lens, h, hk, dk, dv, dtype, True)
    for x, y in zip(a, b):
        np.testing.assert_array_equal(x, y)
    check_linear(hip, lens, h, hk, dk, dv, dtype, True, gap=3, decays=[0.0, -np.inf][:h], in_place=True)


def test_linear_attention_of_two_contexts_at_once(hip):
    """Each context has its stream and its scratch: calls that run beside each other give what each gives alone."""
    import threading

    from pssa_amd import HipDevice

    rng = np.random.default_rng(3)
    n, h, d = 1500, 2, 64
    q, k, v = (rng.normal(0, 1, (n, h, d)) for _ in range(3))
    g = np.full(h, -0.05, np.float32)
    alone, last, _ = run_linear(hip, q, k, v, g, [n], 0.3, None, "f32")
    other = HipDevice(0)
    got = {}

    def work(dev, name):
        got[name] = [run_linear(dev, q, k, v, g, [n], 0.3, None, "f32")[:2] for _ in range(8)]

    threads = [threading.Thread(target=work, args=(dev, i)) for i, dev in enumerate((hip, other, hip))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    other.close()
    assert sorted(got) == [0, 1, 2]
    for results in got.values():
        for out, state in results:
            np.testing.assert_array_equal(out, alone)
            np.testing.assert_array_equal(state, last)


def test_rows_past_one_launch(hip):
    """More rows than the threads of one launch can be counted for: log p of two tokens is -log(1 + e^(other - own)),
    whose rounding is the difference's, the exponential's, the logarithm's and the subtraction's."""
    rows = (1 << 21) + 3
    say("rows past one launch", rows)
    rng = np.random.default_rng(8)
    z = rng.normal(0, 2, (rows, 2)).astype(np.float32)
    t = rng.integers(0, 2, rows).astype(np.uint32)
    at = np.arange(rows)
    d = z[at, 1 - t].astype(np.float64) - z[at, t]
    ref = -np.logaddexp(0.0, d)
    p = 1 / (1 + np.exp(d))
    with Held(hip) as b:
        x, ids = b.up(z), b.up(t)
        lp, tid = b.new(rows, np.float32, 7.0), b.new(rows, np.uint32, 7)
        tlp, tl = b.new(rows, np.float32, 7.0), b.up(np.zeros(rows, np.float32))
        loss, grad = b.new(rows, np.float32, 7.0), b.new((rows, 2), np.float32, 7.0)
        hip.token_logprobs_resident(x.ptr, "f32", rows, 2, ids.ptr, lp.ptr, None, 1, tid.ptr, tlp.ptr)
        hip.distill_resident(x.ptr, "f32", rows, 2, ids.ptr, tl.ptr, 1, loss.ptr, grad.ptr)
        hip.synchronize()
        tol = U32 * 32 * (1 + np.abs(d))
        assert np.all(np.abs(lp.to_host() - ref) <= tol)
        np.testing.assert_array_equal(tid.to_host(), np.argmax(z, 1))
        assert np.all(np.abs(loss.to_host() + ref) <= tol)
        got = grad.to_host()
        assert np.all(np.abs(got[at, t] - (p - 1)) <= tol) and np.all(np.abs(got[at, 1 - t] - (1 - p)) <= tol)


def free_device_bytes():
    import ctypes as C

    free, total = C.c_size_t(), C.c_size_t()
    assert C.CDLL("libamdhip64.so").hipMemGetInfo(C.byref(free), C.byref(total)) == 0
    return free.value


@pytest.mark.parametrize("n,most", [(65535, 2), (400, 900)])
def test_linear_attention_reserved_calls_of_many_ragged_sequences_allocate_nothing(hip, n, most):
    """After a reservation the tables of many sequences of unequal lengths take no memory either; one or two tokens a
    sequence against the recurrence, written out."""
    from pssa_amd import HipDevice
    from pssa_amd.device import _lens

    say("linear reserved", n, "ragged sequences")
    rng = np.random.default_rng(n)
    lens = rng.integers(1, 3, n)
    lens[n // 2] = most
    first = np.cumsum(lens) - lens
    tokens, d, lam = int(lens.sum()), 4, np.float32(-0.5)
    q, k, v = (rng.normal(0, 1, (tokens, d)).astype(np.float32) for _ in range(3))
    c_lens = _lens([int(x) for x in lens])
    others = [HipDevice(0) for _ in range(24)]  # as many tables would be seen in the device's free memory
    with Held(hip) as b:
        x, g = [b.up(a) for a in (q, k, v)], b.up(np.full(1, lam))
        o, s = b.new((tokens, d), np.float32, 7.0), b.new((n, d, d), np.float32, 7.0)
        hip.synchronize()

        def call(dev):
            dev.linear_attention_resident(x[0].ptr, x[1].ptr, x[2].ptr, g.ptr, "f32", 1, d, d, o.ptr, c_lens,
                                          state_out_ptr=s.ptr)
            dev.synchronize()

        call(hip)  # what the runtime sets up for a first call is there
        for dev in others:
            dev.linear_attention_reserve("f32", 1, d, d, c_lens)
        before = free_device_bytes()
        for dev in others:
            call(dev)
        after = free_device_bytes()
        out, state = o.to_host(), s.to_host()
    for dev in others:
        dev.close()
    assert after == before
    f = np.exp(np.float64(lam))
    outer = k.astype(np.float64)[:, :, None] * v[:, None, :]
    second = first[lens == 2] + 1
    sums = outer.copy()
    sums[second] += f * outer[second - 1]
    size = np.abs(outer)
    size[second] += f * size[second - 1]
    short = lens <= 2
    at = np.concatenate([first[short], second])
    ref = np.einsum("td,tdv->tv", q.astype(np.float64), sums)
    bound = np.einsum("td,tdv->tv", np.abs(q).astype(np.float64), size)
    # Four products and their sum, one step of the state with the decay's own rounding.
    assert np.all(np.abs(out[at] - ref[at]) <= U32 * 16 * bound[at])
    ends = first[short] + lens[short] - 1
    assert np.all(np.abs(state[short] - sums[ends]) <= U32 * 8 * size[ends])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("gap", [2, 3])
@pytest.mark.parametrize("length,at,dk,dv", [(150, (100,), 32, 40), (70, (69,), 36, 130), (130, (0, 64, 129), 20, 66),
                                             (700, (300, 301, 640), 32, 40), (700, (63,), 100, 72)])
def test_linear_attention_of_any_alignment_keeps_what_is_not_finite(hip, dtype, gap, length, at, dk, dv):
    """As above with loads of 4 bytes and with rows at any element, which take kernels of their own, whole and in
    segments: values that are not finite in some tokens' v, k or q leave earlier tokens and the other sequence alone."""
    say("linear not finite, any alignment", gap, length, at, dk, dv, dtype)
    rng = np.random.default_rng([gap, length, dk])
    lens, h, hk = [length, 20], 2, 1
    n = sum(lens)
    q, k, v = (rng.normal(0, 1, s) for s in ((n, h, dk), (n, hk, dk), (n, hk, dv)))
    g = np.log(np.array([0.9, 0.99])).astype(np.float32)
    for which, value in (("v", np.nan), ("v", -np.inf), ("k", np.inf), ("k", np.nan), ("q", np.nan)):
        x = {"q": q.copy(), "k": k.copy(), "v": v.copy()}
        for i in at:
            x[which][i, -1, 3] = value
        out, last, held = run_linear(hip, x["q"], x["k"], x["v"], g, lens, 1.0, None, dtype, gap, 1)
        with np.errstate(invalid="ignore"):
            ref, rlast, (size, ssize) = linear64(*held, g, lens, 1.0, None)
        fine, sfine = np.isfinite(ref), np.isfinite(rlast)
        assert fine[:at[0]].all() and fine[length:].all() and not fine.all() and sfine[1].all()
        assert np.isfinite(out[fine]).all() and not np.isfinite(out[~fine]).any(), which
        assert np.isfinite(last[sfine]).all() and not np.isfinite(last[~sfine]).any(), which
        # d_key + 64 terms in a product, one for each of up to 11 chunks' states, powers and products: below 300; two
        # bf16 parts of the state and of the products of q and k where the inputs are bf16.
        low = 3 * 2.0 ** -17 if dtype == "bf16" else 0.0
        tol = (U32 * 300 + low) * size[fine] + (U16 * np.abs(ref[fine]) if dtype == "bf16" else 0)
        assert np.all(np.abs(out[fine] - ref[fine]) <= tol), which
        assert np.all(np.abs(last[sfine] - rlast[sfine]) <= U32 * 300 * ssize[sfine]), which


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("gap", [0, 3])
def test_linear_attention_of_a_prompt_beside_single_tokens(hip, dtype, gap):
    """A prompt and the next token of many streams in one call, more of them than a split call has room for."""
    say("linear prompt beside single tokens", gap, dtype)
    check_linear(hip, [1] * 35 + [900] + [1, 0, 2] * 12, 8, 2, 16, 24, dtype, True, gap)
    check_linear(hip, [1] * 300 + [500] + [1] * 50, 2, 1, 16, 24, dtype, True, gap)


def test_batch_scores_refuse_targets_outside_the_vocabulary(hip):
    """Like a teacher's ids; "no token" and the last token are none of these."""
    from pssa_amd import ModelWeights, PSSAConfig, PSSALayer, Sequence

    say("batch scores refuse targets")
    cfg = PSSAConfig(depth=1, d_vocab=70, d_latent=16, d_state=8, d_mem_key=8, mem_capacity=10)
    layer = PSSALayer(hip, ModelWeights.init(cfg, 1, "baseline"), lanes=2, max_tokens=16)
    ids = np.arange(5, dtype=np.uint32)
    layer.batch_forward([Sequence(0, ids, ids, True)])
    own = layer.token_logprobs(top_k=2)
    for bad in (70, NONE - 1):
        with pytest.raises(HipError, match="outside model vocabulary"):
            layer.token_logprobs(targets=np.array([0, 1, bad, 3, 4], np.uint32))
    got = layer.token_logprobs(targets=np.array([0, 1, 2, 69, NONE], np.uint32), top_k=2)
    np.testing.assert_array_equal(got["logprobs"][:3], own["logprobs"][:3])
    np.testing.assert_array_equal(got["top_ids"], own["top_ids"])
    assert got["logprobs"][4] == 0 and np.isfinite(got["logprobs"]).all()
    layer.close()


# ---------------------------------------------------------------------------
# Rows far apart: offsets past 32 bits


class Rows:
    """Rows of `width` elements at a stride in one device array that is otherwise not set."""

    def __init__(self, hip, rows, ld, dtype):
        self.hip, self.ld, self.dtype = hip, ld, np.dtype(dtype)
        self.buf = hip.empty((rows, ld), dtype)

    def at(self, row, col=0):
        return self.buf.ptr + (row * self.ld + col) * self.dtype.itemsize

    def put(self, a, col=0):
        for r, row in enumerate(a):
            self.buf.write(row, (r * self.ld + col) * self.dtype.itemsize)

    def get(self, rows, width, col=0):
        import ctypes as C

        out = np.empty((rows, width), self.dtype)
        for r in range(rows):
            _abi.call(self.hip._lib.pssa_hip_memcpy, self.hip.handle, out[r].ctypes.data_as(C.c_void_p),
                      C.c_void_p(self.at(r, col)), width * self.dtype.itemsize, _abi.D2H)
        return out


def test_logit_rows_at_far_offsets(hip):
    say("logit rows at far offsets")
    rng = np.random.default_rng(1)
    rows, vocab, ld, k = 6, 1003, (1 << 30) + 5, 8
    stored, held = to_bf16(logits_like(rng, rows, vocab))
    ids, t = teacher(rng, rows, vocab, 12, dead=0.0)
    targets = rng.integers(0, vocab, rows).astype(np.uint32)
    far = Rows(hip, rows, ld, np.uint16)
    with Held(hip) as h:
        far.put(stored)
        di, dt, dg = h.up(ids), h.up(t), h.up(targets)
        lp, loss = h.new(rows, np.float32, 7.0), h.new(rows, np.float32, 7.0)
        ti, tl = h.new((rows, k), np.uint32, 7), h.new((rows, k), np.float32, 7.0)
        hip.token_logprobs_resident(far.buf.ptr, "bf16", rows, vocab, dg.ptr, lp.ptr, None, k, ti.ptr, tl.ptr, ld=ld)
        hip.distill_resident(far.buf.ptr, "bf16", rows, vocab, di.ptr, dt.ptr, 12, loss.ptr, far.buf.ptr, ld=ld)
        hip.synchronize()
        got = [a.to_host() for a in (lp, ti, loss)] + [from_bf16(far.get(rows, vocab))]
    far.buf.close()
    ref, _, _ = log_softmax64(held, 1.0)
    assert np.all(np.abs(got[0] - ref[np.arange(rows), targets]) <= U32 * (4 * np.abs(ref).max() + 100))
    np.testing.assert_array_equal(got[1], top64(held, k))
    near, grad = run_distill(hip, stored, rows, vocab, vocab, ids, t, 1.0, None, "bf16")
    np.testing.assert_array_equal(got[2], near)
    np.testing.assert_array_equal(got[3], from_bf16(grad))


@pytest.mark.parametrize("width", [16, 17])
def test_linear_attention_rows_at_far_offsets(hip, width):
    """q, k, v and the outputs as columns of rows 2^24 elements apart; heads of 17 take the kernel for any width."""
    say("linear rows at far offsets", width)
    rng = np.random.default_rng(width)
    n, ld = 300, (1 << 24) - 8
    x = rng.normal(0, 1, (n, 3 * width)).astype(np.float32)
    stored, held = to_bf16(x)
    g = np.full(1, -0.05, np.float32)
    far = Rows(hip, n, ld, np.uint16)
    with Held(hip) as h:
        far.put(stored)
        dg, s = h.up(g), h.new((1, 1, width, width), np.float32, 7.0)
        hip.linear_attention_resident(far.at(0), far.at(0, width), far.at(0, 2 * width), dg.ptr, "bf16", 1, width, width,
                                      far.at(0, 3 * width + 1), [n], scale=0.5, state_out_ptr=s.ptr, ld_q=ld, ld_k=ld,
                                      ld_v=ld, ld_out=ld)
        hip.synchronize()
        out, state = from_bf16(far.get(n, width, 3 * width + 1)), s.to_host()
    far.buf.close()
    parts = [p.reshape(n, 1, width) for p in np.split(held, 3, 1)]
    ref, rlast, (so, ss) = linear64(*parts, g, [n], 0.5, None)
    part = U32 * (width + 64 + 2 * 5 + 12)
    assert np.all(np.abs(out - ref[:, 0]) <= (part + 3 * 2.0 ** -17) * so[:, 0] + U16 * np.abs(ref[:, 0]) + 1e-30)
    assert np.all(np.abs(state - rlast) <= part * ss + 1e-30)


def test_matvec_w4_rows_at_far_offsets(hip):
    say("w4 rows at far offsets")
    rng = np.random.default_rng(2)
    m, n, k, group, ld = 6, 35, 200, 64, (1 << 30) + 3
    codes, scales, zp, w = w4_inputs(rng, n, k, group, True)
    stored, held = to_bf16(rng.normal(0, 1, (m, k)).astype(np.float32))
    mat = hip.w4_matrix(codes, scales, group, zp)
    far, y = Rows(hip, m, ld, np.uint16), Rows(hip, m, ld, np.float32)
    far.put(stored)
    hip.matvec_w4_resident(far.buf.ptr, "bf16", m, mat, y.buf.ptr, ld_x=ld, ld_y=ld)
    hip.synchronize()
    got = y.get(m, n)
    far.buf.close()
    y.buf.close()
    mat.close()
    assert np.all(np.abs(got - held.astype(np.float64) @ w.T) <= w4_tolerance(held, codes, scales, zp, group))


@pytest.mark.parametrize("dtype,gaps", [("f32", (0, 2, 3)), ("bf16", (0, 2))])
@pytest.mark.parametrize("lens", [[70, 1, 130], [900]])
def test_linear_attention_loads_do_not_change_the_bits(hip, dtype, gaps, lens):
    """Loads of 16 and of 4 bytes feed the same sums (only bf16 rows at odd elements take other ones)."""
    say("linear loads", dtype, lens)
    rng = np.random.default_rng(sum(lens))
    n, h, d = sum(lens), 2, 40
    q, k, v = (rng.normal(0, 1, (n, h, d)) for _ in range(3))
    g = np.full(h, -0.02, np.float32)
    got = [run_linear(hip, q, k, v, g, lens, 0.3, None, dtype, gap)[:2] for gap in gaps]
    for out, state in got[1:]:
        np.testing.assert_array_equal(out, got[0][0])
        np.testing.assert_array_equal(state, got[0][1])
