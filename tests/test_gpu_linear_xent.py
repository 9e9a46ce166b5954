"""GPU: softmax cross-entropy straight from a linear layer's inputs, through the device
C ABI, against the formula in numpy (extended precision).

Bounds.  u = 2^-53.  A logit is off by dz = (K + 3) u (|x||w| + |bias|), largest over its
row below; a probability by p (2 dz + (V + 24) u) (the exponent's error counts for it and
for the sum, exp is good to 2 u, the sum of V terms to V u); a row's loss by 2 dz plus
(V + 8) u and 4 u of its own terms.  fp64 has nothing between 0 and 2^-1074 and rounds
what is below 2^-1022 to multiples of that (extended precision goes on to 1e-4932): a
probability, and what it is multiplied to, may be off by 2^-1022 for this reason.  Products and sums of n terms add n u of the sum of
magnitudes.
"""
import numpy as np
import pytest

from micrograd_b200 import cabi as K

pytestmark = pytest.mark.gpu
U = 2.0 ** -53
LD = np.longdouble
STORE = K.ACC_STORE_A | K.ACC_STORE_B | K.ACC_STORE_C

# (rows, width, classes): single values; one row; odd width, odd classes, both; rows above
# and below every tile; more classes than a CTA has threads, many more than rows.
SHAPES = [(1, 1, 1), (1, 2, 3), (1, 128, 2000), (2, 7, 5), (5, 33, 1001), (16, 64, 10), (32, 64, 1000), (17, 96, 514),
          (33, 128, 4099), (128, 30, 130), (130, 17, 64), (200, 50, 257), (64, 1, 33), (3, 301, 8192), (9, 40, 30011)]


def problem(m, k, v, seed, out_rows=0.1, scale=1.0):
    rng = np.random.default_rng(seed)
    x = np.maximum(rng.standard_normal((m, k)), 0.0) * scale
    w = rng.standard_normal((k, v)) / np.sqrt(k)
    b = 0.1 * rng.standard_normal(v)
    y = rng.integers(0, v, m).astype(np.int32)
    if m > 1:
        y[rng.random(m) < out_rows] = -1
    return rng, x, w, b, y


def reference(x, w, b, y, denom, gloss):
    m, k = x.shape
    v = w.shape[1]
    x, w, b = x.astype(LD), w.astype(LD), b.astype(LD)
    z = x @ w + b
    keep = y >= 0
    at = np.where(keep, y, 0)
    top = z.max(axis=1, keepdims=True)
    e = np.exp(z - top)
    s = e.sum(axis=1, keepdims=True)
    rows = np.where(keep, np.log(s[:, 0]) + top[:, 0] - z[np.arange(m), at], 0)
    dz = (k + 3) * U * (np.abs(x) @ np.abs(w) + np.abs(b)).max(axis=1)
    drow = np.where(keep, 2 * dz + (v + 8) * U + 4 * U * (np.abs(top[:, 0]) + np.abs(np.log(s[:, 0])) + np.abs(z[np.arange(m), at])), 0)
    loss = rows.sum() / denom
    dloss = (drow.sum() + (m + 4) * U * np.abs(rows).sum()) / denom
    c = gloss / denom
    p = e / s
    g = p.copy()
    g[np.arange(m), at] -= 1
    g = g * c * keep[:, None]
    dg = keep[:, None] * (c * (p * (2 * dz[:, None] + (v + 24) * U) + 4 * U * (np.abs(g) / c + p)) + LD(2) ** -1022)
    tiny = LD(2) ** -1022
    out = dict(loss=(loss, dloss),
               gx=(g @ w.T, dg @ np.abs(w).T + (v + 2) * U * (np.abs(g) @ np.abs(w).T) + v * tiny),
               gw=(x.T @ g, np.abs(x).T @ dg + (m + 2) * U * (np.abs(x).T @ np.abs(g)) + m * tiny),
               gb=(g.sum(axis=0), dg.sum(axis=0) + (m + 2) * U * np.abs(g).sum(axis=0)))
    return out


def near(name, got, ref, bound):
    off = np.abs(np.asarray(got).astype(LD) - ref)
    assert np.all(off <= bound), (name, float(np.max(off / np.maximum(bound, 1e-300))))


def call(abi, x, w, b, y, denom, gloss, olds, flags, shift=0):
    """Runs loss and gradients on device copies that start `shift` doubles into their buffers."""
    def put(v):
        a = abi.array(np.concatenate([np.zeros(shift), np.asarray(v, dtype=np.float64).reshape(-1), [55.0]]))
        return a

    m, k = x.shape
    v = w.shape[1]
    dx, dw, dy, dg, loss = put(x), put(w), abi.int_array(y), abi.array([gloss]), abi.empty(1)
    db = None if b is None else put(b)
    out = [None if o is None else put(o) for o in olds]
    abi.mg_linear_xent_fwd_bwd(dx.offset(shift), dw.offset(shift), db and db.offset(shift), dy.ptr, dg.ptr, loss.ptr,
                               *(o and o.offset(shift) for o in out), m, k, v, denom, flags)
    got = []
    for o, like in zip(out, (x, w, w[0])):
        if o is None:
            got.append(None)
            continue
        a = o.numpy()
        assert a[-1] == 55.0 and np.all(a[:shift] == 0)
        got.append(a[shift:-1].reshape(like.shape))
    return float(loss.numpy()[0]), got


@pytest.mark.parametrize("shape", SHAPES)
def test_loss_and_gradients(abi, shape):
    m, k, v = shape
    rng, x, w, b, y = problem(m, k, v, 21)
    olds = [rng.standard_normal(t.shape) for t in (x, w, b)]
    denom, gloss = float(m + 1), 0.7
    ref = reference(x, w, b, y, denom, gloss)
    for flags in (STORE, 0, K.ACC_STORE_B):
        loss, got = call(abi, x, w, b, y, denom, gloss, olds, flags)
        near("loss", loss, *ref["loss"])
        for i, (name, o, old) in enumerate(zip(("gx", "gw", "gb"), got, olds)):
            old = old * (0.0 if flags & (1 << i) else 1.0)
            r, bound = ref[name]
            near(name, o, r + old, bound + 2 * U * (np.abs(r) + np.abs(old)))
        left_out = y < 0
        want = olds[0] * (0.0 if flags & 1 else 1.0)
        assert np.array_equal(got[0][left_out], want[left_out])
    # the loss alone is the same number, and so is a second pass
    dx, dw, db, dy, alone = abi.array(x), abi.array(w), abi.array(b), abi.int_array(y), abi.empty(1)
    abi.mg_linear_xent_fwd(dx.ptr, dw.ptr, db.ptr, dy.ptr, alone.ptr, m, k, v, denom)
    near("loss", alone.numpy()[0], *ref["loss"])
    again = call(abi, x, w, b, y, denom, gloss, olds, flags)
    assert again[0] == loss and all(np.array_equal(a, c) for a, c in zip(again[1], got))
    abi.mg_check_kernel_status()


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("shape", [(5, 300, 5001), (6, 1, 63), (7, 129, 257), (8, 676, 4099), (8, 40, 130), (9, 40, 4099), (6, 5, 1)])
def test_loss_alone_of_five_rows_and_more(abi, shape, shift):
    m, k, v = shape
    rng, x, w, b, y = problem(m, k, v, 31)
    y[1], y[m - 1] = -1, v - 1
    ref = reference(x, w, b, y, 3.0, 1.0)
    x[1] = np.nan  # (left out)
    flat = [abi.array(np.concatenate([np.zeros(shift), t.reshape(-1)])) for t in (x, w, b)]
    dy, loss = abi.int_array(y), abi.empty(1)
    for _ in range(2):
        abi.mg_linear_xent_fwd(*(t.offset(shift) for t in flat), dy.ptr, loss.ptr, m, k, v, 3.0)
        near("loss", loss.numpy()[0], *ref["loss"])
    bare = reference(np.where(np.isnan(x), 0, x), w, 0 * b, y, 3.0, 1.0)
    abi.mg_linear_xent_fwd(flat[0].offset(shift), flat[1].offset(shift), None, dy.ptr, loss.ptr, m, k, v, 3.0)
    near("loss", loss.numpy()[0], *bare["loss"])
    abi.mg_check_kernel_status()


@pytest.mark.parametrize("shape", [(5, 32, 130), (40, 64, 1000), (130, 33, 257)])
def test_each_gradient_alone_and_no_bias(abi, shape):
    m, k, v = shape
    rng, x, w, b, y = problem(m, k, v, 22)
    olds = [np.zeros(t.shape) for t in (x, w, b)]
    loss, full = call(abi, x, w, b, y, float(m), 1.0, olds, STORE)
    for i in range(3):
        one, got = call(abi, x, w, b, y, float(m), 1.0, [o if j == i else None for j, o in enumerate(olds)], STORE)
        assert one == loss and np.array_equal(got[i], full[i])
    bare, got = call(abi, x, w, None, y, float(m), 1.0, olds, STORE)
    nil, want = call(abi, x, w, np.zeros(v), y, float(m), 1.0, olds, STORE)
    assert bare == nil and all(np.array_equal(a, c) for a, c in zip(got, want))


@pytest.mark.parametrize("shape", [(6, 32, 130), (140, 64, 1000)])
def test_addresses_off_the_vector_boundaries(abi, shape):
    m, k, v = shape
    rng, x, w, b, y = problem(m, k, v, 23)
    olds = [rng.standard_normal(t.shape) for t in (x, w, b)]
    ref = reference(x, w, b, y, float(m), 1.0)
    loss, got = call(abi, x, w, b, y, float(m), 1.0, olds, 0, shift=1)
    near("loss", loss, *ref["loss"])
    for name, o, old in zip(("gx", "gw", "gb"), got, olds):
        r, bound = ref[name]
        near(name, o, r + old, bound + 2 * U * (np.abs(r) + np.abs(old)))


def test_left_out_rows_may_hold_anything(abi):
    """Rows of a padded batch with NaN and infinities add nothing anywhere; a batch of
    such rows alone has loss 0 and gradients 0."""
    m, k, v = 50, 32, 300
    rng, x, w, b, y = problem(m, k, v, 24, out_rows=0.4)
    olds = [rng.standard_normal(t.shape) for t in (x, w, b)]
    clean = call(abi, x, w, b, y, float(m), 1.0, olds, 0)
    bad = x.copy()
    bad[y < 0] = np.where(rng.random((int((y < 0).sum()), k)) < 0.5, np.nan, np.inf)
    dirty = call(abi, bad, w, b, y, float(m), 1.0, olds, 0)
    assert clean[0] == dirty[0] and all(np.array_equal(a, c) for a, c in zip(clean[1], dirty[1]))
    dx, dw, db, dy, alone = abi.array(bad), abi.array(w), abi.array(b), abi.int_array(y), abi.empty(1)
    abi.mg_linear_xent_fwd(dx.ptr, dw.ptr, db.ptr, dy.ptr, alone.ptr, m, k, v, float(m))
    assert abs(alone.numpy()[0] - clean[0]) <= 1e-12 * abs(clean[0])
    none = np.full(m, -1, dtype=np.int32)
    loss, got = call(abi, bad, w, b, none, float(m), 1.0, olds, STORE)
    assert loss == 0.0 and all(np.all(g == 0.0) for g in got)


def test_labels_outside_the_classes(abi):
    m, k, v = 12, 16, 40
    rng, x, w, b, y = problem(m, k, v, 25, out_rows=0.0)
    olds = [np.zeros(t.shape) for t in (x, w, b)]
    masked = y.copy()
    masked[3] = masked[7] = -1
    want = call(abi, x, w, b, masked, float(m), 1.0, olds, STORE)
    abi.mg_check_kernel_status()
    for wrong in (v, -2, 2 ** 31 - 1):
        y[3], y[7] = wrong, -1
        got = call(abi, x, w, b, y, float(m), 1.0, olds, STORE)
        assert got[0] == want[0] and all(np.array_equal(a, c) for a, c in zip(got[1], want[1]))
        with pytest.raises(K.MgError, match="fault code 101"):
            abi.mg_check_kernel_status()
        abi.mg_check_kernel_status()


def test_large_and_infinite_logits(abi):
    """Logits of some thousands (exp would overflow), a class at -inf (probability 0), and
    NaN where the formula has none: a row whose input is NaN spoils itself and the sums."""
    m, k, v = 7, 16, 100
    rng, x, w, b, y = problem(m, k, v, 26, out_rows=0.0, scale=2000.0)
    ref = reference(x, w, b, y, float(m), 1.0)
    olds = [np.zeros(t.shape) for t in (x, w, b)]
    loss, got = call(abi, x, w, b, y, float(m), 1.0, olds, STORE)
    near("loss", loss, *ref["loss"])
    for name, o in zip(("gx", "gw", "gb"), got):
        near(name, o, *ref[name])
    x /= 2000.0
    b[5] = -np.inf
    y[y == 5] = 6
    loss, got = call(abi, x, w, b, y, float(m), 1.0, olds, STORE)
    few = np.delete(np.arange(v), 5)
    labels = np.searchsorted(few, y).astype(np.int32)
    ref = reference(x, w[:, few], b[few], labels, float(m), 1.0)
    near("loss", loss, *ref["loss"])
    near("gx", got[0], *ref["gx"])
    near("gw", got[1][:, few], *ref["gw"])
    assert np.all(got[1][:, 5] == 0) and got[2][5] == 0
    x[2, 3] = np.nan
    loss, got = call(abi, x, w, b, y, float(m), 1.0, olds, STORE)
    assert np.isnan(loss) and np.all(np.isnan(got[0][2])) and np.all(np.isfinite(got[0][[0, 1, 3, 4, 5, 6]]))


def test_gradient_against_differences(abi):
    """Central differences of the loss along one direction: with h = 1e-4 the formula's
    error is h^2 / 6 times the third derivative, at most 8 max|dz|^3 here; rounding adds
    1e-14 loss / h."""
    m, k, v = 11, 24, 70
    rng, x, w, b, y = problem(m, k, v, 27)
    olds = [np.zeros(t.shape) for t in (x, w, b)]
    _, got = call(abi, x, w, b, y, float(m), 1.0, olds, STORE)
    step = [rng.standard_normal(t.shape) for t in (x, w, b)]
    slope = sum(float((g * s).sum()) for g, s in zip(got, step))
    h = 1e-4
    ends = [call(abi, x + t * step[0], w + t * step[1], b + t * step[2], y, float(m), 1.0, [None, None, olds[2]], STORE)[0]
            for t in (h, -h)]
    dz = np.abs(step[0] @ w + x @ step[1] + step[2]).max() + 6 * np.abs(step[0] @ step[1]).max()
    assert abs((ends[0] - ends[1]) / (2 * h) - slope) <= h * h / 6 * 8 * dz ** 3 + 1e-14 * abs(ends[0]) / h * 4


def test_rows_in_several_blocks(abi):
    """More logits than the workspace holds at a time: 300 rows of 1 200 002 classes are
    handled in blocks of 128 rows or fewer.  Classes beyond the first 40 have a bias that
    gives them no probability, so the small problem's numbers are the whole one's."""
    m, k, v, few = 300, 2, 1200002, 40
    rng, x, w, b, y = problem(m, k, few, 28)
    wide_w, wide_b = np.zeros((k, v)), np.full(v, -1e4)
    wide_w[:, :few], wide_b[:few] = w, b
    olds = [rng.standard_normal(x.shape), np.zeros((k, v)), np.ones(v)]
    ref = reference(x, w, b, y, float(m), 1.0)
    loss, got = call(abi, x, wide_w, wide_b, y, float(m), 1.0, olds, K.ACC_STORE_B)
    slack = 1 + v / few  # the bounds' terms in the number of classes
    near("loss", loss, ref["loss"][0], ref["loss"][1] * slack)
    near("gx", got[0], ref["gx"][0] + olds[0], ref["gx"][1] * slack + 4 * U * np.abs(olds[0]))
    near("gw", got[1][:, :few], ref["gw"][0], ref["gw"][1] * slack)
    near("gb", got[2][:few], ref["gb"][0] + 1, ref["gb"][1] * slack + 4 * U)
    assert np.all(got[1][:, few:] == 0) and np.all(got[2][few:] == 1)
    abi.mg_check_kernel_status()


def test_many_rows_of_few_classes(abi):
    """More rows than one block takes (262 144), three classes: every row's gradient from
    the formula, and sums to the bounds' accuracy."""
    m, k, v = 600001, 2, 3
    rng, x, w, b, y = problem(m, k, v, 29)
    z = x @ w + b
    e = np.exp(z - z.max(axis=1, keepdims=True))
    p = e / e.sum(axis=1, keepdims=True)
    keep, at = y >= 0, np.where(y >= 0, y, 0)
    loss = -(np.log(p[np.arange(m), at]) * keep).sum() / m
    p[np.arange(m), at] -= 1
    p *= keep[:, None] / m
    got_loss, got = call(abi, x, w, b, y, float(m), 1.0, [np.zeros(t.shape) for t in (x, w, b)], STORE)
    assert abs(got_loss - loss) <= 4 * m * U * loss
    # per row: a few roundings of logits below 10 and probabilities below 1
    assert np.abs(got[0] - p @ w.T).max() <= 200 * U / m
    assert np.abs(got[1] - x.T @ p).max() <= 4 * m * U * (np.abs(x).T @ np.abs(p)).max()
    assert np.abs(got[2] - p.sum(axis=0)).max() <= 4 * m * U * np.abs(p).sum(axis=0).max()
    abi.mg_check_kernel_status()


def test_empty(abi):
    loss, gw = abi.array([3.0]), abi.array([2.0] * 6)
    abi.mg_linear_xent_fwd(None, None, None, None, loss.ptr, 0, 2, 3, 1.0)
    assert loss.numpy()[0] == 0.0
    abi.mg_linear_xent_fwd_bwd(None, None, None, None, None, loss.ptr, None, gw.ptr, None, 0, 2, 3, 1.0, 0)
    assert np.all(gw.numpy() == 2.0)
    abi.mg_linear_xent_fwd_bwd(None, None, None, None, None, loss.ptr, None, gw.ptr, None, 0, 2, 3, 1.0, STORE)
    assert np.all(gw.numpy() == 0.0)
    # no inputs at all: the bias alone decides
    b, y = np.log(np.array([1.0, 2.0, 5.0])), abi.int_array([2, 0])
    db = abi.array(b)
    abi.mg_linear_xent_fwd(None, None, db.ptr, y.ptr, loss.ptr, 2, 0, 3, 2.0)
    assert abs(loss.numpy()[0] - (np.log(8 / 5) + np.log(8)) / 2) <= 1e-15
