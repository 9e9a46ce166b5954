"""GPU: group norm with an activation, channels last, through the device C ABI against
the formula in numpy (sums in extended precision).

Bounds.  u = 2^-53 is half a step of fp64.  A sum of n terms in any order is off by at
most n u sum|terms|; a product, quotient or root adds u of its result; exp and the
sigmoid built on it are good to 8 u.  From there, with E values in a group:
  mean   E u mean|x|                             (dm)
  rstd   (E / 2 + 8) u rstd + rstd^3 dm^2 / 2    (variance around the computed mean)
  unit   rstd (dm + 2 u (|x| + |mean|)) + |unit| drstd / rstd
  z      |gamma| dunit + 2 u (|z| + |beta| + |gamma unit|)
  y      1.1 dz + 10 u |y|                       (|relu'| <= 1, |silu'| < 1.1)
and for the gradients, which are given mean and rstd (dm = drstd = 0):
  gz     |gy| (dz / 2 + 24 u)                    (|silu''| <= 1/2, |act'| < 1.1)
  sums   the terms' own errors plus n u sum|terms|
"""
import numpy as np
import pytest

from micrograd_b200 import cabi as K

pytestmark = pytest.mark.gpu
U = 2.0 ** -53
LD = np.longdouble

# (samples, positions, groups, channels per group): single values, one value a group,
# odd counts, groups that cross every vector and warp width, one group, many samples,
# groups in several pieces.
SHAPES = [(1, 1, 1, 1), (3, 1, 5, 1), (2, 7, 1, 1), (1, 196, 8, 8), (5, 1, 16, 64), (33, 13, 6, 5),
          (2, 9, 3, 33), (1, 300, 1, 64), (130, 3, 2, 2), (7, 1, 1, 1000), (2, 50, 64, 1), (3, 64, 4, 16),
          (1, 5000, 2, 3), (2, 1500, 1, 24), (700, 2, 4, 8), (1, 1024, 2, 128), (3, 1023, 1, 127),
          (2, 1, 3, 4099), (9, 785, 2, 10), (1, 40000, 1, 3)]


def act(z, kind):
    if kind == K.ACT_RELU:
        return np.maximum(z, 0), (z > 0).astype(LD)
    if kind == K.ACT_SILU:
        s = 1 / (1 + np.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    return z, np.ones_like(z)


def make(shape, seed, offset=1.0):
    n, p, g, d = shape
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((n, p, g, d)) * (0.5 + rng.random((g, d))) + offset * rng.standard_normal((g, d))
    return rng, x, 1 + 0.1 * rng.standard_normal(g * d), 0.1 * rng.standard_normal(g * d)


def stats(x, eps):
    x = x.astype(LD)
    mean = x.mean(axis=(1, 3))
    var = ((x - mean[:, None, :, None]) ** 2).mean(axis=(1, 3))
    return mean, 1 / np.sqrt(var + LD(eps))


def forward(x, gamma, beta, eps, kind):
    n, p, g, d = x.shape
    E = p * d
    mean, rstd = stats(x, eps)
    ga, be = gamma.reshape(g, d).astype(LD), beta.reshape(g, d).astype(LD)
    m, r = mean[:, None, :, None], rstd[:, None, :, None]
    unit = (x - m) * r
    z = unit * ga + be
    y, _ = act(z, kind)
    dm = (E + 2) * U * np.abs(x).mean(axis=(1, 3))
    dr = (E / 2 + 8) * U * rstd + rstd ** 3 * dm ** 2 / 2
    dunit = r * (dm[:, None, :, None] + 2 * U * (np.abs(x) + np.abs(m))) + np.abs(unit) * dr[:, None, :, None] / r
    dz = np.abs(ga) * dunit + 2 * U * (np.abs(z) + np.abs(be) + np.abs(ga * unit))
    return (y, mean, rstd), (1.1 * dz + 10 * U * np.abs(y), dm, dr)


def backward(x, gamma, beta, mean, rstd, gy, kind):
    n, p, g, d = x.shape
    E = p * d
    x, gy = x.astype(LD), gy.astype(LD)
    ga, be = gamma.reshape(g, d).astype(LD), beta.reshape(g, d).astype(LD)
    m, r = mean[:, None, :, None].astype(LD), rstd[:, None, :, None].astype(LD)
    unit = (x - m) * r
    z = unit * ga + be
    _, slope = act(z, kind)
    gz = gy * slope
    u = gz * ga
    m1, m2 = u.mean(axis=(1, 3), keepdims=True), (u * unit).mean(axis=(1, 3), keepdims=True)
    gx = r * (u - m1 - unit * m2)
    dunit = r * 2 * U * (np.abs(x) + np.abs(m)) + 2 * U * np.abs(unit)
    dz = np.abs(ga) * dunit + 2 * U * (np.abs(z) + np.abs(be) + np.abs(ga * unit))
    dgz = np.abs(gy) * (dz / 2 + 24 * U)
    du = dgz * np.abs(ga) + 2 * U * np.abs(u)
    dm1 = (du + (E + 2) * U * np.abs(u)).mean(axis=(1, 3), keepdims=True)
    dm2 = (du * np.abs(unit) + np.abs(u) * dunit + (E + 4) * U * np.abs(u * unit)).mean(axis=(1, 3), keepdims=True)
    dgx = r * (du + dm1 + np.abs(unit) * dm2 + dunit * np.abs(m2) + 6 * U * (np.abs(u) + np.abs(m1) + np.abs(unit * m2)))
    dgb = (dgz + (n * p + 2) * U * np.abs(gz)).sum(axis=(0, 1))
    dgg = (dgz * np.abs(unit) + np.abs(gz) * dunit + (n * p + 4) * U * np.abs(gz * unit)).sum(axis=(0, 1))
    return (gx, (gz * unit).sum(axis=(0, 1)), gz.sum(axis=(0, 1))), (dgx, dgg, dgb)


def near(got, ref, bound):
    ref, bound = np.asarray(ref).reshape(-1), np.asarray(bound).reshape(-1)
    off = np.abs(got.reshape(-1).astype(LD) - ref)
    worst = int(np.argmax(off - bound))
    assert np.all(off <= bound), (worst, float(got.reshape(-1)[worst]), float(ref[worst]), float(bound[worst]))


def call_fwd(abi, x, gamma, beta, eps, kind):
    n, p, g, d = x.shape
    dx, y, mean, rstd = abi.array(x), abi.empty(x.size), abi.empty(n * g), abi.empty(n * g)
    dg, db = (None if v is None else abi.array(v) for v in (gamma, beta))
    abi.mg_group_norm_fwd(dx.ptr, dg and dg.ptr, db and db.ptr, y.ptr, mean.ptr, rstd.ptr, n, p, g * d, g, eps, kind)
    return y.numpy(), mean.numpy(), rstd.numpy()


@pytest.mark.parametrize("kind", [K.ACT_NONE, K.ACT_RELU, K.ACT_SILU])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(abi, shape, kind):
    _, x, gamma, beta = make(shape, 11)
    got = call_fwd(abi, x, gamma, beta, 1e-5, kind)
    ref, bound = forward(x, gamma, beta, 1e-5, kind)
    for a, b, c in zip(got, ref, bound):
        near(a, b, c)
    again = call_fwd(abi, x, gamma, beta, 1e-5, kind)
    assert all(np.array_equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("kind", [K.ACT_NONE, K.ACT_RELU, K.ACT_SILU])
@pytest.mark.parametrize("shape", SHAPES)
def test_backward(abi, shape, kind):
    n, p, g, d = shape
    rng, x, gamma, beta = make(shape, 12)
    gy = rng.standard_normal(x.shape)
    mean, rstd = (v.astype(np.float64) for v in stats(x, 1e-5))
    ref, bound = backward(x, gamma, beta, mean, rstd, gy, kind)
    dev = [abi.array(v) for v in (x, gamma, beta, mean, rstd, gy)]
    olds = [rng.standard_normal(v.size) for v in (x, gamma, gamma)]
    for flags in (0, K.ACC_STORE_A | K.ACC_STORE_B | K.ACC_STORE_C, K.ACC_STORE_B):
        out = [abi.array(v) for v in olds]
        abi.mg_group_norm_bwd(*(v.ptr for v in dev), *(v.ptr for v in out), n, p, g * d, g, kind, flags)
        for i, (o, old, r, b) in enumerate(zip(out, olds, ref, bound)):
            old = np.zeros_like(old) if flags & (1 << i) else old
            near(o.numpy(), r.reshape(-1) + old, b.reshape(-1) + 2 * U * (np.abs(old) + np.abs(r.reshape(-1))))
    # each output alone is what it is beside the others
    full = [o.numpy() for o in out]
    for i in range(3):
        alone = abi.array(olds[i])
        abi.mg_group_norm_bwd(*(v.ptr for v in dev), *(alone.ptr if j == i else None for j in range(3)),
                              n, p, g * d, g, kind, flags)
        assert np.array_equal(alone.numpy(), full[i])


def test_gradient_against_differences(abi):
    """d/dt of sum(gy * y(x + t v, gamma + t a, beta + t b)) at 0 by central differences of
    the forward kernel: with h = 1e-4 the formula's error is h^2 / 6 times a third
    derivative that is below 200 sum|gy| here, and rounding adds 1e-15 sum|gy y| / h."""
    shape = (3, 20, 4, 6)
    rng, x, gamma, beta = make(shape, 13)
    gy, v = rng.standard_normal(x.shape), rng.standard_normal(x.shape)
    a, b = rng.standard_normal(gamma.size), rng.standard_normal(beta.size)
    n, p, g, d = shape
    _, mean, rstd = call_fwd(abi, x, gamma, beta, 1e-5, K.ACT_SILU)
    dev = [abi.array(t) for t in (x, gamma, beta, mean, rstd, gy)]
    out = [abi.empty(t.size) for t in (x, gamma, beta)]
    abi.mg_group_norm_bwd(*(t.ptr for t in dev), *(t.ptr for t in out), n, p, g * d, g, K.ACT_SILU, 7)
    slope = sum(float(np.dot(o.numpy(), t.reshape(-1))) for o, t in zip(out, (v, a, b)))
    h = 1e-4
    ends = [float(np.dot(call_fwd(abi, x + s * v, gamma + s * a, beta + s * b, 1e-5, K.ACT_SILU)[0], gy.reshape(-1)))
            for s in (h, -h)]
    total = np.abs(gy).sum()
    assert abs((ends[0] - ends[1]) / (2 * h) - slope) <= (h * h / 6 * 200 + 1e-11) * total


def test_no_parameters_and_large_offset(abi):
    """gamma and beta left out; and values far from zero, where a variance taken as a
    difference of squares would lose everything."""
    shape = (4, 37, 3, 10)
    _, x, _, _ = make(shape, 14, offset=0.0)
    x = x * 1e-3 + 1e6
    one, nil = np.ones(30), np.zeros(30)
    got = call_fwd(abi, x, None, None, 1e-12, K.ACT_NONE)
    ref, bound = forward(x, one, nil, 1e-12, K.ACT_NONE)
    for a, b, c in zip(got, ref, bound):
        near(a, b, c)
    same = call_fwd(abi, x, one, nil, 1e-12, K.ACT_NONE)
    assert np.array_equal(got[0], same[0])


@pytest.mark.parametrize("shape", [(1, 196, 8, 8), (40, 1, 4, 64), (2, 1500, 1, 24)])
def test_infinities_and_nan_stay_in_their_group(abi, shape):
    n, p, g, d = shape
    _, x, gamma, beta = make(shape, 15)
    clean = call_fwd(abi, x, gamma, beta, 1e-5, K.ACT_SILU)
    bad = x.copy()
    bad[0, p // 2, 0, 0] = np.nan
    bad[n - 1, p - 1, g - 1, d - 1] = np.inf
    y, mean, rstd = (v.reshape(w) for v, w in zip(call_fwd(abi, bad, gamma, beta, 1e-5, K.ACT_SILU),
                                                  (x.shape, (n, g), (n, g))))
    hit = np.zeros((n, g), dtype=bool)
    hit[0, 0] = hit[n - 1, g - 1] = True
    assert np.all(np.isnan(rstd[hit])) and np.array_equal(rstd[~hit], clean[2].reshape(n, g)[~hit])
    rows = y.transpose(0, 2, 1, 3)
    assert np.all(np.isnan(rows[hit]))
    assert np.array_equal(rows[~hit], clean[0].reshape(x.shape).transpose(0, 2, 1, 3)[~hit])


def test_equal_values_and_offset_pointers(abi):
    """A constant group: unit is 0 and rstd 1/sqrt(eps).  The same data from an address
    that is only 8-byte aligned."""
    n, p, g, d = 2, 11, 3, 4
    x = np.full((n, p, g, d), 2.5)
    y, mean, rstd = call_fwd(abi, x, None, None, 1e-4, K.ACT_NONE)
    assert np.all(y == 0) and np.all(mean == 2.5) and np.all(np.abs(rstd - 100.0) <= 100 * 4 * U)
    _, x, gamma, beta = make((n, p, g, d), 16)
    want = call_fwd(abi, x, gamma, beta, 1e-5, K.ACT_RELU)
    dx = abi.array(np.concatenate([[0.0], x.reshape(-1)]))
    y, mean, rstd = abi.zeros(x.size + 3), abi.empty(n * g), abi.empty(n * g)
    dg, db = abi.array(gamma), abi.array(beta)
    abi.mg_group_norm_fwd(dx.offset(1), dg.ptr, db.ptr, y.offset(1), mean.ptr, rstd.ptr, n, p, g * d, g, 1e-5, K.ACT_RELU)
    ref, bound = forward(x, gamma, beta, 1e-5, K.ACT_RELU)
    near(y.numpy()[1:-2], ref[0], bound[0])
    assert np.all(y.numpy()[[0, -2, -1]] == 0)  # nothing around the output is touched
    near(mean.numpy(), want[1].astype(LD), bound[1])


@pytest.mark.parametrize("p,g,d", [(1, 16, 64), (500, 2, 20), (40000, 1, 3)])
def test_offsets_beyond_32_bits(abi, p, g, d):
    """2.2e9 values, in each of the forms: the last samples are what they are alone."""
    c = g * d
    n = 2 ** 31 // (p * c) + max(1, 6000000 // (p * c))
    few = max(1, min(64, 200000 // (p * c)))
    size, tail = n * p * c, few * p * c
    x, y = abi.empty(size), abi.empty(size)
    abi.mg_fill_uniform01(x.ptr, size, 9, 0)
    mean, rstd = abi.empty(n * g), abi.empty(n * g)
    abi.mg_group_norm_fwd(x.ptr, None, None, y.ptr, mean.ptr, rstd.ptr, n, p, c, g, 1e-5, K.ACT_SILU)
    xt, yt = np.empty(tail), np.empty(tail)
    abi.mg_download(xt.ctypes.data, x.offset(size - tail), tail)
    abi.mg_download(yt.ctypes.data, y.offset(size - tail), tail)
    ref, bound = forward(xt.reshape(few, p, g, d), np.ones(c), np.zeros(c), 1e-5, K.ACT_SILU)
    near(yt, ref[0], bound[0])
    # backward with x as the upstream gradient
    gg, gb = abi.empty(c), abi.empty(c)
    abi.mg_group_norm_bwd(x.ptr, None, None, mean.ptr, rstd.ptr, x.ptr, y.ptr, gg.ptr, gb.ptr, n, p, c, g, K.ACT_SILU, 7)
    abi.mg_download(yt.ctypes.data, y.offset(size - tail), tail)
    m, r = np.empty(few * g), np.empty(few * g)
    abi.mg_download(m.ctypes.data, mean.offset((n - few) * g), few * g)
    abi.mg_download(r.ctypes.data, rstd.offset((n - few) * g), few * g)
    v = xt.reshape(few, p, g, d)
    ref, bound = backward(v, np.ones(c), np.zeros(c), m.reshape(few, g), r.reshape(few, g), v, K.ACT_SILU)
    near(yt, ref[0], bound[0])


def test_empty(abi):
    keep = abi.array([3.0] * 8)
    for n, p in ((0, 5), (5, 0)):
        abi.mg_group_norm_fwd(None, None, None, None, None, None, n, p, 8, 2, 1e-5, K.ACT_NONE)
        abi.mg_group_norm_bwd(None, None, None, None, None, None, None, keep.ptr, None, n, p, 8, 2, K.ACT_NONE, 0)
        assert np.all(keep.numpy() == 3.0)
    abi.mg_group_norm_bwd(None, None, None, None, None, None, None, keep.ptr, None, 0, 5, 8, 2, K.ACT_NONE, K.ACC_STORE_B)
    assert np.all(keep.numpy() == 0.0)
