"""GPU: group norm, 8-bit activations and the linear cross-entropy through the Tensor API,
each alone and together as a training step uses them, against numpy.

Tolerances: the kernels' own bounds are tested at the C ABI.  Here values that pass
through at most eight products and sums of at most 800 terms each, all well conditioned,
are compared normwise: 1e-11 is 100 times 800 half steps of fp64.
"""
import numpy as np
import pytest

from conftest import norm_err

pytestmark = pytest.mark.gpu
TOL = 1e-11
B = 64


def q8(x):
    m, n = x.shape
    nb = -(-n // B)
    full = np.zeros((m, nb * B))
    full[:, :n] = x
    blocks = full.reshape(m, nb, B)
    top = np.abs(blocks).max(axis=2, keepdims=True)
    inverse = np.divide(127.0, top, out=np.zeros_like(top), where=top > 0)
    codes = np.rint(blocks * inverse)
    codes = np.where(codes == 0, np.sign(blocks), codes)
    return (codes * (top / 127.0)).reshape(m, -1)[:, :n]


def silu(z):
    s = 1 / (1 + np.exp(-z))
    return z * s, s * (1 + z * (1 - s))


def group_norm(x, w, b, groups, eps):
    n, c = x.shape[0], x.shape[-1]
    v = x.reshape(n, -1, groups, c // groups)
    mean = v.mean(axis=(1, 3), keepdims=True)
    rstd = 1 / np.sqrt(v.var(axis=(1, 3), keepdims=True) + eps)
    unit = ((v - mean) * rstd).reshape(x.shape)
    return unit * w + b, unit, rstd


def group_norm_back(gz, unit, rstd, w, groups):
    n, c = gz.shape[0], gz.shape[-1]
    axes = tuple(range(gz.ndim - 1))
    u = (gz * w).reshape(n, -1, groups, c // groups)
    un = unit.reshape(u.shape)
    gx = rstd * (u - u.mean(axis=(1, 3), keepdims=True) - un * (u * un).mean(axis=(1, 3), keepdims=True))
    return gx.reshape(gz.shape), (gz * unit).sum(axis=axes), gz.sum(axis=axes)


def linear(api, w, b):
    lin = api.Linear(*w.shape)
    lin.weights().set_data(w)
    lin.bias().set_data(b)
    return lin


def xent(x, w, b, y):
    z = x @ w + b
    e = np.exp(z - z.max(axis=1, keepdims=True))
    keep = y >= 0
    at = np.where(keep, y, 0)
    p = e / e.sum(axis=1, keepdims=True)
    rows = np.arange(len(y))
    loss = -(np.log(p[rows, at]) * keep).sum() / len(y)
    p[rows, at] -= 1
    return loss, p * keep[:, None] / len(y)


@pytest.mark.parametrize("shape,groups,act", [((6, 40), 5, "silu"), ((3, 7, 5, 24), 4, "relu"), ((2, 130, 6), 6, "none")])
def test_group_norm_node(api, shape, groups, act):
    rng = np.random.default_rng(1)
    c = shape[-1]
    x, w, b, g = rng.standard_normal(shape), 1 + 0.1 * rng.standard_normal(c), rng.standard_normal(c), rng.standard_normal(shape)
    norm = api.GroupNorm(groups, c, 1e-5)
    assert np.all(norm.weights().data() == 1) and np.all(norm.bias().data() == 0)
    norm.weights().set_data(w)
    norm.bias().set_data(b)
    t, gt = api.Tensor(list(shape), x), api.Tensor(list(shape), g)
    y = norm.forward(t, act)
    assert y.shape() == list(shape)
    z, unit, rstd = group_norm(x, w, b, groups, 1e-5)
    want, slope = silu(z) if act == "silu" else (np.maximum(z, 0), (z > 0) * 1.0) if act == "relu" else (z, np.ones_like(z))
    assert norm_err(y.data(), want.reshape(-1)) <= TOL
    for sweep in (1, 2):  # the second sweep accumulates
        y.zero_grad()
        y.mul(gt).sum().backward()
        gx, gw, gb = group_norm_back(g * slope, unit, rstd, w, groups)
        for got, ref in ((t.grad(), gx), (norm.weights().grad(), gw), (norm.bias().grad(), gb)):
            assert norm_err(got, sweep * ref.reshape(-1)) <= TOL
    with pytest.raises(ValueError, match="groups of equal size"):
        api.GroupNorm(3, 10)
    with pytest.raises(ValueError, match="eps"):
        api.GroupNorm(2, 10, -1.0)
    with pytest.raises(ValueError, match="samples, ..., channels"):
        norm.forward(api.Tensor([4, c + 1]))
    with pytest.raises(ValueError, match="samples, ..., channels"):
        norm.forward(api.Tensor([c]))


def test_linear_cross_entropy_node(api):
    rng = np.random.default_rng(2)
    m, k, v = 21, 30, 333
    x, w, b = rng.standard_normal((m, k)), rng.standard_normal((k, v)) / 5, rng.standard_normal(v)
    y = rng.integers(0, v, m).astype(np.int32)
    y[[3, 11]] = -1
    head, t = linear(api, w, b), api.Tensor([m, k], x)
    ref, p = xent(x, w, b, y)
    for labels in (y, api.Tensor([m], y.astype(np.float64))):
        loss = api.linear_cross_entropy(t, head, labels)
        assert abs(loss.data()[0] - ref) <= TOL * ref
        for v_ in (t, head.weights(), head.bias()):
            v_.zero_grad()
        loss.mul(3.0).backward()  # an upstream gradient other than 1
        for got, want in ((t.grad(), p @ w.T), (head.weights().grad(), x.T @ p), (head.bias().grad(), p.sum(axis=0))):
            assert norm_err(got, 3 * want.reshape(-1)) <= TOL
    # the same as the loss of the logits, for rows that are all kept
    y2 = np.abs(y)
    two = api.softmax_cross_entropy(head.forward(t), y2).data()[0]
    assert abs(api.linear_cross_entropy(t, head, y2).data()[0] - two) <= TOL * two
    # parts that need no gradient get none; a loss without any is a loss all the same
    t.zero_grad()
    t.set_requires_grad(False)
    head.bias().zero_grad()
    loss = api.linear_cross_entropy(t, head, y, 7.0)
    loss.backward()
    assert np.all(t.grad() == 0) and norm_err(head.bias().grad(), p.sum(axis=0) * m / 7) <= TOL
    for v_ in (head.weights(), head.bias()):
        v_.set_requires_grad(False)
    assert abs(api.linear_cross_entropy(t, head, y).data()[0] - ref) <= TOL * ref
    with pytest.raises(ValueError, match="one label per row"):
        api.linear_cross_entropy(t, head, y[:-1])
    with pytest.raises(ValueError, match="layer's width"):
        api.linear_cross_entropy(api.Tensor([m, k + 1]), head, y)


def test_a_gradient_required_after_the_loss_is_refused(api):
    rng = np.random.default_rng(3)
    head = linear(api, rng.standard_normal((12, 9)), rng.standard_normal((1, 9)))
    x = api.Tensor([5, 12], rng.standard_normal((5, 12)))
    x.set_requires_grad(False)
    loss = api.linear_cross_entropy(x, head, np.arange(5))
    x.set_requires_grad(True)
    with pytest.raises(RuntimeError, match="did not when the loss was computed"):
        loss.backward()
    assert not np.any(head.weights().grad())


def test_keep_8bit_values_and_uses(api):
    rng = np.random.default_rng(3)
    m, n = 37, 150
    x = rng.standard_normal((m, n)) * np.exp(rng.standard_normal((m, 1)))
    t = api.Tensor([m, n], x)
    assert not t.kept_8bit()
    t.keep_8bit()
    want = q8(x)
    assert t.kept_8bit() and np.array_equal(t.data().reshape(m, n), want) and t.kept_8bit()
    assert t.at([3, 5]) == want[3, 5]
    # any operation reads the kept values; the codes stay
    assert np.array_equal(t.add(1.0).data().reshape(m, n), want + 1.0) and t.kept_8bit()
    t.keep_8bit()
    assert np.array_equal(t.data().reshape(m, n), want)
    # relu of it, and its gradient, from the codes
    g = rng.standard_normal((m, n))
    t.relu().mul(api.Tensor([m, n], g)).sum().backward()
    assert np.array_equal(t.grad().reshape(m, n), g * (want > 0))
    # a product's gradient
    w = api.Tensor([n, 11], rng.standard_normal((n, 11)))
    t.matmul(w).sum().backward()
    assert norm_err(w.grad(), np.repeat(want.sum(axis=0)[:, None], 11, axis=1).reshape(-1)) <= TOL
    # writing ends it
    t.set_at([0, 0], 5.0)
    assert not t.kept_8bit() and t.data()[0] == 5.0 and np.array_equal(t.data()[1:], want.reshape(-1)[1:])
    t.keep_8bit()
    t.copy_from_host(x)
    assert not t.kept_8bit() and np.array_equal(t.data(), x.reshape(-1))
    # vectors, scalars, logical zeros and empty tensors
    v = api.Tensor([70], x.reshape(-1)[:70])
    v.keep_8bit()
    assert np.array_equal(v.data(), q8(x.reshape(-1)[None, :70])[0])
    zero = api.Tensor([4, 4])
    zero.keep_8bit()
    assert np.all(zero.data() == 0)
    api.Tensor([0, 4]).keep_8bit()


def test_keep_8bit_frees_memory(api, abi):
    import ctypes as C
    free, total = C.c_size_t(), C.c_size_t()

    def pool_used():
        abi.mg_sync()
        abi.mg_mem_info(C.byref(free), C.byref(total))
        return total.value - free.value

    # 40 activations of 64 MiB need more than the pool has; kept in 8 bits they fit the
    # room that four of them take.
    n = 8 << 20
    held = []
    x = api.Tensor([n // 1024, 1024])  # (one operand for all: a graph node keeps its operands)
    base = pool_used()
    for _ in range(40):
        t = x.add(1.0)
        t.keep_8bit()
        held.append(t)
    assert pool_used() - base <= 40 * (n + n // 8) * 1.2 + 6 * 8 * n
    assert held[7].at([5, 9]) == 1.0


def test_parameters_in_a_shared_buffer_are_refused(api):
    lin = api.Linear(6, 4)
    opt = api.SGD([lin.weights(), lin.bias()], 0.1)
    opt.enable_allreduce()
    with pytest.raises(RuntimeError, match="shared with other tensors"):
        lin.weights().keep_8bit()


def model(api, seed, width=100, hidden=96, classes=517):
    rng = np.random.default_rng(seed)
    w = [rng.standard_normal(s) / np.sqrt(s[0]) for s in ((width, hidden), (hidden, 72), (72, classes))]
    b = [0.1 * rng.standard_normal(s.shape[1]) for s in w]
    gw, gb = 1 + 0.1 * rng.standard_normal(hidden), 0.1 * rng.standard_normal(hidden)
    layers = [linear(api, *p) for p in zip(w, b)]
    norm = api.GroupNorm(8, hidden)
    norm.weights().set_data(gw)
    norm.bias().set_data(gb)
    params = [t for lin in layers for t in (lin.weights(), lin.bias())] + [norm.weights(), norm.bias()]
    return rng, w, b, gw, gb, layers, norm, params


def step(api, x, y, layers, norm, opt):
    """Linear, group norm with SiLU, linear with ReLU, linear cross-entropy; the activations
    wait for the backward pass in 8 bits."""
    a = layers[0].forward(x)
    h = norm.forward(a, "silu")
    r = layers[1].forward_relu(h)
    h.keep_8bit()
    loss = api.linear_cross_entropy(r, layers[2], y)
    r.keep_8bit()
    opt.zero_grad()
    loss.backward()
    return loss


def reference_step(x, y, w, b, gw, gb):
    a = x @ w[0] + b[0]
    z, unit, rstd = group_norm(a, gw, gb, 8, 1e-5)
    h, slope = silu(z)
    r = np.maximum(h @ w[1] + b[1], 0)
    loss, p = xent(r, w[2], b[2], y)
    g2, gb2 = r.T @ p, p.sum(axis=0)
    gr = (p @ w[2].T) * (r > 0)
    g1, gb1 = q8(h).T @ gr, gr.sum(axis=0)  # the only product that reads an 8-bit activation
    ga, ggw, ggb = group_norm_back((gr @ w[1].T) * slope, unit, rstd, gw, 8)
    return loss, [x.T @ ga, ga.sum(axis=0), g1, gb1, g2, gb2, ggw, ggb]


def test_a_training_step_of_all_three(api, abi):
    rng, w, b, gw, gb, layers, norm, params = model(api, 4)
    m, lr = 130, 0.05
    opt = api.SGD(params, lr)
    values = [t.data().copy() for t in params]
    for it in range(3):
        x = rng.standard_normal((m, 100))
        y = rng.integers(0, 517, m).astype(np.int32)
        y[:5] = -1
        t = api.Tensor([m, 100], x)
        t.set_requires_grad(False)
        loss = step(api, t, y, layers, norm, opt)
        shaped = [v.reshape(s.shape) for v, s in zip(values, [w[0], b[0], w[1], b[1], w[2], b[2], gw, gb])]
        ref, grads = reference_step(x, y, shaped[0:6:2], shaped[1:6:2], shaped[6], shaped[7])
        assert abs(loss.data()[0] - ref) <= TOL * ref
        for p, g in zip(params, grads):
            assert norm_err(p.grad(), g.reshape(-1)) <= TOL
        opt.step()
        values = [v - lr * p.grad() for v, p in zip(values, params)]
        for v, p in zip(values, params):
            assert np.array_equal(v, p.data())
    abi.mg_check_kernel_status()


@pytest.mark.parametrize("m", [48, 3, 1])
def test_the_step_recorded_and_replayed(api, abi, m):
    """Replays give what the same steps give one launch at a time, bit for bit, also while
    another graph of the same parameters is alive."""
    rng, *_, layers, norm, params = model(api, 5)
    opt = api.SGD(params, 0.05)
    start = [p.data().copy() for p in params]
    xs = [rng.standard_normal((m, 100)) for _ in range(4)]
    ys = [rng.integers(-1, 517, m).astype(np.float64) for _ in range(4)]

    def fresh():
        for p, v in zip(params, start):
            p.set_data(v)

    x, y = api.Tensor([m, 100], xs[0]), api.Tensor([m], ys[0])
    x.set_requires_grad(False)
    eager = []
    for a, c in zip(xs, ys):
        x.copy_from_host(a)
        y.copy_from_host(c)
        eager.append(step(api, x, y, layers, norm, opt).data()[0])
        opt.step()
    want = [p.data().copy() for p in params]

    fresh()
    x.copy_from_host(xs[0])
    y.copy_from_host(ys[0])
    got = [step(api, x, y, layers, norm, opt).data()[0]]
    opt.step()
    alive = layers[0].forward(x).sum()  # an eager graph of the same leaves
    outside = api.Tensor([m, 100], xs[0])
    outside.keep_8bit()
    outside_values = outside.data().copy()
    rec = api.RecordedStep()
    rec.begin()
    loss = step(api, x, y, layers, norm, opt)
    opt.step()
    with pytest.raises(RuntimeError, match="made before the recording"):
        x.keep_8bit()
    with pytest.raises(RuntimeError, match="other side"):
        outside.add(1.0)
    rec.end()
    assert outside.kept_8bit() and np.array_equal(outside.data(), outside_values)
    for a, c in zip(xs[1:], ys[1:]):
        x.copy_from_host(a)
        y.copy_from_host(c)
        rec.replay()
        got.append(loss.data()[0])
    assert got == eager
    assert all(np.array_equal(p.data(), v) for p, v in zip(params, want))
    assert np.isfinite(alive.data()[0])
    del loss
    abi.mg_check_kernel_status()
