"""GPU: the operators for larger models at the edges of what they accept."""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest

from micrograd_b200 import cabi as K
from test_gpu_group_norm import backward, call_fwd, make, near, stats
from test_gpu_linear_xent import problem, reference
from test_gpu_q8 import Packed, activation, encode

pytestmark = pytest.mark.gpu
U = 2.0 ** -53
LD = np.longdouble
STORE = K.ACC_STORE_A | K.ACC_STORE_B | K.ACC_STORE_C
MAX = np.finfo(np.float64).max


def silu(z):
    """z / (1 + exp(-z)) and its derivative in extended precision."""
    z = z.astype(LD)
    with np.errstate(all="ignore"):
        e = np.exp(-z)
        s = 1 / (1 + e)
        return z / (1 + e), s * (1 + z * (1 - s))


# Channel counts that take the warp form, the tile form and the general form.
FORMS = {"warp": (3, 1, 8), "tile": (2, 40, 40), "general": (2, 1, 4200)}


def silu_of(abi, form, z):
    """silu(z) and silu'(z) as group norm computes them for the channels' values z: with
    gamma = 0 a channel's z is its beta, and with one sample's gy = 1 at one position, and 0
    elsewhere, gbeta is the derivative."""
    n, p, c = FORMS[form]
    ys, slopes = [], []
    for at in range(0, len(z), c):
        beta = np.zeros(c)
        part = z[at:at + c]
        beta[:len(part)] = part
        x = np.random.default_rng(at).standard_normal((n, p, 1, c))
        y, mean, rstd = call_fwd(abi, x, np.zeros(c), beta, 1e-5, K.ACT_SILU)
        y = y.reshape(n * p, c)
        assert all(np.array_equal(row, y[0], equal_nan=True) for row in y)
        gy = np.zeros((n * p, c))
        gy[-1] = 1.0
        dev = [abi.array(v) for v in (x, np.zeros(c), beta, mean, rstd, gy)]
        gx, gg, gb = abi.empty(x.size), abi.empty(c), abi.empty(c)
        abi.mg_group_norm_bwd(*(v.ptr for v in dev), gx.ptr, gg.ptr, gb.ptr, n, p, c, 1, K.ACT_SILU, STORE)
        if np.all(np.isfinite(part)):
            assert not np.any(gx.numpy())
        ys.append(y[0][:len(part)])
        slopes.append(gb.numpy()[:len(part)])
    return np.concatenate(ys), np.concatenate(slopes)


@pytest.mark.parametrize("form", list(FORMS))
def test_silu_far_out(abi, form):
    """The bounds: the sigmoid is good to 8 u where exp(z) is a normal number, and counts as
    0 below exp(-708) = 3.3e-308: at most 745 * 3.3e-308 of a value or a derivative is lost
    there, and nothing above 2^-1074 further out.  The derivative is s (1 + z (1 - s)): with s
    off by 8 u s, 1 - s is off by 8 u s and what it is multiplied to by 8 u s |z|, so that with
    the three roundings the derivative is good to 24 u s (1 + |z|), also where 1 - s is small."""
    out = np.array([30, 600, 699.9999, 700, 705, 707.9, 708, 709, 709.8, 745, 746, 1e4, 1e10, 1e300, MAX])
    z = np.concatenate([[0.0, 1e-300], out, -out])
    y, slope = silu_of(abi, form, z)
    ref, dref = silu(z)
    near(y, ref, 10 * U * np.abs(ref) + 745 * 3.4e-308)
    far = np.minimum(np.abs(z), 746.0)
    near(slope, dref, 24 * U * (1 + far) / (1 + np.exp(np.minimum(-z, 700.0))) + 746 * 3.4e-308)
    y, slope = silu_of(abi, form, np.array([np.inf, -np.inf, np.nan]))
    assert y[0] == np.inf and np.all(np.isnan(y[1:])) and np.all(np.isnan(slope))


@pytest.mark.parametrize("form", list(FORMS))
def test_silu_over_its_range(abi, form):
    rng = np.random.default_rng(5)
    z = np.concatenate([rng.uniform(-708, 708, 150), rng.standard_normal(150) * 4, rng.standard_normal(60) * 1e-8])
    y, slope = silu_of(abi, form, z)
    ref, dref = silu(z)
    near(y, ref, 10 * U * np.abs(ref))
    s = 1 / (1 + np.exp(-z.astype(LD)))
    near(slope, dref, 24 * U * s * (1 + np.abs(z)))


@pytest.mark.parametrize("n", [64, 66, 65, 127])
def test_codes_between_two_steps(abi, n):
    """Values at or beside half a step, where one rounding more or less is another code:
    whole and half numbers under whole maxima, so that x (127 / max) is exactly a half or
    next to one."""
    rng = np.random.default_rng(n)
    m = 600
    top = np.concatenate([[5, 7, 9, 10, 3, 1], rng.integers(1, 2000, m - 6)]).astype(np.float64)[:, None]
    x = np.rint(rng.uniform(-1, 1, (m, n)) * 2 * top) / 2
    for c in range(0, n, 64):  # every block has its maximum and both of its halves
        x[:, c] = top[:, 0]
        if c + 2 < n:
            x[:, c + 1], x[:, c + 2] = top[:, 0] / 2, -top[:, 0] / 2
    want_codes, want_scales = encode(x)
    dx, packed = abi.array(x), Packed(abi, m, n)
    abi.mg_q8_pack(dx.ptr, packed.codes.ptr, packed.scales.ptr, m, n)
    codes, scales = packed.read()
    assert np.array_equal(codes, want_codes) and np.array_equal(scales, want_scales)


def recorded(api, body):
    """`body` as a recorded step, which is closed whatever happens in it."""
    rec = api.RecordedStep()
    rec.begin()
    try:
        out = body()
    finally:
        rec.end()
    return rec, out


def test_a_buffer_that_a_recorded_step_uses_is_not_given_up(api, abi):
    rng = np.random.default_rng(7)
    m, n = 20, 70
    first, second = rng.standard_normal((2, m, n))
    x, w = api.Tensor([m, n], first), api.Tensor([n, 8], rng.standard_normal((n, 8)))
    x.set_requires_grad(False)
    warm = x.matmul(w).sum()
    del warm
    rec, out = recorded(api, lambda: x.matmul(w).sum())
    for t in (x, w):
        with pytest.raises(RuntimeError, match="a recorded step uses"):
            t.keep_8bit()
        assert not t.kept_8bit()
    x.copy_from_host(second)
    rec.replay()
    want = float((second @ w.data().reshape(n, 8)).sum())
    assert abs(out.data()[0] - want) <= 1e-11 * np.abs(second).sum()
    # a tensor that no step uses may still be kept
    other = api.Tensor([m, n], first)
    other.keep_8bit()
    assert other.kept_8bit()
    # the fp64 form of a kept tensor, once a step has read it, stays where it is
    other.add(1.0)
    rec2, out2 = recorded(api, lambda: other.add(1.0))
    other.keep_8bit()
    filler = [api.Tensor([m, n], np.full((m, n), 9.0)) for _ in range(4)]
    rec2.replay()
    assert np.array_equal(out2.data(), other.data() + 1.0) and len(filler) == 4
    # ... and is given up once no step is left that may use it
    count = abi.mg_graph_count()
    rec2.abandon()
    assert abi.mg_graph_count() == count - 1
    if count == 1:  # (no other test has left one)
        x.keep_8bit()
        assert x.kept_8bit()
    abi.mg_check_kernel_status()


@pytest.mark.parametrize("use", ["product", "mask"])
def test_codes_made_before_a_recording_are_not_read_by_it(api, abi, use):
    """A write outside the step gives such codes up, and replays would go on reading them."""
    rng = np.random.default_rng(8)
    m, n = 12, 70
    t = api.Tensor([m, n], rng.standard_normal((m, n)))
    w = api.Tensor([n, 5], rng.standard_normal((n, 5)))
    loss = (t.matmul(w) if use == "product" else t.relu()).sum()
    if use == "product":
        t.set_requires_grad(False)
    t.keep_8bit()
    values = []

    def body():
        with pytest.raises(RuntimeError, match="other side"):
            loss.backward()
        with pytest.raises(RuntimeError):  # (and the host does not read them into the step)
            values.append(t.data())

    rec, _ = recorded(api, body)
    assert t.kept_8bit() and not values and np.all(np.isfinite(t.data()))
    abi.mg_check_kernel_status()


def test_a_write_during_a_recording_loses_no_kept_values(api, abi):
    rng = np.random.default_rng(12)
    m, n = 9, 130
    x = rng.standard_normal((m, n))
    t, p = api.Tensor([m, n], x), api.Tensor([m, n], x)
    opt = api.SGD([p], 0.5)
    p.sum().backward()
    opt.step()  # (once before the recording)
    for v in (t, p):
        v.keep_8bit()
    kept, before = t.data().copy(), p.data().copy()
    p.add(0.0)  # (its fp64 form exists, for the step below)

    def body():
        for write in (lambda: t.copy_from_host(x), lambda: t.set_at([0, 0], 3.0)):
            with pytest.raises(RuntimeError):
                write()
        opt.step()

    rec, _ = recorded(api, body)
    assert t.kept_8bit() and np.array_equal(t.data(), kept)
    assert not p.kept_8bit()
    for _ in range(2):
        rec.replay()
        before = before - 0.5  # (rounded step by step, as the kernel does)
        assert np.array_equal(p.data(), before)
    t.copy_from_host(x)  # (gives up the parked codes, too)
    assert not t.kept_8bit() and np.array_equal(t.data(), x.reshape(-1))
    abi.mg_check_kernel_status()


def test_a_recorded_product_outlives_the_table_cache(abi):
    """Products of 600 other shapes, more than the cache of split contractions holds, run
    between a recording and its replays."""
    rng = np.random.default_rng(11)
    m, n, k = 4100, 64, 48  # weight gradient: the contraction over m is split
    a, g = rng.standard_normal((m, k)), rng.standard_normal((m, n))
    da, dg, out = abi.array(a), abi.array(g), abi.empty(k * n)
    abi.mg_gemm_tn(da.ptr, dg.ptr, out.ptr, m, n, k, 0)
    want = out.numpy()
    codes, scales = encode(a)
    packed, out8 = Packed(abi, m, k, codes, scales), abi.empty(k * n)
    abi.mg_gemm_tn_q8(packed.codes.ptr, packed.scales.ptr, dg.ptr, out8.ptr, m, n, k, 0)
    want8 = out8.numpy()
    step = C.c_int()
    abi.mg_graph_begin()
    abi.mg_gemm_tn(da.ptr, dg.ptr, out.ptr, m, n, k, 0)
    abi.mg_gemm_tn_q8(packed.codes.ptr, packed.scales.ptr, dg.ptr, out8.ptr, m, n, k, 0)
    abi.mg_graph_end(C.byref(step))
    big, small = abi.zeros(16 * 1300 * 16), abi.empty(256)
    for i in range(600):
        abi.mg_gemm_tn(big.ptr, big.ptr, small.ptr, 16 * (600 + i), 16, 16, 0)
    for _ in range(3):
        abi.mg_fill(out.ptr, 7.0, k * n)
        abi.mg_fill(out8.ptr, 7.0, k * n)
        abi.mg_graph_launch(step.value)
        assert np.array_equal(out.numpy(), want) and np.array_equal(out8.numpy(), want8)
    # ... and the same products, one launch at a time, are still what they were
    abi.mg_gemm_tn(da.ptr, dg.ptr, out.ptr, m, n, k, 0)
    assert np.array_equal(out.numpy(), want)
    abi.mg_graph_destroy(step.value)
    for i in range(600):  # (without a recorded step the tables go again)
        abi.mg_gemm_tn(big.ptr, big.ptr, small.ptr, 16 * (600 + i), 16, 16, 0)
    abi.mg_gemm_tn(da.ptr, dg.ptr, out.ptr, m, n, k, 0)
    assert np.array_equal(out.numpy(), want)
    abi.mg_check_kernel_status()


def memory_growth(setup, small, call):
    """Bytes by which the device's used memory grows in `call`, in a process of its own;
    `small` has run all of its kernels before."""
    code = ("import ctypes as C, sys\nsys.path.insert(0, %r)\nimport micrograd_b200\nabi = micrograd_b200.load_abi()\nabi.mg_init(-1)\n"
            "def used():\n    f, t = C.c_size_t(), C.c_size_t()\n    abi.mg_sync()\n    abi.mg_mem_info(C.byref(f), C.byref(t))\n"
            "    return t.value - f.value\n%s\n%s\nbefore = used()\n%s\nprint(used() - before)\n"
            % (os.path.dirname(os.path.dirname(os.path.abspath(__file__))), setup, small, call))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    return int(r.stdout.split()[-1])


def test_workspace_of_the_masked_input_gradient(abi):
    """3 million rows of 17 columns (copied to 32 in the workspace, 768 MB as a whole) are
    taken in pieces of at most 256 MiB; the pool may add 64."""
    setup = ("m, n, k = 3000001, 17, 2\ng, w, dx, codes = abi.zeros(m * n), abi.zeros(n * k), abi.empty(m * k), abi.zeros(m * k // 8 + 1)")
    call = "abi.mg_gemm_nt_q8(g.ptr, w.ptr, dx.ptr, %s, n, k, 0, codes.ptr)"
    assert memory_growth(setup, call % 1000, call % "m") <= (256 + 64) << 20


def test_masked_input_gradient_in_pieces(abi):
    """The rows at the ends of the pieces (a piece holds 256 MiB / 8 / 32 = 1 048 576 rows)
    and the last one, with and without accumulation."""
    m, n, k = 2100003, 17, 3
    piece = 1 << 20
    rows = np.array([0, 1, piece - 1, piece, piece + 1, 2 * piece - 1, 2 * piece, m - 1])
    rng = np.random.default_rng(9)
    g, w = rng.standard_normal((m, n)), rng.standard_normal((k, n))
    codes, old = rng.integers(-2, 3, (m, k)).astype(np.int8), rng.standard_normal((m, k))
    packed, dg, dw = Packed(abi, m, k, codes, np.zeros(1)), abi.array(g), abi.array(w)
    for acc in (0, 1):
        out = abi.array(old)
        abi.mg_gemm_nt_q8(dg.ptr, dw.ptr, out.ptr, m, n, k, acc, packed.codes.ptr)
        got = out.numpy((m, k))
        ref = (g @ w.T) * (codes > 0) + acc * old
        bound = (2 * n + 6) * U * (np.abs(g) @ np.abs(w).T + np.abs(old))  # (numpy's own errors too)
        assert np.all(np.abs(got - ref) <= bound)
        exact = (g[rows].astype(LD) @ w.T.astype(LD)) * (codes[rows] > 0) + acc * old[rows]
        assert np.all(np.abs(got[rows] - exact) <= bound[rows])


def test_workspace_of_the_weight_gradient(abi):
    """100 000 rows of 16 kept and 1001 other columns (copied to 1008, 806 MB as a whole): at
    most 256 MiB for each; the pool may add 64."""
    setup = "m, n, k = 100000, 1001, 16\ng, codes, scales, dw = abi.zeros(m * n), abi.zeros(m * k // 8 + 1), abi.zeros(m), abi.empty(n * k)"
    call = "abi.mg_gemm_tn_q8(codes.ptr, scales.ptr, g.ptr, dw.ptr, %s, n, k, 0)"
    assert memory_growth(setup, call % 1000, call % "m") <= (512 + 64) << 20


def test_weight_gradient_in_pieces(abi):
    """Rows of 1008 doubles in the workspace: pieces of 33 280 rows."""
    m, n, k = 70001, 1001, 10
    rng, x = activation(m, k, 14)
    codes, scales = encode(x)
    g, old = rng.standard_normal((m, n)), rng.standard_normal((k, n))
    values = codes * np.repeat(scales, 64, axis=1)[:, :k]
    packed, dg = Packed(abi, m, k, codes, scales), abi.array(g)
    bound = (2 * m + 8) * U * (np.abs(values).T @ np.abs(g) + np.abs(old))  # (numpy's own errors too)
    for acc in (0, 1):
        out = abi.array(old)
        abi.mg_gemm_tn_q8(packed.codes.ptr, packed.scales.ptr, dg.ptr, out.ptr, m, n, k, acc)
        assert np.all(np.abs(out.numpy((k, n)) - (values.T @ g + old * acc)) <= bound)


def test_workspace_of_the_norm_of_wide_rows(abi):
    """16 384 rows of 2049 channels in one group.  Channel sums of each row would take 537 MB;
    what a call needs does not grow with the data, and the pool may add 64 MiB."""
    setup = ("n, c = 16384, 2049\nx, gy, gx = abi.zeros(n * c), abi.zeros(n * c), abi.empty(n * c)\n"
             "m, r, gg, gb = abi.zeros(n), abi.zeros(n), abi.empty(c), abi.empty(c)")
    call = ("abi.mg_group_norm_bwd(x.ptr, None, None, m.ptr, r.ptr, gy.ptr, gx.ptr, gg.ptr, gb.ptr, %s, 1, c, 1, 2, 7)")
    assert memory_growth(setup, call % 10, call % "n") <= (16 + 64) << 20


@pytest.mark.parametrize("p", [1, 2])
def test_norm_gradients_of_many_wide_rows(abi, p):
    """Gradients of each row, and the channels' sums over all of them added to what was there."""
    d = 2049
    n = 9000
    rng = np.random.default_rng(10)
    x = abi.empty(n * p * d)
    gy = abi.empty(n * p * d)
    abi.mg_fill_uniform01(x.ptr, n * p * d, 3, 0)
    abi.mg_fill_uniform01(gy.ptr, n * p * d, 4, 0)
    xv, gv = x.numpy((n, p, 1, d)), gy.numpy((n, p, 1, d))
    gamma, beta = 1 + 0.1 * rng.standard_normal(d), 0.1 * rng.standard_normal(d)
    mean, rstd = xv.mean(axis=(1, 3)), 1 / np.sqrt(xv.var(axis=(1, 3)) + 1e-5)
    m4, r4 = mean[:, None, :, None], rstd[:, None, :, None]
    olds = [rng.standard_normal(v.shape) for v in (gamma, gamma)]
    dev = [abi.array(v) for v in (gamma, beta, mean, rstd)]
    gx, gg, gb = abi.empty(n * p * d), abi.array(olds[0]), abi.array(olds[1])
    abi.mg_group_norm_bwd(x.ptr, *(v.ptr for v in dev), gy.ptr, gx.ptr, gg.ptr, gb.ptr, n, p, d, 1, K.ACT_RELU, K.ACC_STORE_A)
    unit = (xv - m4) * r4
    gz = gv * (unit * gamma + beta > 0)
    # (all of this is well conditioned: sums of at most 18 000 terms of one size)
    for got, ref, old, size in ((gg, (gz * unit).sum(axis=(0, 1))[0], olds[0], np.abs(gz * unit).sum(axis=(0, 1))[0]),
                                (gb, gz.sum(axis=(0, 1))[0], olds[1], np.abs(gz).sum(axis=(0, 1))[0])):
        assert np.all(np.abs(got.numpy() - (ref + old)) <= 2 * (n * p + 40) * U * (size + np.abs(old)))
    got = gx.numpy((n, p, 1, d))
    for i in (0, 1, 7, 8, 295, 296, 4500, n - 1):
        ref, bound = backward(xv[i:i + 1], gamma, beta, mean[i:i + 1], rstd[i:i + 1], gv[i:i + 1], K.ACT_RELU)
        near(got[i], ref[0], bound[0])
    u = gz * gamma
    full = r4 * (u - u.mean(axis=(1, 3), keepdims=True) - unit * (u * unit).mean(axis=(1, 3), keepdims=True))
    assert np.abs(got - full).max() <= 1e-11 * np.abs(full).max()


@pytest.mark.parametrize("shifts", [(0, 0, 0), (1, 1, 1), (0, 0, 1), (0, 1, 0), (1, 0, 0)])
@pytest.mark.parametrize("m", [1, 2, 3, 4])
def test_few_rows_off_the_vector_boundaries(abi, m, shifts):
    """Even class counts, whose rows of w and gw are taken in pairs where the addresses of
    both allow it: x, w and gw start `shifts` doubles behind a boundary."""
    k, v = 70, 130
    rng, x, w, b, y = problem(m, k, v, 40 + m, out_rows=0.0)
    if m > 2:
        y[1] = -1
    ref = reference(x, w, b, y, float(m), 0.8)
    olds = [rng.standard_normal(t.shape) for t in (x, w, b)]

    def put(t, shift):
        return abi.array(np.concatenate([np.zeros(shift), t.reshape(-1), [55.0]]))

    sx, sw, sg = shifts
    dx, dw, db, dy, dg, loss = put(x, sx), put(w, sw), abi.array(b), abi.int_array(y), abi.array([0.8]), abi.empty(1)
    for flags in (0, STORE):
        out = [put(olds[0], 0), put(olds[1], sg), put(olds[2], 0)]
        abi.mg_linear_xent_fwd_bwd(dx.offset(sx), dw.offset(sw), db.ptr, dy.ptr, dg.ptr, loss.ptr,
                                   out[0].ptr, out[1].offset(sg), out[2].ptr, m, k, v, float(m), flags)
        assert abs(LD(loss.numpy()[0]) - ref["loss"][0]) <= ref["loss"][1]
        for name, o, old, s in zip(("gx", "gw", "gb"), out, olds, (0, sg, 0)):
            a = o.numpy()
            assert a[-1] == 55.0 and not np.any(a[:s])
            r, bound = ref[name]
            was = 0 * old if flags else old
            assert np.all(np.abs(a[s:-1].reshape(old.shape).astype(LD) - (r + was)) <= bound + 2 * U * (np.abs(r) + np.abs(was)))
    abi.mg_check_kernel_status()


@pytest.mark.parametrize("which", ["x", "gy", "gx", "all"])
@pytest.mark.parametrize("shape", [(9, 3, 4, 8), (5, 1, 3, 64), (3, 50, 2, 12), (2, 6, 1, 4200)])
def test_norm_gradients_off_the_vector_boundaries(abi, shape, which):
    """x, gy and gx start one and two doubles behind a 32-byte boundary, one at a time and
    together, in the warp form (twice), the tile form and the general form."""
    n, p, g, d = shape
    rng, x, gamma, beta = make(shape, 41)
    gy, old = rng.standard_normal(x.shape), rng.standard_normal(x.shape)
    mean, rstd = (v.astype(np.float64) for v in stats(x, 1e-5))
    ref, bound = backward(x, gamma, beta, mean, rstd, gy, K.ACT_SILU)
    params = [abi.array(v) for v in (gamma, beta, mean, rstd)]
    for shift in (1, 2):
        s = [shift if which in (name, "all") else 0 for name in ("x", "gy", "gx")]
        for flags in (0, K.ACC_STORE_A):
            dx, dgy, dgx = (abi.array(np.concatenate([np.zeros(k), v.reshape(-1), [55.0]])) for k, v in zip(s, (x, gy, old)))
            gg, gb = abi.empty(g * d), abi.empty(g * d)
            abi.mg_group_norm_bwd(dx.offset(s[0]), *(v.ptr for v in params), dgy.offset(s[1]), dgx.offset(s[2]), gg.ptr, gb.ptr,
                                  n, p, g * d, g, K.ACT_SILU, flags | K.ACC_STORE_B | K.ACC_STORE_C)
            got = dgx.numpy()
            assert got[-1] == 55.0 and not np.any(got[:s[2]])
            was = np.zeros(x.size) if flags else old.reshape(-1)
            near(got[s[2]:-1], ref[0].reshape(-1) + was, bound[0].reshape(-1) + 2 * U * (np.abs(was) + np.abs(ref[0].reshape(-1))))
            near(gg.numpy(), ref[1], bound[1])
            near(gb.numpy(), ref[2], bound[2])


@pytest.mark.parametrize("shape", [(9, 3, 4, 8), (3, 50, 2, 12)])
def test_norm_off_the_vector_boundaries(abi, shape):
    n, p, g, d = shape
    _, x, gamma, beta = make(shape, 42)
    want = call_fwd(abi, x, gamma, beta, 1e-5, K.ACT_RELU)
    dg, db = abi.array(gamma), abi.array(beta)
    for sx, sy in ((2, 0), (0, 2), (1, 0), (0, 1), (2, 2)):
        dx = abi.array(np.concatenate([np.zeros(sx), x.reshape(-1)]))
        y, mean, rstd = abi.array(np.full(sy + x.size + 1, 55.0)), abi.empty(n * g), abi.empty(n * g)
        abi.mg_group_norm_fwd(dx.offset(sx), dg.ptr, db.ptr, y.offset(sy), mean.ptr, rstd.ptr, n, p, g * d, g, 1e-5, K.ACT_RELU)
        got = y.numpy()
        assert got[-1] == 55.0 and np.all(got[:sy] == 55.0)
        # (another vector width adds the group's values up in another order)
        e = p * d
        assert np.abs(got[sy:-1] - want[0]).max() <= 8 * (e + 20) * U * max(1.0, np.abs(x).max()) * want[2].max() * 1.5
        assert np.abs(mean.numpy() - want[1]).max() <= 2 * e * U * np.abs(x).max()


def test_a_refusal_during_a_recording_forgets_nothing(api, abi):
    """A tensor that the step being recorded uses is refused then, and afterwards too; the
    fp64 form of a kept one that it reads stays."""
    rng = np.random.default_rng(15)
    x, y = (api.Tensor([6, 70], rng.standard_normal((6, 70))) for _ in range(2))
    y.keep_8bit()
    y.add(1.0)  # (its fp64 form)

    def body():
        out = x.add(1.0), y.add(1.0)
        with pytest.raises(RuntimeError, match="made before the recording"):
            x.keep_8bit()
        y.keep_8bit()
        return out

    rec, (of_x, of_y) = recorded(api, body)
    with pytest.raises(RuntimeError, match="a recorded step uses"):
        x.keep_8bit()
    y.keep_8bit()
    filler = [api.Tensor([6, 70], np.full((6, 70), 9.0)) for _ in range(4)]
    rec.replay()
    assert np.array_equal(of_x.data(), x.data() + 1.0) and np.array_equal(of_y.data(), y.data() + 1.0) and len(filler) == 4
    rec.abandon()


@pytest.mark.parametrize("use", ["product", "mask", "layer"])
def test_a_refused_gradient_is_not_marked_as_written(api, abi, use):
    rng = np.random.default_rng(16)
    t = api.Tensor([12, 70], rng.standard_normal((12, 70)))
    w = api.Tensor([70, 5], rng.standard_normal((70, 5)))
    head = api.Linear(70, 5)
    leaf = {"product": w, "mask": t, "layer": head.weights()}[use]
    out = t.matmul(w) if use == "product" else t.relu() if use == "mask" else head.forward(t)
    if use != "mask":
        t.set_requires_grad(False)
    loss = out.sum()
    t.keep_8bit()

    def body():
        with pytest.raises(RuntimeError, match="other side"):
            loss.backward()

    recorded(api, body)[0].abandon()
    assert not np.any(leaf.grad())  # (a logical zero: there is no buffer to read)
