"""GPU: activations kept in 8 bits, through the device C ABI, against the definition in
numpy.  Codes, scales and values are exact: the definition names every rounding
(quotient, product, nearest whole number).  Products with 8-bit operands: u = 2^-53,
a contraction of n terms is off by at most (n + 2) u sum|terms|.
"""
import numpy as np
import pytest

from micrograd_b200 import cabi as K

pytestmark = pytest.mark.gpu
U = 2.0 ** -53
B = K.Q8_BLOCK
MAX_SCALE = float.fromhex("0x1.0204081020407p+1017")  # 127 steps of it are finite


def encode(x):
    m, n = x.shape
    nb = -(-n // B)
    full = np.zeros((m, nb * B))
    full[:, :n] = x
    blocks = full.reshape(m, nb, B)
    top = np.abs(blocks).max(axis=2)
    with np.errstate(all="ignore"):
        inverse = np.where(top >= 1e-300, 127.0 / top, 0.0)
        codes = np.rint(blocks * inverse[:, :, None])
        codes = np.where(codes == 0, np.sign(blocks), codes)
        scales = np.where(inverse > 0, np.minimum(top / 127.0, MAX_SCALE), 0.0)
        finite = np.isfinite(top)
        codes = np.where(finite[:, :, None], codes, np.nan_to_num(np.sign(blocks)))
        scales = np.where(finite, scales, np.nan)
    return codes.reshape(m, -1)[:, :n].astype(np.int8), scales


def decode(codes, scales):
    return codes * np.repeat(scales, B, axis=1)[:, :codes.shape[1]]


class Packed:
    def __init__(self, abi, m, n, codes=None, scales=None):
        self.abi, self.m, self.n = abi, m, n
        words = (m * n + 7) // 8 + 1
        raw = np.full(words * 8, 77, dtype=np.int8)
        if codes is not None:
            raw[:m * n] = codes.reshape(-1)
        self.codes = abi.array(raw.view(np.float64))
        self.scales = abi.array(np.full(m * -(-n // B) + 1, -5.0) if scales is None else scales)

    def read(self):
        raw = self.codes.numpy().view(np.int8)
        assert np.all(raw[self.m * self.n:] == 77)  # nothing behind the codes is written
        nb = -(-self.n // B)
        scales = self.scales.numpy()
        assert np.all(scales[self.m * nb:] == -5.0)
        return raw[:self.m * self.n].reshape(self.m, self.n), scales[:self.m * nb].reshape(self.m, nb)


def activation(m, n, seed, relu=True):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((m, n)) * np.exp(rng.standard_normal((m, 1)))
    return rng, (np.maximum(x, 0.0) if relu else x)


SHAPES = [(1, 1), (1, 63), (1, 64), (1, 65), (3, 128), (33, 785), (5, 130), (2, 4096), (64, 66), (257, 100), (7, 2),
          (1000, 1), (513, 192), (31, 68)]


@pytest.mark.parametrize("relu", [True, False])
@pytest.mark.parametrize("shape", SHAPES)
def test_pack_and_unpack(abi, shape, relu):
    m, n = shape
    _, x = activation(m, n, 1, relu)
    x.reshape(-1)[:: 7] *= 1e-4  # values below half a step keep their sign
    want_codes, want_scales = encode(x)
    dx, packed, back = abi.array(x), Packed(abi, m, n), abi.array(np.full(m * n + 2, 9.0))
    abi.mg_q8_pack(dx.ptr, packed.codes.ptr, packed.scales.ptr, m, n)
    codes, scales = packed.read()
    assert np.array_equal(codes, want_codes) and np.array_equal(scales, want_scales)
    assert np.array_equal(np.sign(codes), np.sign(x))
    abi.mg_q8_unpack(packed.codes.ptr, packed.scales.ptr, back.ptr, m, n)
    got = back.numpy()
    assert np.array_equal(got[:-2].reshape(m, n), decode(codes, scales)) and np.all(got[-2:] == 9.0)
    step = np.repeat(scales, B, axis=1)[:, :n]
    off = np.abs(got[:-2].reshape(m, n) - x)
    # half a step, a whole one for what is kept from 0, and the roundings of scale and inverse
    assert np.all(off <= np.where(np.abs(x) >= step / 2, 0.5, 1.0) * step + 127 * 4 * U * step)


def test_addresses_off_the_vector_boundaries(abi):
    m, n = 37, 192
    _, x = activation(m, n, 2, relu=False)
    want = encode(x)
    for shift in (1, 2, 3):
        dx = abi.array(np.concatenate([np.zeros(shift), x.reshape(-1)]))
        raw, scales, back = abi.array(np.zeros((m * n + 16) // 8 + 1)), abi.empty(m * 3 + shift), abi.empty(m * n + shift)
        abi.mg_q8_pack(dx.offset(shift), raw.ptr + shift, scales.offset(shift), m, n)
        assert np.array_equal(raw.numpy().view(np.int8)[shift:shift + m * n].reshape(m, n), want[0])
        assert np.array_equal(scales.numpy()[shift:].reshape(m, 3), want[1])
        abi.mg_q8_unpack(raw.ptr + shift, scales.offset(shift), back.offset(shift), m, n)
        assert np.array_equal(back.numpy()[shift:].reshape(m, n), decode(*want))


def test_special_blocks(abi):
    """Zeros, the smallest and largest numbers, infinities and NaN, each in a block beside
    ordinary ones."""
    x = np.ones((8, 3 * B))
    x[0, B:2 * B] = 0.0
    x[1, B] = 5e-324
    x[1, B + 1:2 * B] = 0.0
    x[2, B:2 * B] = -1e-301
    x[3, B:2 * B] = 1.7e308
    x[3, B + 1] = -1.7976931348623157e308
    x[4, B + 3] = np.inf
    x[5, B + 3] = -np.inf
    x[6, B + 3] = np.nan
    x[7, B:2 * B] = -0.0
    want_codes, want_scales = encode(x)
    m, n = x.shape
    dx, packed, back = abi.array(x), Packed(abi, m, n), abi.empty(m * n)
    abi.mg_q8_pack(dx.ptr, packed.codes.ptr, packed.scales.ptr, m, n)
    codes, scales = packed.read()
    assert np.array_equal(codes, want_codes) and np.array_equal(scales, want_scales, equal_nan=True)
    abi.mg_q8_unpack(packed.codes.ptr, packed.scales.ptr, back.ptr, m, n)
    y = back.numpy((m, n))
    assert np.array_equal(y, decode(codes, scales), equal_nan=True)
    assert np.all(y[:, :B] == 1.0) and np.all(y[:, 2 * B:] == 1.0)
    assert np.all(y[[0, 1, 2, 7], B:2 * B] == 0.0) and np.all(codes[2, B:2 * B] == -1) and codes[1, B] == 1
    assert np.all(np.isfinite(y[3])) and np.all(np.isnan(y[4:7, B:2 * B]))


# (rows, kept columns, other columns): one row, ten classes, odd sizes, tiles that end
# inside a block, long contractions that are split over the SMs.
PRODUCTS = [(1, 1, 1), (16, 10, 1), (1, 64, 130), (33, 785, 17), (128, 128, 128), (1000, 66, 10), (257, 100, 96),
            (640, 256, 200), (4096, 128, 10), (5000, 192, 64), (300, 1024, 130), (999, 34, 33), (2048, 130, 258),
            (129, 112, 2), (777, 320, 16)]


@pytest.mark.parametrize("shape", PRODUCTS)
def test_weight_gradient(abi, shape):
    m, k, n = shape
    rng, x = activation(m, k, 3, relu=False)
    codes, scales = encode(x)
    g, old = rng.standard_normal((m, n)), rng.standard_normal((k, n))
    values = decode(codes, scales)
    ref = (values.T.astype(np.longdouble) @ g.astype(np.longdouble))
    bound = (m + 4) * U * (np.abs(values).T @ np.abs(g))
    packed, dg = Packed(abi, m, k, codes, scales), abi.array(g)
    for acc in (0, 1):
        out = abi.array(old)
        abi.mg_gemm_tn_q8(packed.codes.ptr, packed.scales.ptr, dg.ptr, out.ptr, m, n, k, acc)
        off = np.abs(out.numpy((k, n)) - (ref + old * acc))
        assert np.all(off <= bound + acc * U * (np.abs(old) + np.abs(ref)))
        again = abi.array(old)
        abi.mg_gemm_tn_q8(packed.codes.ptr, packed.scales.ptr, dg.ptr, again.ptr, m, n, k, acc)
        assert np.array_equal(out.numpy(), again.numpy())
    abi.mg_check_kernel_status()


@pytest.mark.parametrize("shape", PRODUCTS)
def test_masked_input_gradient(abi, shape):
    m, k, n = shape
    rng, x = activation(m, k, 4, relu=True)
    codes, scales = encode(x)
    g, w, old = rng.standard_normal((m, n)), rng.standard_normal((k, n)), rng.standard_normal((m, k))
    mask = codes > 0
    assert np.array_equal(mask, x > 0)
    ref = (g.astype(np.longdouble) @ w.T.astype(np.longdouble)) * mask
    bound = (n + 2) * U * (np.abs(g) @ np.abs(w).T)
    packed, dg, dw = Packed(abi, m, k, codes, scales), abi.array(g), abi.array(w)
    for acc in (0, 1):
        out = abi.array(old)
        abi.mg_gemm_nt_q8(dg.ptr, dw.ptr, out.ptr, m, n, k, acc, packed.codes.ptr)
        got = out.numpy((m, k))
        assert np.all(np.abs(got - (ref + old * acc)) <= bound + acc * U * (np.abs(old) + np.abs(ref)))
        assert np.array_equal(got[~mask], (old * acc)[~mask])
    abi.mg_check_kernel_status()


def test_a_bad_block_reaches_its_own_rows_of_the_gradient_only(abi):
    m, k, n = 200, 192, 24
    rng, x = activation(m, k, 5)
    x[17, 70] = np.nan
    codes, scales = encode(x)
    g = rng.standard_normal((m, n))
    packed, dg, out = Packed(abi, m, k, codes, scales), abi.array(g), abi.empty(k * n)
    abi.mg_gemm_tn_q8(packed.codes.ptr, packed.scales.ptr, dg.ptr, out.ptr, m, n, k, 0)
    got = out.numpy((k, n))
    assert np.all(np.isnan(got[64:128])) and np.all(np.isfinite(got[:64])) and np.all(np.isfinite(got[128:]))


@pytest.mark.parametrize("n", [1, 5, 1024, 100003])
def test_relu_backward(abi, n):
    rng = np.random.default_rng(n)
    codes = rng.integers(-127, 128, n).astype(np.int8)
    codes[rng.random(n) < 0.3] = 0
    g, old = rng.standard_normal(n), rng.standard_normal(n)
    packed, dg = Packed(abi, 1, n, codes, np.zeros(1)), abi.array(g)
    for flags in (0, K.ACC_STORE_A):
        out = abi.array(old)
        abi.mg_relu_bwd_q8(packed.codes.ptr, dg.ptr, out.ptr, n, flags)
        assert np.array_equal(out.numpy(), g * (codes > 0) + (0 if flags else old))


@pytest.mark.parametrize("off", [1, 2, 3])
def test_relu_backward_off_the_vector_boundaries(abi, off):
    rng = np.random.default_rng(off)
    n = 1003
    codes, g, old = rng.integers(-3, 4, n + off).astype(np.int8), rng.standard_normal(n), rng.standard_normal(n)
    packed, dg, out = Packed(abi, 1, n + off, codes, np.zeros(1)), abi.array(g), abi.array(old)
    abi.mg_relu_bwd_q8(packed.codes.ptr + off, dg.ptr, out.ptr, n, 0)
    assert np.array_equal(out.numpy(), g * (codes[off:] > 0) + old)
    shifted, kept = abi.array(np.concatenate([np.zeros(off), g])), abi.array(np.concatenate([np.zeros(off), old]))
    abi.mg_relu_bwd_q8(packed.codes.ptr, shifted.ptr + 8 * off, kept.ptr + 8 * off, n, 0)
    assert np.array_equal(kept.numpy()[off:], g * (codes[:n] > 0) + old)
    assert not np.any(kept.numpy()[:off])


def test_offsets_beyond_32_bits(abi):
    """2.2e9 values: the last rows are packed and read back like the first."""
    m, n = 2 ** 31 // 1000 + 70000, 1000
    x = abi.empty(m * n)
    abi.mg_fill_uniform01(x.ptr, m * n, 3, 0)
    codes, scales = abi.empty(m * n // 8 + 1), abi.empty(m * 16)
    abi.mg_q8_pack(x.ptr, codes.ptr, scales.ptr, m, n)
    rows = 64
    tail = np.empty(rows * n)
    abi.mg_download(tail.ctypes.data, x.offset((m - rows) * n), rows * n)
    want = encode(tail.reshape(rows, n))
    got = np.empty(rows * n // 8)
    abi.mg_download(got.ctypes.data, codes.ptr + (m - rows) * n, rows * n // 8)
    assert np.array_equal(got.view(np.int8).reshape(rows, n), want[0])
    s = np.empty(rows * 16)
    abi.mg_download(s.ctypes.data, scales.offset((m - rows) * 16), rows * 16)
    assert np.array_equal(s.reshape(rows, 16), want[1])
    abi.mg_fill(x.ptr, 0.0, m * n)
    abi.mg_q8_unpack(codes.ptr, scales.ptr, x.ptr, m, n)
    abi.mg_download(tail.ctypes.data, x.offset((m - rows) * n), rows * n)
    assert np.array_equal(tail.reshape(rows, n), decode(*want))
    # the ReLU mask and the two products read the codes there as well
    g = abi.empty(m)
    abi.mg_fill(g.ptr, 0.0, m)
    abi.mg_fill(g.offset(m - 1), 1.0, 1)
    dw, w, dx = abi.empty(n), abi.array(np.ones(n)), x
    abi.mg_gemm_tn_q8(codes.ptr, scales.ptr, g.ptr, dw.ptr, m, 1, n, 0)
    assert np.array_equal(dw.numpy(), decode(*want)[-1])
    abi.mg_gemm_nt_q8(g.ptr, w.ptr, dx.ptr, m, 1, n, 0, codes.ptr)
    abi.mg_download(tail.ctypes.data, dx.offset((m - rows) * n), rows * n)
    assert np.array_equal(tail.reshape(rows, n)[-1], (want[0][-1] > 0) * 1.0) and not tail[:-n].any()


def test_empty(abi):
    out = abi.array([4.0] * 6)
    for m, n in ((0, 5), (5, 0)):
        abi.mg_q8_pack(None, None, None, m, n)
        abi.mg_q8_unpack(None, None, None, m, n)
    abi.mg_relu_bwd_q8(None, None, None, 0, 0)
    abi.mg_gemm_tn_q8(None, None, None, out.ptr, 0, 2, 3, 1)
    assert np.all(out.numpy() == 4.0)
    abi.mg_gemm_tn_q8(None, None, None, out.ptr, 0, 2, 3, 0)
    assert np.all(out.numpy() == 0.0)
