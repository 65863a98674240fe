"""The 8-bit rows and products on the GPU (include/lunelette_serving.h) against their
definitions in 64 bits."""
import numpy as np
import pytest

import lunelette_amd as lh

import q8_oracle as q8

pytestmark = pytest.mark.gpu


# ---- rows ----

def upload(x, pad, offset):
    """Rows of x, padded, `offset` elements into a buffer: (buffer, pointer, stride)."""
    tokens, width = x.shape
    buf = np.full(offset + tokens * (width + pad), np.nan, np.float32)
    buf[offset:].reshape(tokens, width + pad)[:, :width] = x
    d = lh.DeviceBuffer.from_array(buf)
    return d, d.ptr + 4 * offset, width + pad


class Codes:
    """Outputs in 8 bits, padded and guarded."""

    def __init__(self, tokens, width, pad=0):
        self.tokens, self.width, self.stride = tokens, width, q8.up16(width) + 16 * pad
        self.codes = lh.DeviceBuffer.from_array(np.full(tokens * self.stride + 16, 0x5a, np.int8))
        self.scales = lh.DeviceBuffer.from_array(np.full(tokens + 1, 7.25, np.float32))

    def get(self):
        codes = self.codes.download(np.int8)
        assert np.all(codes[self.tokens * self.stride:] == 0x5a)
        codes = codes[:self.tokens * self.stride].reshape(self.tokens, self.stride)
        assert np.all(codes[:, self.width:] == 0x5a), "wrote between the rows"
        scales = self.scales.download(np.float32)
        assert scales[self.tokens] == 7.25
        return codes[:, :self.width], scales[:self.tokens]


def run_rows(gpu, x, pad=0, offset=0, code_pad=0, stream=None):
    tokens, width = x.shape
    keep, ptr, stride = upload(x, pad, offset)
    out = Codes(tokens, width, code_pad)
    lh.check(gpu.lh_q8_rows(ptr, stride, width, tokens, out.codes.ptr, out.stride, out.scales.ptr,
                            stream))
    lh.check(gpu.lh_device_synchronize())
    return out.get()


def run_silu(gpu, gate, up, pad=0, offset=0, code_pad=0):
    tokens, width = gate.shape
    both, ptr, stride = upload(np.concatenate([gate, up], axis=1), pad, offset)
    out = Codes(tokens, width, code_pad)
    lh.check(gpu.lh_q8_silu(ptr, stride, ptr + 4 * width, stride, width, tokens, out.codes.ptr,
                            out.stride, out.scales.ptr, None))
    lh.check(gpu.lh_device_synchronize())
    return out.get()


def run_norm(gpu, x, add, gamma, kept="own", pad=0, offset=0, code_pad=0):
    """kept: where h goes: "own", "x", "add" or None. Returns (h or None, codes, scales)."""
    tokens, width = x.shape
    d_x, x_ptr, xs = upload(x, pad, offset)
    d_a, a_ptr, adds = (None, None, 0) if add is None else upload(add, pad + 1, offset)
    d_g = lh.DeviceBuffer.from_array(np.concatenate([np.zeros(offset, np.float32), gamma]))
    d_h, h_ptr, hs = upload(np.zeros_like(x), pad + 2, offset)
    if kept != "own":
        h_ptr, hs = {"x": (x_ptr, xs), "add": (a_ptr, adds), None: (None, 0)}[kept]
        d_h = {"x": d_x, "add": d_a, None: None}[kept]
    out = Codes(tokens, width, code_pad)
    lh.check(gpu.lh_q8_norm(x_ptr, xs, a_ptr, adds, d_g.ptr + 4 * offset, h_ptr, hs, width, tokens,
                            out.codes.ptr, out.stride, out.scales.ptr, None))
    lh.check(gpu.lh_device_synchronize())
    h = None
    if kept:
        h = d_h.download(np.float32)[offset:].reshape(tokens, hs)
        assert np.isnan(h[:, width:]).all(), "wrote between the rows"
        h = h[:, :width]
    return (h,) + out.get()


WIDTHS = [(1, 1), (3, 2), (1, 16), (2, 63), (5, 64), (3, 65), (2, 1023), (2, 1024), (3, 1025),
          (7, 1371), (1, 3072), (70, 3072), (3, 4096), (1, 4097), (2, 8193), (3, 9216), (1, 16384),
          (2, 16385), (1, 65536), (300, 33)]


@pytest.mark.parametrize("tokens,width", WIDTHS)
def test_rows(gpu, tokens, width):
    rng = np.random.default_rng(tokens + width)
    x = (rng.normal(size=(tokens, width)) * np.exp(rng.normal(size=width))).astype(np.float32)
    got = run_rows(gpu, x)
    q8.check_rows(*got, x.astype(np.float64))
    for how in (dict(pad=3, offset=1), dict(pad=4, code_pad=1)):
        again = run_rows(gpu, x, **how)
        assert np.array_equal(again[0], got[0]) and np.array_equal(again[1], got[1])


@pytest.mark.parametrize("width", [w + d for w in (256, 512, 768, 1024, 2048, 3072, 4096, 6144, 8192,
                                                  12288, 16384, 24576, 32768)
                                   for d in (-1, 0, 1)])
def test_row_widths(gpu, width):
    """To either side of each way to hold a row, a number of rows that fills no workgroup."""
    rng = np.random.default_rng(width)
    x = (rng.normal(size=(6, width)) * np.exp(rng.normal(size=width))).astype(np.float32)
    y = rng.normal(size=(6, width)).astype(np.float32)
    gamma = (1 + 0.3 * rng.normal(size=width)).astype(np.float32)
    q8.check_rows(*run_rows(gpu, x), x.astype(np.float64))
    q8.check_rows(*run_silu(gpu, x, y), q8.silu(x, y))
    h, v = q8.norm(x, y, gamma)
    got = run_norm(gpu, x, y, gamma, kept="x", pad=1)
    assert np.array_equal(got[0], h)
    q8.check_rows(got[1], got[2], v)


def test_rows_ties_and_ranges(gpu):
    """Halves go to even codes, whatever the scale; constant, zero, subnormal, largest
    and nonfinite rows."""
    rng = np.random.default_rng(1)
    width = 600
    x = rng.normal(size=(14, width)).astype(np.float32)
    for r, s in ((0, 1.0), (1, 3.0), (2, 7 * 2.0 ** -20)):
        x[r] = (rng.integers(-126, 126, size=width) + 0.5) * s
        x[r, 7] = 127 * s
    x[3] = 0
    x[4] = -0.0
    x[5] = -2.75
    x[6] *= np.float32(1e-42)
    x[7] *= np.float32(1e38)
    x[8] = 0
    x[8, 599] = np.float32(1e-45)
    x[9, 0] = np.inf
    x[10, 599] = -np.inf
    x[11, 300] = np.nan
    x[12] = 0
    x[12, 5] = 3.4e38
    x[13] *= np.float32(2.0 ** -140)
    codes, scales = run_rows(gpu, x)
    want, scale, _ = q8.quantize(x.astype(np.float64))
    assert np.array_equal(codes, want)
    assert np.array_equal(scales, scale, equal_nan=True)
    assert list(np.nonzero(np.isnan(scales))[0]) == [9, 10, 11]
    assert np.all(np.abs(codes[:3].astype(int)) % 2 == (np.arange(width) == 7))
    assert np.all(codes[5] == -127)


@pytest.mark.parametrize("tokens,width", WIDTHS)
def test_silu(gpu, tokens, width):
    rng = np.random.default_rng(tokens * 3 + width)
    gate = (2 * rng.normal(size=(tokens, width))).astype(np.float32)
    up = (rng.normal(size=(tokens, width)) * np.exp(rng.normal(size=width))).astype(np.float32)
    got = run_silu(gpu, gate, up)
    q8.check_rows(*got, q8.silu(gate, up))
    for how in (dict(pad=3, offset=1), dict(pad=4, code_pad=1)):
        again = run_silu(gpu, gate, up, **how)
        assert np.array_equal(again[0], got[0]) and np.array_equal(again[1], got[1])


def test_silu_ranges(gpu):
    rng = np.random.default_rng(2)
    width = 300
    gate = rng.normal(size=(12, width)).astype(np.float32)
    up = rng.normal(size=(12, width)).astype(np.float32)
    gate[0] *= 1000                      # where the exponential ends
    gate[1] = -np.abs(gate[1]) * 80      # values far below the row's largest
    gate[2] *= np.float32(1e30)
    up[2] *= np.float32(1e20)            # v past FP32
    gate[3] = np.float32(-3e38)
    gate[4, 3] = np.inf
    gate[5, 4] = -np.inf
    up[6, 299] = np.inf
    up[7, 0] = np.nan
    gate[8] = 0
    gate[9] *= np.float32(1e-30)
    up[9] *= np.float32(1e-30)           # v past the smallest
    gate[10] *= np.float32(1e25)
    up[10] *= np.float32(1e13)           # v near the largest
    gate[11] = -800
    up[11] = np.float32(3e38)
    codes, scales = run_silu(gpu, gate, up)
    v = q8.silu(gate, up)
    v[4:8] = np.nan                      # an Inf or NaN in either
    q8.check_rows(codes, scales, v)
    assert list(np.nonzero(np.isnan(scales))[0]) == [2, 4, 5, 6, 7]


@pytest.mark.parametrize("width", [200, 500, 700, 1001, 2000, 3000, 4000, 6000, 8000, 12000, 16001,
                                   24000, 32000, 40000])
def test_nonfinite_anywhere(gpu, width):
    """One Inf or NaN in a row, in every part of it, in each input; the rows between stay."""
    at = sorted({0, 3, 255, 256, width // 3, width // 2, 3 * width // 4, width - 2, width - 1}
                & set(range(width)))
    tokens = 2 * len(at) + 1
    rng = np.random.default_rng(width)
    x, second = (rng.normal(size=(tokens, width)).astype(np.float32) for _ in range(2))
    gamma = rng.normal(size=width).astype(np.float32)
    for odd in (np.float32(np.nan), np.float32(np.inf), np.float32(-np.inf)):
        for place in (0, 1):
            both = [x.copy(), second.copy()]
            for i, c in enumerate(at):
                both[place][2 * i + 1, c] = odd
            bad = np.arange(tokens) % 2 == 1
            h, v = q8.norm(both[0], both[1], gamma)
            got = run_norm(gpu, both[0], both[1], gamma)
            v[bad] = np.nan
            q8.check_rows(*got[1:], v)
            got = run_silu(gpu, *both)
            v = q8.silu(*both)
            v[bad] = np.nan
            q8.check_rows(*got, v)
            if not place:
                got = run_rows(gpu, both[0])
                q8.check_rows(*got, both[0].astype(np.float64))
                assert np.array_equal(np.isnan(got[1]), bad) and not got[0][bad].any()


@pytest.mark.parametrize("tokens,width", WIDTHS)
def test_norm(gpu, tokens, width):
    rng = np.random.default_rng(tokens * 5 + width)
    x = (rng.normal(size=(tokens, width)) * np.exp(rng.normal(size=width))).astype(np.float32)
    add = rng.normal(size=(tokens, width)).astype(np.float32)
    gamma = (1 + 0.3 * rng.normal(size=width)).astype(np.float32)
    h, v = q8.norm(x, add, gamma)
    first = run_norm(gpu, x, add, gamma)
    assert np.array_equal(first[0], h)
    q8.check_rows(first[1], first[2], v)
    for how in (dict(kept="x"), dict(kept="add", pad=3, offset=1), dict(kept=None, pad=4),
                dict(kept="own", pad=1, offset=2, code_pad=1)):
        again = run_norm(gpu, x, add, gamma, **how)
        assert again[0] is None or np.array_equal(again[0], h)
        assert np.array_equal(again[1], first[1]) and np.array_equal(again[2], first[2])
    for kept in ("own", "x", None):
        alone = run_norm(gpu, x, None, gamma, kept=kept)
        assert alone[0] is None or np.array_equal(alone[0], x)
        q8.check_rows(alone[1], alone[2], q8.norm(x, None, gamma)[1])


def test_norm_ranges(gpu):
    """Rows far from 1, zero rows (the 1e-5 counts), and nonfinite ones, in their own
    rows only."""
    rng = np.random.default_rng(3)
    width = 500
    x = rng.normal(size=(11, width)).astype(np.float32)
    add = rng.normal(size=(11, width)).astype(np.float32)
    gamma = rng.normal(size=width).astype(np.float32)
    x[0], add[0] = 0, 0
    add[1] = -x[1]
    x[2] *= np.float32(1e-30)
    add[2] *= np.float32(1e-30)
    x[3] *= np.float32(1e37)
    x[4], add[4] = np.float32(3e38), np.float32(2e38)   # the sum overflows
    x[5, 3] = np.inf
    add[6, 4] = np.nan
    x[7, 1], add[7, 1] = np.inf, -np.inf
    x[8] = 5
    x[9, 0] = np.float32(1e6)
    h, v = q8.norm(x, add, gamma)
    v[4:8] = np.nan
    got = run_norm(gpu, x, add, gamma)
    assert np.array_equal(got[0], h, equal_nan=True)
    q8.check_rows(got[1], got[2], v)
    assert list(np.nonzero(np.isnan(got[2]))[0]) == [4, 5, 6, 7]
    # Weights that take the values past FP32, or are not finite.
    for odd in (np.float32(3e38), np.float32(np.inf), np.float32(np.nan)):
        g = gamma.copy()
        g[499] = odd
        h, v = q8.norm(x[8:], add[8:], g)
        got = run_norm(gpu, x[8:], add[8:], g)
        q8.check_rows(got[1], got[2], v)


# ---- products ----

SIZES = [(1, 1, 1), (16, 64, 1), (17, 65, 3), (5, 16, 16), (33, 200, 17), (100, 4096, 1),
         (3072, 4096, 1), (640, 1371, 2), (50, 2080, 33), (64, 1024, 64), (70, 65536, 2),
         (129, 127, 65), (2051, 544, 130), (1030, 9216, 9), (300, 8192, 24), (256, 512, 128),
         (513, 640, 257), (1000, 96, 500), (16, 9216, 300), (5003, 1371, 77), (4100, 640, 10),
         (1111, 3333, 111)]


@pytest.mark.parametrize("rows,cols,tokens", SIZES)
def test_matvec(gpu, rows, cols, tokens):
    rng = np.random.default_rng(rows * 7 + cols + tokens)
    codes, scales = q8.random_weights(rng, rows, cols)
    x = rng.integers(-128, 128, size=(tokens, cols), dtype=np.int8)
    x_scales = rng.uniform(0.01, 0.1, size=tokens).astype(np.float32)
    packed = q8.pack(gpu, codes, scales)
    want = q8.product(codes, scales, x, x_scales)
    for how in ({}, dict(x_pad=1, y_pad=3), dict(y_pad=4, y_offset=1)):
        got = q8.matvec(gpu, packed, x, x_scales, rows, **how)
        assert np.array_equal(got, want), how


@pytest.mark.parametrize("tokens", list(range(1, 18)) + [31, 32, 33, 48, 63, 64, 65, 96, 127, 128,
                                                         129, 255, 256, 257, 511, 512, 513])
def test_matvec_token_counts(gpu, tokens):
    """To either side of each way to run a product."""
    rows, cols = 1040, 1216
    rng = np.random.default_rng(tokens)
    codes, scales = q8.random_weights(rng, rows, cols)
    x = rng.integers(-128, 128, size=(tokens, cols), dtype=np.int8)
    x_scales = rng.uniform(0.01, 0.1, size=tokens).astype(np.float32)
    got = q8.matvec(gpu, q8.pack(gpu, codes, scales), x, x_scales, rows)
    assert np.array_equal(got, q8.product(codes, scales, x, x_scales))


@pytest.mark.parametrize("rows,cols,tokens", [(64, 65536, 1), (64, 65536, 40), (64, 65536, 300)])
def test_matvec_largest_sums(gpu, rows, cols, tokens):
    """Codes of -128 throughout: sums of 2^30."""
    codes = np.full((rows, cols), -128, np.int8)
    codes[1::2] = 127
    x = np.full((tokens, cols), -128, np.int8)
    scales, x_scales = np.ones(rows, np.float32), np.ones(tokens, np.float32)
    got = q8.matvec(gpu, q8.pack(gpu, codes, scales), x, x_scales, rows)
    assert np.all(got[:, 0] == 2.0 ** 30)
    assert np.array_equal(got, q8.product(codes, scales, x, x_scales))


@pytest.mark.parametrize("tokens", [3, 40, 300])
def test_matvec_scales(gpu, tokens):
    """Scales of 0, NaN and of every size, in their own rows and columns."""
    rows, cols = 70, 320
    rng = np.random.default_rng(tokens)
    codes, scales = q8.random_weights(rng, rows, cols)
    x = rng.integers(-128, 128, size=(tokens, cols), dtype=np.int8)
    x_scales = rng.uniform(0.01, 0.1, size=tokens).astype(np.float32)
    scales[[0, 1, 2, 3]] = 0, np.nan, 1e-38, 1e30
    x_scales[[0, 1, 2]] = np.nan, 0, 1e-30
    got = q8.matvec(gpu, q8.pack(gpu, codes, scales), x, x_scales, rows)
    assert np.array_equal(got, q8.product(codes, scales, x, x_scales), equal_nan=True)
    assert np.isnan(got[0]).all() and np.isnan(got[:, 1]).all()


def test_quantized_weights(gpu):
    """lh_q8_quantize equals the packed codes of the definition."""
    rows, cols = 37, 333
    rng = np.random.default_rng(4)
    w = rng.normal(size=(rows, cols)).astype(np.float32)
    w[3] = 0
    w[4, 332] = np.nan
    w[5] *= np.float32(1e-42)
    w[6] = rng.integers(-126, 126, size=cols) + 0.5
    w[6, 0] = 127
    w[7, 0] = np.inf
    codes, scales, _ = q8.quantize(w.astype(np.float64))
    d_w = lh.DeviceBuffer.from_array(w)
    packed = lh.DeviceBuffer(gpu.lh_q8_bytes(rows, cols))
    lh.check(gpu.lh_memset_device(packed.ptr, 0xff, packed.nbytes))
    lh.check(gpu.lh_q8_quantize(d_w.ptr, rows, cols, packed.ptr, None))
    lh.check(gpu.lh_device_synchronize())
    want = q8.pack(gpu, codes, scales)
    assert np.array_equal(packed.download(np.uint32), want.download(np.uint32))


@pytest.mark.parametrize("rows,cols", [(16, 5), (17, 1000), (3, 1500), (40, 2049)])
def test_quantized_nonfinite_anywhere(gpu, rows, cols):
    """One Inf or NaN in every other row, wherever it stands; packed codes from any address."""
    rng = np.random.default_rng(rows * cols)
    w = rng.normal(size=(rows, cols)).astype(np.float32)
    for r in range(0, rows, 2):
        w[r, r * (cols - 1) // max(1, rows - 1)] = (np.nan, np.inf, -np.inf)[r // 2 % 3]
    codes, scales, _ = q8.quantize(w.astype(np.float64))
    assert np.isnan(scales[::2]).all() and np.isfinite(scales[1::2]).all()
    d_w = lh.DeviceBuffer.from_array(np.concatenate([np.zeros(1, np.float32), w.ravel()]))
    d_s = lh.DeviceBuffer.from_array(scales)
    packed = [lh.DeviceBuffer(gpu.lh_q8_bytes(rows, cols)) for _ in range(4)]
    for p in packed:
        lh.check(gpu.lh_memset_device(p.ptr, 0xff, p.nbytes))
    lh.check(gpu.lh_q8_quantize(d_w.ptr + 4, rows, cols, packed[0].ptr, None))
    for p, offset in zip(packed[1:], (0, 1, 7)):
        d_c = lh.DeviceBuffer.from_array(np.concatenate([np.zeros(offset, np.int8), codes.ravel()]))
        lh.check(gpu.lh_q8_pack(d_c.ptr + offset, d_s.ptr, rows, cols, p.ptr, None))
        lh.check(gpu.lh_device_synchronize())
    for p in packed[:1] + packed[2:]:
        assert np.array_equal(p.download(np.uint8), packed[1].download(np.uint8))


def test_matvec_large_offsets(gpu):
    """Outputs and weights past 2^32 bytes."""
    rng = np.random.default_rng(5)
    rows, cols, tokens = 40, 64, 65535
    codes, scales = q8.random_weights(rng, rows, cols)
    x = rng.integers(-128, 128, size=(tokens, cols), dtype=np.int8)
    x_scales = rng.uniform(0.01, 0.1, size=tokens).astype(np.float32)
    stride = 17000
    packed = q8.pack(gpu, codes, scales)
    d_x, d_s = lh.DeviceBuffer.from_array(x), lh.DeviceBuffer.from_array(x_scales)
    y = lh.DeviceBuffer(4 * stride * tokens)
    need = gpu.lh_q8_scratch(rows, cols, tokens)
    scratch = lh.DeviceBuffer(max(16, need))
    lh.check(gpu.lh_q8_matvec(packed.ptr, d_x.ptr, cols, d_s.ptr, y.ptr, stride, rows, cols, tokens,
                              scratch.ptr, need, None))
    lh.check(gpu.lh_device_synchronize())
    want = q8.product(codes, scales, x, x_scales)
    for t in (0, 1, 40000, 65534):
        got = np.empty(rows, np.float32)
        lh.check(gpu.lh_memcpy_dtoh(got.ctypes.data, y.ptr + 4 * stride * t, got.nbytes))
        assert np.array_equal(got, want[t])
    del y
    # Weights: codes of 70000 rows x 65536 columns, made on the device.
    rows, cols, tokens = 70000, 65536, 2
    packed = lh.DeviceBuffer(gpu.lh_q8_bytes(rows, cols))
    lh.check(gpu.lh_memset_device(packed.ptr, 0, packed.nbytes))
    last = packed.ptr + (rows // 16 - 1) * (cols // 64) * 1024
    lh.check(gpu.lh_memset_device(last, 3, (cols // 64) * 1024))
    ones = np.ones(rows, np.float32)
    lh.check(gpu.lh_memcpy_htod(packed.ptr + rows // 16 * (cols // 64) * 1024, ones.ctypes.data,
                                ones.nbytes))
    x = np.ones((tokens, cols), np.int8)
    got = q8.matvec(gpu, packed, x, np.ones(tokens, np.float32), rows)
    assert np.all(got[:, :-16] == 0) and np.all(got[:, -16:] == 3 * cols)
