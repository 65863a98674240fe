"""Products of 8-bit rows by every kernel that runs them: the sizes here reach each one, on the
CPU by its choice, and on the GPU its outputs equal the formula's bit for bit."""
import ctypes

import numpy as np
import pytest

import lunelette_amd as lh

import q8_oracle as q8

# (rows, cols, tokens): (kernel, column splits). Kernels 0 to 3 stream the weights, with two
# tiles of rows a workgroup in 1 and 3 and two of tokens in 2 and 3; 4 to 8 are tiles in
# LDS of 64 x 32 (rows by tokens), 64 x 64, 64 x 128, 128 x 128 and 192 x 128.
WAYS = {
    (1111, 3333, 16): (0, 1), (3072, 4096, 4): (0, 1), (6144, 512, 4): (0, 1),
    (6144, 512, 5): (1, 1), (6129, 1000, 16): (1, 1), (6145, 70, 9): (1, 1),
    (1040, 1216, 17): (2, 1), (6128, 333, 32): (2, 1),
    (6145, 300, 24): (3, 1), (6200, 130, 32): (3, 1), (6160, 1371, 17): (3, 1),
    (2051, 544, 130): (4, 1), (3000, 2000, 129): (4, 1), (404, 3126, 180): (4, 5),
    (2500, 1371, 300): (5, 1), (2049, 700, 1025): (5, 1), (872, 4223, 202): (5, 4),
    # One step of columns, an odd and an even number of them, splits.
    (2048, 64, 1024): (6, 1), (917, 311, 1157): (6, 1), (4001, 1400, 260): (6, 1),
    (1500, 6000, 200): (6, 5),
    # Whole last tiles and parts of one, which leave by other stores.
    (7000, 100, 400): (7, 1), (4158, 313, 760): (7, 1), (5000, 1000, 700): (7, 1),
    (3200, 64, 2500): (7, 1), (1025, 9000, 1000): (7, 3),
    (9000, 64, 500): (8, 1), (4608, 900, 1111): (8, 1), (4610, 900, 1111): (8, 1),
    (9217, 520, 513): (8, 1), (2795, 346, 1504): (8, 1), (2858, 16322, 135): (8, 8),
}


def way(rows, cols, tokens):
    splits = ctypes.c_uint32()
    return lh.test_lib().lunelette_metal_test_q8_way(rows, cols, tokens,
                                                     ctypes.byref(splits)), splits.value


def test_every_kernel_is_reached():
    assert {size: way(*size) for size in WAYS} == WAYS
    assert {kernel for kernel, _ in WAYS.values()} == set(range(9))
    for kernel, height in ((7, 128), (8, 192)):
        last = {rows % height == 0 for (rows, _, _), (k, s) in WAYS.items()
                if k == kernel and s == 1}
        assert last == {True, False}


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,tokens", WAYS)
def test_matvec_by_every_kernel(gpu, rows, cols, tokens):
    rng = np.random.default_rng(rows + 3 * cols + 7 * tokens)
    codes, scales = q8.random_weights(rng, rows, cols)
    x = rng.integers(-128, 128, size=(tokens, cols), dtype=np.int8)
    x_scales = rng.uniform(0.01, 0.1, size=tokens).astype(np.float32)
    packed = q8.pack(gpu, codes, scales)
    want = q8.product(codes, scales, x, x_scales)
    for how in ({}, dict(x_pad=1, y_pad=3, y_offset=1)):
        got = q8.matvec(gpu, packed, x, x_scales, rows, **how)
        assert np.array_equal(got, want), how
