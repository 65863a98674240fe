"""The batched serving operators on the GPU where values differ by many powers of two
or are not finite: what a token does not see, unlikely positions, the largest keys, and
rows whose elements span the range of FP32."""
import numpy as np
import pytest

import lunelette_amd as lh

import serving_oracle as so
from test_gpu_serving import KINDS, close

pytestmark = pytest.mark.gpu

# (head dim, query heads, tokens, positions before them): a tile of a prompt from its
# start and after a prefix, and each of the tiles of few rows.
CALLS = [(128, 3, 48, 0), (64, 4, 40, 75), (64, 2, 150, 20), (128, 1, 16, 75), (64, 1, 7, 30),
         (128, 1, 3, 40), (64, 4, 1, 100)]


def filled(gpu, kind, dim, heads, k, v, page=32):
    """A sequence of one KV head with these keys and values [n][dim], and what the
    cache holds of them."""
    n = k.shape[0]
    seq = so.Sequences(gpu, kind, dim, heads, 1, page, [n], np.random.default_rng(n))
    seq.append(seq.batch([n], [n]), k[:, None], v[:, None])
    return seq, so.cache_values(k[:, None], kind), so.cache_values(v[:, None], kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,heads,count,prefix", CALLS[:-1])
@pytest.mark.parametrize("power", [13, 24, 60, 100])
def test_paged_hidden_values_take_no_part(gpu, kind, dim, heads, count, prefix, power):
    """A value far larger than the others at a position that only the last tokens
    see: the tokens before it keep their precision."""
    if kind == lh.CACHE_F16 and power > 13:
        pytest.skip("past FP16")
    rng = np.random.default_rng(dim + count)
    n = prefix + count
    k, v = (rng.normal(size=(n, dim)).astype(np.float32) for _ in range(2))
    v[n - 2] *= np.float32(2.0 ** power)
    seq, keys, values = filled(gpu, kind, dim, heads, k, v)
    q = rng.normal(size=(count, heads, dim)).astype(np.float32)
    got = seq.attention(seq.batch([count], [n]), q, 0.125)
    for t in range(count):
        want, off = so.attention(q[t], keys, values, prefix + t, 0.125)
        close(got[t], want, off)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,heads,count,prefix", CALLS)
@pytest.mark.parametrize("where", ["first", "middle", "raised"])
def test_paged_unlikely_positions_take_no_part(gpu, kind, dim, heads, count, prefix, where):
    """A visible position of hardly any probability (e^-40) whose value is far larger
    than the others costs them no precision, whether it comes before them, among them,
    or had nearly all of the probability until they came."""
    rng = np.random.default_rng(dim + count + len(where))
    before = 70
    n = before + prefix + count
    k = np.zeros((n, dim), np.float32)
    v = rng.normal(size=(n, dim)).astype(np.float32)
    at = {"first": 3, "middle": 45, "raised": 10}[where]
    # Scores 0 and -40; "raised": 0 up to position 39 and 40 from there on.
    if where == "raised":
        k[40:, 0] = 320
    else:
        k[at, 0] = -320
    v[at] *= np.float32(2.0 ** (13 if kind == lh.CACHE_F16 else 30))
    seq, keys, values = filled(gpu, kind, dim, heads, k, v)
    q = np.zeros((count, heads, dim), np.float32)
    q[..., 0] = 1
    got = seq.attention(seq.batch([count], [n]), q, 0.125)
    for t in range(count):
        last = before + prefix + t
        want, _ = so.attention(q[t], keys, values, last, 0.125)
        # Equal scores of all positions that count: the exponential's two steps, the
        # sums, and planes to 2^-31 of the largest product at each position.
        p = np.exp((keys[:last + 1, 0, 0].astype(np.float64) -
                    keys[:last + 1, 0, 0].max()) * 0.125)
        p /= p.sum()
        size = p @ (3 * np.abs(values[:last + 1, 0]).max(-1).astype(np.float64))
        off = size * (2.0 ** -20 + ((last + 1) / 16 + 64) * so.EPS32)
        close(got[t], want, np.full_like(want, off))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,heads,count,prefix", CALLS)
@pytest.mark.parametrize("at", [0, 10, 45])
@pytest.mark.parametrize("inf", [np.inf, -np.inf, 7e4])
def test_paged_infinite_keys(gpu, kind, dim, heads, count, prefix, at, inf):
    """Tokens that see a key with an Inf (or what FP16 rounds to it) give NaN,
    whatever the sign and size of their queries there; the others do not notice."""
    rng = np.random.default_rng(dim + count + at)
    before = 70 if prefix or count == 1 else 0
    n = before + prefix + count
    k, v = (rng.normal(size=(n, dim)).astype(np.float32) for _ in range(2))
    k[at, 5] = inf
    seq, keys, values = filled(gpu, kind, dim, heads, k, v)
    q = rng.normal(size=(count, heads, dim)).astype(np.float32)
    q[..., 5] = np.ldexp(q[..., 5], -rng.integers(0, 45, size=(count, heads)))
    q[-1, 0, 5] = 0
    got = seq.attention(seq.batch([count], [n]), q, 0.125)
    if np.isfinite(keys).all():
        return   # 4 bits hold 7e4
    for t in range(count):
        last = before + prefix + t
        if last >= at:
            assert np.isnan(got[t]).all(), t
            continue
        want, off = so.attention(q[t], keys, values, last, 0.125)
        close(got[t], want, off)


@pytest.mark.parametrize("dim,heads,count,prefix", CALLS)
def test_paged_largest_halves(gpu, dim, heads, count, prefix):
    """FP16's largest keys and values are finite."""
    rng = np.random.default_rng(dim + count)
    n = 70 + prefix + count
    k, v = (rng.choice(np.float32([-65504, 65504, 1]), size=(n, dim)) for _ in range(2))
    seq, keys, values = filled(gpu, lh.CACHE_F16, dim, heads, k, v)
    q = (rng.normal(size=(count, heads, dim)) * 1e-5).astype(np.float32)
    got = seq.attention(seq.batch([count], [n]), q, 0.125)
    for t in range(count):
        want, off = so.attention(q[t], keys, values, 70 + prefix + t, 0.125)
        close(got[t], want, off)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,heads,count,prefix", CALLS)
@pytest.mark.parametrize("at", [0, 10, 45])
@pytest.mark.parametrize("inf", [np.inf, -np.inf])
def test_paged_infinite_values(gpu, kind, dim, heads, count, prefix, at, inf):
    """Tokens that see a value with an Inf give NaN, of FP16 pages in that element
    alone."""
    rng = np.random.default_rng(dim + count + at)
    before = 70 if prefix or count == 1 else 0
    n = before + prefix + count
    k, v = (rng.normal(size=(n, dim)).astype(np.float32) for _ in range(2))
    v[at, 5] = inf
    seq, keys, values = filled(gpu, kind, dim, heads, k, v)
    q = rng.normal(size=(count, heads, dim)).astype(np.float32)
    got = seq.attention(seq.batch([count], [n]), q, 0.125)
    finite = np.where(np.isfinite(values), values, 0)
    for t in range(count):
        last = before + prefix + t
        want, off = so.attention(q[t], keys, finite, last, 0.125)
        if last >= at:
            want[:, 5 if kind == lh.CACHE_F16 else slice(None)] = np.nan
        close(got[t], want, off)


@pytest.mark.parametrize("dim,heads,count,prefix", CALLS)
@pytest.mark.parametrize("power", [-110, -60, 60, 104, 110, 120])
def test_paged_keys_of_every_size(gpu, dim, heads, count, prefix, power):
    """4-bit keys up to the end of FP32 with queries that bring the scores back to
    a common size."""
    rng = np.random.default_rng(dim + count)
    n = 70 + prefix + count
    k, v = (rng.normal(size=(n, dim)).astype(np.float32) for _ in range(2))
    k = np.ldexp(k, power)
    seq, keys, values = filled(gpu, lh.CACHE_Q4, dim, heads, k, v)
    q = np.ldexp(rng.normal(size=(count, heads, dim)).astype(np.float32), -power)
    got = seq.attention(seq.batch([count], [n]), q, 0.125)
    for t in range(count):
        want, off = so.attention(q[t], keys, values, 70 + prefix + t, 0.125)
        close(got[t], want, off)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,heads,count,prefix", CALLS)
@pytest.mark.parametrize("size,scale", [(1e-38, 1e-20), (1e-38, 1e38), (1e38, 1e-38),
                                        (1e-44, 1.0)])
def test_paged_ends_of_the_scale(gpu, kind, dim, heads, count, prefix, size, scale):
    """Queries and scales at the ends of FP32 whose scores vanish or are common ones."""
    rng = np.random.default_rng(dim + count)
    n = 70 + prefix + count
    k, v = (rng.normal(size=(n, dim)).astype(np.float32) for _ in range(2))
    seq, keys, values = filled(gpu, kind, dim, heads, k, v)
    q = (rng.uniform(-1, 1, size=(count, heads, dim)) * size).astype(np.float32)
    scale = float(np.float32(scale))
    got = seq.attention(seq.batch([count], [n]), q, scale)
    for t in range(count):
        want, off = so.attention(q[t], keys, values, 70 + prefix + t, scale)
        close(got[t], want, off)


@pytest.mark.parametrize("tokens", [1, 8, 16, 40, 64, 100])
@pytest.mark.parametrize("group", [32, 128])
def test_q4_matvec_large_beside_zero_weights(gpu, group, tokens):
    """Weights of 0 (code 8) with large scales under large x: nothing of them in y,
    which holds what the other 128-column blocks give."""
    rows, cols = 48, 512
    rng = np.random.default_rng(tokens)
    codes, scales = so.q4_random(rng, rows, cols, group)
    codes[:, 128:256] = 8
    scales[:, 128 // group:256 // group] = so.bf16(np.float32(1e16))
    x = rng.normal(size=(tokens, cols)).astype(np.float32)
    x[:, 128:256] *= np.float32(1e30)
    w = so.q4_weights(codes, scales, group)
    got = so.q4_run(gpu, so.q4_on_device(gpu, codes, scales, group), x, rows, cols, group)
    close(got, x.astype(np.float64) @ w.T, so.q4_bound(w, x))


@pytest.mark.parametrize("rows,cols,group,tokens", [
    (200, 8320, 64, 129), (90, 16640, 128, 140), (61, 20608, 32, 150), (2051, 1088, 64, 200),
    (700, 2176, 128, 131), (8300, 640, 128, 70), (8300, 576, 64, 128), (33, 65536, 128, 129)])
def test_q4_matvec_many_tokens(gpu, rows, cols, group, tokens):
    """Products whose planes a launch of their own makes: every group size, ragged
    token tiles, column splits, rows of x past what a thread of that launch holds."""
    rng = np.random.default_rng(rows + tokens)
    codes, scales = so.q4_random(rng, rows, cols, group)
    x = (rng.normal(size=(tokens, cols)) * np.exp(rng.normal(size=cols))).astype(np.float32)
    w = so.q4_weights(codes, scales, group)
    packed = so.q4_on_device(gpu, codes, scales, group)
    got = so.q4_run(gpu, packed, x, rows, cols, group, x_pad=3, y_pad=1)
    close(got, x.astype(np.float64) @ w.T, so.q4_bound(w, x))


@pytest.mark.parametrize("rows,tokens", [(48, 100), (48, 130), (8300, 70)])
def test_q4_matvec_special_rows_of_many(gpu, rows, tokens):
    """Rows of every magnitude, a zero row, and rows with an Inf or NaN, which stay
    their own row's, past 64 tokens."""
    cols, group = 384, 64
    rng = np.random.default_rng(tokens)
    codes, scales = so.q4_random(rng, rows, cols, group)
    x = rng.normal(size=(tokens, cols)).astype(np.float32)
    for first in (0, 50, tokens - 6):
        x[first] = 0
        x[first + 1] *= np.float32(1e36)
        x[first + 2] *= np.float32(1e-36)
        x[first + 3, 100] = -np.inf
        x[first + 4, 383] = np.nan
        x[first + 5, 11] = 1e5
    packed = so.q4_on_device(gpu, codes, scales, group)
    w = so.q4_weights(codes, scales, group)
    got = so.q4_run(gpu, packed, x, rows, cols, group)
    odd = ~np.isfinite(x).all(1)
    x = np.where(np.isfinite(x), x, 0)
    want = x.astype(np.float64) @ w.T
    want[odd] = np.nan
    # Elements below 2^-16 of their row's largest carry 2^-38 of that instead.
    bound = so.q4_bound(w, x) + np.abs(w).sum(1) * 2.0 ** -38 * np.abs(x).max(
        1, keepdims=True).astype(np.float64)
    close(got, want, bound)


@pytest.mark.parametrize("tokens", [1, 9, 16, 40, 100, 130])
def test_q4_matvec_planes_of_single_columns(gpu, tokens):
    """Rows with one weight each, x of every size down to 2^-40 of the token's
    largest: each element by itself to 2^-22 of itself or 2^-38 of the largest."""
    rows, cols, group = 256, 640, 32
    rng = np.random.default_rng(tokens)
    codes = np.full((rows, cols), 8, np.uint8)
    at = rng.integers(0, cols, size=rows)
    codes[np.arange(rows), at] = rng.choice(np.uint8([0, 1, 7, 9, 15]), size=rows)
    scales = so.bf16(rng.uniform(0.5, 2.0, size=(rows, cols // group)))
    x = np.ldexp(rng.normal(size=(tokens, cols)), rng.integers(-40, 1, size=(tokens, cols)))
    x = x.astype(np.float32)
    x[:, 3] = 1
    w = so.q4_weights(codes, scales, group)
    got = so.q4_run(gpu, so.q4_on_device(gpu, codes, scales, group), x, rows, cols, group)
    largest = np.abs(x).max(1, keepdims=True).astype(np.float64)
    one = np.abs(x).astype(np.float64)[:, at]
    # Two products, the group's scale and the power of two back: five roundings.
    off = np.maximum(one * 2.0 ** -22, largest * 2.0 ** -38) + 5 * so.EPS32 * one
    close(got, x.astype(np.float64) @ w.T, off * np.abs(w).max(1))


@pytest.mark.parametrize("group", [64, 128])
def test_q4_quantize_groups(gpu, group):
    """Rounded weights with the larger groups and columns that end inside a block."""
    rows, cols = 35, 3 * group
    rng = np.random.default_rng(group)
    w = rng.normal(size=(rows, cols)).astype(np.float32)
    w[3, :group] = 0
    w[5, group + 3] = -np.inf
    w[6] *= np.float32(1e30)
    w[7, :group] = np.float32(1e-44)
    blocks = w.reshape(rows, -1, group)
    with np.errstate(invalid="ignore", divide="ignore"):
        scales = so.bf16(np.abs(blocks).max(-1) / np.float32(7))
        scales[~np.isfinite(blocks).all(-1)] = np.nan
        code = np.rint(np.clip(blocks / scales[..., None], -7, 7))
    code = np.where(scales[..., None] > 0, code, 0.0)
    want = (code * scales[..., None]).reshape(rows, cols)
    packed = lh.DeviceBuffer(gpu.lh_q4_bytes(rows, cols, group))
    d_w = lh.DeviceBuffer.from_array(w)
    lh.check(gpu.lh_q4_quantize(d_w.ptr, rows, cols, group, packed.ptr, None))
    got = so.q4_run(gpu, packed, np.eye(cols, dtype=np.float32), rows, cols, group).T
    odd = np.isnan(want).any(1)
    assert list(np.nonzero(odd)[0]) == [5]
    assert np.array_equal(got[~odd], want[~odd].astype(np.float32))
    assert np.isnan(got[5]).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,heads,count", [(64, 2, 1), (128, 1, 3)])
def test_paged_most_splits(gpu, kind, dim, heads, count):
    """As many splits as one token's attention is ever cut into."""
    n = 133003
    rng = np.random.default_rng(dim)
    k, v = (rng.normal(size=(n, dim)).astype(np.float32) for _ in range(2))
    seq, keys, values = filled(gpu, kind, dim, heads, k, v, page=256)
    q = rng.normal(size=(count, heads, dim)).astype(np.float32)
    got = seq.attention(seq.batch([count], [n]), q, 0.125)
    for t in range(count):
        want, off = so.attention(q[t], keys, values, n - count + t, 0.125)
        close(got[t], want, off)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,heads,count,prefix", CALLS)
@pytest.mark.parametrize("scale", [1.0, 1e15, 1e38])
def test_paged_zero_queries(gpu, kind, dim, heads, count, prefix, scale):
    """A query of zeros has scores of 0 at any scale: the mean of what it sees."""
    rng = np.random.default_rng(dim + count)
    n = 70 + prefix + count
    k = (rng.normal(size=(n, dim)) * 1e4).astype(np.float32)
    v = rng.normal(size=(n, dim)).astype(np.float32)
    seq, keys, values = filled(gpu, kind, dim, heads, k, v)
    q = np.zeros((count, heads, dim), np.float32)
    q[::2] = -0.0
    scale = float(np.float32(scale))
    got = seq.attention(seq.batch([count], [n]), q, scale)
    for t in range(count):
        want, off = so.attention(q[t], keys, values, 70 + prefix + t, scale)
        close(got[t], want, off)
