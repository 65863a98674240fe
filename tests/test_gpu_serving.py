"""The batched serving operators on the GPU (include/lunelette_serving.h) against
their definitions in 64 bits: 4-bit products, log probabilities, the paged cache
with its append and attention, and one decode step made of all of them."""
import ctypes

import numpy as np
import pytest

import lunelette_amd as lh

import serving_oracle as so

pytestmark = pytest.mark.gpu
KINDS = [pytest.param(lh.CACHE_F16, id="f16"), pytest.param(lh.CACHE_Q4, id="q4")]


def close(got, want, off):
    got = got.astype(np.float64)
    both = np.isnan(want) & np.isnan(got)
    same = got == want
    with np.errstate(invalid="ignore"):
        worst = np.where(both | same, 0.0, np.abs(got - want) - off)
    assert np.all(worst <= 0), (float(np.nanmax(worst)), int((~(worst <= 0)).sum()))


# ---- 4-bit weights ----

@pytest.mark.parametrize("rows,cols,group,tokens", [
    (1, 32, 32, 1), (16, 128, 128, 1), (17, 96, 32, 3), (100, 4096, 128, 1), (33, 256, 64, 17),
    (3072, 4096, 64, 1), (40, 160, 32, 16), (64, 1024, 128, 33), (50, 2080, 32, 65),
    (70, 65536, 128, 2), (2051, 544, 32, 130), (1030, 9216, 64, 9), (8, 192, 64, 5),
    (5000, 64, 64, 2), (31, 12288, 32, 40)])
def test_q4_matvec(gpu, rows, cols, group, tokens):
    rng = np.random.default_rng(rows * 7 + cols)
    codes, scales = so.q4_random(rng, rows, cols, group)
    x = (rng.normal(size=(tokens, cols)) * np.exp(rng.normal(size=cols))).astype(np.float32)
    packed = so.q4_on_device(gpu, codes, scales, group)
    w = so.q4_weights(codes, scales, group)
    got = so.q4_run(gpu, packed, x, rows, cols, group)
    close(got, x.astype(np.float64) @ w.T, so.q4_bound(w, x))
    # Strides and a start off the 16-byte boundary change nothing.
    again = so.q4_run(gpu, packed, x, rows, cols, group, x_pad=3, y_pad=5, offset=1)
    assert np.array_equal(again.view(np.uint32), got.view(np.uint32))


@pytest.mark.parametrize("rows,cols,group,tokens", [
    (33000, 128, 32, 1), (33000, 128, 64, 3), (33003, 384, 128, 7), (9000, 384, 64, 16),
    (4100, 640, 128, 10), (2000, 2048, 32, 24), (2000, 2080, 32, 48), (777, 5120, 128, 64),
    (300, 8192, 32, 64), (16, 4160, 64, 31), (600, 4096, 128, 8), (600, 4096, 128, 9)])
def test_q4_matvec_turns_and_splits(gpu, rows, cols, group, tokens):
    """Workgroups with several turns of row tiles, tokens to either side of each
    way to run a product, column splits of odd lengths."""
    rng = np.random.default_rng(rows + tokens)
    codes, scales = so.q4_random(rng, rows, cols, group)
    x = rng.normal(size=(tokens, cols)).astype(np.float32)
    w = so.q4_weights(codes, scales, group)
    packed = so.q4_on_device(gpu, codes, scales, group)
    got = so.q4_run(gpu, packed, x, rows, cols, group, x_pad=1, y_pad=2)
    close(got, x.astype(np.float64) @ w.T, so.q4_bound(w, x))


@pytest.mark.parametrize("rows,tokens", [(1000, 65), (1000, 96), (1000, 97), (1000, 128),
                                         (1000, 129), (8192, 80), (8193, 80), (8, 128)])
def test_q4_matvec_two_token_groups(gpu, rows, tokens):
    """Past 64 tokens, to either side of where a launch of its own makes the planes."""
    cols, group = 1056, 32
    rng = np.random.default_rng(rows + tokens)
    codes, scales = so.q4_random(rng, rows, cols, group)
    x = rng.normal(size=(tokens, cols)).astype(np.float32)
    w = so.q4_weights(codes, scales, group)
    packed = so.q4_on_device(gpu, codes, scales, group)
    got = so.q4_run(gpu, packed, x, rows, cols, group, x_pad=2, y_pad=1)
    close(got, x.astype(np.float64) @ w.T, so.q4_bound(w, x))


@pytest.mark.parametrize("tokens", [2, 30, 70])
def test_q4_matvec_ties(gpu, tokens):
    """x halfway between two FP16 values: the second plane has the rest."""
    rows, cols, group = 32, 640, 32
    rng = np.random.default_rng(tokens)
    codes, scales = so.q4_random(rng, rows, cols, group)
    x = (1 + (2 * rng.integers(0, 1024, size=(tokens, cols)) + 1) * 2.0 ** -11).astype(np.float32)
    x *= rng.choice([-1, 1], size=x.shape)
    w = so.q4_weights(codes, scales, group)
    got = so.q4_run(gpu, so.q4_on_device(gpu, codes, scales, group), x, rows, cols, group)
    close(got, x.astype(np.float64) @ w.T, so.q4_bound(w, x))


@pytest.mark.parametrize("tokens", [6, 40])
def test_q4_matvec_ranges_and_special_rows(gpu, tokens):
    """Rows of every magnitude, a zero row, and rows with an Inf or NaN, which
    stay their own row's."""
    rows, cols, group = 48, 384, 32
    rng = np.random.default_rng(tokens)
    codes, scales = so.q4_random(rng, rows, cols, group)
    x = rng.normal(size=(tokens, cols)).astype(np.float32)
    x[0] = 0
    x[1] *= np.float32(1e36)
    x[2] *= np.float32(1e-36)
    x[3, 100] = np.inf
    x[4, 7] = np.nan
    x[5, 11] = 1e5    # one column far above the rest
    packed = so.q4_on_device(gpu, codes, scales, group)
    w = so.q4_weights(codes, scales, group)
    got = so.q4_run(gpu, packed, x, rows, cols, group)
    x = np.where(np.isfinite(x), x, 0)
    want = x.astype(np.float64) @ w.T
    want[3:5] = np.nan
    # Elements below 2^-16 of their row's largest carry 2^-38 of that instead.
    bound = so.q4_bound(w, x) + np.abs(w).sum(1) * 2.0 ** -38 * np.abs(x).max(
        1, keepdims=True).astype(np.float64)
    close(got, want, bound)


def test_q4_quantize(gpu):
    """The packed form of rounded FP32 weights equals that of the codes and
    scales of the definition, read through products with unit vectors."""
    rows, cols, group = 35, 160, 32
    rng = np.random.default_rng(2)
    w = rng.normal(size=(rows, cols)).astype(np.float32)
    w[3, :32] = 0
    w[4, 32:64] = np.float32(1e-45)
    w[5, 70] = np.nan
    w[6] *= np.float32(1e30)
    blocks = w.reshape(rows, -1, group)
    with np.errstate(invalid="ignore"):
        scales = so.bf16(np.abs(blocks).max(-1) / np.float32(7))
        scales[~np.isfinite(blocks).all(-1)] = np.nan
        code = np.rint(np.clip(blocks / scales[..., None], -7, 7))
    code = np.where(scales[..., None] > 0, code, 0.0)
    want = (code * scales[..., None]).reshape(rows, cols)
    packed = lh.DeviceBuffer(gpu.lh_q4_bytes(rows, cols, group))
    d_w = lh.DeviceBuffer.from_array(w)
    lh.check(gpu.lh_q4_quantize(d_w.ptr, rows, cols, group, packed.ptr, None))
    got = so.q4_run(gpu, packed, np.eye(cols, dtype=np.float32), rows, cols, group)
    nan = np.isnan(want).any(1)
    assert list(np.nonzero(nan)[0]) == [5]
    assert np.array_equal(got.T[~nan], want[~nan].astype(np.float32))
    assert np.isnan(got.T[5]).all()


# ---- log probabilities ----

def run_logprobs(gpu, x, tokens, top, pad=0, offset=0, entropy=True, stream=None):
    rows, vocab = x.shape
    stride = vocab + pad
    buf = np.full(offset + rows * stride, np.nan, np.float32)
    buf[offset:].reshape(rows, stride)[:, :vocab] = x
    d_x = lh.DeviceBuffer.from_array(buf)
    d_t = None if tokens is None else lh.DeviceBuffer.from_array(np.asarray(tokens, np.int64))
    outs = [lh.DeviceBuffer.from_array(np.full(n + 2, 7.25, np.float32))
            for n in (rows, rows, rows * top)]
    ids = lh.DeviceBuffer.from_array(np.full(rows * top + 2, 77, np.int64))
    need = gpu.lh_logprobs_scratch(rows, vocab, top)
    scratch = lh.DeviceBuffer(max(16, need))
    lh.check(gpu.lh_memset_device(scratch.ptr, 0xff, scratch.nbytes))
    lh.check(gpu.lh_logprobs(d_x.ptr + 4 * offset, stride, rows, vocab, d_t and d_t.ptr,
                             outs[0].ptr if d_t else None, outs[1].ptr if entropy else None, top,
                             ids.ptr if top else None, outs[2].ptr if top else None, scratch.ptr,
                             need, stream))
    lh.check(gpu.lh_device_synchronize())
    got = [o.download(np.float32) for o in outs]
    got_ids = ids.download(np.int64)
    for g, n in zip(got, (rows if d_t else 0, rows if entropy else 0, rows * top)):
        assert np.all(g[n:] == 7.25)
    assert np.all(got_ids[rows * top:] == 77)
    return (got[0][:rows], got[1][:rows], got_ids[:rows * top].reshape(rows, top),
            got[2][:rows * top].reshape(rows, top))


def check_logprobs(gpu, x, tokens, top, **how):
    lp, entropy, ids, tops = run_logprobs(gpu, x, tokens, top, **how)
    for r in range(x.shape[0]):
        want = so.logprobs(x[r], -1 if tokens is None else tokens[r], top)
        off = want[4]
        assert np.array_equal(ids[r], want[2]), r
        close(tops[r], want[3], off[2])
        if tokens is not None:
            close(lp[r:r + 1], np.array([want[0]]), off[0])
        if how.get("entropy", True):
            close(entropy[r:r + 1], np.array([want[1]]), off[1])
    return lp, entropy, ids, tops


@pytest.mark.parametrize("rows,vocab,top", [
    (1, 1, 1), (1, 131072, 20), (2, 2, 64), (5, 77, 64), (3, 1000, 5), (7, 4097, 1),
    (40, 5003, 64), (1, 151936, 64), (300, 2048, 3), (9, 8192, 0), (2, 300001, 33)])
def test_logprobs(gpu, rows, vocab, top):
    rng = np.random.default_rng(rows + vocab)
    x = (2.5 * rng.normal(size=(rows, vocab))).astype(np.float32)
    x[::3, vocab // 2] += 18            # almost certain rows
    tokens = rng.integers(0, vocab, size=rows)
    tokens[::2] = vocab // 2
    got = check_logprobs(gpu, x, tokens, top)
    again = check_logprobs(gpu, x, tokens, top, pad=3, offset=1)
    for a, b in zip(got, again):
        assert np.array_equal(a.view(np.uint8), b.view(np.uint8))


def orders(rng, vocab):
    """Rows whose order is hard on a selection."""
    up = np.linspace(-30, 30, vocab).astype(np.float32)
    ties = rng.integers(0, 5, size=vocab).astype(np.float32)
    zeros = np.where(rng.random(vocab) < 0.5, np.float32(0.0), np.float32(-0.0))
    masked = np.full(vocab, -np.inf, np.float32)
    masked[rng.integers(0, vocab, size=9)] = rng.normal(size=9).astype(np.float32)
    lowest = np.full(vocab, np.finfo(np.float32).min, np.float32)
    lowest[[1, vocab - 1]] = 3.5, -2
    clustered = rng.normal(size=vocab).astype(np.float32)
    clustered[vocab // 3:vocab // 3 + 100] += 10
    large = (rng.normal(size=vocab) * 1e37).astype(np.float32)
    return np.stack([up, up[::-1], np.full(vocab, 1.5, np.float32), ties, zeros, masked, lowest,
                     clustered, large])


@pytest.mark.parametrize("vocab,top", [(3000, 64), (70001, 20), (131072, 64), (515, 7)])
def test_logprobs_orders_ties_and_masks(gpu, vocab, top):
    x = orders(np.random.default_rng(vocab), vocab)
    check_logprobs(gpu, x, [0, vocab - 1, -1, 5, 7, 3, vocab, -2, 2 ** 40], top)


def test_logprobs_without_a_distribution(gpu):
    """Nothing but masks, NaN and +Inf: in their own rows only."""
    x = np.random.default_rng(3).normal(size=(6, 9000)).astype(np.float32)
    x[1] = -np.inf
    x[2, 8999] = np.nan
    x[3, 0] = np.inf
    x[4] = -np.inf
    x[4, 4500] = 2.0
    x[5] = np.nan
    lp, entropy, ids, tops = check_logprobs(gpu, x, [1, 2, 3, 4, 4500, -1], 4)
    assert lp[4] == 0 and entropy[4] == 0 and list(ids[4]) == [4500, -1, -1, -1]
    assert np.isneginf(lp[1]) and entropy[1] == 0 and np.isneginf(tops[1]).all()


def test_logprobs_outputs_left_out(gpu):
    x = np.random.default_rng(4).normal(size=(3, 5000)).astype(np.float32)
    check_logprobs(gpu, x, None, 8)
    check_logprobs(gpu, x, [1, 2, 3], 0, entropy=False)
    check_logprobs(gpu, x, None, 0)


# ---- paged cache ----

SHAPES = [(128, 32, 8, 64), (64, 14, 2, 32), (128, 24, 4, 96), (64, 3, 3, 256), (128, 5, 1, 128),
          (64, 64, 1, 32), (128, 40, 2, 32)]


def tables(rng, positions, dim):
    half = dim // 2
    angle = np.arange(positions)[:, None] * 1e4 ** (-np.arange(half) / half)
    angle = np.concatenate([angle, angle], axis=1)
    return (np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32),
            rng.uniform(0.5, 2, size=positions).astype(np.float32))


class Run:
    """Steps of ragged sequences with the host's copy of keys and values."""

    def __init__(self, gpu, kind, dim, heads, kv_heads, page, lengths, seed):
        rng = self.rng = np.random.default_rng(seed)
        self.seq = so.Sequences(gpu, kind, dim, heads, kv_heads, page, lengths, rng)
        self.cos, self.sin, self.factor = tables(rng, max(lengths + [1]), dim)
        self.keys = [np.zeros((0, kv_heads, dim), np.float32) for _ in lengths]
        self.values = [np.zeros((0, kv_heads, dim), np.float32) for _ in lengths]

    def step(self, counts):
        s, rng = self.seq, self.rng
        before = [k.shape[0] for k in self.keys]
        lengths = [b + c for b, c in zip(before, counts)]
        batch = s.batch(counts, lengths)
        n = sum(counts)
        spread = np.exp(rng.normal(size=s.dim))
        q = rng.normal(size=(n, s.heads, s.dim)).astype(np.float32)
        k = (rng.normal(size=(n, s.kv_heads, s.dim)) * spread).astype(np.float32)
        v = rng.normal(size=(n, s.kv_heads, s.dim)).astype(np.float32)
        pos = np.concatenate([np.arange(b, l) for b, l in zip(before, lengths)])
        out = s.append(batch, k, v, q, self.cos, self.sin, self.factor)
        turned = so.rotate(q, self.cos[pos], self.sin[pos]) * self.factor[pos][:, None, None]
        close(out, turned, np.abs(turned) * so.EPS32 * (1 + 1e-6) + 1e-13)
        held_k = so.cache_values(so.rotate(k, self.cos[pos], self.sin[pos]), s.kind)
        held_v = so.cache_values(v, s.kind)
        at = 0
        for i, c in enumerate(counts):
            self.keys[i] = np.concatenate([self.keys[i], held_k[at:at + c]])
            self.values[i] = np.concatenate([self.values[i], held_v[at:at + c]])
            at += c
        return batch, out, lengths

    def check_cache(self):
        """The whole history, read back."""
        lengths = [k.shape[0] for k in self.keys]
        batch = self.seq.batch(lengths, lengths)
        keys, values = self.seq.read(batch)
        assert np.array_equal(keys, np.concatenate(self.keys))
        assert np.array_equal(values, np.concatenate(self.values))

    def check_attention(self, batch, q, counts, **how):
        s = self.seq
        scale = float(np.float32(1 / np.sqrt(s.dim)))
        got = s.attention(batch, q, scale, **how)
        at = 0
        for i, c in enumerate(counts):
            length = self.keys[i].shape[0]
            for t in range(c):
                want, off = so.attention(q[at], self.keys[i], self.values[i], length - c + t,
                                         scale)
                close(got[at], want, off)
                at += 1
        return got


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,heads,kv_heads,page", SHAPES)
def test_paged_steps(gpu, kind, dim, heads, kv_heads, page):
    """A ragged prompt, single tokens (one sequence rests), a short append: the
    cache's rows and the attention after each."""
    run = Run(gpu, kind, dim, heads, kv_heads, page, [230, 64, 33, 97, 3], dim + heads)
    for counts in ([200, 31, 1, 64, 0], [1, 1, 1, 1, 1], [1, 0, 1, 1, 1], [5, 32, 30, 7, 1],
                   [1, 0, 0, 1, 0]):
        batch, q, _ = run.step(counts)
        run.check_cache()
        run.check_attention(batch, q, counts)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("length", [1, 2, 31, 32, 33, 127, 128, 129, 1000, 4097])
def test_paged_single_token_lengths(gpu, kind, length):
    run = Run(gpu, kind, 128, 32, 8, 64, [length], length)
    if length > 1:
        run.step([length - 1])
    batch, q, _ = run.step([1])
    got = run.check_attention(batch, q, [1])
    again = run.check_attention(batch, q, [1], q_pad=5, out_pad=3)
    assert np.array_equal(got.view(np.uint32), again.view(np.uint32))


@pytest.mark.parametrize("kind", KINDS)
def test_paged_many_sequences(gpu, kind):
    """More sequences than the chip has units, of very different lengths."""
    lengths = [int(l) for l in np.random.default_rng(9).integers(1, 200, size=300)] + [2500]
    run = Run(gpu, kind, 64, 4, 2, 32, lengths, 5)
    run.step([l - 1 for l in lengths])
    counts = [1] * len(lengths)
    batch, q, _ = run.step(counts)
    run.check_cache()
    run.check_attention(batch, q, counts)


@pytest.mark.parametrize("kind", KINDS)
def test_paged_prompt_chunk(gpu, kind):
    """A chunk of a prompt after a prefix, checked at rows over the chunk."""
    run = Run(gpu, kind, 128, 32, 8, 64, [1500], 21)
    run.step([1191])
    batch, q, _ = run.step([309])
    s, scale = run.seq, float(np.float32(1 / np.sqrt(128)))
    got = s.attention(batch, q, scale)
    for t in (0, 1, 15, 16, 17, 150, 151, 307, 308):
        want, off = so.attention(q[t], run.keys[0], run.values[0], 1191 + t, scale)
        close(got[t], want, off)


@pytest.mark.parametrize("kind", KINDS)
def test_paged_larger_than_the_bounds(gpu, kind):
    """max_query and max_length size the launch only."""
    run = Run(gpu, kind, 128, 4, 2, 32, [150, 80], 4)
    run.step([60, 70])
    batch, q, _ = run.step([90, 10])
    batch.max_query = batch.max_length = 1
    run.check_attention(batch, q, [90, 10])
    keys, values = run.seq.read(batch)
    assert np.array_equal(keys[:90], run.keys[0][60:])
    assert np.array_equal(values[90:], run.values[1][70:])


@pytest.mark.parametrize("kind", KINDS)
def test_paged_rows_without_a_place(gpu, kind):
    """Sequences at negative positions, with bad page ids and past their table,
    beside a good one; rows behind the last sequence stay."""
    dim, heads, kv = 64, 6, 2
    rng = np.random.default_rng(8)
    seq = so.Sequences(gpu, kind, dim, heads, kv, 32, [96, 96, 96, 96], rng)
    seq.table[1, 1] = seq.pages          # the second page of sequence 1
    seq.table[2, 0] = -5
    counts, lengths = [40, 40, 40, 40], [40, 40, 30, 110]
    before = seq.memory.download(np.uint8)
    batch = seq.batch(counts, lengths, tokens=165)
    n = batch.tokens
    k, v = (rng.normal(size=(n, kv, dim)).astype(np.float32) for _ in range(2))
    q = rng.normal(size=(n, heads, dim)).astype(np.float32)
    out = seq.append(batch, k, v, q)
    assert np.array_equal(out[:80], q[:80]) and np.array_equal(out[120:160], q[120:160])
    assert np.isnan(out[80:90]).all()    # the ten negative positions
    assert np.array_equal(out[90:120], q[90:120])
    assert np.all(out[160:] == 7.25)
    keys, values = seq.read(batch)
    for got, rows in ((keys, k), (values, v)):
        held = so.cache_values(rows, kind)
        assert np.array_equal(got[:72], held[:72])       # 40 rows, then 32 on a page
        assert np.isnan(got[72:120]).all()
        assert np.array_equal(got[120:146], held[120:146])   # 70..95 on the table
        assert np.isnan(got[146:160]).all()
        assert np.all(got[160:] == 7.25)
    # Only the pages of the batch changed.
    after = seq.memory.download(np.uint8)
    used = {int(t) for t in (seq.table[0, :2].tolist() + [seq.table[1, 0]] +
                             seq.table[3, 2:3].tolist())}
    size = before.size // seq.pages
    for p in range(seq.pages):
        if p not in used:
            assert np.array_equal(before[p * size:(p + 1) * size], after[p * size:(p + 1) * size])
    got = seq.attention(batch, q, 0.125)
    held_k, held_v = so.cache_values(k, kind), so.cache_values(v, kind)
    for i, first in ((0, 0), (1, 40)):
        for t in (0, 1, 31):
            want, off = so.attention(q[first + t], held_k[first:first + 40],
                                     held_v[first:first + 40], t, 0.125)
            close(got[first + t], want, off)
    assert np.isnan(got[72:80]).all()                    # sees the missing page
    assert np.all(got[80:90] == 0)                       # sees nothing
    assert np.isnan(got[90:120]).all()
    assert np.isnan(got[146:160]).all()                  # past the table
    assert np.all(got[160:] == 7.25)


@pytest.mark.parametrize("kind", KINDS)
def test_paged_positions_past_the_rotation(gpu, kind):
    rng = np.random.default_rng(12)
    seq = so.Sequences(gpu, kind, 64, 2, 1, 32, [64], rng, fill=0)
    batch = seq.batch([40], [40])
    cos, sin, factor = tables(rng, 33, 64)
    k, v = (rng.normal(size=(40, 1, 64)).astype(np.float32) for _ in range(2))
    q = rng.normal(size=(40, 2, 64)).astype(np.float32)
    out = seq.append(batch, k, v, q, cos, sin, factor)
    assert np.isfinite(out[:33]).all() and np.isnan(out[33:]).all()
    keys, values = seq.read(batch)
    held = so.cache_values(so.rotate(k[:33], cos, sin), kind)
    assert np.array_equal(keys[:33], held)
    assert np.all(keys[33:] == 0) and np.all(values[33:] == 0)   # not appended


@pytest.mark.parametrize("kind", KINDS)
def test_paged_special_vectors(gpu, kind):
    """Constant and zero vectors, wide ranges, Inf and NaN; positions that a
    token does not see may hold anything."""
    rng = np.random.default_rng(6)
    dim, n = 64, 48
    seq = so.Sequences(gpu, kind, dim, 2, 1, 64, [64], rng)
    k, v = (rng.normal(size=(n, 1, dim)).astype(np.float32) for _ in range(2))
    for a in (k, v):
        a[0] = 0
        a[1] = 3.14159
        a[2] = -1e-3
        a[3, 0, 5] = 1000
        a[4] *= np.float32(1e-6)
        a[5] = np.float32(1e-42)
        a[40, 0, 3] = np.inf
        a[41, 0, 9] = np.nan
        a[42, 0, 1], a[42, 0, 2] = 3e38, -3.4e38
    batch = seq.batch([n], [n])
    seq.append(batch, k, v)
    keys, values = seq.read(batch)
    assert np.array_equal(keys, so.cache_values(k, kind), equal_nan=True)
    assert np.array_equal(values, so.cache_values(v, kind), equal_nan=True)
    q = rng.normal(size=(n, 2, dim)).astype(np.float32)
    got = seq.attention(batch, q, 0.125)
    for t in range(40):
        want, off = so.attention(q[t], keys, values, t, 0.125)
        close(got[t], want, off)
    assert np.isnan(got[41:]).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,heads,count", [
    (128, 1, 3), (64, 1, 4), (128, 1, 5), (64, 2, 4), (128, 3, 3), (64, 1, 16), (128, 1, 17),
    (64, 4, 8), (128, 1, 32), (128, 3, 11), (64, 1, 129), (128, 1, 129)])
def test_paged_row_tiles(gpu, kind, dim, heads, count):
    """To either side of every number of rows in a tile, after a prefix; the last
    position, which only the last token sees, has an Inf among its values."""
    prefix = 75
    rng = np.random.default_rng(dim + heads + count)
    n = prefix + count
    seq = so.Sequences(gpu, kind, dim, heads, 1, 32, [n], rng)
    k, v = (rng.normal(size=(n, 1, dim)).astype(np.float32) for _ in range(2))
    v[n - 1, 0, 5] = np.inf
    seq.append(seq.batch([n], [n]), k, v)
    held_k, held_v = so.cache_values(k, kind), so.cache_values(v, kind)
    q = rng.normal(size=(count, heads, dim)).astype(np.float32)
    got = seq.attention(seq.batch([count], [n]), q, 0.125)
    for t in range(count - 1):
        want, off = so.attention(q[t], held_k[:n - 1], held_v[:n - 1], prefix + t, 0.125)
        close(got[t], want, off)
    if kind == lh.CACHE_Q4:
        assert np.isnan(got[-1]).all()
        return
    held_v[n - 1, 0, 5] = 0
    want, off = so.attention(q[-1], held_k, held_v, n - 1, 0.125)
    want[:, 5] = np.nan
    close(got[-1], want, off)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128])
def test_paged_prompts_from_the_start(gpu, kind, dim):
    """Prompts at position 0, one query head a KV head: the rows of a tile end in
    different blocks."""
    run = Run(gpu, kind, dim, 2, 2, 64, [200, 129, 90], dim)
    batch, q, _ = run.step([200, 129, 90])
    got = run.check_attention(batch, q, [200, 129, 90])
    for _ in range(5):
        again = run.seq.attention(batch, q, float(np.float32(1 / np.sqrt(dim))))
        assert np.array_equal(again.view(np.uint32), got.view(np.uint32))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("count", [3, 40])
@pytest.mark.parametrize("size,scale", [(1e-30, 1e-9), (1e30, 1e-31), (0.0, 1.0), (1e-6, 1e6),
                                        (100.0, 3.0)])
def test_paged_query_sizes(gpu, kind, count, size, scale):
    """Queries and scales whose product alone is of a common size, or vanishes,
    and scores that leave one position."""
    rng = np.random.default_rng(count)
    n, dim = 100, 128
    seq = so.Sequences(gpu, kind, dim, 2, 1, 64, [n], rng)
    k, v = (rng.normal(size=(n, 1, dim)).astype(np.float32) for _ in range(2))
    seq.append(seq.batch([n], [n]), k, v)
    held_k, held_v = so.cache_values(k, kind), so.cache_values(v, kind)
    q = (rng.normal(size=(count, 2, dim)) * size).astype(np.float32)
    scale = float(np.float32(scale))
    got = seq.attention(seq.batch([count], [n]), q, scale)
    for t in range(count):
        want, off = so.attention(q[t], held_k, held_v, n - count + t, scale)
        close(got[t], want, off)


def test_paged_large_offsets(gpu):
    """A cache past 2^32 bytes: the last pages' bytes are their own."""
    rng = np.random.default_rng(31)
    seq = so.Sequences(gpu, lh.CACHE_F16, 128, 8, 8, 1024, [1000], rng, spare=1100)
    assert seq.memory.nbytes > 2 ** 32
    for page in (seq.pages - 1, 3):
        seq.table[0, 0] = page
        batch = seq.batch([1000], [1000])
        k, v = (rng.normal(size=(1000, 8, 128)).astype(np.float32) for _ in range(2))
        seq.append(batch, k, v)
        held = so.cache_values(k, seq.kind), so.cache_values(v, seq.kind)
        if page != 3:
            first = (batch, held, seq.table.copy())
    for batch, held in ((first[0], first[1]), (batch, held)):
        keys, values = seq.read(batch)
        assert np.array_equal(keys, held[0]) and np.array_equal(values, held[1])
    one = seq.batch([1], [1000], table=first[2])
    q = rng.normal(size=(1, 8, 128)).astype(np.float32)
    want, off = so.attention(q[0], first[1][0], first[1][1], 999, 0.1)
    close(seq.attention(one, q, float(np.float32(0.1)))[0], want, off)


# ---- streams, graphs, and all of it together ----

def test_two_streams_at_once(gpu):
    """Calls on two streams with scratch of their own, again and again."""
    rng = np.random.default_rng(14)
    streams = [gpu.lh_stream_create() for _ in range(2)]
    x = [rng.normal(size=(20, 30000)).astype(np.float32) for _ in streams]
    want = [run_logprobs(gpu, a, [3] * 20, 10) for a in x]
    need = gpu.lh_logprobs_scratch(20, 30000, 10)
    bufs = []
    for a in x:
        bufs.append([lh.DeviceBuffer.from_array(a),
                     lh.DeviceBuffer.from_array(np.full(20, 3, np.int64)),
                     lh.DeviceBuffer(80), lh.DeviceBuffer(80), lh.DeviceBuffer(1600),
                     lh.DeviceBuffer(800), lh.DeviceBuffer(max(16, need))])
    for _ in range(20):
        for s, b in zip(streams, bufs):
            lh.check(gpu.lh_logprobs(b[0].ptr, 30000, 20, 30000, b[1].ptr, b[2].ptr, b[3].ptr, 10,
                                     b[4].ptr, b[5].ptr, b[6].ptr, need, s))
    for s in streams:
        lh.check(gpu.lh_stream_synchronize(s))
    for w, b in zip(want, bufs):
        assert np.array_equal(b[2].download(np.float32), w[0])
        assert np.array_equal(b[3].download(np.float32), w[1])
        assert np.array_equal(b[4].download(np.int64).reshape(20, 10), w[2])
        assert np.array_equal(b[5].download(np.float32).reshape(20, 10), w[3])
    for s in streams:
        gpu.lh_stream_destroy(s)


class Decoder:
    """One decode step of a batch, made of the operators: 4-bit q|k|v, append,
    attention, 4-bit o, tied head, log probabilities."""
    HEADS, KV, DIM, HIDDEN, VOCAB, GROUP = 8, 2, 128, 512, 1500, 64

    def __init__(self, gpu, kind, lengths, rng):
        self.gpu, self.n = gpu, len(lengths)
        self.qkv = (self.HEADS + 2 * self.KV) * self.DIM
        self.seq = so.Sequences(gpu, kind, self.DIM, self.HEADS, self.KV, 32,
                                [l + 8 for l in lengths], rng)
        self.cos, self.sin, _ = tables(rng, max(lengths) + 8, self.DIM)
        self.w = [so.q4_random(rng, r, c, self.GROUP) for r, c in
                  ((self.qkv, self.HIDDEN), (self.HIDDEN, self.HEADS * self.DIM))]
        self.packed = [so.q4_on_device(gpu, c, s, self.GROUP) for c, s in self.w]
        self.head = so.bf16(rng.normal(size=(self.VOCAB, self.HIDDEN)).astype(np.float32))
        n = self.n
        shapes = {"x": n * self.HIDDEN, "qkv": n * self.qkv, "att": n * self.HEADS * self.DIM,
                  "o": n * self.HIDDEN, "logits": n * self.VOCAB, "lp": n, "entropy": n,
                  "top": n * 5}
        self.d = {k: lh.DeviceBuffer(4 * v) for k, v in shapes.items()}
        self.d["ids"] = lh.DeviceBuffer(8 * n * 5)
        self.d["tokens"] = lh.DeviceBuffer.from_array(np.arange(n, dtype=np.int64))
        self.d["head"] = lh.DeviceBuffer.from_array(
            (self.head.view(np.uint32) >> 16).astype(np.uint16))
        self.d["cos"] = lh.DeviceBuffer.from_array(self.cos)
        self.d["sin"] = lh.DeviceBuffer.from_array(self.sin)
        for i, l in enumerate(lengths):
            k, v = (rng.normal(size=(l - 1, self.KV, self.DIM)).astype(np.float32)
                    for _ in range(2))
            b = self.seq.batch([l - 1], [l - 1], table=self.seq.table[i:i + 1])
            self.seq.append(b, k, v)
        self.length = lh.DeviceBuffer.from_array(np.asarray(lengths, np.int32))
        self.batch = self.seq.batch([1] * n, lengths)
        self.batch.length = self.length.ptr
        self.batch.max_length = max(lengths) + 8
        self.sizes = [gpu.lh_q4_scratch(self.HIDDEN, n),
                      gpu.lh_paged_attention_scratch(ctypes.byref(self.seq.cache),
                                                     ctypes.byref(self.batch), self.HEADS),
                      gpu.lh_q4_scratch(self.HEADS * self.DIM, n),
                      gpu.lh_logprobs_scratch(n, self.VOCAB, 5)]
        self.scratch = lh.DeviceBuffer(max(self.sizes + [16]))

    def step(self, stream):
        g, d, n, w = self.gpu, self.d, self.n, self.HEADS * self.DIM
        cache, batch = ctypes.byref(self.seq.cache), ctypes.byref(self.batch)
        s, size = self.scratch.ptr, self.scratch.nbytes
        qkv, kv = d["qkv"].ptr, self.KV * self.DIM
        lh.check(g.lh_q4_matvec(self.packed[0].ptr, d["x"].ptr, self.HIDDEN, qkv, self.qkv,
                                self.qkv, self.HIDDEN, self.GROUP, n, s, size, stream))
        lh.check(g.lh_paged_append(cache, batch, self.HEADS, qkv, self.qkv, qkv + 4 * w, self.qkv,
                                   qkv + 4 * (w + kv), self.qkv, d["cos"].ptr, d["sin"].ptr,
                                   self.cos.shape[0], None, qkv, self.qkv, stream))
        lh.check(g.lh_paged_attention(cache, batch, self.HEADS, qkv, self.qkv, 0.0625,
                                      d["att"].ptr, w, s, size, stream))
        lh.check(g.lh_q4_matvec(self.packed[1].ptr, d["att"].ptr, w, d["o"].ptr, self.HIDDEN,
                                self.HIDDEN, w, self.GROUP, n, s, size, stream))
        lh.check(g.lh_bf16_matvec(d["head"].ptr, d["o"].ptr, d["logits"].ptr, self.VOCAB,
                                  self.HIDDEN, n, stream))
        lh.check(g.lh_logprobs(d["logits"].ptr, self.VOCAB, n, self.VOCAB, d["tokens"].ptr,
                               d["lp"].ptr, d["entropy"].ptr, 5, d["ids"].ptr, d["top"].ptr, s,
                               size, stream))

    def outputs(self):
        lh.check(self.gpu.lh_device_synchronize())
        out = {k: self.d[k].download(np.float32) for k in
               ("qkv", "att", "o", "logits", "lp", "entropy", "top")}
        out["ids"] = self.d["ids"].download(np.int64)
        return out


@pytest.mark.parametrize("kind", KINDS)
def test_decode_step_of_all_operators(gpu, kind):
    rng = np.random.default_rng(77)
    lengths = [130, 1, 64, 33, 257]
    dec = Decoder(gpu, kind, lengths, rng)
    x = rng.normal(size=(dec.n, dec.HIDDEN)).astype(np.float32)
    dec.d["x"].upload(x)
    dec.step(None)
    out = dec.outputs()
    n, w, kv = dec.n, dec.HEADS * dec.DIM, dec.KV * dec.DIM
    # Each stage against its definition on the rows that it was given.
    w0 = so.q4_weights(*dec.w[0], dec.GROUP)
    raw = x.astype(np.float64) @ w0.T
    bound = so.q4_bound(w0, x)
    pos = np.asarray(lengths) - 1
    qkv = out["qkv"].reshape(n, -1)
    close(qkv[:, w:], raw[:, w:], bound[:, w:])          # k and v as they were projected
    turned = so.rotate(raw[:, :w].reshape(n, dec.HEADS, dec.DIM), dec.cos[pos], dec.sin[pos])
    close(qkv[:, :w], turned.reshape(n, w), 2 * bound[:, :w].max() + 1e-6 * np.abs(raw).max())
    full = dec.seq.batch(lengths, lengths)
    keys, values = dec.seq.read(full)
    at = 0
    for i, l in enumerate(lengths):
        k = so.rotate(qkv[i:i + 1, w:w + kv].reshape(1, dec.KV, dec.DIM), dec.cos[pos[i]][None],
                      dec.sin[pos[i]][None])
        assert np.array_equal(keys[at + l - 1], so.cache_values(k, kind)[0])
        want, off = so.attention(qkv[i, :w].reshape(dec.HEADS, dec.DIM), keys[at:at + l],
                                 values[at:at + l], l - 1, 0.0625)
        close(out["att"].reshape(n, dec.HEADS, dec.DIM)[i], want, off)
        at += l
    w1 = so.q4_weights(*dec.w[1], dec.GROUP)
    att = out["att"].reshape(n, w)
    close(out["o"].reshape(n, -1), att.astype(np.float64) @ w1.T, so.q4_bound(w1, att))
    for r in range(n):
        want = so.logprobs(out["logits"].reshape(n, -1)[r], r, 5)
        assert np.array_equal(out["ids"].reshape(n, 5)[r], want[2])
        close(out["lp"][r:r + 1], np.array([want[0]]), want[4][0])
        close(out["entropy"][r:r + 1], np.array([want[1]]), want[4][1])


class Graph:
    """The calls that a function makes on a stream, captured."""

    def __init__(self, record):
        self.hip = ctypes.CDLL(lh.LIBRARY)   # the HIP runtime that it links
        for name in ("hipStreamBeginCapture", "hipStreamEndCapture", "hipGraphInstantiate",
                     "hipGraphLaunch"):
            getattr(self.hip, name).restype = ctypes.c_int
        self.stream = lh.lib().lh_stream_create()
        s = ctypes.c_void_p(self.stream)
        assert self.hip.hipStreamBeginCapture(s, 0) == 0
        record(self.stream)
        graph, self.exec = ctypes.c_void_p(), ctypes.c_void_p()
        assert self.hip.hipStreamEndCapture(s, ctypes.byref(graph)) == 0
        assert self.hip.hipGraphInstantiate(ctypes.byref(self.exec), graph, None, None,
                                            ctypes.c_size_t(0)) == 0

    def launch(self):
        assert self.hip.hipGraphLaunch(self.exec, ctypes.c_void_p(self.stream)) == 0
        lh.check(lh.lib().lh_stream_synchronize(self.stream))


@pytest.mark.parametrize("kind", KINDS)
def test_captured_step_follows_the_lengths(gpu, kind):
    """A captured step replayed while the sequences grow equals eager steps of
    another copy, bit for bit."""
    lengths = [30, 63, 5]
    a = Decoder(gpu, kind, lengths, np.random.default_rng(5))
    b = Decoder(gpu, kind, lengths, np.random.default_rng(5))
    graph = Graph(a.step)
    rng = np.random.default_rng(6)
    for turn in range(6):
        x = rng.normal(size=(a.n, a.HIDDEN)).astype(np.float32)
        now = np.asarray([l + turn for l in lengths], np.int32)
        for dec in (a, b):
            dec.d["x"].upload(x)
            dec.length.upload(now)
        graph.launch()
        b.step(None)
        got, want = a.outputs(), b.outputs()
        for name in want:
            assert np.array_equal(got[name], want[name]), (turn, name)


class Chunk:
    """Products, append and attention of a chunk of tokens, with scratch of their own."""

    def __init__(self, gpu, kind, count, rng):
        self.gpu, self.count = gpu, count
        self.cols, self.rows, self.group = 2048, 6 * 128, 32
        self.seq = so.Sequences(gpu, kind, 128, 4, 1, 64, [700 + count], rng)
        self.packed = so.q4_on_device(gpu, *so.q4_random(rng, self.rows, self.cols, self.group),
                                      self.group)
        k, v = (rng.normal(size=(700, 1, 128)).astype(np.float32) for _ in range(2))
        self.seq.append(self.seq.batch([700], [700]), k, v)
        self.batch = self.seq.batch([count], [700 + count])
        self.x = lh.DeviceBuffer(4 * count * self.cols)
        self.qkv = lh.DeviceBuffer(4 * count * self.rows)
        self.out = lh.DeviceBuffer(4 * count * 512)
        self.sizes = [gpu.lh_q4_scratch(self.cols, count), gpu.lh_paged_attention_scratch(
            ctypes.byref(self.seq.cache), ctypes.byref(self.batch), 4)]
        self.scratch = lh.DeviceBuffer(max(self.sizes + [16]))

    def step(self, stream):
        g, n, size = self.gpu, self.count, self.scratch.nbytes
        cache, batch = ctypes.byref(self.seq.cache), ctypes.byref(self.batch)
        q = self.qkv.ptr
        lh.check(g.lh_q4_matvec(self.packed.ptr, self.x.ptr, self.cols, q, self.rows, self.rows,
                                self.cols, self.group, n, self.scratch.ptr, size, stream))
        lh.check(g.lh_paged_append(cache, batch, 4, q, self.rows, q + 2048, self.rows, q + 2560,
                                   self.rows, None, None, 0, None, q, self.rows, stream))
        lh.check(g.lh_paged_attention(cache, batch, 4, q, self.rows, 0.0625, self.out.ptr, 512,
                                      self.scratch.ptr, size, stream))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("counts", [(5, 40), (100, 150)])
def test_captured_chunks_on_two_streams(gpu, kind, counts):
    """Two captured chunks replayed at once, again and again, equal eager ones."""
    chunks = [Chunk(gpu, kind, c, np.random.default_rng(c)) for c in counts]
    eager = [Chunk(gpu, kind, c, np.random.default_rng(c)) for c in counts]
    graphs = [Graph(c.step) for c in chunks]
    rng = np.random.default_rng(1)
    for turn in range(4):
        for c, e in zip(chunks, eager):
            x = rng.normal(size=(c.count, c.cols)).astype(np.float32)
            c.x.upload(x)
            e.x.upload(x)
        for g in graphs:
            assert g.hip.hipGraphLaunch(g.exec, ctypes.c_void_p(g.stream)) == 0
        for e in eager:
            e.step(None)
        lh.check(gpu.lh_device_synchronize())
        for c, e in zip(chunks, eager):
            want = e.out.download(np.float32)
            assert np.isfinite(want).all()
            assert np.array_equal(c.out.download(np.float32), want), turn
            assert np.array_equal(c.qkv.download(np.float32), e.qkv.download(np.float32)), turn
