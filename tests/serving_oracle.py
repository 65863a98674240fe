"""The batched serving operators (include/lunelette_serving.h) in 64 bits, from
their definitions, and device helpers for their tests."""
import ctypes

import numpy as np

import lunelette_amd as lh

EPS32 = 2.0 ** -24   # half a step of FP32, relative


def bf16(v):
    """FP32 values rounded to BF16, ties to even, as FP32."""
    u = np.asarray(v, np.float32).view(np.uint32).astype(np.uint64)
    return (((u + 0x7fff + ((u >> 16) & 1)) >> 16) << 16).astype(np.uint32).view(np.float32)


# ---- 4-bit weights ----

def q4_random(rng, rows, cols, group):
    codes = rng.integers(0, 16, size=(rows, cols), dtype=np.uint8)
    scales = bf16(rng.uniform(0.5, 2.0, size=(rows, cols // group)) * 0.01)
    return codes, scales


def q4_weights(codes, scales, group):
    return (codes.astype(np.float64) - 8) * np.repeat(scales.astype(np.float64), group, axis=1)


def q4_on_device(gpu, codes, scales, group):
    rows, cols = codes.shape
    packed = lh.DeviceBuffer(gpu.lh_q4_bytes(rows, cols, group))
    two = lh.DeviceBuffer.from_array(codes[:, 0::2] | (codes[:, 1::2] << 4))
    bits = lh.DeviceBuffer.from_array((scales.view(np.uint32) >> 16).astype(np.uint16))
    lh.check(gpu.lh_q4_pack(two.ptr, bits.ptr, rows, cols, group, packed.ptr, None))
    lh.check(gpu.lh_device_synchronize())
    return packed


def q4_run(gpu, packed, x, rows, cols, group, x_pad=0, y_pad=0, offset=0, stream=None):
    """y [tokens][rows] of x [tokens][cols], rows of x and y padded, x starting
    `offset` elements into its buffer; checks that the padding stays."""
    tokens = x.shape[0]
    xs, ys = cols + x_pad, rows + y_pad
    buf = np.full(offset + tokens * xs, np.nan, np.float32)
    buf[offset:].reshape(tokens, xs)[:, :cols] = x
    d_x = lh.DeviceBuffer.from_array(buf)
    d_y = lh.DeviceBuffer.from_array(np.full(tokens * ys + 4, 7.25, np.float32))
    need = gpu.lh_q4_scratch(cols, tokens)
    scratch = lh.DeviceBuffer(max(16, need))
    lh.check(gpu.lh_q4_matvec(packed.ptr, d_x.ptr + 4 * offset, xs, d_y.ptr, ys, rows, cols, group,
                              tokens, scratch.ptr, need, stream))
    lh.check(gpu.lh_device_synchronize())
    y = d_y.download(np.float32)
    assert np.all(y[tokens * ys:] == 7.25)
    y = y[:tokens * ys].reshape(tokens, ys)
    assert np.all(y[:, rows:] == 7.25), "wrote between the rows"
    return y[:, :rows]


def q4_bound(w, x):
    """What y may be off: x in planes to 2^-22 of itself, then at most one
    rounding for every two of a 32-column product's sums, 40 for the sums inside
    one, across groups and across waves."""
    cols = w.shape[1]
    magnitude = np.abs(x).astype(np.float64) @ np.abs(w).T
    return magnitude * (2.0 ** -22 + (2 * cols / 32 + 40) * EPS32) + 1e-37


# ---- log probabilities ----

def logprobs(row, token, top):
    """(ln p of token, entropy, ids, ln p of ids, allowed error of each)."""
    x = np.asarray(row, np.float64)
    n = x.size
    bad = np.isnan(x).any() or np.isposinf(x).any()
    if bad:
        nan = np.float64(np.nan)
        return nan, nan, np.full(top, -1), np.full(top, nan), (0, 0, np.zeros(top))
    if np.all(np.isneginf(x)):
        lp = -np.inf if 0 <= token < n else (0.0 if token == -1 else np.nan)
        return lp, 0.0, np.full(top, -1), np.full(top, -np.inf), (0, 0, np.zeros(top))
    d = x - x.max()
    first = int(np.argmax(d))
    e = np.exp(d)
    rest = np.delete(e, first)
    with np.errstate(invalid="ignore"):
        distance = np.where(rest > 0, -np.delete(d, first), 0.0)
    z1 = rest.sum()                       # Z - 1 without the cancellation
    log_z = np.log1p(z1)
    p = rest / (1 + z1)
    lp = d - log_z
    entropy = log_z + (p * distance).sum()
    # exp in FP32: two steps, plus its argument's rounding; sums in 64 bits.
    each = p * (distance * EPS32 + 2.0 ** -21)
    # The sum that holds the largest token's 1 rounds to 2^-53 at each of its
    # additions: at most those of a lane's n / 64 terms and the joins.
    wide = (n / 64 + 64) * 2.0 ** -53
    off_z = each.sum() + wide
    off_h = (each * (1 + distance)).sum() + 2.0 ** -22 * entropy + wide
    order = np.lexsort((np.arange(n), -(x + 0.0)))
    order = order[~np.isneginf(x[order])][:top]
    ids = np.concatenate([order, np.full(top - order.size, -1, np.int64)])
    tops = np.concatenate([lp[order], np.full(top - order.size, -np.inf)])
    with np.errstate(invalid="ignore"):
        off_top = np.where(np.isfinite(tops), off_z + 2.0 ** -23 * np.abs(tops), 0.0)
    if token == -1:
        given, off = 0.0, 0.0
    elif not 0 <= token < n:
        given, off = np.nan, 0.0
    else:
        given = lp[token]
        off = off_z + 2.0 ** -23 * abs(given) if np.isfinite(given) else 0.0
    return given, entropy, ids, tops, (off, off_h, off_top)


# ---- paged cache ----

def rotate(x, cos, sin):
    """x [n][heads][dim] by rows cos, sin [n][dim], in 64 bits."""
    half = x.shape[-1] // 2
    x, c, s = x.astype(np.float64), cos[:, None].astype(np.float64), sin[:, None].astype(np.float64)
    return np.concatenate([x[..., :half] * c[..., :half] - x[..., half:] * s[..., :half],
                           x[..., half:] * c[..., half:] + x[..., :half] * s[..., half:]], axis=-1)


def cache_values(rows, kind):
    """What the cache holds of rows [...][dim] (64 bits)."""
    rows = np.asarray(rows, np.float64)
    if kind == lh.CACHE_F16:
        with np.errstate(over="ignore"):
            return rows.astype(np.float32).astype(np.float16).astype(np.float32)
    with np.errstate(all="ignore"):
        z = bf16(rows.min(-1, keepdims=True).astype(np.float32))
        step = ((rows.max(-1, keepdims=True) - z) / 15).astype(np.float32)
        s = np.where(step > 0, bf16(step), np.float32(0))
        code = np.clip(np.rint((rows - z) / s), 0, 15)
        code = np.where(s > 0, code, 0.0)
        value = (code * s.astype(np.float64) + z).astype(np.float32)
        fine = np.isfinite(rows).all(-1, keepdims=True) & np.isfinite(z) & np.isfinite(s)
    return np.where(fine, value, np.float32(np.nan))


class Sequences:
    """Sequences over one cache, with the host's copy of what it holds."""

    def __init__(self, gpu, kind, dim, heads, kv_heads, page, lengths, rng, spare=2, fill=0xff):
        self.gpu, self.kind, self.dim = gpu, kind, dim
        self.heads, self.kv_heads, self.page = heads, kv_heads, page
        self.n = len(lengths)
        need = [max(0, -(-l // page)) for l in lengths]
        self.width = max(need + [1])
        self.pages = sum(need) + spare
        order = rng.permutation(self.pages)
        self.table = np.full((self.n, self.width), -1, np.int32)
        at = 0
        for i, k in enumerate(need):
            self.table[i, :k] = order[at:at + k]
            at += k
        c = self.cache = lh.PagedCache()
        c.kind, c.kv_heads, c.head_dim, c.page_size, c.pages = kind, kv_heads, dim, page, self.pages
        nbytes = gpu.lh_paged_cache_bytes(ctypes.byref(c))
        self.memory = lh.DeviceBuffer(nbytes)
        lh.check(gpu.lh_memset_device(self.memory.ptr, fill, nbytes))
        c.data = self.memory.ptr
        self.keep = []

    def batch(self, counts, lengths, tokens=None, table=None):
        """A call in which sequence i brings its last counts[i] of lengths[i]."""
        start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        table = self.table if table is None else table
        b = lh.PagedBatch()
        bufs = [lh.DeviceBuffer.from_array(a) for a in
                (start, np.asarray(lengths, np.int32), np.ascontiguousarray(table, np.int32))]
        b.sequences, b.tokens = len(counts), int(start[-1]) if tokens is None else tokens
        b.tokens = max(1, b.tokens)
        b.table_width = table.shape[1]
        b.max_query, b.max_length = max(1, max(counts)), max(1, max(lengths))
        b.query_start, b.length, b.table = (x.ptr for x in bufs)
        self.keep.append(bufs)
        return b

    def append(self, batch, k, v, q=None, cos=None, sin=None, factor=None, stream=None):
        """k, v [tokens][kv_heads][dim], q [tokens][heads][dim]; returns q out."""
        gpu, kv, width = self.gpu, self.kv_heads * self.dim, self.heads * self.dim
        bufs = [None if a is None else lh.DeviceBuffer.from_array(np.asarray(a, np.float32))
                for a in (k, v, q, cos, sin, factor)]
        ptr = [b and b.ptr for b in bufs]
        out = None
        if q is not None:
            out = lh.DeviceBuffer.from_array(np.full(q.size, 7.25, np.float32))
        lh.check(gpu.lh_paged_append(
            ctypes.byref(self.cache), ctypes.byref(batch), self.heads if q is not None else 0,
            ptr[2], width, ptr[0], kv, ptr[1], kv, ptr[3], ptr[4],
            0 if cos is None and factor is None else (cos if cos is not None else factor).shape[0],
            ptr[5], out and out.ptr, width, stream))
        lh.check(gpu.lh_device_synchronize())
        return None if q is None else out.download(np.float32).reshape(q.shape)

    def read(self, batch):
        kv, n = self.kv_heads * self.dim, batch.tokens
        out = [lh.DeviceBuffer.from_array(np.full(n * kv, 7.25, np.float32)) for _ in range(2)]
        lh.check(self.gpu.lh_paged_read(ctypes.byref(self.cache), ctypes.byref(batch), out[0].ptr,
                                        kv, out[1].ptr, kv, None))
        lh.check(self.gpu.lh_device_synchronize())
        return [o.download(np.float32).reshape(n, self.kv_heads, self.dim) for o in out]

    def attention(self, batch, q, scale, q_pad=0, out_pad=0, stream=None):
        width, n = self.heads * self.dim, batch.tokens
        buf = np.full((n, width + q_pad), np.nan, np.float32)
        buf[:, :width] = q.reshape(n, width)
        d_q = lh.DeviceBuffer.from_array(buf)
        out = lh.DeviceBuffer.from_array(np.full((n, width + out_pad), 7.25, np.float32))
        need = self.gpu.lh_paged_attention_scratch(ctypes.byref(self.cache), ctypes.byref(batch),
                                                   self.heads)
        scratch = lh.DeviceBuffer(max(16, need))
        lh.check(self.gpu.lh_memset_device(scratch.ptr, 0xff, scratch.nbytes))
        lh.check(self.gpu.lh_paged_attention(
            ctypes.byref(self.cache), ctypes.byref(batch), self.heads, d_q.ptr, width + q_pad,
            scale, out.ptr, width + out_pad, scratch.ptr, need, stream))
        lh.check(self.gpu.lh_device_synchronize())
        got = out.download(np.float32).reshape(n, width + out_pad)
        assert np.all(got[:, width:] == 7.25), "wrote between the rows"
        return got[:, :width].reshape(n, self.heads, self.dim)


def attention(q, keys, values, last, scale):
    """One token's row q [heads][dim] over keys, values [length][kv_heads][dim]
    up to position last, in 64 bits, and what it may be off.

    Scores: q in planes to 2^-22, dim products and sums of FP32, the offset and
    scale of 4-bit codes (whose parts are up to three times the largest
    value): delta. A probability is off by 2 delta and exp's two steps, the sum
    over positions by a rounding for every 16 of them, 64 for the joins."""
    heads, dim = q.shape
    group = heads // keys.shape[1]
    out, off = np.zeros((heads, dim)), np.zeros((heads, dim))
    if last < 0:
        return out, off
    for h in range(heads):
        k = keys[:last + 1, h // group].astype(np.float64)
        v = values[:last + 1, h // group].astype(np.float64)
        s = k @ q[h].astype(np.float64) * scale
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h] = p @ v
        size = scale * np.abs(q[h]).astype(np.float64).sum() * 3 * np.abs(k).max(-1)
        delta = (size * (2.0 ** -22 + (dim + 8) * EPS32)).max()
        magnitude = p @ (3 * np.abs(v).max(-1))
        off[h] = magnitude * (2 * delta + 2.0 ** -20 + ((last + 1) / 16 + 64) * EPS32)
    return out, off
