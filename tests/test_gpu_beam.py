"""Beam search on the GPU (include/lunelette_serving.h): the choice against its definition
in 64 bits, the reordering of tables and pages, and a search over layers of 8-bit
products, eager and captured."""
import ctypes

import numpy as np
import pytest

import lunelette_amd as lh

import q8_oracle as q8
import serving_oracle as so
from test_gpu_serving import Graph, KINDS, close, orders, tables

pytestmark = pytest.mark.gpu


# ---- the choice ----

class Choice:
    """Buffers of a call, guarded."""

    def __init__(self, gpu, logits, scores, done, stop, keep, groups, beams, pad=0, offset=0):
        self.gpu, self.keep, self.groups, self.beams, self.stop = gpu, keep, groups, beams, stop
        rows, self.vocab = logits.shape
        self.stride = self.vocab + pad
        buf = np.full(offset + rows * self.stride, np.nan, np.float32)
        buf[offset:].reshape(rows, self.stride)[:, :self.vocab] = logits
        self.x = lh.DeviceBuffer.from_array(buf)
        self.x_ptr = self.x.ptr + 4 * offset
        self.scores = lh.DeviceBuffer.from_array(np.asarray(scores, np.float32))
        self.done = None if done is None else lh.DeviceBuffer.from_array(
            np.asarray(done, np.uint8))
        n = self.n = groups * keep
        self.parent = lh.DeviceBuffer.from_array(np.full(n + 1, 77, np.int32))
        self.token = lh.DeviceBuffer.from_array(np.full(n + 1, 77, np.int64))
        self.score = lh.DeviceBuffer.from_array(np.full(n + 1, 7.25, np.float32))
        self.ended = lh.DeviceBuffer.from_array(np.full(n + 1, 77, np.uint8))
        self.need = gpu.lh_beam_scratch(groups, beams, self.vocab, keep)
        self.scratch = lh.DeviceBuffer(max(16, self.need))
        lh.check(gpu.lh_memset_device(self.scratch.ptr, 0xff, self.scratch.nbytes))

    def call(self, stream=None):
        lh.check(self.gpu.lh_beam_select(
            self.x_ptr, self.stride, self.groups, self.beams, self.vocab, self.scores.ptr,
            self.done and self.done.ptr, self.stop, self.keep, self.parent.ptr, self.token.ptr,
            self.score.ptr, self.ended.ptr, self.scratch.ptr, self.need, stream))

    def get(self):
        lh.check(self.gpu.lh_device_synchronize())
        out = (self.parent.download(np.int32), self.token.download(np.int64),
               self.score.download(np.float32), self.ended.download(np.uint8))
        for got, guard in zip(out, (77, 77, 7.25, 77)):
            assert got[self.n] == guard
        return [got[:self.n].reshape(self.groups, self.keep) for got in out]


def check_choice(gpu, logits, scores, done, stop, keep, groups, beams, **how):
    """Against the definition, as far as the inputs decide."""
    call = Choice(gpu, logits, scores, done, stop, keep, groups, beams, **how)
    call.call()
    got = call.get()
    none = np.zeros(groups * beams, np.uint8)
    parent, token, score, ended, off, decided = q8.select(
        logits, np.asarray(scores, np.float32), none if done is None else done, stop, keep, groups,
        beams)
    assert decided.mean() >= 0.5   # the inputs say something
    close(got[2], score, off)
    for g, want in ((got[0], parent), (got[1], token), (got[3], ended)):
        assert np.array_equal(g[decided], want[decided])
    return got


@pytest.mark.parametrize("groups,beams,vocab,keep", [
    (1, 1, 1, 1), (1, 1, 131072, 1), (1, 4, 131072, 4), (3, 5, 1000, 10), (2, 64, 70, 64),
    (1, 64, 5003, 64), (7, 3, 4097, 6), (16, 8, 2048, 16), (2, 2, 3, 64), (40, 16, 515, 16),
    (1, 2, 300001, 4), (300, 1, 77, 5), (1, 1, 5, 64), (5, 33, 1025, 33), (2, 7, 151936, 14)])
def test_select(gpu, groups, beams, vocab, keep):
    rng = np.random.default_rng(groups + vocab)
    n = groups * beams
    logits = (2.5 * rng.normal(size=(n, vocab))).astype(np.float32)
    logits[::3, vocab // 2] += 18            # almost certain rows
    scores = (-12 + 2 * rng.normal(size=n)).astype(np.float32)
    done = (rng.random(n) < 0.2).astype(np.uint8)
    got = check_choice(gpu, logits, scores, done, vocab // 2, keep, groups, beams)
    again = check_choice(gpu, logits, scores, done, vocab // 2, keep, groups, beams, pad=3,
                         offset=1)
    for a, b in zip(got, again):
        assert np.array_equal(a.view(np.uint8), b.view(np.uint8))
    check_choice(gpu, logits, scores, None, -1, keep, groups, beams)


@pytest.mark.parametrize("beams,keep", [(1, 1), (2, 64), (64, 2), (3, 42), (3, 43), (43, 3), (16, 8),
                                        (8, 17), (64, 3), (16, 64), (17, 64)])
def test_select_numbers_of_candidates(gpu, beams, keep):
    """To either side of 128 and of 1024 candidates in a group's lists, with equal logits in a
    row, finished beams and beams without a score."""
    rng = np.random.default_rng(beams * keep)
    groups, vocab = 3, 900
    n = groups * beams
    logits = (np.round(8 * rng.normal(size=(n, vocab))) / 4).astype(np.float32)
    scores = (-5 + 3 * rng.normal(size=n)).astype(np.float32)
    check_choice(gpu, logits, scores, None, 7, keep, groups, beams)
    done = rng.random(n) < 0.3
    scores[rng.random(n) < 0.3] = -np.inf
    check_choice(gpu, logits, scores, done, 7, keep, groups, beams)


@pytest.mark.parametrize("vocab,keep", [(3000, 64), (70001, 20), (131072, 64), (515, 7)])
def test_select_orders_ties_and_masks(gpu, vocab, keep):
    """Rows whose order is hard on a selection, one at a time in a group."""
    x = orders(np.random.default_rng(vocab), vocab)
    check_choice(gpu, x, np.linspace(-3, -9, 9), None, 5, keep, 9, 1)


def test_select_equal_beams(gpu):
    """Beams of equal rows and scores: every token of the first before those of the
    second with the same score; and scores of -0."""
    rng = np.random.default_rng(8)
    row = rng.normal(size=2000).astype(np.float32)
    logits = np.stack([row, row, row, row - 100])
    got = check_choice(gpu, logits, [-1, -1, -1, -1], None, -1, 12, 1, 4)
    equal = got[0][0][got[0][0] < 3]       # the last beam's logits are rounded otherwise
    assert np.array_equal(equal, np.tile([0, 1, 2], 3)[:equal.size])
    got = check_choice(gpu, np.zeros((4, 1), np.float32), [0.0, -0.0, 0.0, -0.0], None, -1, 4, 1, 4)
    assert list(got[0][0]) == [0, 1, 2, 3]
    flat = np.full((2, 5000), 1.5, np.float32)
    got = check_choice(gpu, flat, [-2, -2], None, -1, 64, 1, 2)
    assert np.all(got[0] == 0) and np.array_equal(got[1][0], np.arange(64))


def test_select_without_candidates(gpu):
    """Beams of score -Inf and rows of nothing but masks have none; what rows are not
    read may hold anything; one bad beam takes its group, and no other."""
    rng = np.random.default_rng(9)
    groups, beams, vocab = 9, 3, 2500
    logits = rng.normal(size=(groups * beams, vocab)).astype(np.float32)
    scores = rng.normal(size=groups * beams).astype(np.float32)
    done = np.zeros(groups * beams, np.uint8)
    scores[0:3] = -np.inf                    # nothing at all
    logits[0:3] = np.nan
    logits[4] = -np.inf                      # a row of masks beside two others
    scores[7:9] = -np.inf                    # a first step
    logits[7:9] = np.nan
    done[10], logits[10] = 1, np.inf         # a finished beam's row
    logits[13, 2499] = np.nan                # bad groups
    logits[15, 0] = np.inf
    scores[19] = np.nan
    scores[23], done[23] = np.inf, 1
    logits[24:27] = -np.inf                  # one token left of three rows
    logits[25, 777] = -3
    got = check_choice(gpu, logits, scores, done, 777, 5, groups, beams)
    assert np.all(got[0][0] == -1) and np.isneginf(got[2][0]).all()
    assert np.all(got[0][2] == 0)
    for g in (4, 5, 6, 7):
        assert np.all(got[0][g] == -1) and np.isnan(got[2][g]).all()
    assert list(got[1][8]) == [777, -1, -1, -1, -1] and list(got[3][8]) == [1, 0, 0, 0, 0]


@pytest.mark.parametrize("rows,vocab", [(256, 70001), (40, 131072), (9, 1500)])
def test_a_nan_or_inf_anywhere_in_a_row(gpu, rows, vocab):
    """The scan of a row, which log probabilities share, in every chunk and round of it."""
    rng = np.random.default_rng(rows)
    x = rng.normal(size=(rows, vocab)).astype(np.float32)
    bad = np.arange(rows) % 5 != 0
    for r in np.nonzero(bad)[0]:
        x[r, r * (vocab - 1) // (rows - 1)] = (np.nan, np.inf)[r % 2]
    x[::5, 1::2] = -np.inf
    for keep in (1, 4, 64):
        call = Choice(gpu, x, np.zeros(rows), None, -1, keep, rows, 1)
        call.call()
        parent, _, score, _ = call.get()
        assert np.array_equal(np.isnan(score), np.repeat(bad[:, None], keep, 1))
        assert np.array_equal(parent < 0, np.isnan(score))
    d_x = lh.DeviceBuffer.from_array(x)
    for top in (0, 4):
        need = gpu.lh_logprobs_scratch(rows, vocab, top)
        scratch = lh.DeviceBuffer(max(16, need))
        tokens = lh.DeviceBuffer.from_array(np.zeros(rows, np.int64))
        out = [lh.DeviceBuffer.from_array(np.zeros(rows, np.float32)) for _ in range(2)]
        ids = lh.DeviceBuffer.from_array(np.zeros(rows * 4, np.int64))
        best = lh.DeviceBuffer.from_array(np.zeros(rows * 4, np.float32))
        lh.check(gpu.lh_logprobs(d_x.ptr, vocab, rows, vocab, tokens.ptr, out[0].ptr, out[1].ptr,
                                 top, ids.ptr if top else None, best.ptr if top else None,
                                 scratch.ptr, need, None))
        lh.check(gpu.lh_device_synchronize())
        for o in out:
            assert np.array_equal(np.isnan(o.download(np.float32)), bad)
        if top:
            assert np.array_equal(ids.download(np.int64).reshape(rows, 4) < 0,
                                  np.repeat(bad[:, None], 4, 1))


def test_select_all_finished(gpu):
    rng = np.random.default_rng(10)
    logits = np.full((6, 9), np.nan, np.float32)
    scores = np.array([-3, -1, -np.inf, -2, -2, -2], np.float32)
    got = check_choice(gpu, logits, scores, np.ones(6, np.uint8), 4, 3, 2, 3)
    assert np.array_equal(got[0], [[1, 0, -1], [0, 1, 2]])
    assert np.array_equal(got[3], [[1, 1, 0], [1, 1, 1]])


def test_select_far_scores(gpu):
    """Scores from the ends of FP32 beside common ones."""
    rng = np.random.default_rng(11)
    logits = rng.normal(size=(8, 700)).astype(np.float32)
    scores = np.array([-3e38, 3e38, -1, 1e-42, -1e10, -2, 0, 5], np.float32)
    call = Choice(gpu, logits, scores, None, -1, 6, 2, 4)
    call.call()
    parent, token, score, _ = call.get()
    assert np.all(parent[0] == 1) and np.all(score[0] == np.float32(3e38))
    # Tokens of the far beam have equal scores in 64 bits: the larger logit first.
    assert np.array_equal(token[0], np.argsort(-logits[1], kind="stable")[:6])
    want = q8.select(logits, scores, np.zeros(8), -1, 6, 2, 4)
    assert np.array_equal(parent[1], want[0][1]) and np.array_equal(token[1], want[1][1])


def test_select_on_two_streams(gpu):
    rng = np.random.default_rng(12)
    streams = [gpu.lh_stream_create() for _ in range(2)]
    calls = []
    for _ in streams:
        logits = rng.normal(size=(12, 40000)).astype(np.float32)
        calls.append(Choice(gpu, logits, rng.normal(size=12), None, 3, 8, 3, 4))
    want = []
    for c in calls:
        c.call()
        want.append(c.get())
    for _ in range(20):
        for s, c in zip(streams, calls):
            c.call(s)
    for s in streams:
        lh.check(gpu.lh_stream_synchronize(s))
    for w, c in zip(want, calls):
        for a, b in zip(w, c.get()):
            assert np.array_equal(a, b)
    for s in streams:
        gpu.lh_stream_destroy(s)


# ---- the reordering ----

class Layers:
    """Alike caches of several layers, filled with random bytes."""

    def __init__(self, gpu, layers, kind, kv_heads, dim, page, pages, rng):
        self.gpu = gpu
        self.caches = (lh.PagedCache * layers)()
        self.memory, self.host = [], []
        for c in self.caches:
            c.kind, c.kv_heads, c.head_dim, c.page_size, c.pages = kind, kv_heads, dim, page, pages
            nbytes = gpu.lh_paged_cache_bytes(ctypes.byref(c))
            self.host.append(rng.integers(0, 256, size=(pages, nbytes // pages), dtype=np.uint8))
            self.memory.append(lh.DeviceBuffer.from_array(self.host[-1]))
            c.data = self.memory[-1].ptr


def run_reorder(gpu, layers, parent, lengths, table, in_place=False, stream=None):
    groups, beams = parent.shape
    bufs = [lh.DeviceBuffer.from_array(np.asarray(a, np.int32)) for a in (parent, lengths, table)]
    out = bufs[2] if in_place else lh.DeviceBuffer.from_array(
        np.full(table.size + 4, 77, np.int32))
    lh.check(gpu.lh_beam_reorder(layers.caches, len(layers.caches), groups, beams, bufs[0].ptr,
                                 bufs[1].ptr, bufs[2].ptr, out.ptr, table.shape[1], stream))
    lh.check(gpu.lh_device_synchronize())
    got = out.download(np.int32)
    assert in_place or np.all(got[table.size:] == 77)
    if not in_place:
        assert np.array_equal(bufs[2].download(np.int32), table.reshape(-1))
    return got[:table.size].reshape(table.shape)


def own_pages(rng, groups, beams, page, lengths, width):
    """Tables of groups that share their full pages; pages dealt in random order."""
    total = groups * (beams * width + width)
    order = rng.permutation(total).astype(np.int32)
    table = order[:groups * beams * width].reshape(groups * beams, width).copy()
    for g in range(groups):
        full = min(width, max(0, lengths[g * beams]) // page)
        table[g * beams:(g + 1) * beams, :full] = table[g * beams, :full]
    return table, total


def check_reorder(gpu, layers, parent, lengths, table, page, in_place=False):
    got = run_reorder(gpu, layers, parent, lengths, table, in_place)
    want, copies = q8.reorder(parent, lengths, table, page)
    assert np.array_equal(got, want)
    pages = layers.caches[0].pages
    for host, memory in zip(layers.host, layers.memory):
        for a, b in copies:
            if 0 <= a < pages and 0 <= b < pages:
                host[b] = host[a]
        assert np.array_equal(memory.download(np.uint8).reshape(host.shape), host)
    return want, copies


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("groups,beams,layers,kv_heads,dim,page,width", [
    (1, 1, 1, 1, 64, 32, 1), (1, 4, 26, 2, 128, 32, 5), (3, 8, 2, 1, 64, 64, 3),
    (2, 64, 3, 1, 64, 32, 2), (5, 2, 64, 1, 64, 32, 70), (1, 5, 1, 3, 64, 96, 130),
    (9, 3, 4, 1, 128, 32, 2)])
def test_reorder(gpu, kind, in_place, groups, beams, layers, kv_heads, dim, page, width):
    rng = np.random.default_rng(groups * 31 + beams)
    lengths = rng.integers(0, page * width + 1, size=groups).repeat(beams).astype(np.int32)
    lengths[:beams] = page * (width - 1) + 1     # one group with a begun page for sure
    table, pages = own_pages(rng, groups, beams, page, lengths, width)
    caches = Layers(gpu, layers, kind, kv_heads, dim, page, pages, rng)
    for turn in range(3):
        parent = rng.integers(0, beams, size=(groups, beams)).astype(np.int32)
        table, _ = check_reorder(gpu, caches, parent, lengths, table, page, in_place)


@pytest.mark.parametrize("in_place", [False, True])
def test_reorder_families(gpu, in_place):
    """Everyone stays, a permutation, one parent of all (the first and the last), places
    without a parent, ids outside the group."""
    rng = np.random.default_rng(2)
    beams, page, width = 6, 32, 4
    families = [[0, 1, 2, 3, 4, 5], [5, 3, 4, 0, 1, 2], [0] * 6, [5] * 6, [-1] * 6,
                [2, -1, 2, 0, -1, 0], [6, 7, -2, 2 ** 31 - 1, -2 ** 31, 1], [3, 3, 3, 1, 1, -1]]
    groups = len(families)
    for rest in (0, 1, 31):
        lengths = np.full(groups * beams, 2 * page + rest, np.int32)
        table, pages = own_pages(rng, groups, beams, page, lengths, width)
        caches = Layers(gpu, 2, lh.CACHE_Q4, 1, 64, page, pages, rng)
        new, copies = check_reorder(gpu, caches, np.array(families, np.int32), lengths, table, page,
                                    in_place)
        assert np.array_equal(new[:beams], table[:beams])
        assert len(copies) == (0 if rest == 0 else 5 + 5 + 2 + 3)
        # No page from the open one on stands in two places.
        own = new[:, 2:].reshape(-1)
        assert np.unique(own).size == own.size


def test_reorder_odd_lengths_and_pages(gpu):
    """Negative and zero lengths, lengths at and past the table, page ids without a place:
    nothing is read or written out of range, and the rest is as defined."""
    rng = np.random.default_rng(3)
    beams, page, width = 3, 32, 2
    lengths = np.array([-5, 0, 1, 63, 64, 65, 2 ** 31 - 1], np.int32).repeat(beams)
    groups = len(lengths) // beams
    table, pages = own_pages(rng, groups, beams, page, np.maximum(lengths, 0), width)
    table[2 * beams, 0] = -1                     # the page of a parent
    table[3 * beams + 1, 1] = pages + 100        # and of a beam without children
    table[3 * beams + 2, 1] = 2 ** 31 - 1
    caches = Layers(gpu, 1, lh.CACHE_F16, 1, 64, page, pages, rng)
    parent = np.tile(np.array([0, 0, 0], np.int32), (groups, 1))
    check_reorder(gpu, caches, parent, lengths, table, page)


def test_reorder_large_offsets(gpu):
    """Pages past 2^32 bytes."""
    c = (lh.PagedCache * 1)()
    c[0].kind, c[0].kv_heads, c[0].head_dim, c[0].page_size = lh.CACHE_F16, 8, 128, 1024
    c[0].pages = 1100
    nbytes = gpu.lh_paged_cache_bytes(c)
    assert nbytes > 2 ** 32
    memory = lh.DeviceBuffer(nbytes)
    page_bytes = nbytes // 1100
    c[0].data = memory.ptr
    rng = np.random.default_rng(4)
    one = rng.integers(0, 256, size=page_bytes, dtype=np.uint8)
    lh.check(gpu.lh_memset_device(memory.ptr, 0, nbytes))
    lh.check(gpu.lh_memcpy_htod(memory.ptr + 1098 * page_bytes, one.ctypes.data, page_bytes))
    bufs = [lh.DeviceBuffer.from_array(np.array(a, np.int32)) for a in
            ([0, 0], [7, 7], [1098, 1099])]
    out = lh.DeviceBuffer(8)
    lh.check(gpu.lh_beam_reorder(c, 1, 1, 2, bufs[0].ptr, bufs[1].ptr, bufs[2].ptr, out.ptr, 1,
                                 None))
    lh.check(gpu.lh_device_synchronize())
    got = np.empty(page_bytes, np.uint8)
    lh.check(gpu.lh_memcpy_dtoh(got.ctypes.data, memory.ptr + 1099 * page_bytes, page_bytes))
    assert np.array_equal(got, one)


# ---- a search ----

class Search:
    """Steps of a beam search over layers of 8-bit products: norm, q|k|v, append, attention,
    rows, o, norm with the residual, gate|up, SwiGLU, down, and the choice of the next
    beams with the caches' reordering."""
    HEADS, KV, DIM, HIDDEN, INNER, VOCAB, PAGE, LAYERS = 4, 2, 64, 256, 336, 700, 32, 2

    def __init__(self, gpu, kind, groups, beams, capacity, seed):
        rng = np.random.default_rng(seed)
        self.gpu, self.groups, self.beams, self.n = gpu, groups, beams, groups * beams
        self.capacity = capacity
        self.width = self.HEADS * self.DIM
        self.qkv = (self.HEADS + 2 * self.KV) * self.DIM
        self.embedding = rng.normal(size=(self.VOCAB, self.HIDDEN)).astype(np.float32)
        self.cos, self.sin, _ = tables(rng, capacity, self.DIM)
        columns = -(-capacity // self.PAGE)
        order = rng.permutation(self.n * columns).astype(np.int32)
        self.first_table = order.reshape(self.n, columns)
        self.caches = (lh.PagedCache * self.LAYERS)()
        self.d = {}
        self.packed = []
        for i, c in enumerate(self.caches):
            c.kind, c.kv_heads, c.head_dim, c.page_size = kind, self.KV, self.DIM, self.PAGE
            c.pages = self.n * columns
            self.buffer("pages%d" % i, gpu.lh_paged_cache_bytes(ctypes.byref(c)))
            c.data = self.d["pages%d" % i].ptr
            layer = []
            for rows, cols in ((self.qkv, self.HIDDEN), (self.HIDDEN, self.width),
                               (2 * self.INNER, self.HIDDEN), (self.HIDDEN, self.INNER)):
                w = lh.DeviceBuffer.from_array(
                    (rng.normal(size=(rows, cols)) / np.sqrt(cols)).astype(np.float32))
                p = lh.DeviceBuffer(gpu.lh_q8_bytes(rows, cols))
                lh.check(gpu.lh_q8_quantize(w.ptr, rows, cols, p.ptr, None))
                lh.check(gpu.lh_device_synchronize())
                layer.append((p, rows, cols))
            self.packed.append(layer)
            for name in ("g1", "g2"):
                self.put(name + str(i), (1 + 0.2 * rng.normal(size=self.HIDDEN)).astype(np.float32))
        self.put("gn", np.ones(self.HIDDEN, np.float32))
        # The head's weights are the embedding's, in 8 bits.
        e = lh.DeviceBuffer.from_array(self.embedding)
        self.head = lh.DeviceBuffer(gpu.lh_q8_bytes(self.VOCAB, self.HIDDEN))
        lh.check(gpu.lh_q8_quantize(e.ptr, self.VOCAB, self.HIDDEN, self.head.ptr, None))
        lh.check(gpu.lh_device_synchronize())
        n = self.n
        for name, size in (("x", self.HIDDEN), ("qkv", self.qkv), ("att", self.width),
                           ("o", self.HIDDEN), ("gu", 2 * self.INNER), ("down", self.HIDDEN),
                           ("logits", self.VOCAB), ("scales", 1)):
            self.buffer(name, 4 * n * size)
        self.buffer("codes", n * q8.up16(max(self.width, self.INNER, self.HIDDEN)))
        self.put("start", np.arange(n + 1, dtype=np.int32))
        self.put("cos", self.cos)
        self.put("sin", self.sin)
        self.put("table", self.first_table)
        self.put("length", np.ones(n, np.int32))
        for i in range(2):
            scores = np.full((groups, beams), -np.inf, np.float32)
            scores[:, 0] = 0
            self.put("score%d" % i, scores)
            self.put("done%d" % i, np.zeros(n, np.uint8))
        self.buffer("parent", 4 * n)
        self.buffer("token", 8 * n)
        b = self.batch = lh.PagedBatch()
        b.sequences, b.tokens, b.table_width, b.max_query, b.max_length = n, n, columns, 1, capacity
        b.query_start, b.length, b.table = (self.d[k].ptr for k in ("start", "length", "table"))
        sizes = [gpu.lh_q8_scratch(r, c, n) for layer in self.packed for _, r, c in layer]
        sizes += [gpu.lh_q8_scratch(self.VOCAB, self.HIDDEN, n),
                  gpu.lh_beam_scratch(groups, beams, self.VOCAB, beams),
                  gpu.lh_paged_attention_scratch(ctypes.byref(self.caches[0]), ctypes.byref(b),
                                                 self.HEADS)]
        self.buffer("scratch", max(sizes + [16]))

    def buffer(self, name, nbytes):
        self.d[name] = lh.DeviceBuffer(nbytes)

    def put(self, name, array):
        self.d[name] = lh.DeviceBuffer.from_array(array)

    def product(self, weights, rows, cols, out, stream):
        d = self.d
        lh.check(self.gpu.lh_q8_matvec(weights.ptr, d["codes"].ptr, q8.up16(cols), d["scales"].ptr,
                                       d[out].ptr, rows, rows, cols, self.n, d["scratch"].ptr,
                                       d["scratch"].nbytes, stream))

    def norm(self, add, gamma, stream):
        d, h = self.d, self.HIDDEN
        lh.check(self.gpu.lh_q8_norm(d["x"].ptr, h, add and d[add].ptr, h if add else 0,
                                     d[gamma].ptr, d["x"].ptr if add else None, h if add else 0, h,
                                     self.n, d["codes"].ptr, h, d["scales"].ptr, stream))

    def step(self, stream, turn):
        """x holds the tokens' embeddings, length the lengths with them."""
        g, d, n, w, kv = self.gpu, self.d, self.n, self.width, self.KV * self.DIM
        batch = ctypes.byref(self.batch)
        codes, scales, scratch = d["codes"].ptr, d["scales"].ptr, d["scratch"]
        add = None
        for i, layer in enumerate(self.packed):
            cache = ctypes.byref(self.caches[i])
            self.norm(add, "g1%d" % i, stream)
            self.product(*layer[0], "qkv", stream)
            qkv = d["qkv"].ptr
            lh.check(g.lh_paged_append(cache, batch, self.HEADS, qkv, self.qkv, qkv + 4 * w,
                                       self.qkv, qkv + 4 * (w + kv), self.qkv, d["cos"].ptr,
                                       d["sin"].ptr, self.capacity, None, qkv, self.qkv, stream))
            lh.check(g.lh_paged_attention(cache, batch, self.HEADS, qkv, self.qkv, 0.125,
                                          d["att"].ptr, w, scratch.ptr, scratch.nbytes, stream))
            lh.check(g.lh_q8_rows(d["att"].ptr, w, w, n, codes, q8.up16(w), scales, stream))
            self.product(*layer[1], "o", stream)
            self.norm("o", "g2%d" % i, stream)
            self.product(*layer[2], "gu", stream)
            lh.check(g.lh_q8_silu(d["gu"].ptr, 2 * self.INNER, d["gu"].ptr + 4 * self.INNER,
                                  2 * self.INNER, self.INNER, n, codes, q8.up16(self.INNER),
                                  scales, stream))
            self.product(*layer[3], "down", stream)
            add = "down"
        self.norm(add, "gn", stream)
        self.product(self.head, self.VOCAB, self.HIDDEN, "logits", stream)
        now, then = turn % 2, 1 - turn % 2
        lh.check(g.lh_beam_select(
            d["logits"].ptr, self.VOCAB, self.groups, self.beams, self.VOCAB,
            d["score%d" % now].ptr, d["done%d" % now].ptr, 13, self.beams, d["parent"].ptr,
            d["token"].ptr, d["score%d" % then].ptr, d["done%d" % then].ptr, scratch.ptr,
            scratch.nbytes, stream))
        lh.check(g.lh_beam_reorder(self.caches, self.LAYERS, self.groups, self.beams,
                                   d["parent"].ptr, d["length"].ptr, d["table"].ptr,
                                   d["table"].ptr, self.batch.table_width, stream))

    def feed(self, tokens, length):
        self.d["x"].upload(self.embedding[tokens])
        self.d["length"].upload(np.full(self.n, length, np.int32))

    def cache_rows(self, layer, length):
        """Keys and values of all sequences, [n][length][kv][dim]."""
        start = lh.DeviceBuffer.from_array(np.arange(self.n + 1, dtype=np.int32) * length)
        b = lh.PagedBatch()
        b.sequences, b.tokens, b.table_width = self.n, self.n * length, self.batch.table_width
        b.max_query, b.max_length = length, length
        b.query_start, b.length, b.table = start.ptr, self.d["length"].ptr, self.d["table"].ptr
        kv = self.KV * self.DIM
        out = [lh.DeviceBuffer(4 * b.tokens * kv) for _ in range(2)]
        lh.check(self.gpu.lh_paged_read(ctypes.byref(self.caches[layer]), ctypes.byref(b),
                                        out[0].ptr, kv, out[1].ptr, kv, None))
        lh.check(self.gpu.lh_device_synchronize())
        return [o.download(np.float32).reshape(self.n, length, self.KV, self.DIM) for o in out]


def search_on(search, prompts, steps, step):
    """Prompts token by token through every beam's row (all rows alike), then steps of the
    search by `step`. Yields after each: (turn, length, rows of logits)."""
    tokens = np.repeat(prompts[:, 0], search.beams)
    histories = [[int(t)] for t in tokens]
    turn = 0
    for length in range(1, prompts.shape[1] + steps):
        search.feed(tokens, length)
        step(turn)
        lh.check(search.gpu.lh_device_synchronize())
        logits = search.d["logits"].download(np.float32).reshape(search.n, -1)
        if length < prompts.shape[1]:
            # Still the prompt: every beam goes on as itself, nothing is chosen.
            tokens = np.repeat(prompts[:, length], search.beams)
            for h, t in zip(histories, tokens):
                h.append(int(t))
            scores = np.full((search.groups, search.beams), -np.inf, np.float32)
            scores[:, 0] = 0
            for i in range(2):
                search.d["score%d" % i].upload(scores)
                search.d["done%d" % i].upload(np.zeros(search.n, np.uint8))
            yield turn, length, logits, histories, None
            turn += 1
            continue
        parent = search.d["parent"].download(np.int32)
        token = search.d["token"].download(np.int64)
        score = search.d["score%d" % (1 - turn % 2)].download(np.float32)
        rows = [search.beams * (i // search.beams) + p for i, p in enumerate(parent)]
        tokens = np.where(token < 0, 0, token)   # a finished beam goes on with any token
        yield turn, length, logits, histories, (parent, token, score)
        histories = [histories[r] + [int(t)] for r, t in zip(rows, tokens)]
        turn += 1


@pytest.mark.parametrize("kind", KINDS)
def test_search_follows_its_hypotheses(gpu, kind):
    """Every step's beams hold the caches of their own hypotheses: the first layer's rows, which
    hang on a token and its position alone, bit for bit those that the token was appended
    with; scores are sums along the hypotheses."""
    groups, beams, steps = 2, 4, 45
    prompts = np.random.default_rng(1).integers(20, 700, size=(groups, 30))
    s = Search(gpu, kind, groups, beams, 80, 3)
    given = {}        # (token, position) -> the first layer's cache rows
    sums = None       # of each hypothesis, in 64 bits

    def step(turn):
        s.step(None, turn)

    for turn, length, logits, histories, chosen in search_on(s, prompts, steps, step):
        if chosen is None:
            continue
        parent, token, score = chosen
        assert np.all(parent >= 0)
        rows = np.arange(s.n) // beams * beams + parent
        if sums is None:
            sums = [(0.0, False, 0.0)] * s.n
        following = []
        for i, r in enumerate(rows):
            total, ended, off = sums[r]
            if ended:
                assert token[i] == -1
                following.append((total, True, off))
                continue
            lp, _, _, _, errors = so.logprobs(logits[r], int(token[i]), 1)
            # A choice adds a log probability to an FP32 score and rounds it again.
            off = off + errors[0] + 2.0 ** -23 * (abs(total) + abs(lp))
            following.append((total + lp, bool(token[i] == 13), off))
            assert abs(score[i] - (total + lp)) <= off
        sums = following
        keys, values = s.cache_rows(0, length)
        for i, r in enumerate(rows):
            for at, t in enumerate(histories[r]):
                row = (keys[i, at], values[i, at])
                known = given.setdefault((t, at), row)
                assert np.array_equal(known[0], row[0]) and np.array_equal(known[1], row[1])
        for layer in range(s.LAYERS):
            assert all(np.isfinite(a).all() for a in s.cache_rows(layer, length))
    # Branches were taken: hypotheses of a group that share a part and differ after it.
    assert len(given) > groups * (30 + steps)


@pytest.mark.parametrize("kind", KINDS)
def test_search_of_one_beam_is_greedy(gpu, kind):
    """One beam: the likeliest token each time, and the products' rows do not depend on how many
    tokens there are."""
    prompts = np.random.default_rng(2).integers(20, 700, size=(3, 5))
    s = Search(gpu, kind, 3, 1, 40, 5)
    for _, _, logits, _, chosen in search_on(s, prompts, 20, lambda turn: s.step(None, turn)):
        if chosen is not None:
            live = chosen[1] >= 0
            assert np.array_equal(chosen[1][live], logits.argmax(1)[live])


@pytest.mark.parametrize("kind", KINDS)
def test_captured_search_equals_eager(gpu, kind):
    """Two captured steps (scores from one array to the other and back), replayed in turn,
    with eager work between them, equal eager steps of another copy bit for bit."""
    prompts = np.random.default_rng(4).integers(20, 700, size=(2, 3))
    a, b = (Search(gpu, kind, 2, 3, 40, 7) for _ in range(2))
    graphs = [Graph(lambda stream, t=t: a.step(stream, t)) for t in range(2)]
    first = search_on(a, prompts, 30, lambda turn: graphs[turn % 2].launch())
    second = search_on(b, prompts, 30, lambda turn: b.step(None, turn))
    for got, want in zip(first, second):
        assert np.array_equal(got[2], want[2]), got[0]
        if want[4] is not None:
            for x, y in zip(got[4], want[4]):
                assert np.array_equal(x, y), got[0]
        for layer in range(a.LAYERS):
            for x, y in zip(a.cache_rows(layer, got[1]), b.cache_rows(layer, want[1])):
                assert np.array_equal(x, y), got[0]


def test_rows_and_products_on_two_streams(gpu):
    """Norm, rows and products of two sizes at once, each with buffers of its own."""
    rng = np.random.default_rng(13)
    streams = [gpu.lh_stream_create() for _ in range(2)]
    jobs = []
    for tokens, cols, rows in ((9, 3000, 700), (150, 1200, 900)):
        codes, scales = q8.random_weights(rng, rows, cols)
        x = rng.normal(size=(tokens, cols)).astype(np.float32)
        need = gpu.lh_q8_scratch(rows, cols, tokens)
        d = [lh.DeviceBuffer.from_array(x), lh.DeviceBuffer(tokens * q8.up16(cols)),
             lh.DeviceBuffer(4 * tokens), lh.DeviceBuffer(4 * tokens * rows),
             lh.DeviceBuffer(max(16, need)), q8.pack(gpu, codes, scales)]
        c, s, _ = q8.quantize(x.astype(np.float64))
        jobs.append((d, need, rows, cols, tokens, q8.product(codes, scales, c, s)))
    for _ in range(20):
        for stream, (d, need, rows, cols, tokens, _) in zip(streams, jobs):
            lh.check(gpu.lh_q8_rows(d[0].ptr, cols, cols, tokens, d[1].ptr, q8.up16(cols), d[2].ptr,
                                    stream))
            lh.check(gpu.lh_q8_matvec(d[5].ptr, d[1].ptr, q8.up16(cols), d[2].ptr, d[3].ptr, rows,
                                      rows, cols, tokens, d[4].ptr, need, stream))
    for s in streams:
        lh.check(gpu.lh_stream_synchronize(s))
    for d, _, rows, _, tokens, want in jobs:
        assert np.array_equal(d[3].download(np.float32).reshape(tokens, rows), want)
    for s in streams:
        gpu.lh_stream_destroy(s)
