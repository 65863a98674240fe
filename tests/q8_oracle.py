"""The 8-bit and beam search operators (include/lunelette_serving.h) in 64 bits, from
their definitions, and device helpers for their tests."""
import numpy as np

import lunelette_amd as lh

import serving_oracle as so


def up16(n):
    return (n + 15) // 16 * 16


# ---- 8-bit rows ----

def quantize(v):
    """(codes, scales) of 64-bit rows v [tokens][width] that may hold Inf and NaN, and
    where a code lies so near a border that the last bits of v decide."""
    with np.errstate(all="ignore"):
        scale = (np.abs(v).max(1) / 127).astype(np.float32)
        bad = ~np.isfinite(v).all(1) | ~np.isfinite(scale)
        quotient = v / scale.astype(np.float64)[:, None]
        code = np.rint(np.clip(quotient, -127, 127))
        near = np.abs(np.abs(quotient - np.floor(quotient)) - 0.5) < 1e-9
    none = bad | ~(scale > 0)
    code[none] = 0
    near[none] = False
    return code.astype(np.int8), np.where(bad, np.float32(np.nan), scale), near


def norm(x, add, gamma):
    """(h, v) of lh_q8_norm."""
    with np.errstate(all="ignore"):
        h = x if add is None else x + add
        wide = h.astype(np.float64)
        mean = (wide * wide).sum(1, keepdims=True) / h.shape[1]
        return h, gamma.astype(np.float64) * (wide / np.sqrt(mean + 1e-5))


def silu(gate, up):
    g = gate.astype(np.float64)
    with np.errstate(all="ignore"):
        return g / (1 + np.exp(-g)) * up.astype(np.float64)


def check_rows(codes, scales, v):
    """Codes and scales against values v. The 64-bit values may differ in their last
    bits, which can turn a scale whose quotient lies on a border of FP32, or a code
    that does: by one step then."""
    want, scale, near = quantize(v)
    assert np.array_equal(np.isnan(scales), np.isnan(scale))
    fine = ~np.isnan(scale)
    assert np.all(np.abs(scales[fine].view(np.int32) - scale[fine].view(np.int32)) <= 1)
    assert np.all(np.abs(codes.astype(int) - want) <= near.astype(int))
    # That is the exception: no row here is made of borders.
    assert near.mean() < 0.01


# ---- 8-bit products ----

def product(codes, scales, x, x_scales):
    """y as the header writes it: exact sums, then three FP32 roundings."""
    sums = np.rint(x.astype(np.float64) @ codes.astype(np.float64).T)   # exact below 2^53
    with np.errstate(all="ignore"):
        return x_scales[:, None] * (scales[None] * sums.astype(np.float32))


def pack(gpu, codes, scales):
    rows, cols = codes.shape
    packed = lh.DeviceBuffer(gpu.lh_q8_bytes(rows, cols))
    lh.check(gpu.lh_memset_device(packed.ptr, 0xff, packed.nbytes))
    c, s = lh.DeviceBuffer.from_array(codes), lh.DeviceBuffer.from_array(scales)
    lh.check(gpu.lh_q8_pack(c.ptr, s.ptr, rows, cols, packed.ptr, None))
    lh.check(gpu.lh_device_synchronize())
    return packed


def matvec(gpu, packed, x, x_scales, rows, x_pad=0, y_pad=0, y_offset=0, stream=None):
    """y [tokens][rows] of codes x [tokens][cols]: rows of x padded with any codes, the
    last one ending on its last 16-byte word, rows of y padded and checked."""
    tokens, cols = x.shape
    xs, ys = up16(cols) + 16 * x_pad, rows + y_pad
    buf = np.full((tokens, xs), 0x55, np.int8)
    buf[:, :cols] = x
    d_x = lh.DeviceBuffer.from_array(buf.reshape(-1)[:(tokens - 1) * xs + up16(cols)])
    d_s = lh.DeviceBuffer.from_array(x_scales)
    d_y = lh.DeviceBuffer.from_array(np.full(y_offset + tokens * ys + 4, 7.25, np.float32))
    need = gpu.lh_q8_scratch(rows, cols, tokens)
    scratch = lh.DeviceBuffer(max(16, need))
    lh.check(gpu.lh_memset_device(scratch.ptr, 0xff, scratch.nbytes))
    lh.check(gpu.lh_q8_matvec(packed.ptr, d_x.ptr, xs, d_s.ptr, d_y.ptr + 4 * y_offset, ys, rows,
                              cols, tokens, scratch.ptr, need, stream))
    lh.check(gpu.lh_device_synchronize())
    y = d_y.download(np.float32)
    assert np.all(y[:y_offset] == 7.25) and np.all(y[y_offset + tokens * ys:] == 7.25)
    y = y[y_offset:y_offset + tokens * ys].reshape(tokens, ys)
    assert np.all(y[:, rows:] == 7.25), "wrote between the rows"
    return y[:, :rows]


def random_weights(rng, rows, cols):
    codes = rng.integers(-128, 128, size=(rows, cols), dtype=np.int8)
    return codes, (rng.uniform(0.5, 2, size=rows) * 1e-3).astype(np.float32)


# ---- beam search ----

def select(logits, scores, done, stop, keep, groups, beams):
    """(parent, token, score, done, allowed error of the scores, whether a place is decided)
    of lh_beam_select, in 64 bits. Candidates of two beams whose scores are nearer than
    twice the errors of both may change places: their places are not decided, and
    their scores may be off by that distance too."""
    parent = np.full((groups, keep), -1, np.int32)
    token = np.full((groups, keep), -1, np.int64)
    score = np.full((groups, keep), -np.inf)
    ended = np.zeros((groups, keep), np.uint8)
    off, decided = np.zeros((groups, keep)), np.ones((groups, keep), bool)
    for g in range(groups):
        found = []   # score, beam, place in its row, token, error
        bad = False
        for b in range(beams):
            r = g * beams + b
            s = float(scores[r])
            bad |= np.isnan(s) or s == np.inf
            if done[r]:
                if s > -np.inf:
                    found.append((s, b, 0, -1, 0.0))
                continue
            if s == -np.inf:
                continue
            _, _, ids, lp, errors = so.logprobs(logits[r], -1, keep)
            bad |= bool(np.isnan(lp).any())
            found += [(s + v, b, i, int(t), float(e)) for i, (t, v, e) in
                      enumerate(zip(ids, lp, errors[2])) if t >= 0]
        if bad:
            score[g] = np.nan
            continue
        found.sort(key=lambda f: (-f[0], f[1], f[2]))
        for k, f in enumerate(found[:keep]):
            score[g, k], parent[g, k], token[g, k] = f[0], f[1], f[3]
            off[g, k] = f[4] + 2.0 ** -23 * abs(f[0])
            ended[g, k] = done[g * beams + f[1]] or (f[3] >= 0 and f[3] == stop)
        for k, (f, other) in enumerate(zip(found[:keep], found[1:])):
            distance = f[0] - other[0]
            if other[1] != f[1] and 0 < distance < 2 * (f[4] + other[4]):
                for place in (k, k + 1):
                    if place < keep:
                        decided[g, place] = False
                        off[g, place] += distance
    return parent, token, score, ended, off, decided


def reorder(parent, lengths, table, page):
    """(new table, [(from, to)] pages) of lh_beam_reorder."""
    groups, beams = parent.shape
    new, copies = table.copy(), []
    for g in range(groups):
        rows = slice(g * beams, (g + 1) * beams)
        old = table[rows]
        length = max(0, int(lengths[g * beams]))
        column = length // page
        valid = [int(p) if 0 <= p < beams else -1 for p in parent[g]]
        free = [b for b in range(beams) if b not in valid]
        taken = set()
        for k, p in enumerate(valid):
            if p >= 0 and p not in taken:
                taken.add(p)
                owner = p
            else:
                owner = free.pop(0)
                if p >= 0 and length % page and column < table.shape[1]:
                    copies.append((int(old[p][column]), int(old[owner][column])))
            source = owner if p < 0 else p
            new[rows.start + k, :column] = old[source][:column]
            new[rows.start + k, column:] = old[owner][column:]
    return new, copies
