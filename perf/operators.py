"""Timed workloads of the batched 4-bit serving operators.

What a program that serves several sequences from little memory has the GPU
do besides the forward path of one sequence:

- products with 4-bit weights and group scales (lh_q4_matvec): one decode
  token, a decode batch, a short prompt;
- keys and values appended to a paged cache, rotated on the way, with the
  queries (lh_paged_append), and the rows read back (lh_paged_read);
- attention over the paged cache, FP16 rows or 4-bit codes
  (lh_paged_attention): one long sequence, ragged decode batches, a prompt's
  chunk after a long prefix;
- log probabilities of given tokens with the entropy and the top alternatives
  of logit rows (lh_logprobs): one served token, a scored prompt, a
  vocabulary of another size of which a mask leaves a part.

Activations and logits are FP32, as everywhere in this framework. The plain
forms compute in 32 bits; the rotation, the 4-bit codes of the cache and the
sums over a vocabulary in 64.
"""
import ctypes
import math

import torch

own = False

HEADS, KV_HEADS, DIM = 32, 8, 128   # the model's attention


# ---- cases ------------------------------------------------------------------

def _q4(name, rows, cols, group, tokens):
    return {"name": name, "op": "q4", "rows": rows, "cols": cols, "group": group,
            "tokens": tokens}


def _logprobs(name, rows, vocab, stride, top, masked):
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "stride": stride,
            "top": top, "masked": masked}


def _paged(name, op, kind, sequences, shortest, longest, query, page, heads=HEADS,
           kv_heads=KV_HEADS, dim=DIM):
    return {"name": name, "op": op, "kind": kind, "sequences": sequences, "shortest": shortest,
            "longest": longest, "query": query, "page": page, "heads": heads,
            "kv_heads": kv_heads, "dim": dim}


def listed():
    return [
        # One generated token through the o projection.
        _q4("q4_o_1", 3072, 4096, 128, 1),
        # gate and up of a decode batch, the finest groups.
        _q4("q4_gateup_8", 18432, 3072, 32, 8),
        # A short prompt through the down projection, a ragged number of tokens.
        _q4("q4_down_45", 3072, 9216, 64, 45),
        # One served token: its log probability and twenty alternatives.
        _logprobs("logprobs_1", 1, 131072, 131072, 20, False),
        # A scored prompt chunk.
        _logprobs("logprobs_256", 256, 131072, 131072, 5, False),
        # Another vocabulary in padded rows, part of it masked, the most alternatives.
        _logprobs("logprobs_37", 37, 50021, 50176, 64, True),
        # One decode step of a batch into the 4-bit cache.
        _paged("append_q4_48", "append", "q4", 48, 65, 4352, 1, 64),
        # Prompt chunks of several sequences into FP16 pages.
        _paged("append_f16_4x256", "append", "f16", 4, 300, 4352, 256, 32),
        # One sequence deep in a long session.
        _paged("attention_q4_1", "attention", "q4", 1, 15999, 15999, 1, 64),
        # A ragged decode batch over FP16 pages.
        _paged("attention_f16_32", "attention", "f16", 32, 37, 4352, 1, 64),
        # A prompt's chunk after a long prefix.
        _paged("attention_q4_prompt", "attention", "q4", 1, 4352, 4352, 256, 128),
        # A large decode batch of long sequences.
        _paged("attention_q4_64", "attention", "q4", 64, 1003, 17920, 1, 64),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    case = _draw(rng)
    del case["name"]
    return case


def _draw(rng):
    which = rng.random()
    if which < 0.27:
        group = rng.choice((32, 64, 128))
        tokens = _log_int(rng, 1, 64)
        rows = _log_int(rng, 64, 18432)
        cols = group * _log_int(rng, 1, 16384 // group)
        # No dearer than the listed gate and up.
        while rows * cols > 18432 * 3072:
            rows //= 2
        return _q4(None, rows, cols, group, tokens)
    if which < 0.5:
        vocab = rng.choice((131072, _log_int(rng, 1000, 151936), _log_int(rng, 1000, 151936)))
        rows = _log_int(rng, 1, 256)
        while rows * vocab > 256 * 131072:
            rows //= 2
        return _logprobs(None, rows, vocab, vocab + rng.choice((0, 0, 3, 64)),
                         rng.choice((1, 5, 20, 64)), rng.random() < 0.3)
    heads, kv_heads, dim = rng.choice(((32, 8, 128), (32, 8, 128), (16, 16, 64), (24, 4, 128),
                                       (14, 2, 64), (8, 1, 128)))
    kind, page = rng.choice(("q4", "f16")), rng.choice((32, 64, 128, 256))
    if which < 0.68:
        if rng.random() < 0.5:
            sequences, query = _log_int(rng, 1, 64), 1
        else:
            sequences, query = _log_int(rng, 1, 8), _log_int(rng, 2, 256)
        op = "append"
    else:
        op = "attention"
        if rng.random() < 0.65:
            sequences, query = _log_int(rng, 1, 64), 1
        else:
            sequences, query = _log_int(rng, 1, 4), _log_int(rng, 2, 96)
    longest = _log_int(rng, max(16, query), 17920 if query == 1 else 4352)
    # No dearer than the listed large batch.
    row = 2 * kv_heads * (dim // 2 + 4 if kind == "q4" else 2 * dim)
    while query == 1 and sequences * longest * row > 400e6:
        longest //= 2
    return _paged(None, op, kind, sequences, _log_int(rng, max(1, min(query, longest)), longest),
                  longest, query, page, heads, kv_heads, dim)


def _lengths(case):
    """Lengths after the call, from the longest down to the shortest, and the
    tokens that each sequence brings."""
    n = case["sequences"]
    ratio = case["shortest"] / case["longest"]
    lengths = [max(1, int(round(case["longest"] * ratio ** (i / max(1, n - 1)))))
               for i in range(n)]
    if case["query"] == 1:
        return lengths, [1] * n
    counts = [max(1, (case["query"] * (n - i)) // n) for i in range(n)]
    return lengths, [min(c, l) for c, l in zip(counts, lengths)]


# ---- inputs -----------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _q4_inputs(case, seed):
    """Codes of normally distributed weights (two to a byte, the even column in
    the low bits) and BF16 scales of about 0.01."""
    g = _generator(seed)
    rows, cols = case["rows"], case["cols"]
    codes = torch.empty(rows, cols // 2, dtype=torch.uint8, device="cuda")
    for r in range(0, rows, 4096):
        n = min(4096, rows - r)
        c = _normal(g, n, cols).mul_(2.4).round_().clamp_(-8, 7).add_(8).to(torch.uint8)
        codes[r:r + n] = c[:, 0::2] | (c[:, 1::2] << 4)
    scales = (0.01 * torch.exp(0.3 * _normal(g, rows, cols // case["group"]))).bfloat16()
    spread = torch.exp(0.5 * _normal(g, cols))
    return codes, scales, _normal(g, case["tokens"], cols) * spread


def _logit_inputs(case, seed):
    """Logits with the spread of a language model's, some rows almost certain
    of one token; the given tokens are likely ones or any."""
    g = _generator(seed)
    rows, vocab = case["rows"], case["vocab"]
    buffer = torch.zeros(rows, case["stride"], device="cuda")
    x = buffer[:, :vocab]
    x.copy_(2.5 * _normal(g, rows, vocab))
    tokens = torch.randint(vocab, (rows,), device="cuda", generator=g)
    sure = torch.rand(rows, device="cuda", generator=g) * 25
    likely = torch.randint(vocab, (rows,), device="cuda", generator=g)
    x.scatter_add_(1, likely[:, None], sure[:, None])
    tokens = torch.where(torch.arange(rows, device="cuda") % 2 == 0, likely, tokens)
    if case["masked"]:
        keep = torch.rand(vocab, device="cuda", generator=g) < 0.4
        keep[tokens] = True
        x.masked_fill_(~keep, -math.inf)
    return x, tokens


class _Batch:
    """The sequences of a call: pages dealt in random order."""

    def __init__(self, case, seed):
        g = _generator(seed)
        self.lengths, self.counts = _lengths(case)
        page = case["page"]
        self.need = [(n + page - 1) // page for n in self.lengths]
        self.width = max(self.need)
        self.pages = sum(self.need) + 3
        order = torch.randperm(self.pages, device="cuda", generator=g).int()
        self.table = torch.full((len(self.lengths), self.width), -1, dtype=torch.int32,
                                device="cuda")
        at = 0
        for i, n in enumerate(self.need):
            self.table[i, :n] = order[at:at + n]
            at += n
        starts = [0]
        for c in self.counts:
            starts.append(starts[-1] + c)
        self.starts = starts
        self.tokens = starts[-1]
        self.query_start = torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.length = torch.tensor(self.lengths, dtype=torch.int32, device="cuda")

    def positions(self):
        return torch.cat([torch.arange(l - c, l) for l, c in zip(self.lengths, self.counts)]
                         ).cuda()


def _rotation_table(case):
    """cos and sin rows of the positions, [longest][dim], the halves alike."""
    half = case["dim"] // 2
    inverse = 1e6 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    angle = torch.arange(case["longest"], dtype=torch.float64, device="cuda")[:, None] * inverse
    angle = torch.cat([angle, angle], dim=1)
    return angle.cos().float(), angle.sin().float()


def _append_inputs(case, seed, tokens):
    """Rows of a fused q|k|v projection; some channels of k and v larger."""
    g = _generator(seed + 1)
    q, kv = case["heads"] * case["dim"], case["kv_heads"] * case["dim"]
    x = _normal(g, tokens, q + 2 * kv) * torch.exp(0.5 * _normal(g, q + 2 * kv))
    cos, sin = _rotation_table(case)
    factor = 1 + 0.1 * torch.log1p(torch.arange(case["longest"], device="cuda") // 16384)
    return x, cos, sin, factor


def _history(case, seed, index, length):
    """A sequence's keys (rotated already) and values, [length][kv_heads][dim]."""
    g = _generator(seed + 2 + index)
    out = []
    for spread in (0.5, 0.3):
        s = torch.exp(spread * _normal(g, case["kv_heads"], case["dim"]))
        out.append(_normal(g, length, case["kv_heads"], case["dim"]) * s)
    return out


# ---- a program's state ------------------------------------------------------

def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _scratch(nbytes):
    return torch.empty(max(16, int(nbytes)), dtype=torch.uint8, device="cuda")


class _Q4:
    def __init__(self, case, seed):
        self.case = case
        self.codes, self.scales, self.x = _q4_inputs(case, seed)
        if own:
            import lunelette_amd as lh
            self.lh, self.lib = lh, lh.lib()
            rows, cols, group = case["rows"], case["cols"], case["group"]
            # A program lays its weights out once, when it loads them.
            self.packed = _scratch(self.lib.lh_q4_bytes(rows, cols, group))
            lh.check(self.lib.lh_q4_pack(self.codes.data_ptr(), self.scales.data_ptr(), rows,
                                         cols, group, self.packed.data_ptr(), _stream()))
            self.scratch = _scratch(self.lib.lh_q4_scratch(cols, case["tokens"]))
            self.y = torch.empty(case["tokens"], rows, device="cuda")

    def run(self):
        c = self.case
        if not own:
            low, high = self.codes & 15, self.codes >> 4
            w = torch.stack([low, high], dim=2).view(c["rows"], -1, c["group"]).float() - 8
            w = w * self.scales.float()[:, :, None]
            return self.x @ w.view(c["rows"], c["cols"]).t()
        self.lh.check(self.lib.lh_q4_matvec(
            self.packed.data_ptr(), self.x.data_ptr(), c["cols"], self.y.data_ptr(), c["rows"],
            c["rows"], c["cols"], c["group"], c["tokens"], self.scratch.data_ptr(),
            self.scratch.numel(), _stream()))
        return self.y


class _Logprobs:
    def __init__(self, case, seed):
        self.case = case
        self.x, self.tokens = _logit_inputs(case, seed)
        if own:
            import lunelette_amd as lh
            self.lh, self.lib = lh, lh.lib()
            rows, top = case["rows"], case["top"]
            self.scratch = _scratch(self.lib.lh_logprobs_scratch(rows, case["vocab"], top))
            self.logprob = torch.empty(rows, device="cuda")
            self.entropy = torch.empty(rows, device="cuda")
            self.top_ids = torch.empty(rows, top, dtype=torch.int64, device="cuda")
            self.top = torch.empty(rows, top, device="cuda")

    def run(self):
        c = self.case
        if not own:
            shifted = self.x - self.x.amax(1, keepdim=True)
            e = torch.exp(shifted)
            z = e.sum(1, dtype=torch.float64)
            log_z = torch.log(z)
            weighted = torch.where(e > 0, e * shifted, 0.0).sum(1, dtype=torch.float64)
            given = shifted.gather(1, self.tokens[:, None])[:, 0].double() - log_z
            ids = torch.sort(self.x, dim=1, descending=True, stable=True).indices[:, :c["top"]]
            top = shifted.gather(1, ids).double() - log_z[:, None]
            return {"logprob": given.float(), "entropy": (log_z - weighted / z).float(),
                    "top_ids": ids, "top": top.float()}
        self.lh.check(self.lib.lh_logprobs(
            self.x.data_ptr(), c["stride"], c["rows"], c["vocab"], self.tokens.data_ptr(),
            self.logprob.data_ptr(), self.entropy.data_ptr(), c["top"], self.top_ids.data_ptr(),
            self.top.data_ptr(), self.scratch.data_ptr(), self.scratch.numel(), _stream()))
        return {"logprob": self.logprob, "entropy": self.entropy, "top_ids": self.top_ids,
                "top": self.top}


def _quantize(rows):
    """4-bit codes of 64-bit vectors [..][dim] with a BF16 scale and zero each."""
    z = rows.amin(-1, keepdim=True).float().bfloat16().double()
    s = ((rows.amax(-1, keepdim=True) - z) / 15).float().bfloat16().double().clamp(min=0)
    code = torch.round((rows - z) / s).clamp(0, 15)
    code = torch.where(s > 0, code, 0.0).to(torch.uint8)
    return code, torch.cat([s, z], dim=-1).bfloat16()


def _dequantize(code, sz):
    sz = sz.float()
    return code.float() * sz[..., :1] + sz[..., 1:]


class _PlainCache:
    """Pages of [page][kv_heads][dim] rows: half values, or codes (two to a
    byte) with a scale and a zero."""

    def __init__(self, case, pages):
        self.q4, self.page = case["kind"] == "q4", case["page"]
        shape = (2, pages, case["page"], case["kv_heads"])
        dim = case["dim"]
        if self.q4:
            self.codes = torch.zeros(*shape, dim // 2, dtype=torch.uint8, device="cuda")
            self.sz = torch.zeros(*shape, 2, dtype=torch.bfloat16, device="cuda")
        else:
            self.rows = torch.zeros(*shape, dim, dtype=torch.half, device="cuda")

    def put(self, which, page, slot, rows):
        """Rows [n][kv_heads][dim] in 64 bits to slots of pages."""
        if self.q4:
            code, sz = _quantize(rows)
            self.codes[which, page, slot] = code[..., 0::2] | (code[..., 1::2] << 4)
            self.sz[which, page, slot] = sz
        else:
            self.rows[which, page, slot] = rows.float().half()

    def get(self, which, page, slot=None):
        at = (which, page) if slot is None else (which, page, slot)
        if not self.q4:
            return self.rows[at].float()
        packed = self.codes[at]
        code = torch.stack([packed & 15, packed >> 4], dim=-1).flatten(-2)
        return _dequantize(code, self.sz[at])


class _Paged:
    def __init__(self, case, seed):
        self.case = case
        self.batch = b = _Batch(case, seed)
        if own:
            self._own_cache()
        else:
            self.cache = _PlainCache(case, b.pages)
        tokens, width = b.tokens, case["heads"] * case["dim"]
        if case["op"] == "append":
            self.x, self.cos, self.sin, self.factor = _append_inputs(case, seed, tokens)
            pos = b.positions()
            owner = torch.repeat_interleave(torch.arange(len(b.counts), device="cuda"),
                                            torch.tensor(b.counts, device="cuda"))
            self.position, self.slot = pos, pos % case["page"]
            self.page_of = b.table[owner, pos // case["page"]].long()
            if own:
                kv = case["kv_heads"] * case["dim"]
                self.q_out = torch.empty(tokens, width, device="cuda")
                self.keys = torch.empty(tokens, kv, device="cuda")
                self.values = torch.empty(tokens, kv, device="cuda")
            return
        self.q = _normal(_generator(seed + 1), tokens, width)
        self.scale = 1 / math.sqrt(case["dim"])
        for i, length in enumerate(b.lengths):
            k, v = _history(case, seed, i, length)
            if own:
                self._own_fill(i, length, k, v)
            else:
                p = torch.arange(length, device="cuda")
                page, slot = b.table[i].long()[p // case["page"]], p % case["page"]
                self.cache.put(0, page, slot, k.double())
                self.cache.put(1, page, slot, v.double())
        if own:
            self.scratch = _scratch(self.lib.lh_paged_attention_scratch(
                ctypes.byref(self.cache), ctypes.byref(self.own_batch), case["heads"]))
            self.out = torch.empty(tokens, width, device="cuda")

    # The framework's cache and batch.

    def _own_batch(self, start, length, table, sequences, tokens, query, longest):
        b = self.lh.PagedBatch()
        b.sequences, b.tokens, b.table_width = sequences, tokens, table.shape[-1]
        b.max_query, b.max_length = query, longest
        b.query_start, b.length, b.table = start.data_ptr(), length.data_ptr(), table.data_ptr()
        return b

    def _own_cache(self):
        import lunelette_amd as lh
        self.lh, self.lib = lh, lh.lib()
        case, b = self.case, self.batch
        c = self.cache = lh.PagedCache()
        c.kind = lh.CACHE_Q4 if case["kind"] == "q4" else lh.CACHE_F16
        c.kv_heads, c.head_dim = case["kv_heads"], case["dim"]
        c.page_size, c.pages = case["page"], b.pages
        self.memory = torch.zeros(self.lib.lh_paged_cache_bytes(ctypes.byref(c)),
                                  dtype=torch.uint8, device="cuda")
        c.data = self.memory.data_ptr()
        self.own_batch = self._own_batch(b.query_start, b.length, b.table, len(b.lengths),
                                         b.tokens, max(b.counts), max(b.lengths))

    def _own_fill(self, index, length, k, v):
        """Earlier calls brought this sequence's rows, rotated already."""
        case = self.case
        start = torch.tensor([0, length], dtype=torch.int32, device="cuda")
        total = torch.tensor([length], dtype=torch.int32, device="cuda")
        one = self._own_batch(start, total, self.batch.table[index], 1, length, length, length)
        kv = case["kv_heads"] * case["dim"]
        self.lh.check(self.lib.lh_paged_append(
            ctypes.byref(self.cache), ctypes.byref(one), 0, None, 0, k.data_ptr(), kv,
            v.data_ptr(), kv, None, None, 0, None, None, 0, _stream()))

    def run(self):
        return self._append() if self.case["op"] == "append" else self._attention()

    def _append(self):
        case = self.case
        heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
        at = (0, heads * dim, (heads + kv_heads) * dim, (heads + 2 * kv_heads) * dim)
        if own:
            row, x = at[3], self.x.data_ptr()
            self.lh.check(self.lib.lh_paged_append(
                ctypes.byref(self.cache), ctypes.byref(self.own_batch), heads, x, row,
                x + 4 * at[1], row, x + 4 * at[2], row, self.cos.data_ptr(),
                self.sin.data_ptr(), case["longest"], self.factor.data_ptr(),
                self.q_out.data_ptr(), heads * dim, _stream()))
            self.lh.check(self.lib.lh_paged_read(
                ctypes.byref(self.cache), ctypes.byref(self.own_batch), self.keys.data_ptr(),
                kv_heads * dim, self.values.data_ptr(), kv_heads * dim, _stream()))
            return {"q": self.q_out, "keys": self.keys, "values": self.values}
        n = self.x.shape[0]
        q, k, v = (self.x[:, at[i]:at[i + 1]].reshape(n, -1, dim).double() for i in range(3))
        cos = self.cos[self.position].double()[:, None]
        sin = self.sin[self.position].double()[:, None]

        def rotate(u):
            half = dim // 2
            return u * cos + torch.cat([-u[..., half:], u[..., :half]], dim=-1) * sin

        q = rotate(q) * self.factor[self.position].double()[:, None, None]
        self.cache.put(0, self.page_of, self.slot, rotate(k))
        self.cache.put(1, self.page_of, self.slot, v)
        return {"q": q.float().view(n, -1),
                "keys": self.cache.get(0, self.page_of, self.slot).view(n, -1),
                "values": self.cache.get(1, self.page_of, self.slot).view(n, -1)}

    def _attention(self):
        case, b = self.case, self.batch
        if own:
            width = case["heads"] * case["dim"]
            self.lh.check(self.lib.lh_paged_attention(
                ctypes.byref(self.cache), ctypes.byref(self.own_batch), case["heads"],
                self.q.data_ptr(), width, self.scale, self.out.data_ptr(), width,
                self.scratch.data_ptr(), self.scratch.numel(), _stream()))
            return self.out
        kv_heads, dim, group = case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"]
        out = torch.empty_like(self.q)
        for i, (length, count) in enumerate(zip(b.lengths, b.counts)):
            page = b.table[i, :b.need[i]].long()
            k = self.cache.get(0, page).flatten(0, 1)[:length].permute(1, 2, 0).contiguous()
            v = self.cache.get(1, page).flatten(0, 1)[:length].permute(1, 0, 2).contiguous()
            rows = slice(b.starts[i], b.starts[i + 1])
            q = self.q[rows].view(count, kv_heads, group, dim).permute(1, 0, 2, 3)
            s = torch.matmul(q.reshape(kv_heads, count * group, dim), k) * self.scale
            s = s.view(kv_heads, count, group, length)
            last = torch.arange(length - count, length, device="cuda")
            hidden = torch.arange(length, device="cuda")[None, :] > last[:, None]
            s = s.masked_fill(hidden[None, :, None], -math.inf)
            e = torch.exp(s - s.amax(-1, keepdim=True))
            p = (e / e.sum(-1, keepdim=True)).view(kv_heads, count * group, length)
            o = torch.matmul(p, v).view(kv_heads, count, group, dim)
            out[rows] = o.permute(1, 0, 2, 3).reshape(count, -1)
        return out


def prepare(case, seed):
    kinds = {"q4": _Q4, "logprobs": _Logprobs, "append": _Paged, "attention": _Paged}
    return kinds[case["op"]](case, int(seed))


def run(state):
    return state.run()


# ---- what a pass cannot do without --------------------------------------------

def work(case):
    if case["op"] == "q4":
        rows, cols, tokens = case["rows"], case["cols"], case["tokens"]
        return {"bytes": rows * cols // 2 + 2 * rows * (cols // case["group"]) +
                4 * tokens * (rows + cols), "flops": 2 * rows * cols * tokens}
    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        # A subtraction, an exponential, two sums and a product for each logit.
        return {"bytes": 4 * rows * vocab + rows * (16 + 12 * case["top"]),
                "flops": 5 * rows * vocab}
    lengths, counts = _lengths(case)
    tokens, q = sum(counts), case["heads"] * case["dim"]
    kv = case["kv_heads"] * case["dim"]
    vector = case["dim"] // 2 + 4 if case["kind"] == "q4" else 2 * case["dim"]
    row = 2 * case["kv_heads"] * vector          # a position's keys and values
    if case["op"] == "append":
        # Rows of q, k, v and of the rotation in; q and the cache out; the cache
        # in and its values out.
        return {"bytes": tokens * (4 * (q + 2 * kv) + 8 * case["dim"] + 4 * q + 2 * row + 8 * kv),
                "flops": tokens * (3 * q + 3 * kv + 4 * kv)}
    pairs = sum(c * l - c * (c - 1) // 2 for l, c in zip(lengths, counts))
    return {"bytes": row * sum(lengths) + 8 * tokens * q, "flops": 4 * q * pairs}


# ---- the same in 64 bits ------------------------------------------------------

def exact(case, seed):
    seed = int(seed)
    return {"q4": _exact_q4, "logprobs": _exact_logprobs, "append": _exact_append,
            "attention": _exact_attention}[case["op"]](case, seed)


def _exact_q4(case, seed):
    codes, scales, x = _q4_inputs(case, seed)
    out = torch.zeros(case["tokens"], case["rows"], dtype=torch.float64, device="cuda")
    x, s, group = x.double(), scales.double(), case["group"]
    for j in range(case["cols"] // group):
        block = codes[:, j * group // 2:(j + 1) * group // 2]
        even, odd = (block % 16).double() - 8, (block // 16).double() - 8
        part = x[:, j * group:(j + 1) * group]
        out += (part[:, 0::2] @ even.t() + part[:, 1::2] @ odd.t()) * s[:, j]
    return out


def _exact_logprobs(case, seed):
    x, tokens = _logit_inputs(case, seed)
    n, top = case["rows"], case["top"]
    out = {"logprob": [], "entropy": [], "top_ids": [], "top": []}
    for r in range(n):
        row = x[r].double()
        p = row - torch.logsumexp(row, 0)
        live = p[p > -math.inf]
        out["logprob"].append(p[tokens[r]])
        out["entropy"].append(-(live.exp() * live).sum())
        # Of equal logits the lowest ids: the k-th largest value is a threshold,
        # and of those that equal it the first fill the list.
        limit = torch.topk(row, top).values[-1]
        above = (row > limit).nonzero()[:, 0]
        equal = (row == limit).nonzero()[:, 0][:top - len(above)]
        above = above[torch.argsort(row[above], descending=True, stable=True)]
        ids = torch.cat([above, equal])
        out["top_ids"].append(ids)
        out["top"].append(p[ids])
    return {k: torch.stack(v) for k, v in out.items()}


def _exact_cache(rows, kind):
    """The values that a cache of this kind holds of rows [..][dim]."""
    if kind == "f16":
        return rows.float().half().double()
    low = rows.min(-1).values.float().bfloat16().double().unsqueeze(-1)
    high = rows.max(-1).values.unsqueeze(-1)
    step = ((high - low) / 15).float().bfloat16().double()
    steps = ((rows - low) / step).round().clamp(0, 15)
    return low + step * steps


def _exact_append(case, seed):
    b = _Batch(case, seed)
    x, cos, sin, factor = _append_inputs(case, seed, b.tokens)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    half = dim // 2
    pos = b.positions()
    x = x.double().view(b.tokens, heads + 2 * kv_heads, dim)
    c, s = cos.double()[pos][:, None, :half], sin.double()[pos][:, None, :half]
    turned = torch.empty_like(x[:, :heads + kv_heads])
    first, second = x[:, :heads + kv_heads, :half], x[:, :heads + kv_heads, half:]
    turned[..., :half] = first * c - second * s
    turned[..., half:] = second * c + first * s
    q = turned[:, :heads] * factor.double()[pos][:, None, None]
    return {"q": q.flatten(1), "keys": _exact_cache(turned[:, heads:], case["kind"]).flatten(1),
            "values": _exact_cache(x[:, heads + kv_heads:], case["kind"]).flatten(1)}


def _exact_attention(case, seed):
    b = _Batch(case, seed)
    kv_heads, dim = case["kv_heads"], case["dim"]
    group = case["heads"] // kv_heads
    q = _normal(_generator(seed + 1), b.tokens, case["heads"] * dim).double()
    q = q.view(b.tokens, case["heads"], dim)
    out = torch.empty_like(q)
    for i, (length, count) in enumerate(zip(b.lengths, b.counts)):
        k, v = (_exact_cache(t.double(), case["kind"]) for t in _history(case, seed, i, length))
        seen = torch.arange(length - count, length, device="cuda")
        visible = torch.arange(length, device="cuda")[None, :] <= seen[:, None]
        for h in range(case["heads"]):
            s = q[b.starts[i]:b.starts[i + 1], h] @ k[:, h // group].t() / math.sqrt(dim)
            p = torch.softmax(s.masked_fill(~visible, -math.inf), dim=1)
            out[b.starts[i]:b.starts[i + 1], h] = p @ v[:, h // group]
    return out.view(b.tokens, -1)
