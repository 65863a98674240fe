"""Timed workloads of 8-bit layers and beam search for batched serving.

What a program that serves many sequences or beams at a time has the GPU do
besides the paged cache, in layers of 8-bit weights and activations:

- products of 8-bit rows with 8-bit weights, a scale for each token and for
  each output channel (lh_q8_matvec): one decode token, a few requests' beams,
  prompts of many tokens;
- the rows that they take: RMSNorm of a residual sum (lh_q8_norm), SwiGLU and
  plain rows (lh_q8_silu, lh_q8_rows), rounded to 8 bits with a scale each;
- the choice of the next hypotheses over beams and vocabulary (lh_beam_select);
- the paged caches' reordering after it (lh_beam_reorder).

Activations, logits and scores are FP32, as everywhere in this framework. The
plain forms compute in 32 bits; values that are rounded to codes, sums over a
vocabulary and the scores that are compared in 64. Codes are returned as the
values that they stand for.
"""
import ctypes
import math

import torch

own = False

EPSILON = 1e-5   # of the RMSNorm, as in lh_rmsnorm


# ---- cases ------------------------------------------------------------------

def _product(name, rows, cols, tokens):
    return {"name": name, "op": "product", "rows": rows, "cols": cols, "tokens": tokens}


def _rows(name, op, width, tokens, pad=0):
    """op: "norm" (with the residual's addition), "first_norm" (without),
    "silu" or "rows". pad: elements between the FP32 rows."""
    return {"name": name, "op": op, "width": width, "tokens": tokens, "pad": pad}


def _select(name, groups, beams, vocab, stride, keep, first=False, done=0.0, masked=False):
    """first: one beam of a group has a score yet. done: share of finished beams."""
    return {"name": name, "op": "select", "groups": groups, "beams": beams, "vocab": vocab,
            "stride": stride, "keep": keep, "first": first, "done": done, "masked": masked}


def _reorder(name, groups, beams, layers, kind, page, shortest, longest, kv_heads=8, dim=128):
    return {"name": name, "op": "reorder", "groups": groups, "beams": beams, "layers": layers,
            "kind": kind, "page": page, "shortest": shortest, "longest": longest,
            "kv_heads": kv_heads, "dim": dim}


def listed():
    return [
        # One generated token through gate and up.
        _product("q8_gateup_1", 18432, 3072, 1),
        # Three requests of eight beams through the down projection.
        _product("q8_down_24", 3072, 9216, 24),
        # Odd sizes all around, more tokens than one tile has.
        _product("q8_odd_77", 5003, 1371, 77),
        # Prompts through gate and up.
        _product("q8_gateup_2048", 18432, 3072, 2048),
        # The norm before a projection: a decode token, and prompts.
        _rows("norm_1", "norm", 3072, 1),
        _rows("norm_4096", "norm", 3072, 4096),
        # The attention's outputs before the o projection, in padded rows.
        _rows("rows_50", "rows", 4096, 50, 3),
        # gate and up of prompts, side by side in the product's rows.
        _rows("silu_2048", "silu", 9216, 2048),
        # The first choice after a prompt: one beam, four to fill.
        _select("select_first_1x4", 1, 4, 131072, 131072, 4, first=True),
        # A batch of requests, two candidates a beam, some beams finished.
        _select("select_16x8", 16, 8, 131072, 131072, 16, done=0.15),
        # One request's beams in a 4-bit cache of all layers.
        _reorder("reorder_q4_1x4", 1, 4, 26, "q4", 64, 1003, 1003),
        # A batch of requests in FP16 pages.
        _reorder("reorder_f16_8x8", 8, 8, 26, "f16", 64, 65, 4321),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    case = _draw(rng)
    del case["name"]
    return case


def _draw(rng):
    which = rng.random()
    if which < 0.4:
        rows, cols = _log_int(rng, 16, 18432), _log_int(rng, 16, 16384)
        tokens = _log_int(rng, 1, 2048)
        # No dearer than the listed prompts, nor in weights.
        while rows * cols > 18432 * 3072:
            rows //= 2
        while rows * cols * tokens > 18432 * 3072 * 2048:
            tokens //= 2
        return _product(None, rows, cols, tokens)
    if which < 0.65:
        op = rng.choice(("norm", "norm", "first_norm", "silu", "rows"))
        width, tokens = _log_int(rng, 16, 16384), _log_int(rng, 1, 4096)
        while width * tokens > 3072 * 4096:
            tokens //= 2
        return _rows(None, op, width, tokens, rng.choice((0, 0, 1, 4)))
    if which < 0.85:
        groups, beams = _log_int(rng, 1, 32), rng.choice((1, 2, 3, 4, 5, 8, 8, 16))
        vocab = rng.choice((131072, _log_int(rng, 1000, 151936)))
        while groups > 1 and groups * beams * vocab > 128 * 131072:
            groups //= 2
        return _select(None, groups, beams, vocab, vocab + rng.choice((0, 0, 3, 64)),
                       rng.choice((beams, 2 * beams)), rng.random() < 0.15,
                       rng.choice((0.0, 0.2)), rng.random() < 0.3)
    groups, beams = _log_int(rng, 1, 8), rng.choice((2, 3, 4, 5, 8))
    layers = rng.choice((26, _log_int(rng, 1, 32)))
    kv_heads, dim = rng.choice(((8, 128), (8, 128), (16, 64), (2, 64), (1, 128)))
    kind, page = rng.choice(("q4", "f16")), rng.choice((32, 64, 128))
    longest = _log_int(rng, 16, 4352)
    case = _reorder(None, groups, beams, layers, kind, page, _log_int(rng, 1, longest), longest,
                    kv_heads, dim)
    # No dearer than the listed batch.
    while case["layers"] > 1 and _copies(case) * case["layers"] * _page_bytes(case) > \
            32 * 26 * 64 * 8 * 512:
        case["layers"] //= 2
    return case


# ---- inputs -----------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _round_up(n, to):
    return (n + to - 1) // to * to


def _product_inputs(case, seed):
    """Codes and scales of normally distributed weights, and of activations some
    channels of which are larger. The activations' rows lie on 16-byte words."""
    g = _generator(seed)
    rows, cols, tokens = case["rows"], case["cols"], case["tokens"]
    codes = torch.empty(rows, cols, dtype=torch.int8, device="cuda")
    for r in range(0, rows, 4096):
        n = min(4096, rows - r)
        codes[r:r + n] = _normal(g, n, cols).mul_(32).round_().clamp_(-127, 127).to(torch.int8)
    scales = 3e-4 * torch.exp(0.3 * _normal(g, rows))
    v = _normal(g, tokens, cols) * torch.exp(0.5 * _normal(g, cols))
    x_scales = v.abs().amax(1) / 127
    x = torch.zeros(tokens, _round_up(cols, 16), dtype=torch.int8, device="cuda")
    x[:, :cols] = torch.round(v / x_scales[:, None]).to(torch.int8)
    return codes, scales, x, x_scales


def _row_inputs(case, seed):
    """FP32 rows in padded buffers: [tokens][width] views. norm: the residual and
    what a layer adds to it, and the norm's weights; silu: gate and up, two parts
    of a product's rows."""
    g = _generator(seed)
    op, width, tokens, pad = case["op"], case["width"], case["tokens"], case["pad"]
    wide = 2 * width if op == "silu" else width
    x = torch.empty(tokens, wide + pad, device="cuda")[:, :wide]
    x.copy_(_normal(g, tokens, wide) * torch.exp(0.5 * _normal(g, wide)))
    if op == "silu":
        return x[:, :width], x[:, width:], None
    if op == "rows":
        return x, None, None
    gamma = 1 + 0.2 * _normal(g, width)
    if op == "first_norm":
        return x, None, gamma
    add = torch.empty(tokens, width + pad, device="cuda")[:, :width]
    add.copy_(0.3 * _normal(g, tokens, width))
    return x, add, gamma


def _select_inputs(case, seed):
    """Logits with the spread of a language model's, some rows almost certain of
    one token; scores of hypotheses of some length."""
    g = _generator(seed)
    groups, beams, vocab = case["groups"], case["beams"], case["vocab"]
    n = groups * beams
    x = torch.zeros(n, case["stride"], device="cuda")[:, :vocab]
    x.copy_(2.5 * _normal(g, n, vocab))
    likely = torch.randint(vocab, (n,), device="cuda", generator=g)
    sure = torch.rand(n, device="cuda", generator=g) * 20
    x.scatter_add_(1, likely[:, None], sure[:, None])
    if case["masked"]:
        keep = torch.rand(vocab, device="cuda", generator=g) < 0.4
        keep[:max(1, 2 * case["keep"])] = True
        x.masked_fill_(~keep, -math.inf)
    scores = -12 + 2 * _normal(g, n)
    done = torch.rand(n, device="cuda", generator=g) < case["done"]
    if case["first"]:
        done[:] = False
        scores.view(groups, beams)[:, 0] = 0
        scores.view(groups, beams)[:, 1:] = -math.inf
    return x, scores, done, int(likely[0])


def _page_bytes(case):
    """A page of one layer: the keys' and values' codes of all KV heads, in 4 bits
    with a scale and a zero for each of their vectors."""
    dim = case["dim"]
    vector = dim // 2 + 4 if case["kind"] == "q4" else 2 * dim
    return case["kv_heads"] * case["page"] * 2 * vector


def _lengths(case):
    """Positions of each group's beams, from the longest down to the shortest."""
    n, ratio = case["groups"], case["shortest"] / case["longest"]
    return [max(1, int(round(case["longest"] * ratio ** (i / max(1, n - 1))))) for i in range(n)]


def _alive(case):
    """Beams of a group that have children: half of them."""
    return (case["beams"] + 1) // 2


def _copies(case):
    """Pages of a layer that are copied: one for each child but a parent's first,
    where the group's open page holds anything."""
    return sum((case["beams"] - _alive(case)) for n in _lengths(case) if n % case["page"])


class _Beams:
    """Requests over a common prompt, whose pages all tables share; each beam has
    an open page and one for later of its own. Pages are dealt in random order."""

    def __init__(self, case, seed):
        g = _generator(seed)
        groups, beams, page = case["groups"], case["beams"], case["page"]
        self.lengths = _lengths(case)
        full = [n // page for n in self.lengths]
        width = max(full) + 2
        self.pages = max(full) + 2 * groups * beams + 1
        order = torch.randperm(self.pages, device="cuda", generator=g).int()
        self.table = torch.full((groups * beams, width), -1, dtype=torch.int32, device="cuda")
        at = max(full)
        for i, n in enumerate(full):
            rows = self.table[i * beams:(i + 1) * beams]
            rows[:, :n] = order[:n]
            rows[:, n:n + 2] = order[at:at + 2 * beams].view(beams, 2)
            at += 2 * beams
        self.length = torch.tensor(self.lengths, dtype=torch.int32, device="cuda"
                                   ).repeat_interleave(beams)
        # Half of the beams go on; their children stand in any order.
        alive = _alive(case)
        chosen = torch.rand(groups, beams, device="cuda", generator=g).argsort(1)[:, :alive]
        more = torch.randint(alive, (groups, beams - alive), device="cuda", generator=g)
        parent = torch.cat([chosen, chosen.gather(1, more)], dim=1)
        mixed = torch.rand(groups, beams, device="cuda", generator=g).argsort(1)
        self.parent = parent.gather(1, mixed).int()
        self.memory = torch.randint(256, (case["layers"], self.pages, _page_bytes(case)),
                                    dtype=torch.uint8, device="cuda", generator=g)


# ---- a program's state ------------------------------------------------------

def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _scratch(nbytes):
    return torch.empty(max(16, int(nbytes)), dtype=torch.uint8, device="cuda")


class _Product:
    def __init__(self, case, seed):
        self.case = case
        self.codes, self.scales, self.x, self.x_scales = _product_inputs(case, seed)
        if own:
            import lunelette_amd as lh
            self.lh, self.lib = lh, lh.lib()
            rows, cols = case["rows"], case["cols"]
            # A program lays its weights out once, when it loads them.
            self.packed = _scratch(self.lib.lh_q8_bytes(rows, cols))
            lh.check(self.lib.lh_q8_pack(self.codes.data_ptr(), self.scales.data_ptr(), rows,
                                         cols, self.packed.data_ptr(), _stream()))
            need = self.lib.lh_q8_scratch(rows, cols, case["tokens"])
            self.scratch = _scratch(need)
            self.y = torch.empty(case["tokens"], rows, device="cuda")

    def run(self):
        c = self.case
        if not own:
            x = self.x[:, :c["cols"]].float() * self.x_scales[:, None]
            return x @ (self.codes.float() * self.scales[:, None]).t()
        self.lh.check(self.lib.lh_q8_matvec(
            self.packed.data_ptr(), self.x.data_ptr(), self.x.stride(0), self.x_scales.data_ptr(),
            self.y.data_ptr(), c["rows"], c["rows"], c["cols"], c["tokens"],
            self.scratch.data_ptr(), self.scratch.numel(), _stream()))
        return self.y


class _Rows:
    def __init__(self, case, seed):
        self.case = case
        self.x, self.second, self.gamma = _row_inputs(case, seed)
        if own:
            import lunelette_amd as lh
            self.lh, self.lib = lh, lh.lib()
            tokens, width = case["tokens"], case["width"]
            self.codes = torch.empty(tokens, _round_up(width, 16), dtype=torch.int8,
                                     device="cuda")
            self.scales = torch.empty(tokens, device="cuda")
            if case["op"] == "norm":
                self.sum = torch.empty(tokens, width, device="cuda")

    def run(self):
        op, width, tokens = self.case["op"], self.case["width"], self.case["tokens"]
        x, second, gamma = self.x, self.second, self.gamma
        if not own:
            out = {}
            if op == "silu":
                v = x.double()
                v = v / (1 + torch.exp(-v)) * second.double()
            elif op == "rows":
                v = x.double()
            else:
                if op == "norm":
                    out["sum"] = x = x + second
                v = x.double()
                mean = (v * v).sum(1, keepdim=True) / width
                v = gamma.double() * (v / torch.sqrt(mean + EPSILON))
            scale = (v.abs().amax(1, keepdim=True) / 127).float()
            out["values"] = torch.round(v / scale.double()).clamp(-127, 127).float() * scale
            return out
        codes, scales, stream = self.codes.data_ptr(), self.scales.data_ptr(), _stream()
        if op == "silu":
            self.lh.check(self.lib.lh_q8_silu(
                x.data_ptr(), x.stride(0), second.data_ptr(), second.stride(0), width, tokens,
                codes, self.codes.stride(0), scales, stream))
        elif op == "rows":
            self.lh.check(self.lib.lh_q8_rows(x.data_ptr(), x.stride(0), width, tokens, codes,
                                              self.codes.stride(0), scales, stream))
        else:
            add = second is not None
            self.lh.check(self.lib.lh_q8_norm(
                x.data_ptr(), x.stride(0), second.data_ptr() if add else None,
                second.stride(0) if add else 0, gamma.data_ptr(),
                self.sum.data_ptr() if add else None, width if add else 0, width, tokens, codes,
                self.codes.stride(0), scales, stream))
        # The values that the codes stand for.
        out = {"values": self.codes[:, :width] * self.scales[:, None]}
        if op == "norm":
            out["sum"] = self.sum
        return out


class _Select:
    def __init__(self, case, seed):
        self.case = case
        self.x, self.scores, self.done, self.stop = _select_inputs(case, seed)
        if own:
            import lunelette_amd as lh
            self.lh, self.lib = lh, lh.lib()
            groups, keep = case["groups"], case["keep"]
            self.scratch = _scratch(self.lib.lh_beam_scratch(groups, case["beams"], case["vocab"],
                                                             keep))
            self.parent = torch.empty(groups, keep, dtype=torch.int32, device="cuda")
            self.token = torch.empty(groups, keep, dtype=torch.int64, device="cuda")
            self.score = torch.empty(groups, keep, device="cuda")
            self.done_out = torch.empty(groups, keep, dtype=torch.bool, device="cuda")

    def run(self):
        c = self.case
        groups, beams, vocab, keep = c["groups"], c["beams"], c["vocab"], c["keep"]
        if own:
            self.lh.check(self.lib.lh_beam_select(
                self.x.data_ptr(), c["stride"], groups, beams, vocab, self.scores.data_ptr(),
                self.done.data_ptr(), self.stop, keep, self.parent.data_ptr(),
                self.token.data_ptr(), self.score.data_ptr(), self.done_out.data_ptr(),
                self.scratch.data_ptr(), self.scratch.numel(), _stream()))
            return {"parent": self.parent, "token": self.token, "score": self.score,
                    "done": self.done_out}
        # A finished beam's one candidate stands behind its tokens' places.
        shifted = self.x - self.x.amax(1, keepdim=True)
        log_z = torch.log(torch.exp(shifted).sum(1, dtype=torch.float64))
        s = self.scores.double()[:, None]
        each = shifted.double() - log_z[:, None] + s
        each = each.masked_fill(self.done[:, None], -math.inf)
        ended = torch.where(self.done[:, None], s, -math.inf)
        each = torch.cat([each, ended], dim=1).view(groups, -1)
        best = torch.sort(each, dim=1, descending=True, stable=True)
        score, place = best.values[:, :keep], best.indices[:, :keep]
        live = score > -math.inf
        beam, token = place // (vocab + 1), place % (vocab + 1)
        token = torch.where(live & (token < vocab), token, -1)
        parent = torch.where(live, beam, -1).int()
        ended = self.done.view(groups, beams).gather(1, beam) & live
        return {"parent": parent, "token": token, "score": score.float(),
                "done": ended | (token == self.stop)}


class _Reorder:
    def __init__(self, case, seed):
        self.case = case
        self.beams = b = _Beams(case, seed)
        if own:
            import lunelette_amd as lh
            self.lh, self.lib = lh, lh.lib()
            self.caches = (lh.PagedCache * case["layers"])()
            for i, c in enumerate(self.caches):
                c.kind = lh.CACHE_Q4 if case["kind"] == "q4" else lh.CACHE_F16
                c.kv_heads, c.head_dim = case["kv_heads"], case["dim"]
                c.page_size, c.pages = case["page"], b.pages
                c.data = b.memory[i].data_ptr()
            self.table = torch.empty_like(b.table)

    def run(self):
        c, b = self.case, self.beams
        groups, beams = c["groups"], c["beams"]
        if own:
            self.lh.check(self.lib.lh_beam_reorder(
                self.caches, c["layers"], groups, beams, b.parent.data_ptr(), b.length.data_ptr(),
                b.table.data_ptr(), self.table.data_ptr(), b.table.shape[1], _stream()))
            return {"table": self.table, "pages": b.memory}
        child = torch.arange(beams, device="cuda")
        parent = b.parent.long()
        has = parent[:, None, :] == child[None, :, None]      # [group][parent][child]
        alive = has.any(2)
        first = has.long().argmax(2)
        keeps = first.gather(1, parent) == child              # a parent's first child
        # The n-th other child takes the pages of the n-th beam without children.
        dead = torch.sort((alive * beams + child).view(groups, beams), dim=1).values
        turn = (torch.cumsum(~keeps, 1) - 1).clamp(min=0)
        owner = torch.where(keeps, parent, dead.gather(1, turn))
        table = b.table.view(groups, beams, -1)
        column = torch.arange(table.shape[2], device="cuda")
        open_column = (b.length.view(groups, beams)[:, :1] // c["page"]).long()
        at = open_column[:, :, None].expand(-1, beams, 1)

        def of(rows):
            return table.gather(1, rows[:, :, None].expand(-1, -1, table.shape[2]))

        from_page, to_page = of(parent).gather(2, at)[..., 0], of(owner).gather(2, at)[..., 0]
        copied = ~keeps & (b.length.view(groups, beams)[:, :1] % c["page"] > 0)
        b.memory[:, to_page[copied].long()] = b.memory[:, from_page[copied].long()]
        new = torch.where(column < open_column[:, :, None], of(parent), of(owner))
        return {"table": new.reshape(b.table.shape), "pages": b.memory}


def prepare(case, seed):
    kinds = {"product": _Product, "select": _Select, "reorder": _Reorder}
    return kinds.get(case["op"], _Rows)(case, int(seed))


def run(state):
    return state.run()


# ---- what a pass cannot do without --------------------------------------------

def work(case):
    op = case["op"]
    if op == "product":
        rows, cols, tokens = case["rows"], case["cols"], case["tokens"]
        return {"bytes": rows * cols + 4 * rows + tokens * (cols + 4) + 4 * tokens * rows,
                "flops": 2 * rows * cols * tokens}
    if op == "select":
        n, vocab = case["groups"] * case["beams"], case["vocab"]
        if case["first"]:
            n = case["groups"]
        # A subtraction, an exponential and a sum for each logit.
        return {"bytes": 4 * n * vocab + 17 * case["groups"] * case["keep"],
                "flops": 3 * n * vocab}
    if op == "reorder":
        table = sum(8 * case["beams"] * (n // case["page"] + 2) for n in _lengths(case))
        return {"bytes": 2 * _copies(case) * case["layers"] * _page_bytes(case) + table,
                "flops": 0}
    elements = case["width"] * case["tokens"]
    if op == "norm":
        # Two rows in, their sum and the values out.
        return {"bytes": 16 * elements + 4 * case["width"], "flops": 8 * elements}
    if op == "silu":
        return {"bytes": 12 * elements, "flops": 8 * elements}
    return {"bytes": 8 * elements, "flops": (6 if op == "first_norm" else 3) * elements}


# ---- the same in 64 bits ------------------------------------------------------

def exact(case, seed):
    seed = int(seed)
    kinds = {"product": _exact_product, "select": _exact_select, "reorder": _exact_reorder}
    return kinds.get(case["op"], _exact_rows)(case, seed)


def _exact_product(case, seed):
    codes, scales, x, x_scales = _product_inputs(case, seed)
    out = torch.empty(case["tokens"], case["rows"], dtype=torch.float64, device="cuda")
    left = x[:, :case["cols"]].double()
    for r in range(0, case["rows"], 2048):
        right = codes[r:r + 2048].double().t().contiguous()
        out[:, r:r + 2048] = (left @ right) * scales[r:r + 2048].double()
    return out.mul_(x_scales.double()[:, None])


def _exact_rows(case, seed):
    x, second, gamma = _row_inputs(case, seed)
    out = {}
    if case["op"] == "silu":
        v = x.double() * torch.sigmoid(x.double()) * second.double()
    elif case["op"] == "rows":
        v = x.double()
    else:
        h = x.double()
        if second is not None:
            # The sum is kept in 32 bits, and its norm is taken of what is kept.
            h = (h + second.double()).float().double()
            out["sum"] = h
        length = torch.linalg.vector_norm(h, dim=1, keepdim=True)
        v = h * gamma.double() / torch.sqrt(length ** 2 / case["width"] + EPSILON)
    step = (v.abs().max(1, keepdim=True).values / 127).float().double()
    out["values"] = step * torch.round(v / step).clamp(-127, 127)
    return out


def _exact_select(case, seed):
    x, scores, done, stop = _select_inputs(case, seed)
    beams, keep = case["beams"], case["keep"]
    out = {"parent": [], "token": [], "score": [], "done": []}
    for g in range(case["groups"]):
        found = []   # (score, beam, token)
        for b in range(beams):
            r = g * beams + b
            s = float(scores[r])
            if bool(done[r]):
                found.append((s, b, -1))
                continue
            if s == -math.inf:
                continue
            p = torch.log_softmax(x[r].double(), 0)
            # The k-th largest is a threshold; stable order by id below it.
            limit = torch.topk(p, min(keep, case["vocab"])).values[-1]
            ids = (p >= limit).nonzero()[:, 0]
            ids = ids[torch.argsort(p[ids], descending=True, stable=True)][:keep]
            found += [(s + v, b, t) for v, t in zip(p[ids].tolist(), ids.tolist())
                      if v > -math.inf]
        found.sort(key=lambda f: (-f[0], f[1]))
        found = found[:keep] + [(-math.inf, -1, -1)] * (keep - len(found))
        out["score"].append([f[0] for f in found])
        out["parent"].append([f[1] for f in found])
        out["token"].append([f[2] for f in found])
        out["done"].append([f[1] >= 0 and (bool(done[g * beams + f[1]]) or f[2] == stop)
                            for f in found])
    types = {"parent": torch.int32, "token": torch.int64, "score": torch.float64,
             "done": torch.bool}
    return {k: torch.tensor(v, dtype=types[k], device="cuda") for k, v in out.items()}


def _exact_reorder(case, seed):
    b = _Beams(case, seed)
    beams, page = case["beams"], case["page"]
    before, after = b.table.tolist(), b.table.tolist()
    pages = b.memory.clone()
    for g, length in enumerate(b.lengths):
        parents = b.parent[g].tolist()
        free = [p for p in range(beams) if p not in parents]
        column, kept = length // page, set()
        for k, p in enumerate(parents):
            source = before[g * beams + p]
            if p in kept:
                owned = before[g * beams + free.pop(0)]
                if length % page:
                    pages[:, owned[column]] = b.memory[:, source[column]]
            else:
                kept.add(p)
                owned = source
            after[g * beams + k] = source[:column] + owned[column:]
    return {"table": torch.tensor(after, dtype=torch.int32, device="cuda"), "pages": pages}
