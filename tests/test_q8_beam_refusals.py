"""Arguments that the 8-bit and beam search operators refuse, on the CPU: every check
comes before the launch, so made-up pointers are never followed."""
import pytest

import lunelette_amd as lh

P = 0x10000   # a 16-byte aligned address that nothing reads
Q, R, S = 2 * P, 3 * P, 4 * P


def rows(l, x=P, xs=100, width=100, tokens=3, codes=Q, cs=112, scales=R):
    return l.lh_q8_rows(x, xs, width, tokens, codes, cs, scales, None)


def silu(l, x=P, xs=100, up=S, us=100, width=100, tokens=3, codes=Q, cs=112, scales=R):
    return l.lh_q8_silu(x, xs, up, us, width, tokens, codes, cs, scales, None)


def norm(l, x=P, xs=100, add=S, adds=100, gamma=5 * P, out=6 * P, outs=100, width=100, tokens=3,
         codes=Q, cs=112, scales=R):
    return l.lh_q8_norm(x, xs, add, adds, gamma, out, outs, width, tokens, codes, cs, scales, None)


def multiply(l, packed=S, x=Q, xs=112, scales=R, y=P, ys=50, r=50, width=100, tokens=3, scratch=P,
            nbytes=1 << 40):
    return l.lh_q8_matvec(packed, x, xs, scales, y, ys, r, width, tokens, scratch, nbytes, None)


BAD_CODES = [dict(width=0), dict(width=65537), dict(tokens=0), dict(tokens=65536),
             dict(scales=None), dict(scales=R + 2)]


@pytest.mark.parametrize("call,codes,stride", [
    (rows, "codes", "cs"), (silu, "codes", "cs"), (norm, "codes", "cs"), (multiply, "x", "xs")])
def test_codes_lie_on_16_bytes(product, call, codes, stride):
    bad = BAD_CODES + [{codes: None}, {codes: Q + 8}, {stride: 96}, {stride: 120},
                       {stride: 2 ** 36 + 16}]
    for change in bad:
        assert call(product, **change) == -1, change
        assert "16-byte" in lh.last_error()


def test_rows_refusals(product):
    for change in (dict(x=None), dict(x=P + 2), dict(xs=99), dict(xs=2 ** 41)):
        assert rows(product, **change) == -1, change
        assert silu(product, **change) == -1, change
        assert norm(product, **change) == -1, change
        assert "width" in lh.last_error()
    for change in (dict(up=None), dict(up=S + 1), dict(us=99)):
        assert silu(product, **change) == -1, change
    for change in (dict(gamma=None), dict(gamma=P + 2), dict(add=S + 2), dict(adds=99),
                   dict(out=P + 2), dict(outs=99)):
        assert norm(product, **change) == -1, change
        assert "gamma" in lh.last_error()


def test_rows_refuse_overlaps(product):
    for change in (dict(codes=P), dict(scales=P)):
        for call in (rows, silu, norm):
            assert call(product, **change) == -1, (call, change)
            assert "overlap" in lh.last_error()
    for change in (dict(codes=S), dict(scales=S)):
        assert silu(product, **change) == -1 and norm(product, **change) == -1
    for change in (dict(out=5 * P), dict(out=Q), dict(out=R)):
        assert norm(product, **change) == -1, change
        assert "overlap" in lh.last_error()
    for change in (dict(out=P, outs=104), dict(out=S, outs=104)):
        assert norm(product, **change) == -1, change
        assert "in place" in lh.last_error()


def test_weights_refusals(product):
    for r, cols in ((0, 64), (2 ** 20 + 1, 64), (16, 0), (16, 65537)):
        assert product.lh_q8_bytes(r, cols) == 0
        assert product.lh_q8_scratch(r, cols, 1) == 0
        assert product.lh_q8_pack(P, P, r, cols, P, None) == -1
        assert "q8_pack" in lh.last_error()
        assert product.lh_q8_quantize(P, r, cols, P, None) == -1
        assert "q8_quantize" in lh.last_error()
    for args in ((None, P, 16, 64, P), (P, None, 16, 64, P), (P, P, 16, 64, None),
                 (P, P, 16, 64, P + 8), (P, P + 2, 16, 64, P)):
        assert product.lh_q8_pack(*args, None) == -1, args
    for args in ((None, 16, 64, P), (P, 16, 64, None), (P + 1, 16, 64, P), (P, 16, 64, P + 8)):
        assert product.lh_q8_quantize(*args, None) == -1, args
    assert product.lh_q8_bytes(17, 65) == 2 * 2 * 1024 + 32 * 4
    assert product.lh_q8_bytes(2 ** 20, 65536) == 2 ** 36 + 2 ** 22
    assert product.lh_q8_scratch(16, 64, 0) == product.lh_q8_scratch(16, 64, 65536) == 0


def test_product_refusals(product):
    for change in (dict(packed=None), dict(packed=S + 8), dict(y=None), dict(y=P + 2),
                   dict(ys=49), dict(r=0), dict(r=2 ** 20 + 1, ys=2 ** 21)):
        assert multiply(product, **change) == -1, change
        assert "rows" in lh.last_error()
    for change in (dict(y=Q), dict(y=R), dict(y=S)):
        assert multiply(product, **change) == -1, change
        assert "overlap" in lh.last_error()
    for r, cols, tokens in ((3072, 9216, 24), (5003, 1371, 77), (64, 65536, 3), (512, 4096, 200)):
        need = product.lh_q8_scratch(r, cols, tokens)
        if need:
            for change in (dict(scratch=None), dict(nbytes=need - 1), dict(scratch=P + 8)):
                assert multiply(product, r=r, ys=r, width=cols, xs=65536, tokens=tokens,
                            **change) == -1, change
                assert "scratch" in lh.last_error()


def select(l, x=P, stride=1000, groups=3, beams=4, vocab=1000, scores=Q, done=R, stop=2, keep=4,
           parent=S, token=5 * P, score=6 * P, out=7 * P, scratch=8 * P, nbytes=1 << 40):
    return l.lh_beam_select(x, stride, groups, beams, vocab, scores, done, stop, keep, parent,
                            token, score, out, scratch, nbytes, None)


def test_select_refusals(product):
    for change in (dict(x=None), dict(x=P + 2), dict(stride=999), dict(groups=0),
                   dict(groups=65536), dict(groups=20000), dict(beams=0), dict(beams=65),
                   dict(vocab=0), dict(vocab=2 ** 24 + 1, stride=2 ** 25), dict(keep=0),
                   dict(keep=65), dict(scores=None), dict(scores=Q + 2)):
        assert select(product, **change) == -1, change
        assert "require logits" in lh.last_error()
    for change in (dict(parent=None), dict(token=None), dict(score=None), dict(parent=S + 2),
                   dict(token=P + 4), dict(score=P + 2)):
        assert select(product, **change) == -1, change
        assert "kept places" in lh.last_error()
    for change in (dict(score=Q), dict(out=R)):
        assert select(product, **change) == -1, change
        assert "overlap" in lh.last_error()
    need = product.lh_beam_scratch(3, 4, 1000, 4)
    assert need
    for change in (dict(scratch=None), dict(nbytes=need - 1), dict(scratch=P + 8)):
        assert select(product, **change) == -1, change
        assert "scratch" in lh.last_error()
    for sizes in ((0, 1, 10, 1), (1, 0, 10, 1), (1, 65, 10, 1), (1, 1, 0, 1), (1, 1, 10, 65),
                  (65535, 2, 10, 1), (1, 1, 10, 0)):
        assert product.lh_beam_scratch(*sizes) == 0


def caches(n, **change):
    out = (lh.PagedCache * n)()
    for c in out:
        c.kind, c.kv_heads, c.head_dim, c.page_size, c.pages, c.data = lh.CACHE_Q4, 8, 128, 64, 10, P
    for k, v in change.items():
        setattr(out[n - 1], k, v)
    return out


def reorder(l, c=None, layers=2, groups=3, beams=4, parent=Q, length=R, table=S, out=5 * P,
            width=6):
    return l.lh_beam_reorder(caches(2) if c is None else c, layers, groups, beams, parent, length,
                             table, out, width, None)


def test_reorder_refusals(product):
    for change in (dict(layers=0), dict(layers=65)):
        assert reorder(product, **change) == -1, change
        assert "layers" in lh.last_error()
    assert product.lh_beam_reorder(None, 1, 1, 1, P, P, P, P, 1, None) == -1
    for change in (dict(data=None), dict(data=P + 8), dict(page_size=48), dict(kind=7)):
        assert reorder(product, c=caches(2, **change)) == -1, change
        assert "cache" in lh.last_error()
    for change in (dict(kind=lh.CACHE_F16), dict(kv_heads=4), dict(head_dim=64),
                   dict(page_size=32), dict(pages=11)):
        assert reorder(product, c=caches(2, **change)) == -1, change
        assert "alike" in lh.last_error()
    for change in (dict(groups=0), dict(groups=65536), dict(groups=20000), dict(beams=0),
                   dict(beams=65), dict(width=0), dict(width=2 ** 20 + 1), dict(parent=None),
                   dict(length=None), dict(table=None), dict(out=None), dict(parent=Q + 2),
                   dict(length=R + 1), dict(table=S + 2), dict(out=P + 2)):
        assert reorder(product, **change) == -1, change
        assert "require parents" in lh.last_error()
    for change in (dict(out=Q), dict(out=R)):
        assert reorder(product, **change) == -1, change
        assert "overlap" in lh.last_error()
