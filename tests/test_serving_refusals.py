"""Arguments that the batched serving operators refuse, on the CPU: every check
comes before the launch, so made-up pointers are never followed."""
import ctypes

import pytest

import lunelette_amd as lh

P = 0x10000   # a 16-byte aligned address that nothing reads


def good_cache(**change):
    c = lh.PagedCache()
    values = dict(kind=lh.CACHE_Q4, kv_heads=8, head_dim=128, page_size=64, pages=10, data=P)
    values.update(change)
    for k, v in values.items():
        setattr(c, k, v)
    return c


def good_batch(**change):
    b = lh.PagedBatch()
    values = dict(sequences=2, tokens=4, table_width=3, max_query=2, max_length=100,
                  query_start=P, length=P, table=P)
    values.update(change)
    for k, v in values.items():
        setattr(b, k, v)
    return b


BAD_CACHES = [dict(kind=2), dict(kind=-1), dict(kv_heads=0), dict(kv_heads=65),
              dict(head_dim=96), dict(head_dim=0), dict(page_size=16), dict(page_size=48),
              dict(page_size=2048), dict(page_size=0), dict(pages=0), dict(pages=2 ** 31)]
BAD_BATCHES = [dict(sequences=0), dict(sequences=65536), dict(tokens=0),
               dict(tokens=2 ** 24 + 1), dict(table_width=0), dict(table_width=2 ** 20 + 1),
               dict(max_query=0), dict(max_length=0)]


def append(l, cache=None, batch=None, heads=32, q=P, qs=4096, k=P, ks=1024, v=P, vs=1024, cos=P,
           sin=P, positions=100, factor=None, out=2 * P, outs=4096):
    return l.lh_paged_append(ctypes.byref(cache or good_cache()),
                             ctypes.byref(batch or good_batch()), heads, q, qs, k, ks, v, vs, cos,
                             sin, positions, factor, out, outs, None)


def attend(l, cache=None, batch=None, heads=32, q=P, qs=4096, scale=0.1, out=2 * P, outs=4096,
           scratch=P, nbytes=1 << 40):
    return l.lh_paged_attention(ctypes.byref(cache or good_cache()),
                                ctypes.byref(batch or good_batch()), heads, q, qs, scale, out,
                                outs, scratch, nbytes, None)


def read(l, cache=None, batch=None, k=P, ks=1024, v=P, vs=1024):
    return l.lh_paged_read(ctypes.byref(cache or good_cache()),
                           ctypes.byref(batch or good_batch()), k, ks, v, vs, None)


@pytest.mark.parametrize("call", [append, attend, read])
def test_paged_calls_refuse_bad_caches_and_batches(product, call):
    for change in BAD_CACHES + [dict(data=None), dict(data=P + 8)]:
        assert call(product, cache=good_cache(**change)) == -1, change
        assert "cache" in lh.last_error()
    for change in BAD_BATCHES + [dict(query_start=None), dict(length=None), dict(table=None),
                                 dict(length=P + 2)]:
        assert call(product, batch=good_batch(**change)) == -1, change
        assert "batch" in lh.last_error()


def test_paged_sizes(product):
    size = product.lh_paged_cache_bytes
    assert size(ctypes.byref(good_cache())) == 10 * 8 * 64 * 2 * (64 + 4)
    assert size(ctypes.byref(good_cache(kind=lh.CACHE_F16, head_dim=64))) == 10 * 8 * 64 * 2 * 128
    assert size(ctypes.byref(good_cache(pages=2 ** 31 - 1, page_size=1024, kv_heads=64))) == \
        (2 ** 31 - 1) * 64 * 1024 * 2 * 68
    for change in BAD_CACHES:
        assert size(ctypes.byref(good_cache(**change))) == 0, change
    need = product.lh_paged_attention_scratch
    for change in BAD_BATCHES:
        assert need(ctypes.byref(good_cache()), ctypes.byref(good_batch(**change)), 32) == 0
    assert need(ctypes.byref(good_cache()), ctypes.byref(good_batch()), 12) == 0


def test_paged_append_refusals(product):
    for change in (dict(heads=12), dict(heads=8 * 65), dict(q=None), dict(out=None),
                   dict(qs=4095), dict(outs=4095), dict(q=P + 2), dict(out=P + 1)):
        assert append(product, **change) == -1, change
        assert "heads" in lh.last_error()
    for change in (dict(k=None), dict(v=None), dict(ks=1023), dict(vs=0), dict(k=P + 2),
                   dict(vs=2 ** 41)):
        assert append(product, **change) == -1, change
        assert "keys and values" in lh.last_error()
    assert append(product, out=P, outs=4100) == -1
    assert "in place" in lh.last_error()
    for change in (dict(cos=None), dict(sin=None), dict(positions=0),
                   dict(cos=None, sin=None, positions=0, factor=P), dict(cos=P + 2)):
        assert append(product, **change) == -1, change
        assert "cos and sin" in lh.last_error()


def test_paged_read_refusals(product):
    for change in (dict(k=None, v=None), dict(ks=1000), dict(vs=1000), dict(k=P + 1)):
        assert read(product, **change) == -1, change
        assert "keys or values" in lh.last_error()


def test_paged_attention_refusals(product):
    for change in (dict(heads=0), dict(heads=12), dict(heads=8 * 65), dict(q=None),
                   dict(out=None), dict(out=P), dict(qs=1), dict(outs=4095), dict(q=P + 2)):
        assert attend(product, **change) == -1, change
        assert "heads" in lh.last_error()
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        assert attend(product, scale=scale) == -1
        assert "scale" in lh.last_error()
    batch = good_batch(max_length=100000, table_width=2000)
    need = product.lh_paged_attention_scratch(ctypes.byref(good_cache()), ctypes.byref(batch), 32)
    if need:
        for change in (dict(scratch=None), dict(nbytes=need - 1), dict(scratch=P + 8)):
            assert attend(product, batch=batch, **change) == -1, change
            assert "scratch" in lh.last_error()


def q4(l, packed=P, x=P, xs=256, y=P, ys=100, rows=100, cols=256, group=64, tokens=3, scratch=P,
       nbytes=1 << 40):
    return l.lh_q4_matvec(packed, x, xs, y, ys, rows, cols, group, tokens, scratch, nbytes, None)


BAD_Q4 = [(0, 256, 64), (2 ** 20 + 1, 256, 64), (100, 0, 64), (100, 65536 + 64, 64),
          (100, 250, 64), (100, 256, 16), (100, 256, 0), (100, 96, 64)]


def test_q4_refuses_its_own_input(product):
    assert q4(product, y=P) == -1
    assert "overlap" in lh.last_error()
    assert q4(product, xs=2 ** 36 + 1) == -1
    assert "stride" in lh.last_error()


def test_q4_refusals(product):
    for rows, cols, group in BAD_Q4:
        assert product.lh_q4_bytes(rows, cols, group) == 0
        assert q4(product, rows=rows, cols=cols, group=group, xs=1 << 20, ys=1 << 21) == -1
        assert product.lh_q4_pack(P, P, rows, cols, group, P, None) == -1
        assert "q4_pack" in lh.last_error()
        assert product.lh_q4_quantize(P, rows, cols, group, P, None) == -1
        assert "q4_quantize" in lh.last_error()
    for change in (dict(packed=None), dict(x=None), dict(y=None), dict(tokens=0),
                   dict(tokens=65536), dict(packed=P + 8), dict(x=P + 2), dict(y=P + 1)):
        assert q4(product, **change) == -1, change
        assert "q4_matvec" in lh.last_error()
    for change in (dict(xs=255), dict(ys=99), dict(xs=2 ** 41)):
        assert q4(product, **change) == -1, change
        assert "stride" in lh.last_error()
    assert product.lh_q4_pack(None, P, 16, 64, 64, P, None) == -1
    assert product.lh_q4_pack(P, None, 16, 64, 64, P, None) == -1
    assert product.lh_q4_pack(P, P, 16, 64, 64, P + 4, None) == -1
    assert product.lh_q4_quantize(P, 16, 64, 64, None, None) == -1
    assert product.lh_q4_bytes(17, 160, 32) == 2 * 2 * (1024 + 128)
    assert product.lh_q4_scratch(0, 1) == product.lh_q4_scratch(64, 0) == 0
    need = product.lh_q4_scratch(256, 64)
    if need:
        for change in (dict(scratch=None), dict(nbytes=need - 1), dict(scratch=P + 8)):
            assert q4(product, tokens=64, **change) == -1, change
            assert "scratch" in lh.last_error()


def logprobs(l, x=P, stride=1000, rows=3, vocab=1000, tokens=P, lp=P, entropy=P, top=5, ids=P,
             tops=P, scratch=P, nbytes=1 << 40):
    return l.lh_logprobs(x, stride, rows, vocab, tokens, lp, entropy, top, ids, tops, scratch,
                         nbytes, None)


def test_logprobs_refusals(product):
    for change in (dict(x=None), dict(rows=0), dict(rows=65536), dict(vocab=0, stride=0),
                   dict(vocab=2 ** 24 + 1, stride=2 ** 25), dict(stride=999), dict(top=65),
                   dict(x=P + 2), dict(stride=2 ** 41)):
        assert logprobs(product, **change) == -1, change
        assert "require logits" in lh.last_error()
    for change in (dict(tokens=None), dict(lp=None), dict(ids=None), dict(tops=None),
                   dict(tokens=None, lp=None, entropy=None, top=0), dict(tokens=P + 4),
                   dict(ids=P + 4), dict(entropy=P + 2)):
        assert logprobs(product, **change) == -1, change
        assert "go together" in lh.last_error()
    for sizes in ((0, 10, 1), (1, 0, 1), (1, 10, 65), (65536, 10, 1)):
        assert product.lh_logprobs_scratch(*sizes) == 0
    need = product.lh_logprobs_scratch(3, 100000, 5)
    if need:
        for change in (dict(scratch=None), dict(nbytes=need - 1), dict(scratch=P + 8)):
            assert logprobs(product, vocab=100000, stride=100000, **change) == -1, change
            assert "scratch" in lh.last_error()
