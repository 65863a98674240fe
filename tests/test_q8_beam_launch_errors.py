"""What a launch of the 8-bit and beam search operators that the HIP runtime refuses leaves
in lh_last_error(), on the CPU as in test_launch_errors.py."""
from test_launch_errors import run

CHILD = r"""
import ctypes, sys
ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
import lunelette_amd as lh
l = lh.lib()
P, Q, R, S, BIG = 0x10000, 0x20000, 0x30000, 0x40000, 1 << 40
caches = (lh.PagedCache * 2)()
for c in caches:
    c.kind, c.kv_heads, c.head_dim, c.page_size, c.pages, c.data = lh.CACHE_Q4, 8, 128, 64, 10, P
calls = {
    "q8 rows": lambda: l.lh_q8_rows(P, 64, 64, 3, Q, 64, R, None),
    "q8 silu": lambda: l.lh_q8_silu(P, 64, S, 64, 64, 3, Q, 64, R, None),
    "q8 norm": lambda: l.lh_q8_norm(P, 64, S, 64, 5 * P, 6 * P, 64, 64, 3, Q, 64, R, None),
    "q8 norm ": lambda: l.lh_q8_norm(P, 9000, None, 0, 5 * P, None, 0, 9000, 3, Q, 9008, R, None),
    "q8 pack": lambda: l.lh_q8_pack(P, Q, 16, 64, R, None),
    "q8 quantize": lambda: l.lh_q8_quantize(P, 16, 64, R, None),
    "beam select": lambda: l.lh_beam_select(P, 64, 2, 3, 64, Q, None, -1, 3, R, S, 5 * P, None,
                                            6 * P, BIG, None),
    "beam reorder": lambda: l.lh_beam_reorder(caches, 2, 1, 3, P, Q, R, R, 4, None),
    "beam reorder ": lambda: l.lh_beam_reorder(caches, 2, 1, 3, P, Q, R, S, 4, None),
}
for i, (rows, cols, tokens) in enumerate(((64, 64, 1), (3072, 9216, 24), (64, 64, 100),
                                          (18432, 3072, 2048), (3072, 9216, 200))):
    calls["q8 matvec" + " " * i] = lambda r=rows, c=cols, t=tokens: l.lh_q8_matvec(
        P, Q, c, R, S, r, r, c, t, 5 * P, BIG, None)
for name, call in calls.items():
    # Twice: a refused launch leaves nothing behind that the next call reports.
    for _ in range(2):
        print(name.strip(), "|", call(), "|", lh.last_error(), flush=True)
"""


def test_refused_launches_keep_the_runtimes_words(tmp_path):
    lines = [line.split(" | ") for line in run(tmp_path, CHILD)]
    assert len(lines) == 28
    for name, status, text in lines:
        assert status == "-1", name
        assert name in text and "invalid configuration" in text, (name, text)
