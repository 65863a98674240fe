"""What a launch that the HIP runtime refuses leaves in lh_last_error(): the runtime's own
words. On the CPU: a library loaded before the product's answers its launches, so no
kernel is ever started and made-up pointers are never followed."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SHIM = r"""
/* Every launch fails with hipErrorInvalidConfiguration, or none does, allocations and
 * waits with hipErrorOutOfMemory; recorded as the runtime does. */
#include <stddef.h>
static __thread int last;
int launch_status = 9;
int hipMalloc(void **p, size_t n)
{
    (void)n;
    *p = NULL;
    return last = 2;
}
int hipHostMalloc(void **p, size_t n, unsigned flags)
{
    (void)flags;
    return hipMalloc(p, n);
}
int hipDeviceSynchronize(void)
{
    return last = 2;
}
int __hipPushCallConfiguration(void)
{
    return 0;
}
int __hipPopCallConfiguration(void)
{
    return 0;
}
int hipLaunchKernel(const void *f, ...)
{
    (void)f;
    if (launch_status) {
        last = launch_status;
    }
    return launch_status;
}
int hipGetLastError(void)
{
    const int e = last;
    last = 0;
    return e;
}
int hipPeekAtLastError(void)
{
    return last;
}
"""

CHILD = r"""
import ctypes, sys
ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
import lunelette_amd as lh
l = lh.lib()
P, BIG = 0x10000, 1 << 40
cache, batch = lh.PagedCache(), lh.PagedBatch()
cache.kind, cache.kv_heads, cache.head_dim, cache.page_size = lh.CACHE_Q4, 8, 128, 64
cache.pages, cache.data = 10, P
batch.sequences, batch.tokens, batch.table_width, batch.max_query = 2, 4, 3, 2
batch.max_length, batch.query_start, batch.length, batch.table = 100, P, P, P
c, b = ctypes.byref(cache), ctypes.byref(batch)
calls = {
    "q4 pack": lambda: l.lh_q4_pack(P, P, 16, 64, 64, P, None),
    "q4 quantize": lambda: l.lh_q4_quantize(P, 16, 64, 64, P, None),
    "q4 matvec": lambda: l.lh_q4_matvec(P, P, 64, 2 * P, 16, 16, 64, 64, 1, P, BIG, None),
    "q4 matvec ": lambda: l.lh_q4_matvec(P, P, 64, 2 * P, 16, 16, 64, 64, 200, P, BIG, None),
    "logprobs": lambda: l.lh_logprobs(P, 64, 1, 64, P, P, P, 0, None, None, P, BIG, None),
    "paged append": lambda: l.lh_paged_append(c, b, 32, P, 4096, P, 1024, P, 1024, P, P, 100,
                                              None, 2 * P, 4096, None),
    "paged read": lambda: l.lh_paged_read(c, b, P, 1024, P, 1024, None),
    "paged attention": lambda: l.lh_paged_attention(c, b, 32, P, 4096, 0.1, 2 * P, 4096, P, BIG,
                                                    None),
    "fp8 matvec": lambda: l.lh_fp8_matvec(P, 1.0, P, 2 * P, 16, 64, 1, 0, None),
    "rmsnorm": lambda: l.lh_rmsnorm(P, P, 2 * P, 64, 1, None),
}
for name, call in calls.items():
    # Twice: a refused launch leaves nothing behind that the next call reports.
    for _ in range(2):
        print(name.strip(), "|", call(), "|", lh.last_error(), flush=True)
"""

AFTER = r"""
import ctypes, sys
shim = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
import lunelette_amd as lh
l = lh.lib()
P = 0x10000
ctypes.c_int.in_dll(shim, "launch_status").value = 0
for fail in (lambda: l.lh_device_alloc(64) is None, lambda: l.lh_host_alloc_pinned(64) is None,
             lambda: l.lh_device_synchronize() == -1):
    print(fail(), "out of memory" in lh.last_error(), l.lh_q4_pack(P, P, 16, 64, 64, P, None),
          l.lh_rmsnorm(P, P, 2 * P, 64, 1, None), flush=True)
"""


def run(tmp_path, program):
    """The lines that a program prints with the answering library loaded first."""
    source, shim = tmp_path / "shim.c", tmp_path / "libshim.so"
    source.write_text(SHIM)
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(shim), str(source)], check=True)
    out = subprocess.run([sys.executable, "-c", program, str(shim)], cwd=ROOT, text=True,
                         stdout=subprocess.PIPE, stderr=subprocess.PIPE, timeout=300)
    assert out.returncode == 0, out.stderr
    return out.stdout.splitlines()


def test_refused_launches_keep_the_runtimes_words(tmp_path):
    lines = [line.split(" | ") for line in run(tmp_path, CHILD)]
    assert len(lines) == 20
    for name, status, text in lines:
        assert status == "-1", name
        assert name in text and "invalid configuration" in text, (name, text)


def test_reported_errors_are_not_the_next_launches(tmp_path):
    """An allocation or wait that failed and said so leaves the next launch its own
    status."""
    assert run(tmp_path, AFTER) == ["True True 0 0"] * 3
