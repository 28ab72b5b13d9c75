"""Entry points of several host threads at once; no GPU."""
import threading

from tbf16 import _ext


def test_workspace_sizes_from_many_threads():
    """What the library keeps per device and per thread is asked for by all of them at the same time."""
    L = _ext.lib()
    shapes = [(M, K, N) for M in (1, 17, 300, 5000) for K in (64, 1000, 4096) for N in (8, 1000, 20000)]

    def ask():
        return [(L.tbf16_linear_i8_ws_bytes(*s), L.tbf16_paged_attn_ws_bytes(s[0], 32, 8, 128, s[2])) for s in shapes]

    got = [None] * 16
    gate = threading.Barrier(len(got))

    def work(i):
        gate.wait()
        got[i] = [ask() for _ in range(20)]

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(got))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    want = ask()
    assert all(g == [want] * 20 for g in got)
