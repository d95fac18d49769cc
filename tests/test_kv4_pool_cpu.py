"""The page pool behind the C entries over a long time."""
import os

from test_kv4_cpu import pool  # noqa: F401  (fixture)


def resident():
    with open("/proc/self/statm") as f:
        return int(f.read().split()[1]) * os.sysconf("SC_PAGE_SIZE")


def test_memory_stays_as_it_is(pool):  # noqa: F811
    """a server's life: a long prefix forked, written to and closed again and again, the pool compacted"""
    p = pool(16384, 4, 8192)
    a = p("open")
    assert p("grow", a, 64 * 8000) == 0

    def turn():
        b = p("fork", a, 64 * 8000)
        assert b >= 0 and p("own", b, 64 * 7990, 16)[0] == 10 and p("grow", b, 64 * 8100) == 0
        assert p("drop", b, 64 * 100, 64 * 7000) == 0 and p("close", b) == 0
        c = p("open")
        assert p("grow", c, 64 * 50) == 0
        assert p("compact", 100) == (0, []) and p("close", c) == 0

    for _ in range(50):
        turn()
    before = resident()
    for _ in range(4000):                                   # (one entry of 8 bytes per page and turn would be 262 MB)
        turn()
    assert resident() - before < 16 << 20 and p("free_pages") == 16384 - 8000
