"""The paged key-value cache on the CPU: the pages' book-keeping against a
model of it, and every refusal that needs no device."""
import ctypes as C
import random

import numpy as np
import pytest

NULL_ARG, STATE_ALLOC = -6, -7


class Model:
    """What the book-keeping says, over the contents of the rows: every page is
    a list of rows, and a sequence reads its rows through its pages."""

    def __init__(self, n_pages, rows):
        self.rows, self.store, self.want = rows, [[None] * rows for _ in range(n_pages)], {}

    def copy(self, src, dst):
        took = [list(self.store[s]) for s in src]
        for t, d in zip(took, dst):
            self.store[d] = t

    def write(self, table, at, values):
        for i, v in enumerate(values):
            self.store[table[(at + i) // self.rows]][(at + i) % self.rows] = v

    def check(self, pages):
        for seq, want in self.want.items():
            t = pages.table(seq)
            assert pages.len(seq) == len(want) and len(t) == -(-len(want) // self.rows)
            assert [self.store[t[i // self.rows]][i % self.rows] for i in range(len(want))] == want


@pytest.mark.parametrize("seed", range(6))
def test_sequences_keep_their_rows(pkg, seed):
    """Random news, forks, extends, trims, frees and compactions: every
    sequence reads back what was written to it, pages in use are exactly those
    that a sequence has, and after a compaction they are the lowest."""
    r = random.Random(seed)
    n_pages, rows = 40, 16
    pages, m = pkg.KvPages(n_pages, rows), Model(n_pages, rows)
    stamp = 0
    for _ in range(400):
        act = r.choice(["new", "fork", "extend", "extend", "extend", "trim", "free", "compact"])
        live = list(m.want)
        if act == "new" or not live:
            m.want[pages.new()] = []
        elif act == "fork":
            s = r.choice(live)
            n = r.randint(0, len(m.want[s]))
            m.want[pages.fork(s, n)] = m.want[s][:n]
        elif act == "extend":
            s, n = r.choice(live), r.randint(0, 40)
            before, table = pages.unused(), list(pages.table(s))
            try:
                src, dst = pages.extend(s, n)
            except MemoryError:
                assert pages.unused() == before and list(pages.table(s)) == table
                continue
            m.copy(src, dst)
            new = list(range(stamp, stamp + n))
            stamp += n
            m.write(pages.table(s), len(m.want[s]), new)
            m.want[s] = m.want[s] + new
        elif act == "trim":
            s = r.choice(live)
            n = r.randint(0, len(m.want[s]))
            pages.trim(s, n)
            m.want[s] = m.want[s][:n]
        elif act == "free":
            s = r.choice(live)
            pages.free(s)
            del m.want[s]
            with pytest.raises(ValueError):
                pages.len(s)
        else:
            src, dst = pages.compact()
            assert not set(src) & set(dst) and len(set(dst)) == len(dst)
            m.copy(src, dst)
            used = {int(p) for s in m.want for p in pages.table(s)}
            assert used == set(range(n_pages - pages.unused()))
        m.check(pages)
        assert len({int(p) for s in m.want for p in pages.table(s)}) == n_pages - pages.unused()


def test_lowest_page_first_and_copy_on_write(pkg):
    p = pkg.KvPages(6, 16)
    a = p.new()
    assert p.extend(a, 20) == ([], []) and list(p.table(a)) == [0, 1]
    b = p.fork(a, 20)
    assert p.unused() == 4
    assert p.extend(b, 1) == ([1], [2]) and list(p.table(b)) == [0, 2]
    assert p.extend(a, 12) == ([], []) and list(p.table(a)) == [0, 1]      # alone on page 1 again
    c = p.fork(a, 32)
    assert p.extend(c, 1) == ([], []) and list(p.table(c)) == [0, 1, 3]    # the shared last page is full
    p.free(a)
    p.free(b)
    assert list(p.table(c)) == [0, 1, 3] and p.unused() == 3
    src, dst = p.compact()
    assert list(src) == [3] and list(dst) == [2] and list(p.table(c)) == [0, 1, 2]


def test_book_keeping_refuses(pkg):
    L = pkg.hip_lib()
    assert not L.l98_kv_pages_open(0, 16) and not L.l98_kv_pages_open(4, 24) and not L.l98_kv_pages_open(4, 8)
    h = L.l98_kv_pages_open(2, 16)
    a, b = C.c_int(), C.c_int()
    out = (C.c_int * 4)()
    try:
        s = L.l98_kv_pages_new(h)
        assert s == 0
        for bad in (-1, 1, 99):
            assert L.l98_kv_pages_len(h, bad) == NULL_ARG
            assert L.l98_kv_pages_fork(h, bad, 0) == NULL_ARG
            assert L.l98_kv_pages_extend(h, bad, 1, a, b) == NULL_ARG
            assert L.l98_kv_pages_trim(h, bad, 0) == NULL_ARG
            assert L.l98_kv_pages_free(h, bad) == NULL_ARG
            assert L.l98_kv_pages_table(h, bad, out, 4) == NULL_ARG
        assert L.l98_kv_pages_extend(h, s, 33, a, b) == STATE_ALLOC and L.l98_kv_pages_len(h, s) == 0
        assert L.l98_kv_pages_extend(h, s, 32, a, b) == 0
        assert L.l98_kv_pages_extend(h, s, 2 ** 31 - 1, a, b) == NULL_ARG
        assert L.l98_kv_pages_extend(h, s, -1, a, b) == NULL_ARG
        assert L.l98_kv_pages_fork(h, s, 33) == NULL_ARG and L.l98_kv_pages_trim(h, s, 33) == NULL_ARG
        assert L.l98_kv_pages_table(h, s, None, 0) == 2 and L.l98_kv_pages_table(h, s, None, 1) == NULL_ARG
        assert L.l98_kv_pages_compact(h, None, None, 0) == 0
        assert L.l98_kv_pages_trim(h, s, 0) == 0
        t = L.l98_kv_pages_new(h)
        assert L.l98_kv_pages_extend(h, s, 1, a, b) == 0 and L.l98_kv_pages_extend(h, t, 1, a, b) == 0
        assert L.l98_kv_pages_free(h, s) == 0
        assert L.l98_kv_pages_compact(h, None, None, 0) == NULL_ARG        # one move, no room for it
        assert L.l98_kv_pages_table(h, t, out, 4) == 1 and out[0] == 1     # and nothing has moved
    finally:
        L.l98_kv_pages_close(h)
    assert L.l98_kv_pages_new(None) == NULL_ARG and L.l98_kv_pages_unused(None) == NULL_ARG


# every refusal below comes before any use of a device: the pointers are made up
FAKE = 1 << 40


def pool_of(pkg, **kw):
    d = dict(data=FAKE, format=0, n_layers=2, n_pages=8, page_rows=16, n_kv_heads=2, head_dim=64)
    d.update(kw)
    return pkg.L98KvPool(*(d[n] for n, _ in pkg.L98KvPool._fields_))


def batch_of(pkg, **kw):
    d = dict(table=FAKE, table_stride=4, table_pages=4, kv_len=FAKE, row0=FAKE, n_seq=2, n_rows=6, max_rows=4,
             max_len=64)
    d.update(kw)
    return pkg.L98KvBatch(*(d[n] for n, _ in pkg.L98KvBatch._fields_))


def rows_of(pkg, heads=2, dim=64, **kw):
    d = dict(p=FAKE, row_stride=heads * dim, head_stride=dim)
    d.update(kw)
    return pkg.L98KvRows(d["p"], d["row_stride"], d["head_stride"])


BAD_POOLS = [dict(format=2), dict(format=-1), dict(n_layers=0), dict(n_layers=1025), dict(n_pages=0),
             dict(page_rows=8), dict(page_rows=24), dict(page_rows=2048), dict(n_kv_heads=0), dict(n_kv_heads=1025),
             dict(head_dim=96), dict(head_dim=256), dict(head_dim=16)]
BAD_BATCHES = [dict(n_seq=-1), dict(n_seq=65536), dict(n_rows=-1), dict(max_rows=-1), dict(max_len=-1),
               dict(table_pages=-1), dict(table_stride=-1)]


def test_calls_refuse(pkg):
    L = pkg.hip_lib()
    err = C.create_string_buffer(200)
    ok, pool, rows = batch_of(pkg), pool_of(pkg), rows_of(pkg)
    q = rows_of(pkg, heads=8)

    def append(p=pool, layer=0, b=ok, k=rows, v=rows, dt=0, fn=L.l98_kv_append):
        return fn(p, layer, b, k, v, dt, None, err, 200)

    def attend(p=pool, layer=0, b=ok, q=q, out=q, heads=8, dt=0, scale=0.125, ws_bytes=1 << 30):
        return L.l98_kv_attend(p, layer, b, q, out, heads, dt, scale, FAKE, ws_bytes, None, err, 200)

    for bad in BAD_POOLS:
        p = pool_of(pkg, **bad)
        assert L.l98_kv_page_bytes(p) == NULL_ARG, bad
        assert append(p=p) == NULL_ARG and append(p=p, fn=L.l98_kv_read) == NULL_ARG and attend(p=p) == NULL_ARG
        assert L.l98_kv_attend_ws_bytes(p, ok, 8, 0) == NULL_ARG
        assert b"pool" in err.value
    for layer in (-1, 2):
        assert append(layer=layer) == NULL_ARG and attend(layer=layer) == NULL_ARG
    for bad in BAD_BATCHES:
        b = batch_of(pkg, **bad)
        assert append(b=b) == NULL_ARG and append(b=b, fn=L.l98_kv_read) == NULL_ARG and attend(b=b) == NULL_ARG, bad
        assert L.l98_kv_attend_ws_bytes(pool, b, 8, 0) == NULL_ARG
    for dt in (-1, 2):
        assert append(dt=dt) == NULL_ARG and attend(dt=dt) == NULL_ARG
        assert L.l98_kv_attend_ws_bytes(pool, ok, 8, dt) == NULL_ARG
    for heads in (0, -2, 3, 34):
        assert attend(heads=heads) == NULL_ARG and L.l98_kv_attend_ws_bytes(pool, ok, heads, 0) == NULL_ARG
    for scale in (float("inf"), float("nan")):
        assert attend(scale=scale) == NULL_ARG
    for bad in (dict(row_stride=-1), dict(head_stride=-64)):
        assert append(k=rows_of(pkg, **bad)) == NULL_ARG and append(v=rows_of(pkg, **bad)) == NULL_ARG
        assert attend(q=rows_of(pkg, **bad)) == NULL_ARG
    for bad in (dict(row_stride=0), dict(head_stride=0), dict(head_stride=32)):   # a written row that overlaps
        assert append(k=rows_of(pkg, **bad), fn=L.l98_kv_read) == NULL_ARG
        assert attend(out=rows_of(pkg, heads=8, **bad)) == NULL_ARG
    # a call without rows is done before it looks at any pointer
    for none in (dict(n_seq=0), dict(n_rows=0), dict(max_rows=0)):
        b = batch_of(pkg, **none)
        assert append(b=b) == 0 and append(b=b, fn=L.l98_kv_read) == 0 and attend(b=b) == 0
        assert L.l98_kv_attend_ws_bytes(pool, b, 8, 0) == 0
    big = batch_of(pkg, n_seq=1, n_rows=8, max_rows=8, max_len=200000, table_pages=20000, table_stride=20000)
    need = L.l98_kv_attend_ws_bytes(pool, big, 8, 1)
    if need:
        assert attend(b=big, dt=1, ws_bytes=need - 1) == NULL_ARG and b"workspace" in err.value


def test_calls_refuse_sizes(pkg):
    """Bounds that the kernels cannot count, scales beyond fp32, and written
    rows and heads that lie in each other; layouts that do not are taken (they
    get as far as the pointers, which are made up)."""
    L = pkg.hip_lib()
    err = C.create_string_buffer(200)
    pool, ok = pool_of(pkg, n_pages=1 << 20), batch_of(pkg)

    def attend(b=ok, out=None, scale=0.125):
        return L.l98_kv_attend(pool, 0, b, rows_of(pkg, heads=8), out or rows_of(pkg, heads=8), 8, 0, scale, FAKE, 1 << 40,
                               None, err, 200)

    far = batch_of(pkg, max_len=2 ** 31 - 1, table_pages=1 << 27, table_stride=1 << 27)
    assert attend(b=far) == NULL_ARG and b"positions" in err.value
    assert L.l98_kv_attend_ws_bytes(pool, far, 8, 0) == NULL_ARG
    lazy = batch_of(pkg, max_len=2 ** 31 - 1)             # the table's end is the bound
    for dt in (0, 1):
        assert L.l98_kv_attend_ws_bytes(pool, lazy, 8, dt) == L.l98_kv_attend_ws_bytes(pool, ok, 8, dt) >= 0
    for scale in (1e38, -3e38):
        assert attend(scale=scale) == NULL_ARG and b"scale" in err.value
    for row, head in ((64, 64), (128, 64), (511, 64), (64, 383), (600, 100), (0, 512), (2 ** 62, 2 ** 62)):
        assert attend(out=rows_of(pkg, row_stride=row, head_stride=head)) == NULL_ARG and b"overlap" in err.value, (row, head)
    for row, head in ((512, 64), (64, 384), (1024, 128), (2 ** 61, 64), (128, 768)):
        assert attend(out=rows_of(pkg, row_stride=row, head_stride=head)) != 0 and b"overlap" not in err.value, (row, head)


def test_copy_refuses(pkg):
    L = pkg.hip_lib()
    err = C.create_string_buffer(200)

    def copy(src, dst, p=pool_of(pkg)):
        a, b = np.array(src, np.int32), np.array(dst, np.int32)
        return L.l98_kv_copy_pages(p, a.ctypes.data_as(pkg._IP), b.ctypes.data_as(pkg._IP), len(src), None, err, 200)

    assert copy([], []) == 0
    for src, dst in (([8], [0]), ([0], [8]), ([-1], [0]), ([0], [-1]), ([0, 1], [2, 2]), ([0], [0]), ([0, 2], [2, 3]),
                     ([0, 1, 2], [3, 4, 1]), (list(range(8)) + [0], list(range(8)) + [0])):
        assert copy(src, dst) == NULL_ARG, (src, dst)
    assert copy([0], [1], pool_of(pkg, head_dim=48)) == NULL_ARG
    assert L.l98_kv_copy_pages(pool_of(pkg), None, None, 1, None, err, 200) == NULL_ARG
    assert L.l98_kv_copy_pages(None, None, None, 0, None, err, 200) == NULL_ARG


def test_page_bytes(pkg):
    L = pkg.hip_lib()
    assert L.l98_kv_page_bytes(pool_of(pkg)) == 2 * 2 * (2 * 16 * 64 + 2 * 16 * 2 * 4)
    assert L.l98_kv_page_bytes(pool_of(pkg, format=1, n_layers=1)) == 2 * 2 * 16 * 64 * 2
    assert pkg.KvPool.page_bytes_of("q8", 64, 4, 128) == 2 * (4 * 64 * 128 + 4 * 64 * 4 * 4)


def test_python_layer_refuses(pkg):
    import torch
    with pytest.raises(ValueError, match="format"):
        pkg.KvPool(torch.zeros(1 << 16, dtype=torch.uint8), "q4", 16, 1, 64)
    with pytest.raises(ValueError, match="limits"):
        pkg.KvPool(torch.zeros(1 << 16, dtype=torch.uint8), "q8", 12, 1, 64)
    with pytest.raises(ValueError, match="GPU"):
        pkg.KvPool(torch.zeros(1 << 16, dtype=torch.uint8), "q8", 16, 1, 64)
    i32 = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="table"):
        pkg.KvBatch(torch.zeros(2, 4, dtype=torch.int32), i32[:2], i32, 2, 1, 64)
    with pytest.raises(ValueError):
        pkg.KvPages(0, 16)
