"""The paged key-value cache on the GPU against its definition in 64 bits.

Tolerances, u = 2^-24 (half a step of fp32, relative), B = 2^-8 (of bf16),
H = 2^-11 (of fp16), for a row with n keys, of width D:

* a score's error: its D products and sums and the scaling, each within u of
  the partial sums, so at most (D + 8) u a with a = max_j |scale| sum_d |q k_j|;
  a bf16 row over a Q8 cache may round the cache's numbers to fp16 (H a more);
* a weight exp(s - m) then is off by twice that (s and m), and by 4 u (|s| + |m|)
  <= 8 u a of the exponent's own arithmetic, all relative; a bf16 row may round
  it to bf16 (B more), and the cache's V to fp16 (H more);
* numerator and denominator are sums of n terms in fp32: at most (n + 64) u each
  of the sum of absolute values;
* a weight is held with a fixed absolute step below some size: for bf16 rows
  over a Q8 cache that of fp16's smallest numbers, at most 2^-25 of the largest
  weight; else at most 2^-38 of it (fp32 itself keeps 2^-126: a value that only
  such weights make up has no relative bound);
* the division and the output's rounding: 2 u of the result, B more for bf16.

So with r = 2 ((D + 16) u + [bf16, q8] H) a + 2 (n + 64) u + [bf16] (2 B + H) the
output is within 2 r sum_j p_j |v_j| + 2 n (2^-38 or 2^-25) max|v| p_max (both
over what the row attends) +
([bf16] B + 2 u) |o|: the weights enter the numerator and the denominator.
"""
import threading

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U, B, H = 2.0 ** -24, 2.0 ** -8, 2.0 ** -11
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
DEV = "cuda"


def say(*a):
    print("[case]", *a, flush=True)


def k_order(d):
    """the dimension at each byte of a Q8 K row"""
    o = np.zeros(d, np.int64)
    for c in range(d // 32):
        for h in range(4):
            for j in range(8):
                o[h * (d // 4) + c * 8 + j] = c * 32 + h * 8 + j
    return o


def v_order(d):
    o = np.zeros(d, np.int64)
    for n in range(16):
        for t in range(d // 16):
            o[n * (d // 16) + t] = t * 16 + n
    return o


def quant(x):
    """codes, scales of x [..., d] by the format's fp32 rule"""
    g = x.astype(np.float32).reshape(*x.shape[:-1], -1, 32)
    am = np.abs(g).max(-1)
    s = (am * np.float32(1.0 / 127.0)).astype(np.float32)
    live = (am > 0) & ~(s < np.float32(1e-30))
    with np.errstate(divide="ignore", over="ignore", invalid="ignore"):
        inv = np.where(live, np.float32(127.0) * (np.float32(1.0) / am), np.float32(0)).astype(np.float32)
    code = np.clip(np.rint(g * inv[..., None]), -127, 127)
    return code, np.where(live, s, np.float32(1)).astype(np.float32)


def bf16(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(torch.bfloat16)


class Cache:
    """A pool whose every byte is 0xFF (NaN as a scale, as bf16) but for the
    rows written here, by the layout's definition."""

    def __init__(self, pkg, fmt, page, hk, dim, n_pages, layers=1, layer=0):
        self.pkg, self.fmt, self.page, self.hk, self.dim, self.layer = pkg, fmt, page, hk, dim, layer
        nbytes = pkg.KvPool.page_bytes_of(fmt, page, hk, dim, layers)
        self.bytes = np.full((n_pages, layers, nbytes // layers), 0xFF, np.uint8)
        self.layers, self.n_pages = layers, n_pages

    def put(self, pid, off, k, v):
        """row `off` of page pid: k, v [hk, dim]; returns the numbers held"""
        blk = self.bytes[pid, self.layer]
        hk, dim, page = self.hk, self.dim, self.page
        n = hk * page * dim
        if self.fmt == "bf16":
            out = []
            for w, x in enumerate((k, v)):
                b = bf16(x)
                blk[w * 2 * n:(w + 1) * 2 * n].view(np.int16).reshape(hk, page, dim)[:, off] = b.view(torch.int16).numpy()
                out.append(b.double().numpy())
            return out
        out = []
        for w, (x, order) in enumerate(((k, k_order(dim)), (v, v_order(dim)))):
            c, s = quant(x)
            blk[w * n:(w + 1) * n].reshape(hk, page, dim)[:, off] = (c.reshape(hk, dim)[:, order] + 128).astype(np.uint8)
            blk[2 * n:].view(np.float32).reshape(2, hk, dim // 32, page)[w, :, :, off] = s
            out.append((c.astype(np.float64) * s[..., None].astype(np.float64)).reshape(hk, dim))
        return out

    def pool(self):
        self.t = torch.from_numpy(self.bytes.reshape(-1).copy()).to(DEV)
        return self.pkg.KvPool(self.t, self.fmt, self.page, self.hk, self.dim, n_layers=self.layers)


class Problem:
    """lens: (new rows, length) of each sequence; holes: {(sequence, page number): id put in the table}."""

    def __init__(self, pkg, fmt, dt, heads, hk, dim, page, lens, seed, holes=None, layers=1, layer=0, spare=3, sharp=1.0,
                 behind=2):
        r = np.random.default_rng(seed)
        self.pkg, self.fmt, self.dt, self.heads, self.hk, self.dim, self.page = pkg, fmt, dt, heads, hk, dim, page
        self.lens = lens
        need = [-(-n // page) for _, n in lens]
        n_pages = sum(need) + spare
        ids = list(r.permutation(n_pages))
        self.cache = Cache(pkg, fmt, page, hk, dim, n_pages, layers, layer)
        width = max(need + [1])
        table = np.full((len(lens), width), -7, np.int32)
        self.kv = []                                  # per sequence: K, V [len, hk, dim], which exist [len]
        for i, (_, n) in enumerate(lens):
            k = r.standard_normal((n, hk, dim))
            v = r.standard_normal((n, hk, dim)) * (0.3 + np.abs(r.standard_normal((1, hk, dim)))) + 0.2
            there = np.ones(n, bool)
            hk_, hv = np.zeros_like(k), np.zeros_like(v)
            for p in range(need[i]):
                table[i, p] = ids.pop()
                for off in range(min(page, n - p * page)):
                    a = p * page + off
                    hk_[a], hv[a] = self.cache.put(table[i, p], off, k[a], v[a])
                if holes and (i, p) in holes:
                    there[p * page:(p + 1) * page] = False
                    table[i, p] = holes[i, p]
            self.kv.append((hk_, hv, there))
        rows = [a for a, _ in lens]
        self.row0 = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.n_rows = int(self.row0[-1])
        self.max_rows, self.max_len = max(rows), max([n for _, n in lens] + [1])
        self.table = torch.from_numpy(table).to(DEV)
        self.kv_len = torch.tensor([n for _, n in lens], dtype=torch.int32, device=DEV)
        self.row0_d = torch.from_numpy(self.row0).to(DEV)
        self.batch = pkg.KvBatch(self.table, self.kv_len, self.row0_d, self.n_rows, self.max_rows, self.max_len)
        q = torch.from_numpy(r.standard_normal((self.n_rows + behind, heads, dim)) * 1.25).to(DT[dt])
        self.q = q.to(DEV)
        self.scale = sharp / np.sqrt(dim)

    def reference(self, q=None):
        """(out, bound) [rows, heads, dim] in 64 bits"""
        q = (self.q if q is None else q).double()
        out = torch.zeros(self.n_rows, self.heads, self.dim, dtype=torch.float64, device=DEV)
        tol = torch.zeros_like(out)
        bf, g = self.dt == "bf16", self.heads // self.hk
        for i, (rows, n) in enumerate(self.lens):
            if rows == 0 or n == 0:
                continue
            k, v, there = (torch.from_numpy(x).to(DEV) for x in self.kv[i])
            pos = torch.arange(n - rows, n, device=DEV)
            seen = (torch.arange(n, device=DEV)[None] <= pos[:, None]) & there[None]
            for h in range(self.heads):
                kh, vh, qh = k[:, h // g], v[:, h // g], q[self.row0[i]:self.row0[i + 1], h]
                s = torch.where(seen, qh @ kh.T * self.scale, -torch.inf)
                a = torch.where(seen, qh.abs() @ kh.abs().T * abs(self.scale), 0.0).amax(1)
                m = s.amax(1, keepdim=True)
                p = torch.where(seen, torch.exp(s - torch.where(torch.isinf(m), 0.0, m)), 0.0)
                l = p.sum(1, keepdim=True)
                p = p / torch.where(l == 0, 1.0, l)
                o = p @ vh
                r = (2 * ((self.dim + 16) * U + (H if bf and self.fmt == "q8" else 0)) * a + 2 * (n + 64) * U +
                     ((2 * B + H) if bf else 0))
                out[self.row0[i]:self.row0[i + 1], h] = o
                largest = torch.where(seen, vh.abs().amax(1), 0.0).amax(1)[:, None]      # of V that the row attends
                low = 2 * n * (2.0 ** -25 if bf and self.fmt == "q8" else 2.0 ** -38) * p.amax(1)[:, None] * largest
                tol[self.row0[i]:self.row0[i + 1], h] = (2 * r[:, None] * (p @ vh.abs()) + low +
                                                         ((B if bf else 0) + 2 * U) * o.abs())
        return out, tol

    def ws(self, pool, q=None):
        n = pool.attend_ws_bytes(self.batch, self.q if q is None else q)
        return torch.full((n,), 0xFF, dtype=torch.uint8, device=DEV)

    def run(self, pool=None, out=None, q=None, **kw):
        pool = pool or self.cache.pool()
        q = self.q if q is None else q
        out = torch.full_like(q, 77.0) if out is None else out
        pool.attend(self.batch, q, out, self.scale, self.ws(pool, q), layer=self.cache.layer, **kw)
        torch.cuda.synchronize()
        return out

    def check(self, out, q=None):
        want, tol = self.reference(q)
        d = (out[:self.n_rows].double() - want).abs()
        worst = float((d / tol.clamp(min=1e-300)).nan_to_num(nan=1e9).max()) if d.numel() else 0.0
        if d.numel():
            bad = ~(d <= tol)
            assert not bool(bad.any()), f"{int(bad.sum())} values off, worst {worst:.3g} times the bound"
            rms = float((d.square().mean() / want.square().mean().clamp(min=1e-300)).sqrt())
            say(f"worst {worst:.3g} of the bound, rms {rms:.3g}")
        assert bool((out[self.n_rows:] == 77.0).all()), "rows behind the last sequence were written"


FEW = [(1, 1), (4, 60), (0, 50), (1, 0), (3, 1), (2, 129), (8, 333), (1, 16), (5, 64), (1, 700)]
PROMPT = [(70, 70), (1, 200), (130, 147), (0, 0), (257, 321), (9, 9), (2, 0), (40, 33)]
SHAPES = [(16, 4, 128), (16, 4, 64), (4, 2, 64), (2, 1, 32), (3, 3, 128), (16, 1, 64), (7, 1, 32)]


@pytest.mark.parametrize("heads,hk,dim", SHAPES)
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("fmt", ["q8", "bf16"])
def test_attend(pkg, fmt, dt, heads, hk, dim):
    """Batches of few rows and of prompts: lengths of zero and one, rows with
    no position (length below the rows), empty sequences, pages that end
    inside a tile; everything unused is NaN."""
    for n, (lens, page) in enumerate(((FEW, 16), (FEW, 64), (PROMPT, 32), (PROMPT, 256), ([(1, 5)], 16), ([(1, 1)], 1024))):
        p = Problem(pkg, fmt, dt, heads, hk, dim, page, lens, seed=n)
        say("attend", fmt, dt, heads, hk, dim, page, lens)
        p.check(p.run())


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("fmt", ["q8", "bf16"])
def test_attend_long(pkg, fmt, dt):
    """Contexts that are split: one sequence among short ones, and long
    prefixes before a chunk of rows."""
    for lens, page in (([(3, 40011), (1, 17), (8, 9000)], 128), ([(100, 9100)], 64), ([(20, 20000), (33, 33)], 32),
                       ([(150, 9100), (1, 5)], 64)):
        say("long", fmt, dt, lens)
        p = Problem(pkg, fmt, dt, 8, 2, 64, page, lens, seed=len(lens))
        p.check(p.run())


@pytest.mark.parametrize("sharp", [0.0, 8.0, -3.0, 300.0])
def test_attend_scales(pkg, sharp):
    """A scale of zero (the mean), negative, and so large that one key takes all."""
    for fmt, dt, lens in (("q8", "bf16", [(90, 300)]), ("bf16", "f32", [(4, 300)]), ("q8", "f32", [(4, 900), (64, 64)]),
                          ("bf16", "bf16", [(3, 1000), (200, 200)]), ("q8", "bf16", [(1300, 1300), (64, 64)]),
                          ("bf16", "bf16", [(1300, 1300), (64, 64)])):
        say("scale", sharp, fmt, dt, lens)
        p = Problem(pkg, fmt, dt, 4, 1, 64, 16, lens, seed=5, sharp=sharp)
        p.check(p.run())


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("fmt", ["q8", "bf16"])
def test_holes(pkg, fmt, dt):
    """Table entries outside the pool: their rows are attended by nobody, a
    row whose every page is one gets zeros."""
    lens = [(4, 100), (60, 70), (1, 30), (2, 200)]
    holes = {(0, 0): -1, (0, 3): 10 ** 6, (1, 2): -2 ** 31, (2, 0): -1, (2, 1): 2 ** 31 - 1, (3, 12): -1}
    for page in (16,):
        say("holes", fmt, dt)
        p = Problem(pkg, fmt, dt, 8, 2, 64, page, lens, seed=9, holes=holes)
        out = p.run()
        p.check(out)
        assert bool((out[64] == 0).all())


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("fmt", ["q8", "bf16"])
@pytest.mark.parametrize("lens", [[(8, 108)], [(150, 190)], [(2000, 2040)]])
def test_nonfinite_rows_ahead(pkg, fmt, dt, lens):
    """Infinities and NaN in K and V at a position: the rows before it are
    what they are without it, bit for bit, the rows that attend it are not finite."""
    rows, n = lens[0]
    at = n - rows // 2 - 1
    p = Problem(pkg, fmt, dt, 4, 2, 64, 16, lens, seed=3)
    clean = p.run()
    p.check(clean)
    before = rows - (n - at)
    pid = int(p.table[0, at // 16])
    blk = p.cache.bytes[pid, 0]
    for bad in (np.inf, -np.inf, np.nan):
        for w in (0, 1):
            say("nonfinite", fmt, dt, lens, bad, "KV"[w])
            keep = blk.copy()
            if fmt == "bf16":
                blk.view(np.int16).reshape(2, 2, 16, 64)[w, :, at % 16, 5] = bf16(np.array([bad])).view(torch.int16).numpy()[0]
            else:
                blk[2 * 2 * 16 * 64:].view(np.float32).reshape(2, 2, 2, 16)[w, :, 1, at % 16] = bad
            out = p.run()
            blk[:] = keep
            assert torch.equal(out[:before], clean[:before])
            if w == 1 or not np.isinf(bad):        # a score of -inf or +inf may leave a finite row
                assert not bool(torch.isfinite(out[before:p.n_rows]).all(-1).any())
            assert bool((out[p.n_rows:] == 77.0).all())


BATCH = [(130, 130 + 37 * (i % 5)) if i % 4 else (i % 7 * 3, i % 7 * 11) for i in range(32)]


@pytest.mark.parametrize("heads,hk,dim,lens", [(16, 4, 32, PROMPT), (20, 4, 64, PROMPT), (28, 4, 128, PROMPT),
                                               (8, 8, 64, [(600, 640), (1, 700), (513, 513), (5, 9)]),
                                               (7, 1, 128, [(300, 3000), (1, 1), (130, 2500)])])
@pytest.mark.parametrize("fmt", ["q8", "bf16"])
def test_attend_some_prompts(pkg, fmt, heads, hk, dim, lens):
    """Prompts that are few, in blocks of 128 rows: whole and split, odd groups."""
    say("some prompts", fmt, heads, hk, dim, lens)
    for page in (16, 128):
        p = Problem(pkg, fmt, "bf16", heads, hk, dim, page, lens, seed=page)
        p.check(p.run())


@pytest.mark.parametrize("heads,hk,dim", [(16, 4, 128), (20, 4, 64), (4, 4, 32)])
@pytest.mark.parametrize("fmt", ["q8", "bf16"])
def test_attend_many_prompts(pkg, fmt, heads, hk, dim):
    """Enough rows for a block of 256 each on every CU: batches of prompts of
    odd lengths with empty ones and single rows between, and with holes."""
    say("many prompts", fmt, heads, hk, dim)
    lens = BATCH if heads > 4 else [(a * 4, n + 3 * a) for a, n in BATCH]
    for page, holes in ((16, None), (64, {(3, 0): -1, (5, 1): 2 ** 31 - 1, (9, 2): 10 ** 6})):
        p = Problem(pkg, fmt, "bf16", heads, hk, dim, page, lens, seed=page, holes=holes)
        p.check(p.run())
        assert torch.equal(p.run(), p.run())


def test_attend_prompts_by_groups(pkg):
    """A table and a bound of the lengths so large that the batch goes through
    its workspace in two groups."""
    say("groups")
    lens = [(60, 60), (1, 900), (0, 0), (40, 700), (33, 34), (70, 300)]
    p = Problem(pkg, "q8", "bf16", 16, 4, 128, 64, lens, seed=6)
    table = torch.full((len(lens), 2048), -1, dtype=torch.int32, device=DEV)
    table[:, :p.table.shape[1]] = p.table
    p.batch = pkg.KvBatch(table, p.kv_len, p.row0_d, p.n_rows, p.max_rows, 131072)
    p.check(p.run())


@pytest.mark.parametrize("fmt", ["q8", "bf16"])
@pytest.mark.parametrize("lens", [[(8, 108)], [(150, 190)], [(150, 190)] * 80, [(2000, 2040)]],
                         ids=["few", "prompt", "prompts", "long prompt"])
def test_huge_rows_ahead(pkg, fmt, lens):
    """Finite K or V of 1e30 at a position, and from there on: a row before it
    does not notice, one that attends it has what the formula says."""
    for dt in ("f32", "bf16"):
        rows, n = lens[0]
        p = Problem(pkg, fmt, dt, 4, 2, 64, 16, lens, seed=3)
        for at, to in ((n - rows // 2 - 1, n - rows // 2), (n - 5, n - 4), (n - rows // 2 - 1, n)):
            for w in (0, 1):
                say("huge", fmt, dt, lens[0], at, to, "KV"[w])
                held = p.cache.bytes.copy(), [tuple(x.copy() for x in y) for y in p.kv]
                r = np.random.default_rng(at)
                for i in range(len(lens)):
                    for a in range(at, to):
                        kv = [x[a] for x in p.kv[i][:2]]
                        kv[w] = r.standard_normal(kv[w].shape) * 1e30
                        got = p.cache.put(int(p.table[i, a // 16]), a % 16, *kv)
                        p.kv[i][w][a] = got[w]
                p.check(p.run())
                p.cache.bytes, p.kv = held


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("lens", [[(150, 560)], [(2, 560)], [(1500, 1560)]])
def test_ranges_of_the_scales(pkg, dt, lens):
    """Q8 values whose size changes from tile to tile and inside one, by 2^-20
    to 2^20, up, down and to zero."""
    for pattern in ([20, -20], [-20, 20], [0, -12, -6, 18, -18], [-20, None, 3], [-90, -60, -20]):
        for run in (64, 16, 5):
            say("ranges", dt, lens, pattern, run)
            p = Problem(pkg, "q8", dt, 4, 2, 64, 16, lens, seed=run)
            k, v, _ = p.kv[0]
            for a in range(len(v)):
                e = pattern[a // run % len(pattern)]
                k[a], v[a] = p.cache.put(int(p.table[0, a // 16]), a % 16, k[a], v[a] * (0.0 if e is None else 2.0 ** e))
            p.check(p.run())


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("fmt", ["q8", "bf16"])
@pytest.mark.parametrize("lens", [[(2, 30000)], [(100, 9100)], [(150, 9100)]])
def test_nan_in_a_whole_split(pkg, fmt, dt, lens):
    """Keys that are all NaN over more than a split's range reach every row."""
    say("nan split", fmt, dt, lens)
    p = Problem(pkg, fmt, dt, 8, 2, 64, 1024, lens, seed=4)
    for page in range(1, 6):
        blk = p.cache.bytes[int(p.table[0, page]), 0]
        if fmt == "bf16":
            blk.view(np.int16).reshape(2, 2, 1024, 64)[0, :, :, 7] = bf16(np.array([np.nan])).view(torch.int16).numpy()[0]
        else:
            blk[2 * 2 * 1024 * 64:].view(np.float32).reshape(2, 2, 2, 1024)[0, :, 1] = np.nan
    out = p.run()
    assert bool(out[:p.n_rows].isnan().all()) and bool((out[p.n_rows:] == 77.0).all())


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 90])
def test_no_keys(pkg, dt, rows):
    """A table of no pages, a bound of no positions, lengths of zero and below:
    the rows are zeros, the others untouched; a bound without an end is the table's."""
    say("no keys", dt, rows)
    p = Problem(pkg, "q8", dt, 8, 2, 64, 16, [(rows, rows + 30), (0, 0), (rows, 2 * rows)], seed=rows)
    pool = p.cache.pool()
    full = p.run(pool)
    none = torch.empty(3, 0, dtype=torch.int32, device=DEV)
    for table, kv_len, max_len in ((none, p.kv_len, p.max_len), (p.table, p.kv_len, 0), (p.table, p.kv_len * 0, p.max_len),
                                   (p.table, p.kv_len - 1000, p.max_len)):
        p.batch = pkg.KvBatch(table, kv_len, p.row0_d, p.n_rows, p.max_rows, max_len)
        out = torch.full_like(p.q, 77.0)
        need = pool.attend_ws_bytes(p.batch, p.q)
        pool.attend(p.batch, p.q, out, p.scale, torch.empty(need, dtype=torch.uint8, device=DEV) if need else None)
        torch.cuda.synchronize()
        assert bool((out[:p.n_rows] == 0).all()) and bool((out[p.n_rows:] == 77.0).all())
        k = torch.full((p.n_rows, 2, 64), 5.0, device=DEV)
        v = k.clone()
        before = pool.data.clone()
        pool.append(p.batch, k, v)
        pool.read(p.batch, k, v)
        torch.cuda.synchronize()
        assert torch.equal(pool.data, before) and bool((k == 0).all()) and bool((v == 0).all())
    p.batch = pkg.KvBatch(p.table, p.kv_len, p.row0_d, p.n_rows, p.max_rows, 2 ** 31 - 1)
    p.check(p.run(pool))
    with pytest.raises(ValueError, match="contiguous"):
        pool.attend(p.batch, p.q, full, p.scale, torch.empty(1 << 20, 2, dtype=torch.uint8, device=DEV)[:, 0])


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("lens", [FEW, PROMPT, PROMPT * 2])
def test_strides_and_alignment(pkg, dt, lens):
    """q and out as slices of wider and of odd arrays, heads before rows, out
    in q's place: the same bits as the contiguous call's."""
    p = Problem(pkg, "q8", dt, 8, 2, 64, 32, lens, seed=21)
    pool = p.cache.pool()
    want = p.run(pool)
    n, e = p.q.shape[0], 8 * 64

    def wide(pad, off):
        flat = torch.zeros(n * (e + pad) + off + 8, dtype=DT[dt], device=DEV)
        return flat[off:off + n * (e + pad)].view(n, e + pad)[:, :e].view(n, 8, 64)

    for kind in ("odd", "wide", "heads first", "gated"):
        say("strides", kind, dt)
        if kind == "heads first":
            q, out = (torch.zeros(8, n, 64, dtype=DT[dt], device=DEV).transpose(0, 1) for _ in range(2))
        elif kind == "gated":                      # [q | gate] of each head, as the model projects them
            q, out = (torch.zeros(n, 8, 128, dtype=DT[dt], device=DEV)[..., :64] for _ in range(2))
        else:
            q, out = (wide(3, 1) if kind == "odd" else wide(64, 0) for _ in range(2))
        q.copy_(p.q)
        out.fill_(77.0)
        assert torch.equal(p.run(pool, out, q), want)
    q = p.q.clone()
    got = p.run(pool, q, q)
    assert torch.equal(got[:p.n_rows], want[:p.n_rows]) and torch.equal(got[p.n_rows:], p.q[p.n_rows:])


def test_bounds_of_the_call(pkg):
    """max_rows, max_len and n_rows below what the arrays say: rows past them
    are left alone, positions past them are not attended."""
    say("bounds")
    p = Problem(pkg, "q8", "f32", 4, 2, 64, 16, [(8, 50), (3, 20)], seed=2)
    pool = p.cache.pool()
    full = p.run(pool)
    for n_rows, max_rows, max_len in ((9, 8, 50), (11, 2, 50), (11, 8, 20), (0, 8, 50), (11, 0, 50)):
        b = pkg.KvBatch(p.table, p.kv_len, p.row0_d, n_rows, max_rows, max_len)
        out = torch.full_like(p.q, 77.0)
        ws = torch.empty(pool.attend_ws_bytes(b, p.q), dtype=torch.uint8, device=DEV)
        pool.attend(b, p.q, out, p.scale, ws)
        torch.cuda.synchronize()
        for i, (r0, rows) in enumerate(((0, 8), (8, 3))):
            for j in range(rows):
                if j >= max_rows or r0 + j >= n_rows:
                    assert bool((out[r0 + j] == 77.0).all()), (n_rows, max_rows, i, j)
                elif max_len >= 50 or i == 1:
                    assert torch.allclose(out[r0 + j], full[r0 + j], rtol=1e-4, atol=1e-5)
                else:
                    assert bool(torch.isfinite(out[r0 + j]).all())


@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("fmt", ["q8", "bf16"])
def test_append_and_read(pkg, fmt, dt, dim):
    """Appended rows' bytes are the layout's definition, nothing else in the
    pool changes, and read gives the numbers back (zeros without a page)."""
    r = np.random.default_rng(dim)
    hk, page, layers, layer = 3, 16, 3, 1
    lens = [(5, 21), (0, 9), (16, 16), (1, 1), (33, 70), (4, 2)]
    say("append", fmt, dt, dim)
    p = Problem(pkg, fmt, dt, hk, hk, dim, page, lens, seed=1, layers=layers, layer=layer,
                holes={(4, 3): -1, (2, 0): 10 ** 7})
    pool = p.cache.pool()
    before = p.cache.bytes.copy()
    k, v = (torch.from_numpy(r.standard_normal((p.n_rows + 2, hk, dim)) * 3).to(DT[dt]) for _ in range(2))
    k[0, 0, :32], v[1, 1, :32] = 0.0, 1e-35           # groups of zeros, and below the smallest scale
    k[2, 2, 3] = 1e30
    table, want = p.table.cpu().numpy(), torch.zeros(p.n_rows, 2, hk, dim, dtype=torch.float64)
    for i, (rows, n) in enumerate(lens):
        for j in range(rows):
            pos = n - rows + j
            if pos < 0 or not 0 <= table[i, pos // page] < p.cache.n_pages:
                continue
            at = p.row0[i] + j
            held = p.cache.put(table[i, pos // page], pos % page, k[at].float().numpy(), v[at].float().numpy())
            want[at] = torch.from_numpy(np.stack(held))
    for order in ("rows", "odd"):
        if order == "odd":
            big = torch.zeros(p.n_rows + 2, 2, hk + 1, dim + 1, dtype=DT[dt], device=DEV)
            kd, vd = big[:, 0, :hk, 1:], big[:, 1, :hk, 1:]
            kd.copy_(k), vd.copy_(v)
        else:
            kd, vd = k.to(DEV), v.to(DEV)
        pool.data.copy_(torch.from_numpy(before.reshape(-1)))
        pool.append(p.batch, kd, vd, layer=layer)
        torch.cuda.synchronize()
        assert np.array_equal(pool.data.cpu().numpy(), p.cache.bytes.reshape(-1)), order
        for od in ("f32", "bf16"):
            ko, vo = (torch.full((p.n_rows + 2, hk, dim + 1), 77.0, dtype=DT[od], device=DEV)[..., order == "odd":][..., :dim]
                      for _ in range(2))
            pool.read(p.batch, ko, vo, layer=layer)
            torch.cuda.synchronize()
            for w, o in enumerate((ko, vo)):
                x = want[:, w].float().to(DT[od])
                assert torch.equal(o[:p.n_rows].cpu(), x), (order, od, w)
                assert bool((o[p.n_rows:] == 77.0).all())


@pytest.mark.parametrize("n_seq,most,hk,dim,page", [(64, 130, 4, 128, 64), (70, 131, 4, 64, 16), (90, 100, 3, 32, 32),
                                                    (2100, 3, 5, 64, 16), (5000, 1, 3, 32, 16), (900, 12, 8, 128, 16)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("fmt", ["q8", "bf16"])
def test_append_and_read_many(pkg, fmt, dt, n_seq, most, hk, dim, page):
    """Calls of many rows against the same rows in small calls, both ways, and
    against the numbers that the format holds."""
    say("append many", fmt, dt, n_seq, most, hk, dim, page)
    r = np.random.default_rng(n_seq)
    rows = r.integers(0, most + 1, n_seq)
    rows[r.integers(n_seq)] = most
    lens = rows + r.integers(0, 40, n_seq)
    need = -(-lens // page)
    n_pages = int(need.sum()) + 3
    ids = r.permutation(n_pages).astype(np.int32)
    table = np.full((n_seq, int(need.max())), -1, np.int32)
    at = 0
    for i in range(n_seq):
        table[i, :need[i]] = ids[at:at + need[i]]
        at += need[i]
    row0 = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    n = int(row0[-1])
    t, kl, r0 = (torch.from_numpy(x.astype(np.int32)).to(DEV) for x in (table, lens, row0))
    size = pkg.KvPool.page_bytes_of(fmt, page, hk, dim)
    big = pkg.KvBatch(t, kl, r0, n, most, int(lens.max()))
    small = [pkg.KvBatch(t[i:i + 50], kl[i:i + 50], r0[i:i + 51].clone(), n, most, int(lens.max())) for i in range(0, n_seq, 50)]
    k, v = (torch.from_numpy(r.standard_normal((n, hk, dim)).astype(np.float32)).to(DT[dt]).to(DEV) for _ in range(2))
    pools = []
    for parts in ([big], small):
        pool = pkg.KvPool(torch.full((n_pages, size), 0xFF, dtype=torch.uint8, device=DEV), fmt, page, hk, dim)
        for b in parts:
            pool.append(b, k, v)
        pools.append(pool)
    torch.cuda.synchronize()
    assert torch.equal(pools[0].data, pools[1].data)
    for parts in ([big], small):
        ko, vo = (torch.full((n + 2, hk, dim), 77.0, device=DEV) for _ in range(2))
        for b in parts:
            pools[0].read(b, ko, vo)
        torch.cuda.synchronize()
        for x, o in ((k, ko), (v, vo)):
            if fmt == "bf16":
                want = x.to(torch.bfloat16).float()
            else:
                code, scale = quant(x.float().cpu().numpy())
                want = torch.from_numpy((code.astype(np.float32) * scale[..., None]).reshape(n, hk, dim)).to(DEV)
            assert torch.equal(o[:n], want) and bool((o[n:] == 77.0).all())


def test_append_nonfinite(pkg):
    """NaN and infinities: a Q8 group with an infinity reads back as NaN, one
    with NaN as zeros (the sessions' rule), the other groups are untouched."""
    say("append nonfinite")
    p = Problem(pkg, "q8", "f32", 1, 1, 64, 16, [(3, 3)], seed=1)
    pool = p.cache.pool()
    k, v = torch.ones(3, 1, 64, device=DEV), torch.ones(3, 1, 64, device=DEV)
    k[0, 0, 3], v[1, 0, 40] = torch.inf, torch.nan
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    pool.append(p.batch, k, v)
    pool.read(p.batch, ko, vo)
    torch.cuda.synchronize()
    assert bool(ko[0, 0, :32].isnan().all()) and bool((ko[0, 0, 32:] == 1).all()) and bool((ko[1:] == 1).all())
    assert bool((vo[1, 0, 32:] == 0).all()) and bool((vo[1, 0, :32] == 1).all()) and bool((vo[0] == 1).all())
    v[1, 0, 32:] = torch.tensor([0x7FC00055, 0x7F800001], dtype=torch.int32, device=DEV).view(torch.float32).repeat(16)
    pool.append(p.batch, k, v)                       # NaN with other bits
    pool.read(p.batch, ko, vo)
    torch.cuda.synchronize()
    assert bool((vo[1, 0, 32:] == 0).all()) and bool((vo[1, 0, :32] == 1).all()) and bool((vo[0] == 1).all())


@pytest.mark.parametrize("layers,page,hk,dim,n", [(1, 16, 1, 32, 1), (3, 16, 2, 64, 5), (2, 64, 4, 128, 40), (1, 16, 1, 32, 1200)])
def test_copy_pages(pkg, layers, page, hk, dim, n):
    """Every byte of every layer, no other page; more pages than one launch holds."""
    say("copy", layers, page, hk, dim, n)
    for fmt in ("q8", "bf16"):
        size = pkg.KvPool.page_bytes_of(fmt, page, hk, dim, layers)
        g = torch.Generator(device=DEV).manual_seed(n)
        t = torch.randint(0, 256, (2 * n + 1, size), dtype=torch.uint8, device=DEV, generator=g)
        pool = pkg.KvPool(t, fmt, page, hk, dim, n_layers=layers)
        perm = torch.randperm(2 * n + 1, generator=torch.Generator().manual_seed(n))
        src, dst = perm[:n], perm[n:2 * n]
        src[n // 2:] = src[0]                          # one page to several places
        want = t.clone()
        want[dst.to(DEV)] = t[src.to(DEV)]
        pool.copy_pages(src.numpy(), dst.numpy())
        torch.cuda.synchronize()
        assert torch.equal(t, want)


def test_far_pages(pkg):
    """Pages past 4 GiB in the pool, for every call."""
    say("far pages")
    page, hk, dim = 64, 4, 128
    size = pkg.KvPool.page_bytes_of("q8", page, hk, dim)
    n_pages = (5 << 30) // size
    t = torch.empty(n_pages, size, dtype=torch.uint8, device=DEV)
    pool = pkg.KvPool(t, "q8", page, hk, dim)
    p = Problem(pkg, "q8", "bf16", 8, hk, dim, page, [(3, 70), (200, 200)], seed=4)
    far = [n_pages - 1 - i for i in range(6)]
    table = torch.tensor([[far[0], far[1], -1, -1], far[2:6]], dtype=torch.int32, device=DEV)
    for i in range(2):
        for k in range((2, 4)[i]):
            t[int(table[i, k])] = torch.from_numpy(p.cache.bytes[int(p.table[i, k])].reshape(-1)).to(DEV)
    p.batch = pkg.KvBatch(table, p.kv_len, p.row0_d, p.n_rows, p.max_rows, p.max_len)
    p.check(p.run(pool))
    wide = torch.full((2, 64), -1, dtype=torch.int32, device=DEV)
    wide[:, :4] = table
    p.batch = pkg.KvBatch(wide, p.kv_len, p.row0_d, p.n_rows, p.max_rows, 4096)      # as prompts
    p.check(p.run(pool))
    pool.copy_pages([far[2], far[3]], [7, far[0] - 6])
    torch.cuda.synchronize()
    assert torch.equal(t[7], t[far[2]]) and torch.equal(t[far[0] - 6], t[far[3]])
    k = torch.randn(p.n_rows, hk, dim, device=DEV)
    ko, vo = torch.empty_like(k), torch.empty_like(k)
    pool.append(p.batch, k, k)
    pool.read(p.batch, ko, vo)
    torch.cuda.synchronize()
    assert torch.equal(ko, vo) and float((ko - k).abs().max()) < float(k.abs().max()) / 127


@pytest.mark.parametrize("lens", [[(4, 3000), (1, 200)], [(300, 2300), (5, 5)]])
def test_streams_graphs_and_workspaces(pkg, lens):
    """On another stream than the current one; captured together with append,
    replayed with new inputs and eager calls between; two graphs that share a
    workspace, one after the other; the same bits every time."""
    say("graphs", lens)
    p = Problem(pkg, "q8", "bf16", 8, 2, 128, 64, lens, seed=8, behind=0)
    pool = p.cache.pool()
    eager = p.run(pool)
    p2 = Problem(pkg, "bf16", "bf16", 8, 2, 128, 64, lens, seed=18, behind=0)
    pool2 = p2.cache.pool()
    eager2 = p2.run(pool2)
    ws = torch.full((max(pool.attend_ws_bytes(p.batch, p.q), pool2.attend_ws_bytes(p2.batch, p2.q)),), 0xFF,
                    dtype=torch.uint8, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = torch.full_like(p.q, 77.0)
    pool.attend(p.batch, p.q, out, p.scale, ws, stream=side)
    side.synchronize()
    assert torch.equal(out, eager)
    q, q2 = p.q.clone(), p2.q.clone()
    k = torch.randn(p.n_rows, 2, 128, device=DEV, dtype=torch.bfloat16)
    o, o2 = torch.empty_like(q), torch.empty_like(q2)
    graphs = []
    for body in (lambda: (pool.append(p.batch, k, k), pool.attend(p.batch, q, o, p.scale, ws)),
                 lambda: pool2.attend(p2.batch, q2, o2, p2.scale, ws)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            body()
        graphs.append(g)
    for n in range(4):
        q.copy_(torch.randn_like(q)), q2.copy_(torch.randn_like(q2)), k.copy_(torch.randn_like(k))
        o.fill_(5.0), o2.fill_(5.0)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        got, got2 = o.clone(), o2.clone()
        pool.append(p.batch, k, k)
        assert torch.equal(got, p.run(pool, q=q)) and torch.equal(got2, p2.run(pool2, q=q2))
    assert torch.equal(p2.run(pool2), eager2)


def test_two_threads(pkg):
    """Two host threads with a stream, outputs and a workspace each, on a
    pool each: what each gets alone."""
    say("two threads")
    ps = [Problem(pkg, "q8", "bf16", 8, 2, 128, 64, lens, seed=2 + i, behind=0)
          for i, lens in enumerate(([(4, 3000), (1, 200)], [(300, 2300), (5, 5)]))]
    pools = [p.cache.pool() for p in ps]
    alone = [p.run(pool) for p, pool in zip(ps, pools)]
    ws = [p.ws(pool) for p, pool in zip(ps, pools)]
    streams = [torch.cuda.Stream() for _ in ps]
    outs = [[torch.full_like(p.q, 77.0) for _ in range(20)] for p in ps]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            for out in outs[i]:
                pools[i].attend(ps[i].batch, ps[i].q, out, ps[i].scale, ws[i], stream=streams[i])
        except Exception as e:                         # (a thread's own exception reaches nobody)
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed
    for i in range(2):
        assert all(torch.equal(o, alone[i]) for o in outs[i])


def test_same_bits_whatever_the_batch(pkg):
    """The same call twice gives the same bits."""
    say("same bits")
    for lens in (FEW, PROMPT, [(5, 30000)]):
        p = Problem(pkg, "q8", "f32", 16, 4, 64, 64, lens, seed=31)
        pool = p.cache.pool()
        assert torch.equal(p.run(pool), p.run(pool))


def test_a_session_of_pages(pkg):
    """The operators together, as a server uses them: a prompt is read in two
    chunks, forked into three samples that go on with drafts of which some rows
    are rejected, one ends, the pool is compacted, the others go on; every
    attention against a cache that is kept apart."""
    say("session of pages")
    r = np.random.default_rng(7)
    hk, heads, dim, page, layers, n_pages = 2, 8, 64, 16, 2, 64
    size = pkg.KvPool.page_bytes_of("q8", page, hk, dim, layers)
    pool = pkg.KvPool(torch.full((n_pages, size), 0xFF, dtype=torch.uint8, device=DEV), "q8", page, hk, dim, n_layers=layers)
    pages = pkg.KvPages(n_pages, page)
    hist = {}                                           # sequence -> per layer lists of (k, v) held

    def step(new):
        """new: {sequence: rows}; appends, attends and checks every layer"""
        seqs = list(new)
        moves = [pages.extend(s, new[s]) for s in seqs]
        pool.copy_pages(sum((a for a, _ in moves), []), sum((b for _, b in moves), []))
        tabs = [pages.table(s) for s in seqs]
        t = np.full((len(seqs), max(len(x) for x in tabs)), -1, np.int32)
        for i, x in enumerate(tabs):
            t[i, :len(x)] = x
        row0 = np.concatenate([[0], np.cumsum([new[s] for s in seqs])]).astype(np.int32)
        lens = [pages.len(s) for s in seqs]
        n = int(row0[-1])
        b = pkg.KvBatch(torch.from_numpy(t).to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV),
                        torch.from_numpy(row0).to(DEV), n, max(new.values()), max(lens))
        for layer in range(layers):
            k, v, q = (torch.from_numpy(r.standard_normal((n, h, dim))).float().to(DEV) for h in (hk, hk, heads))
            out = torch.empty_like(q)
            ws = torch.empty(pool.attend_ws_bytes(b, q), dtype=torch.uint8, device=DEV)
            pool.append(b, k, v, layer=layer)
            pool.attend(b, q, out, 0.125, ws, layer=layer)
            torch.cuda.synchronize()
            for i, s in enumerate(seqs):
                for a in range(row0[i], row0[i + 1]):
                    held = []
                    for x in (k, v):
                        c, sc = quant(x[a].cpu().numpy())
                        held.append((c.astype(np.float64) * sc[..., None]).reshape(hk, dim))
                    hist[s][layer].append(held)
                    kk = torch.from_numpy(np.stack([x[0] for x in hist[s][layer]])).to(DEV)
                    vv = torch.from_numpy(np.stack([x[1] for x in hist[s][layer]])).to(DEV)
                    for h in range(heads):
                        s_ = kk[:, h // 4] @ q[a, h].double() * 0.125
                        want = torch.softmax(s_, 0) @ vv[:, h // 4]
                        bound = torch.softmax(s_, 0) @ vv[:, h // 4].abs()
                        amp = float((kk[:, h // 4].abs() @ q[a, h].double().abs() * 0.125).max())
                        rel = 2 * (2 * (dim + 16) * U * amp + 2 * (len(kk) + 64) * U)
                        assert bool(((out[a, h].double() - want).abs() <= rel * bound + 2 * U * want.abs()).all())

    a = pages.new()
    hist[a] = [[] for _ in range(layers)]
    step({a: 40})
    step({a: 21})
    kids = [a]
    for _ in range(2):
        c = pages.fork(a, 61)
        hist[c] = [list(x) for x in hist[a]]
        kids.append(c)
    for n in range(3):
        step({s: 4 for s in kids})
        for i, s in enumerate(kids):                    # the verify keeps 1 to 3 of the 4 rows
            keep = pages.len(s) - 1 - (n + i) % 3
            pages.trim(s, keep)
            hist[s] = [x[:keep] for x in hist[s]]
    pages.free(a)
    kids.remove(a)
    pool.copy_pages(*pages.compact())
    step({kids[0]: 1, kids[1]: 17})
    step({kids[1]: 1})


def test_pointers_are_refused(pkg):
    """Host memory, null and misaligned pointers are errors, not faults."""
    say("pointers")
    p = Problem(pkg, "q8", "f32", 4, 2, 64, 16, [(2, 40)], seed=2)
    pool = p.cache.pool()
    out, ws = torch.empty_like(p.q), p.ws(pool)
    host = torch.zeros(1 << 16)
    for name, t in (("table", p.table), ("kv_len", p.kv_len), ("row0", p.row0_d)):
        b = pkg.KvBatch(p.table, p.kv_len, p.row0_d, p.n_rows, p.max_rows, p.max_len)
        for bad in (host.data_ptr(), 0, t.data_ptr() + 2):
            setattr(b.c, name, bad)
            with pytest.raises(ValueError, match=name):
                pool.attend(b, p.q, out, 1.0, ws)
    with pytest.raises(ValueError, match="not on a GPU"):
        pool.attend(p.batch, p.q.cpu(), out, 1.0, ws)
    for bad in (p.q.double(), p.q.half()):
        with pytest.raises(ValueError, match="float32"):
            pool.attend(p.batch, bad, bad, 1.0, ws)
    with pytest.raises(ValueError, match="shape"):
        pool.attend(p.batch, p.q[:1], out, 1.0, ws)
    with pytest.raises(ValueError, match="shape"):
        pool.append(p.batch, p.q, p.q)
    rows = pkg.L98KvRows(host.data_ptr(), 256, 64)
    err = pkg.C.create_string_buffer(200)
    good = pkg.L98KvRows(p.q.data_ptr(), 256, 64)
    for q, o in ((rows, good), (good, rows)):
        assert pkg.hip_lib().l98_kv_attend(pool.c, 0, p.batch.c, q, o, 4, 0, 1.0, ws.data_ptr(), ws.numel(), None, err,
                                           200) == -6
        assert b"not device memory" in err.value
    pool.c.data = host.data_ptr()
    with pytest.raises(ValueError, match="device memory"):
        pool.copy_pages([0], [1])
    torch.cuda.synchronize()
