"""The paged key-value cache and the attention that reads it, as timed cases.

A pool holds pages of `page` rows (positions) for `kv_heads` heads of width
`dim`; a sequence is a list of pages (its row of the page table) and a length.
Four operators work on it:

  append  quantizes or rounds new K and V rows into the sequences' pages (and
          `read` gives them back as numbers);
  copy    copies whole pages, as a fork's copy on write or a compaction does;
  few     attention of the newest one to eight rows of each sequence over all
          the rows before them (single tokens, a draft's verify rows);
  prompt  the same for many new rows: whole prompts and their chunks, packed
          one behind the other.

The head counts and widths are those of this repository's models (csrc/synth.h:
16 query heads over 4 KV heads of 64 or 128, 4 over 2 of 64, 2 over 1 of 32),
the contexts those of bench.py (512-token prompts, 4096 tokens in chunks of 512,
32 sessions of 256 to 2048 positions with 4 verify rows each) and longer ones.

A page of one layer, in bytes, n = kv_heads * page * dim:
  bf16  K [kv_heads][page][dim], V the same;
  q8    K codes (n bytes), V codes (n), K scales, V scales (float
        [kv_heads][dim/32][page] each); a code byte is the number + 128, a
        group of 32 values x has the scale max|x| / 127.  A row's bytes are
        ordered for the matrix instructions: of K, byte h*(dim/4) + c*8 + j is
        dimension c*32 + h*8 + j; of V, byte n*(dim/16) + t is dimension
        t*16 + n.
"""
import math
import random

import torch

own = False

F = {"f32": torch.float32, "bf16": torch.bfloat16}


# --------------------------------------------------------------- cases ---

def _c(name, kind, fmt, dt, heads, kv_heads, dim, page, seqs, rows, past):
    d = {"kind": kind, "fmt": fmt, "dt": dt, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
         "seqs": seqs, "rows_lo": rows[0], "rows_hi": rows[1], "past_lo": past[0], "past_hi": past[1]}
    return dict(d, name=name) if name else d


def _copy(name, layers, kv_heads, dim, page, pages, moves):
    d = {"kind": "copy", "fmt": "bf16", "layers": layers, "kv_heads": kv_heads, "dim": dim, "page": page,
         "pages": pages, "moves": moves}
    return dict(d, name=name) if name else d


def listed():
    return [
        # the verify rows of 32 sessions (k = 3) go into the cache
        _c("append_verify_32", "append", "q8", "f32", 16, 4, 128, 64, 32, (4, 4), (256, 2044)),
        # a batch of prompts goes into the cache
        _c("append_prompts", "append", "q8", "bf16", 16, 4, 128, 64, 8, (700, 4096), (0, 0)),
        # eight samples of one prompt start writing: their shared last pages are copied (32 layers)
        _copy("fork_8", 32, 4, 64, 16, 600, 8),
        # a pool is compacted after sessions ended: 400 pages of 8 layers move down
        _copy("compact_400", 8, 4, 128, 64, 1000, 400),
        # one new token of one short session
        _c("token_short", "few", "q8", "f32", 16, 4, 64, 16, 1, (1, 1), (300, 300)),
        # the verify of 32 sessions, 4 rows each, contexts of 256 to 2048
        _c("verify_32", "few", "q8", "f32", 16, 4, 128, 64, 32, (4, 4), (252, 2044)),
        # one new token for each of 100 sessions whose cache is bf16
        _c("tokens_100_bf16", "few", "bf16", "bf16", 16, 4, 128, 32, 100, (1, 1), (1, 4999)),
        # the widest verify (k = 7) far into one very long session
        _c("verify_long", "few", "q8", "bf16", 16, 4, 128, 128, 1, (8, 8), (250007, 250007)),
        # a 512-token prompt
        _c("prompt_512", "prompt", "bf16", "bf16", 16, 4, 64, 64, 1, (512, 512), (0, 0)),
        # prompts of different lengths, packed
        _c("prompts_packed", "prompt", "q8", "bf16", 16, 4, 128, 64, 9, (33, 4001), (0, 0)),
        # the last 512-row chunk of a 4096-token prompt, in fp32
        _c("chunk_f32", "prompt", "q8", "f32", 16, 4, 128, 64, 1, (512, 512), (3584, 3584)),
        # a document as one prompt
        _c("prompt_16384", "prompt", "q8", "bf16", 16, 4, 128, 64, 1, (16384, 16384), (0, 0)),
    ]


def _log(rng, lo, hi):
    return min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["append", "copy", "few", "few", "prompt", "prompt"])
    heads, kv_heads, dim = rng.choice([(16, 4, 128), (16, 4, 64), (4, 2, 64), (2, 1, 32), (8, 8, 64), (12, 1, 128)])
    page = rng.choice([16, 32, 64, 128, 256])
    if kind == "copy":
        layers, pages = rng.choice([1, 4, 8, 24, 32]), _log(rng, 12, 1500)
        size = layers * 4 * kv_heads * page * dim
        pages = max(4, min(pages, (1 << 30) // size))
        return _copy(None, layers, kv_heads, dim, page, pages, max(1, min(pages // 2, _log(rng, 1, 600))))
    fmt, dt = rng.choice(["q8", "q8", "bf16"]), rng.choice(["f32", "bf16", "bf16"])
    if kind == "append":
        seqs, rows = _log(rng, 1, 64), _log(rng, 1, 3000)
        rows = max(1, min(rows, 30000 // seqs))
        return _c(None, kind, fmt, dt, heads, kv_heads, dim, page, seqs, (max(1, rows // 3), rows), (0, _log(rng, 1, 1000)))
    if kind == "few":
        seqs, past = _log(rng, 1, 128), _log(rng, 1, 200000)
        past = max(1, min(past, 400000 // seqs))
        rows = rng.randint(1, 8)
        return _c(None, kind, fmt, dt, heads, kv_heads, dim, page, seqs, (min(rows, rng.randint(1, 8)), rows), (past // 8, past))
    seqs, rows, past = _log(rng, 1, 12), _log(rng, 9, 5000), rng.choice([0, 0, _log(rng, 1, 4000)])
    rows = max(9, min(rows, 12000 // seqs))
    if dt == "f32":
        rows, past = max(9, min(rows, 2000 // seqs)), min(past, 2000)
    return _c(None, kind, fmt, dt, heads, kv_heads, dim, page, seqs, (max(1, rows // 10), rows), (0, past))


def _lens(case):
    """(new rows, rows before them) of each sequence: the case's alone."""
    r = random.Random("%(seqs)d %(rows_lo)d %(rows_hi)d %(past_lo)d %(past_hi)d" % case)
    rows = [r.randint(case["rows_lo"], case["rows_hi"]) for _ in range(case["seqs"])]
    past = [r.randint(case["past_lo"], case["past_hi"]) for _ in range(case["seqs"])]
    rows[-1], past[0] = case["rows_hi"], case["past_hi"]
    return rows, past


def work(case):
    row = case["kv_heads"] * case["dim"]
    if case["kind"] == "copy":
        return {"bytes": 2 * case["moves"] * case["layers"] * 4 * row * case["page"], "flops": 0}
    rows, past = _lens(case)
    held = row * 2 if case["fmt"] == "bf16" else row + row // 32 * 4
    e = 4 if case["dt"] == "f32" else 2
    n = sum(rows)
    if case["kind"] == "append":      # the rows in, the cache written; then read, and the rows out
        return {"bytes": 4 * n * (row * e + held), "flops": 4 * n * row}
    q = case["heads"] * case["dim"]
    pairs = sum(r * p + r * (r + 1) // 2 for r, p in zip(rows, past))
    return {"bytes": 2 * n * q * e + 2 * held * sum(r + p for r, p in zip(rows, past)), "flops": 4 * q * pairs}


# --------------------------------------------------------------- inputs ---

def _k_order(dim):
    """dimension of each byte of a q8 K row"""
    return torch.arange(dim).view(dim // 32, 4, 8).permute(1, 0, 2).reshape(-1)


def _v_order(dim):
    return torch.arange(dim).view(dim // 16, 16).t().reshape(-1)


def _quant(x):
    """codes and scales of groups of 32, all in fp32: the format's rounding"""
    g = x.float().unflatten(-1, (-1, 32))
    amax = g.abs().amax(-1)
    s = amax * (1.0 / 127.0)
    live = (amax > 0) & ~(s < 1e-30)
    s, inv = torch.where(live, s, 1.0), torch.where(live, 127.0 / amax, 0.0)
    return (g * inv[..., None]).round().clamp(-127, 127), s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    hk, dim, page = case["kv_heads"], case["dim"], case["page"]
    st = dict(case)
    if case["kind"] == "copy":
        n = case["pages"]
        st["data"] = normal(n, case["layers"] * 2 * hk * page * dim).to(torch.bfloat16)
        st["at"] = torch.randperm(n, generator=torch.Generator().manual_seed(seed))[: 2 * case["moves"]].to(torch.int32)
        st["src"], st["dst"] = st["at"][: case["moves"]].numpy(), st["at"][case["moves"]:].numpy()
        if own:
            st["pool"] = _package().KvPool(st["data"], "bf16", page, hk, dim, n_layers=case["layers"])
        return st
    rows, past = _lens(case)
    dt = F[case["dt"]]
    lens = [r + p for r, p in zip(rows, past)]
    need = [-(-n // page) for n in lens]
    n_pages = sum(need) + 3
    ids = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(rows), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, k in enumerate(need):
        table[i, :k] = ids[at:at + k]
        at += k
    row0 = [0]
    for r in rows:
        row0.append(row0[-1] + r)
    st.update(table=table, kv_len=torch.tensor(lens, dtype=torch.int32, device="cuda"),
              row0=torch.tensor(row0, dtype=torch.int32, device="cuda"), n_rows=row0[-1], max_rows=max(rows),
              max_len=max(lens), n_pages=n_pages)
    # K and V as a model has them: normed keys, values with channels of different sizes
    k, v = normal(n_pages, hk, page, dim), normal(n_pages, hk, page, dim) * (0.3 + normal(1, hk, 1, dim).abs())
    if case["fmt"] == "bf16":
        st["data"] = torch.stack([k, v], 1).to(torch.bfloat16).reshape(n_pages, -1)
    else:
        parts = []
        for x, order in ((k, _k_order(dim)), (v, _v_order(dim))):
            code, s = _quant(x)
            parts.append(((code.flatten(-2)[..., order] + 128).to(torch.uint8).reshape(n_pages, -1),
                          s.transpose(-1, -2).contiguous().view(torch.uint8).reshape(n_pages, -1)))
        st["data"] = torch.cat([parts[0][0], parts[1][0], parts[0][1], parts[1][1]], 1)
    del k, v
    if case["kind"] == "append":
        st["k"], st["v"] = normal(row0[-1], hk, dim).to(dt), (normal(row0[-1], hk, dim) * 0.7).to(dt)
        st["k_out"], st["v_out"] = torch.empty_like(st["k"]), torch.empty_like(st["v"])
    else:
        st["q"] = (normal(row0[-1], case["heads"], dim) * 1.25).to(dt)
        st["out"] = torch.zeros_like(st["q"])
        st["scale"] = 1.0 / math.sqrt(dim)
    if own:
        P = _package()
        st["pool"] = P.KvPool(st["data"], case["fmt"], page, hk, dim)
        st["batch"] = P.KvBatch(table, st["kv_len"], st["row0"], st["n_rows"], st["max_rows"], st["max_len"])
        if case["kind"] != "append":
            st["ws"] = torch.empty(st["pool"].attend_ws_bytes(st["batch"], st["q"]), dtype=torch.uint8, device="cuda")
    return st


def _package():
    from __graft_entry__ import load_package
    return load_package()


# ----------------------------------------------------------- plain form ---

def _places(st):
    """of each new row: its sequence, its number there, its position"""
    r = torch.arange(st["n_rows"], device="cuda")
    row0, n = st["row0"].long(), st["kv_len"].long()
    i = torch.searchsorted(row0[1:].contiguous(), r, right=True)
    j = r - row0[i]
    return i, j, n[i] - (row0[i + 1] - row0[i]) + j


def _split(st, data):
    """bytes or numbers of pages [..., page bytes] to K and V [..., kv_heads, page, dim] in fp32"""
    hk, dim, page = st["kv_heads"], st["dim"], st["page"]
    lead, n = data.shape[:-1], hk * page * dim
    if st["fmt"] == "bf16":
        x = data.float().reshape(*lead, 2, hk, page, dim)
        return x.select(-4, 0), x.select(-4, 1)
    s = data[..., 2 * n:].contiguous().view(torch.float32).reshape(*lead, 2, hk, dim // 32, page).transpose(-1, -2)
    code = data[..., : 2 * n].reshape(*lead, 2, hk, page, dim).float() - 128.0
    k = code.select(-4, 0).unflatten(-1, (4, dim // 32, 8)).transpose(-2, -3).reshape(*lead, hk, page, dim)
    v = code.select(-4, 1).unflatten(-1, (16, dim // 16)).transpose(-1, -2).reshape(*lead, hk, page, dim)
    sk, sv = s.select(-4, 0)[..., None], s.select(-4, 1)[..., None]
    return (k.unflatten(-1, (-1, 32)) * sk).flatten(-2), (v.unflatten(-1, (-1, 32)) * sv).flatten(-2)


def _plain_append(st):
    hk, dim, page, data = st["kv_heads"], st["dim"], st["page"], st["data"]
    i, _, pos = _places(st)
    at = st["table"][i, pos // page].long()
    off = pos % page
    n = hk * page * dim
    if st["fmt"] == "bf16":
        pool = data.view(-1, 2, hk, page, dim)
        pool[at, 0, :, off] = st["k"].to(torch.bfloat16)
        pool[at, 1, :, off] = st["v"].to(torch.bfloat16)
        return {"k": pool[at, 0, :, off].to(st["k"].dtype), "v": pool[at, 1, :, off].to(st["k"].dtype)}
    codes = data[:, : 2 * n].unflatten(1, (2, hk, page, dim))
    scales = data.view(torch.float32)[:, n // 2:].unflatten(1, (2, hk, dim // 32, page))
    out = {}
    for w, name in enumerate(("k", "v")):
        c, s = _quant(st[name])
        u = (c.flatten(-2) + 128).to(torch.uint8)
        u = u.unflatten(-1, (-1, 4, 8)).transpose(-2, -3) if w == 0 else u.unflatten(-1, (-1, 16)).transpose(-1, -2)
        codes[at, w, :, off] = u.flatten(2)
        scales[at, w, :, :, off] = s
        u, s = codes[at, w, :, off], scales[at, w, :, :, off]
        u = u.unflatten(-1, (4, -1, 8)).transpose(-2, -3) if w == 0 else u.unflatten(-1, (16, -1)).transpose(-1, -2)
        u = u.flatten(2).unflatten(-1, (-1, 32)).float() - 128.0
        out[name] = (u * s[..., None]).flatten(-2).to(st["k"].dtype)
    return out


def _plain_attend(st):
    hk, dim, heads = st["kv_heads"], st["dim"], st["heads"]
    g, n_seq, n_max = heads // hk, st["table"].shape[0], st["max_rows"]
    k, v = _split(st, st["data"][st["table"].clamp(min=0).long()])          # [seqs, pages, kv_heads, page, dim]
    k, v = (x.transpose(1, 2).reshape(n_seq, hk, -1, dim) for x in (k, v))
    row0, n = st["row0"].long(), st["kv_len"].long()
    j = torch.arange(n_max, device="cuda")
    q = st["q"][(row0[:-1, None] + j).clamp(max=st["n_rows"] - 1)].float()
    q = q.view(n_seq, n_max, hk, g, dim).transpose(1, 2).reshape(n_seq, hk, n_max * g, dim)
    pos = (n - (row0[1:] - row0[:-1]))[:, None] + j                         # [seqs, rows]
    key = torch.arange(k.shape[2], device="cuda")
    seen = (key <= pos[..., None]) & (key < n[:, None, None])               # [seqs, rows, keys]
    seen = seen[:, None, :, None].expand(-1, 1, -1, g, -1).reshape(n_seq, 1, n_max * g, -1)
    s = torch.where(seen, torch.matmul(q, k.transpose(-1, -2)) * st["scale"], float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(-1, keepdim=True)
    v = torch.where((key < n[:, None])[:, None, :, None], v, 0.0)
    o = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
    o = o.view(n_seq, hk, n_max, g, dim).transpose(1, 2).reshape(n_seq, n_max, heads, dim)
    i, j, _ = _places(st)
    return o[i, j].to(st["q"].dtype)


def run(st):
    if st["kind"] == "copy":
        if own:
            st["pool"].copy_pages(st["src"], st["dst"])
        else:
            at = st["at"].to("cuda").long()
            st["data"][at[st["moves"]:]] = st["data"][at[: st["moves"]]]
        return st["data"]
    if st["kind"] == "append":
        if own:
            st["pool"].append(st["batch"], st["k"], st["v"])
            st["pool"].read(st["batch"], st["k_out"], st["v_out"])
            return {"k": st["k_out"], "v": st["v_out"]}
        return _plain_append(st)
    if own:
        return st["pool"].attend(st["batch"], st["q"], st["out"], st["scale"], st["ws"])
    return _plain_attend(st)


# ---------------------------------------------------------------- exact ---

def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "copy":
        x = st["data"].clone()
        for a, b in zip(st["src"].tolist(), st["dst"].tolist()):
            x[b] = st["data"][a]
        return x
    hk, dim, page = case["kv_heads"], case["dim"], case["page"]
    if case["kind"] == "append":
        # a code is the format's fp32 decision; the number it stands for is code * scale
        def held(x):
            if case["fmt"] == "bf16":
                return x.to(torch.bfloat16).double()
            a = x.float().reshape(-1, 32)
            big = a.abs().max(1, keepdim=True).values
            return (torch.round(a * (127.0 / big)).double() * (big * (1.0 / 127.0)).double()).reshape(x.shape)
        return {"k": held(st["k"]), "v": held(st["v"])}
    rows, past = _lens(case)
    out = torch.zeros(st["n_rows"], case["heads"], dim, dtype=torch.float64, device="cuda")
    n, r0, group = hk * page * dim, 0, case["heads"] // hk
    for i, (r, p) in enumerate(zip(rows, past)):
        pages = st["data"][st["table"][i, : -(-(r + p) // page)].long()]
        for h in range(hk):
            kv = []
            for w in range(2):
                if case["fmt"] == "bf16":
                    x = pages.view(-1, 2, hk, page, dim)[:, w, h].double()
                else:
                    b = pages[:, w * n:(w + 1) * n].reshape(-1, hk, page, dim)[:, h].double() - 128
                    x = torch.empty_like(b)
                    x[..., (_v_order if w else _k_order)(dim).cuda()] = b
                    s = pages[:, 2 * n:].contiguous().view(torch.float32).view(-1, 2, hk, dim // 32, page)[:, w, h]
                    x *= s.double().transpose(-1, -2).repeat_interleave(32, -1)
                kv.append(x.reshape(-1, dim)[: r + p])
            for lo in range(0, r, 4096):
                hi = min(r, lo + 4096)
                key, pos = torch.arange(p + hi, device="cuda"), torch.arange(p + lo, p + hi, device="cuda")
                for y in range(group):
                    q = st["q"][r0 + lo:r0 + hi, h * group + y].double()
                    s = (q @ kv[0][: p + hi].T) * st["scale"]
                    s.masked_fill_(key[None] > pos[:, None], float("-inf"))
                    out[r0 + lo:r0 + hi, h * group + y] = torch.softmax(s, 1) @ kv[1][: p + hi]
        r0 += r
    return out
