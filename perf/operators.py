"""The measured calls of the paged KV cache and the attention that reads it.

Kinds:

  attend  ops.tree_attention_paged: the rows (tree nodes, or a causal chunk) of a batch of sequences over a prefix that
          all of them share and over each sequence's own pages, with plain, capped, biased or windowed scores
  tables  ops.page_tables: pages given to growing sequences, their block tables, the slots of the new rows
  write   ops.kv_write_paged: K/V rows into the slots of their pages, from a contiguous cache or a fused q/k/v block
  commit  ops.kv_compact_paged: every sequence's accepted rows moved together, through its block table

``run`` is the framework's call where ``own`` is true and the plain form (elementary torch operations in 32 bits, one
rounding at the end) where it is not; ``exact`` is the definition in 64 bits.

The head layouts are those of the configured models (tiny fp32 Llama, 4 query and 2 KV heads of 64; Llama-2-7B, 32 and
32 of 128; Qwen2.5-14B, 40 and 8 of 128) and 16 heads of 64 for an attention with a distance bias.
"""

import math
import zlib

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}
HEADS = {"tiny": (4, 2, 64), "7b": (32, 32, 128), "14b": (40, 8, 128), "bias64": (16, 16, 64)}


def listed():
    return [
        # the smallest attention: a small fp32 model's trees over a short shared prompt, bound by launches
        {"name": "attend-tiny-fp32", "kind": "attend", "heads": "tiny", "dtype": "float32", "page": 16, "batch": 2,
         "rows_min": 5, "rows": 8, "prefix": 40, "len_min": 3, "len": 64, "mask": "tree", "cap": 0.0, "window": 0,
         "bias": False},
        # a server's decode step without drafts: one token for each of 64 chats behind one system prompt
        {"name": "attend-decode-14b-B64", "kind": "attend", "heads": "14b", "dtype": "float16", "page": 16,
         "batch": 64, "rows_min": 1, "rows": 1, "prefix": 2000, "len_min": 1, "len": 1500, "mask": "tree", "cap": 0.0,
         "window": 0, "bias": False},
        # a verification step at 7B width: 26-node trees of 16 sequences, every head with its own keys
        {"name": "attend-tree-7b-B16-T26", "kind": "attend", "heads": "7b", "dtype": "bfloat16", "page": 64,
         "batch": 16, "rows_min": 26, "rows": 26, "prefix": 2048, "len_min": 0, "len": 1024, "mask": "tree",
         "cap": 0.0, "window": 0, "bias": False},
        # a target with capped scores and a sliding window, ragged trees over long chats
        {"name": "attend-cap-window-14b-B8", "kind": "attend", "heads": "14b", "dtype": "bfloat16", "page": 32,
         "batch": 8, "rows_min": 9, "rows": 48, "prefix": 1501, "len_min": 100, "len": 4000, "mask": "tree",
         "cap": 50.0, "window": 2048, "bias": False},
        # chunked prompts of four requests with a distance bias, causal, heads of 64
        {"name": "attend-chunk-bias-B4", "kind": "attend", "heads": "bias64", "dtype": "float16", "page": 16,
         "batch": 4, "rows_min": 100, "rows": 700, "prefix": 300, "len_min": 0, "len": 777, "mask": "causal",
         "cap": 0.0, "window": 0, "bias": True},
        # the largest: 64 sequences' trees behind a shared document of 8192 tokens
        {"name": "attend-tree-14b-B64-P8192", "kind": "attend", "heads": "14b", "dtype": "bfloat16", "page": 64,
         "batch": 64, "rows_min": 26, "rows": 26, "prefix": 8192, "len_min": 16, "len": 1000, "mask": "tree",
         "cap": 0.0, "window": 0, "bias": False},
        # the pages of a step: eight sequences grow by a tree each, a few need a page
        {"name": "tables-step-B8", "kind": "tables", "page": 16, "batch": 8, "rows_min": 26, "rows": 26,
         "prefix": 4096, "len_min": 16, "len": 4000, "admit": False},
        # admitting 256 prompts at once: every page of every table is new
        {"name": "tables-admit-B256", "kind": "tables", "page": 16, "batch": 256, "rows_min": 1, "rows": 2000,
         "prefix": 0, "len_min": 0, "len": 0, "admit": True},
        # the new K/V rows of eight trees in one layer, read out of the fused q/k/v block
        {"name": "write-step-14b-M208", "kind": "write", "heads": "14b", "dtype": "bfloat16", "page": 16,
         "layers": 1, "rows": 208, "source": "qkv"},
        # a prefilled prompt of 2000 tokens moved from its contiguous cache into pages, eight layers at 7B width
        {"name": "write-prompt-7b-2000", "kind": "write", "heads": "7b", "dtype": "bfloat16", "page": 64, "layers": 8,
         "rows": 2000, "source": "cache"},
        # the accepted paths of eight sequences of a 14B target, all 48 layers
        {"name": "commit-14b-B8-T26", "kind": "commit", "heads": "14b", "dtype": "bfloat16", "page": 16, "layers": 48,
         "batch": 8, "rows_min": 26, "rows": 26, "prefix": 512, "len_min": 16, "len": 500},
        # wide trees of many sequences at 7B width
        {"name": "commit-7b-B32-T64", "kind": "commit", "heads": "7b", "dtype": "float16", "page": 32, "layers": 8,
         "batch": 32, "rows_min": 40, "rows": 64, "prefix": 0, "len_min": 1, "len": 300},
    ]


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))

    def zlog(hi):  # zero now and then
        return 0 if rng.random() < 0.15 else log(1, hi)

    kind = rng.choice(["attend", "attend", "attend", "attend", "attend", "tables", "write", "commit"])
    page = rng.choice([16, 32, 64, 128])
    c = {"kind": kind, "page": page}
    if kind == "attend":
        heads = rng.choice(["tiny", "7b", "14b", "14b", "bias64"])
        dtype = "float32" if heads == "tiny" else rng.choice(["bfloat16", "float16"])
        causal = rng.random() < 0.3
        small = heads == "tiny"
        batch = log(1, 8 if small else 64)
        rows = log(1, min(700, max(1, 3000 // batch))) if causal else log(1, min(160, max(1, 1800 // batch)))
        if small:
            rows = min(rows, 64)
        length = zlog(600 if small else 4000 if batch <= 16 else 1500)
        c.update(heads=heads, dtype=dtype, batch=batch, rows_min=rng.randint(1, rows), rows=rows,
                 prefix=zlog(500 if small else 8192 if not causal else 2500), len_min=rng.randint(0, length),
                 len=length, mask="causal" if causal else "tree", cap=rng.choice([0.0, 0.0, 0.0, 30.0, 50.0]),
                 window=rng.choice([0, 0, 0, log(16, 4096)]), bias=heads == "bias64" or rng.random() < 0.1)
    elif kind == "tables":
        rows = log(1, 2000)
        length = zlog(8000)
        c.update(batch=log(1, 256), rows_min=rng.randint(1, rows), rows=rows, prefix=zlog(8192),
                 len_min=rng.randint(0, length), len=length, admit=rng.random() < 0.3)
    elif kind == "write":
        source = rng.choice(["qkv", "cache"])
        c.update(heads=rng.choice(["7b", "14b"]), dtype=rng.choice(["bfloat16", "float16", "float32"]),
                 layers=1 if source == "qkv" else rng.randint(1, 4), rows=log(1, 2000), source=source)
    else:
        rows = log(2, 64)
        length = zlog(500)
        c.update(heads=rng.choice(["7b", "14b"]), dtype=rng.choice(["bfloat16", "float16", "float32"]),
                 layers=rng.randint(1, 16), batch=log(1, 32), rows_min=rng.randint(1, rows), rows=rows,
                 prefix=zlog(2000), len_min=rng.randint(0, length), len=length)
    return c


# ------------------------------------------------------------------ inputs
def _sizes(c):
    """A generator that depends on the case alone: its sizes are the same for every seed."""
    return np.random.default_rng(zlib.crc32(repr(sorted((k, v) for k, v in c.items() if k != "name")).encode()))


def _lengths(c, rng):
    """Per sequence: new rows and private cached rows."""
    n = c["batch"]
    rows = rng.integers(c["rows_min"], c["rows"] + 1, n)
    priv = rng.integers(c["len_min"], c["len"] + 1, n)
    return rows.astype(np.int64), priv.astype(np.int64)


def _tree(t, rng):
    """Parents and depths of a drafted tree of t nodes, depth by depth."""
    deep = min(t, int(rng.integers(4, 7)))
    first = max(1, min(t // deep, 8))
    rest = t - first
    widths = [first] + [rest // max(1, deep - 1) + (1 if d >= deep - 1 - rest % max(1, deep - 1) else 0)
                        for d in range(deep - 1)]
    parents, depths, prev, at = [], [], [-1], 0
    for d, w in enumerate(widths):
        if w == 0:
            continue
        pick = sorted(int(rng.integers(0, len(prev))) for _ in range(w))
        parents += [prev[i] for i in pick]
        depths += [d] * w
        prev = list(range(at, at + w))
        at += w
    return parents, depths


def _bits(parents, words):
    out, full = np.zeros((len(parents), words), np.uint64), []
    for t, p in enumerate(parents):
        b = (1 << t) | (full[p] if p >= 0 else 0)
        full.append(b)
        for w in range(words):
            out[t, w] = (b >> (64 * w)) & 0xFFFFFFFFFFFFFFFF
    return out.view(np.int64)


def _ints(a, dtype=torch.int64):
    return torch.as_tensor(np.ascontiguousarray(a)).to(dtype).to(DEV)


def _tables(need, total, rng):
    """A block table with need[b] pages per sequence out of a shuffled pool; the pages left over."""
    perm = rng.permutation(total)
    table = np.full((len(need), max(1, int(max(need)))), -1, np.int64)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at: at + n]
        at += int(n)
    return table, perm[at:]


def _randn(shape, dtype, gen):
    """Normal values, made in pieces so that a large pool needs no fp32 copy of itself."""
    out = torch.empty(shape, dtype=dtype, device=DEV)
    flat = out.view(-1)
    step = 1 << 27
    for i in range(0, flat.numel(), step):
        n = min(step, flat.numel() - i)
        flat[i: i + n] = torch.randn(n, generator=gen, device=DEV, dtype=torch.float32).to(dtype)
    return out


def prepare(case, seed):
    c = case
    rng, size = np.random.default_rng(1000003 * seed + 17), _sizes(c)
    gen = torch.Generator(device=DEV).manual_seed(1000003 * seed + 29)
    ps = c["page"]
    st = {"case": c, "status": torch.zeros(1, dtype=torch.int32, device=DEV)}
    if c["kind"] == "write":
        nh, nkv, hd = HEADS[c["heads"]]
        dt, n, layers = DTYPES[c["dtype"]], c["rows"], c["layers"]
        pages = -(-n // ps) + 3
        order = rng.permutation(pages)
        at = int(rng.integers(0, 2 * ps))  # the rows follow a few that are cached
        idx = np.arange(at, at + n) % (pages * ps)
        st["slots"] = _ints(order[idx // ps] * ps + idx % ps)
        st["k_pool"] = _randn((layers, pages, nkv, ps, hd), dt, gen)
        st["v_pool"] = _randn((layers, pages, nkv, ps, hd), dt, gen)
        if c["source"] == "qkv":
            qkv = _randn((n, (nh + 2 * nkv) * hd), dt, gen)
            st["k"] = qkv[:, nh * hd: (nh + nkv) * hd].view(1, n, nkv, hd)
            st["v"] = qkv[:, (nh + nkv) * hd:].view(1, n, nkv, hd)
        else:
            cap = n + int(size.integers(1, 100))
            st["k"] = _randn((layers, nkv, cap, hd), dt, gen)[:, :, :n].transpose(1, 2)
            st["v"] = _randn((layers, nkv, cap, hd), dt, gen)[:, :, :n].transpose(1, 2)
        return st

    rows, priv = _lengths(c, size)
    row0 = np.concatenate([[0], np.cumsum(rows)])
    m, s0 = int(row0[-1]), c["prefix"]
    st.update(m=m, max_rows=int(rows.max()), max_len=int(priv.max()) + s0, row0=row0, rows=rows, priv=priv)
    st["seq_row0"], st["seq_len"] = _ints(row0, torch.int32), _ints(priv + s0)
    if c["kind"] == "tables":
        held = np.zeros_like(priv) if c["admit"] else -(-priv // ps)
        full = -(-(priv + rows) // ps)
        extra = int((full - held).clip(0).sum()) + int(size.integers(0, 50))
        table, free = _tables(held, int(held.sum()) + extra, rng)
        wide = np.full((c["batch"], int(full.max()) + int(size.integers(0, 4))), -1, np.int64)
        n = min(wide.shape[1], table.shape[1])
        wide[:, :n] = table[:, :n]
        st["table"], st["held"] = _ints(wide, torch.int32), _ints(held, torch.int32)
        st["free"], st["top"] = _ints(free, torch.int32), _ints([len(free)], torch.int32)
        st["held_out"], st["top_out"] = torch.empty_like(st["held"]), torch.empty_like(st["top"])
        return st

    nh, nkv, hd = HEADS[c["heads"]]
    dt = DTYPES[c["dtype"]]
    npre = -(-s0 // ps) if c["kind"] == "attend" else 0
    need = -(-(priv + rows) // ps)
    pages = int(need.sum()) + npre + 2
    table, left = _tables(need, pages, rng)
    st["table"], st["prefix_table"] = _ints(table, torch.int32), _ints(left[:npre], torch.int32)
    if c["kind"] == "commit":
        layers = c["layers"]
        st["k_pool"] = _randn((layers, pages, nkv, ps, hd), dt, gen)
        st["v_pool"] = _randn((layers, pages, nkv, ps, hd), dt, gen)
        acc = np.zeros((c["batch"], 2 + st["max_rows"]), np.int32)
        for b, t in enumerate(rows):
            parents, depths = _tree(int(t), rng)
            node = int(rng.integers(0, t))
            path = [node]
            while parents[path[0]] >= 0:
                path.insert(0, parents[path[0]])
            path = path[: path[0]]  # no accepted row lies where another one moves to: a second pass moves the same rows
            acc[b, 0], acc[b, 1] = len(path), int(rng.integers(0, 32000))
            acc[b, 2: 2 + len(path)] = path
        st["accept"], st["accept_host"] = _ints(acc, torch.int32), acc
        return st

    st["k_pool"] = _randn((pages, nkv, ps, hd), dt, gen)
    st["v_pool"] = _randn((pages, nkv, ps, hd), dt, gen)
    st["q"] = (_randn((m, nh, hd), dt, gen).float() * 1.5).to(dt)
    st["scale"] = hd ** -0.5
    words = -(-st["max_rows"] // 64)
    pos, bits = np.zeros(m, np.int64), np.zeros((m, words), np.int64)
    for b, t in enumerate(rows):
        if c["mask"] == "tree":
            parents, depths = _tree(int(t), rng)
            bits[row0[b]: row0[b + 1]] = _bits(parents, words)
        else:
            depths = range(int(t))
        pos[row0[b]: row0[b + 1]] = s0 + priv[b] + np.asarray(list(depths), np.int64)
    st["positions"] = _ints(pos)
    st["bits"] = _ints(bits) if c["mask"] == "tree" else None
    st["slopes"] = (torch.tensor([2.0 ** (-8.0 * (h + 1) / nh) for h in range(nh)], dtype=torch.float32, device=DEV)
                    if c["bias"] else None)
    if own:
        from parallel_eagle_amd import ops
        st["ws"] = torch.empty(ops.attention_paged_workspace_bytes(m, c["batch"], nh, nkv, hd, st["max_rows"],
                                                                   st["max_len"], s0, dt),
                               dtype=torch.uint8, device=DEV)
    return st


# ------------------------------------------------------------------ the calls
def _own(st):
    from parallel_eagle_amd import _lib, ops
    c = st["case"]
    if c["kind"] == "attend":
        return ops.tree_attention_paged(
            st["q"], st["k_pool"], st["v_pool"], st["table"], st["seq_row0"], st["seq_len"], st["scale"],
            st["max_rows"], st["max_len"], st["status"],
            mask_mode=_lib.PE_MASK_TREE if c["mask"] == "tree" else _lib.PE_MASK_CAUSAL, bits=st["bits"],
            positions=st["positions"], prefix_table=st["prefix_table"], prefix_len=c["prefix"], softcap=c["cap"],
            slopes=st["slopes"], window=c["window"], workspace=st["ws"])
    if c["kind"] == "tables":
        slots = ops.page_tables(st["seq_len"], st["seq_row0"], st["table"], st["held"], st["free"], st["top"],
                                c["page"], st["m"], st["status"], prefix_len=c["prefix"], held_out=st["held_out"],
                                top_out=st["top_out"])
        return {"slots": slots, "table": st["table"], "held": st["held_out"], "top": st["top_out"]}
    if c["kind"] == "write":
        ops.kv_write_paged(st["k"], st["v"], st["k_pool"], st["v_pool"], st["slots"], st["status"])
    else:
        ops.kv_compact_paged(st["k_pool"], st["v_pool"], st["table"], st["seq_len"], st["accept"], st["status"],
                             prefix_len=c["prefix"])
    return {"k": st["k_pool"], "v": st["v_pool"]}


def _gather(pool, table, n, ps):
    """The first n cached rows of a list of pages, [nkv][n][hd] in fp32."""
    x = pool[table[: -(-n // ps)].long()].float()  # [pages][nkv][ps][hd]
    return x.transpose(0, 1).reshape(pool.shape[1], -1, pool.shape[3])[:, :n]


def _plain_attend(st):
    c = st["case"]
    nh, nkv, hd = HEADS[c["heads"]]
    g, ps, s0 = nh // nkv, c["page"], c["prefix"]
    out = torch.empty((st["m"], nh * hd), dtype=st["q"].dtype, device=DEV)
    kp, vp = (_gather(st[x], st["prefix_table"], s0, ps) for x in ("k_pool", "v_pool"))
    for b in range(c["batch"]):
        r0, r1 = int(st["row0"][b]), int(st["row0"][b + 1])
        t, p = r1 - r0, int(st["priv"][b])
        k = torch.cat([kp, _gather(st["k_pool"], st["table"][b], p + t, ps)], dim=1)  # [nkv][s0 + p + t][hd]
        v = torch.cat([vp, _gather(st["v_pool"], st["table"][b], p + t, ps)], dim=1)
        q = st["q"][r0:r1].float().view(t, nkv, g, hd).permute(1, 2, 0, 3).reshape(nkv, g * t, hd)
        s = torch.matmul(q, k.transpose(1, 2).contiguous()).view(nkv, g, t, -1) * st["scale"]
        if c["cap"]:
            s = torch.tanh(s / c["cap"]) * c["cap"]
        pos = st["positions"][r0:r1]
        kpos = torch.cat([torch.arange(s0 + p, device=DEV), pos])
        dist = pos.view(t, 1) - kpos.view(1, -1)
        if c["bias"]:
            s = s - st["slopes"].view(nkv, g, 1, 1) * dist.float()
        u = torch.arange(t, device=DEV)
        if c["mask"] == "tree":
            node = (st["bits"][r0:r1][:, u // 64] >> (u % 64)) & 1 == 1
        else:
            node = u.view(t, 1) >= u.view(1, t)
        see = torch.cat([torch.ones((t, s0 + p), dtype=torch.bool, device=DEV), node], dim=1)
        if c["window"]:
            see = see & (dist < c["window"])
        s = s.masked_fill(~see, -math.inf)
        top = s.amax(-1, keepdim=True).clamp_min(-3e38)
        e = torch.exp(s - top)
        o = torch.matmul(e.view(nkv, g * t, -1), v).view(nkv, g, t, hd) / e.sum(-1, keepdim=True).clamp_min(1e-38)
        out[r0:r1] = o.permute(2, 0, 1, 3).reshape(t, nh * hd).to(out.dtype)
    return out


def _plain_tables(st):
    c, dev = st["case"], DEV
    ps = c["page"]
    row0 = st["seq_row0"].long()
    rows, priv, held = row0[1:] - row0[:-1], st["seq_len"] - c["prefix"], st["held"].long()
    full = (priv + rows + ps - 1) // ps
    need = torch.where(rows > 0, (full - held).clamp_min(0), torch.zeros_like(full))
    off = torch.cumsum(need, 0) - need
    j = torch.arange(st["table"].shape[1], device=dev).view(1, -1)
    i = j - held.view(-1, 1)
    new = (i >= 0) & (i < need.view(-1, 1))
    at = (st["top"].long() - 1 - off.view(-1, 1) - i).clamp(0, st["free"].numel() - 1)
    table = torch.where(new, st["free"][at], st["table"])
    r = torch.arange(st["m"], device=dev)
    b = torch.searchsorted(row0[1:].contiguous(), r, right=True)
    idx = priv[b] + r - row0[b]
    slots = table[b, idx // ps].long() * ps + idx % ps
    return {"slots": slots, "table": table, "held": (held + need).int(), "top": (st["top"] - need.sum()).int()}


def _plain_write(st):
    ps = st["case"]["page"]
    page, at = st["slots"] // ps, st["slots"] % ps
    for pool, src in ((st["k_pool"], st["k"]), (st["v_pool"], st["v"])):
        for i in range(pool.shape[0]):
            pool[i][page, :, at] = src[i]
    return {"k": st["k_pool"], "v": st["v_pool"]}


def _plain_commit(st):
    c = st["case"]
    ps = c["page"]
    n, path = st["accept"][:, 0].long(), st["accept"][:, 2:].long()
    width = path.shape[1]
    i = torch.arange(width, device=DEV).view(1, -1)
    live = i < n.view(-1, 1)
    base = (st["seq_len"] - c["prefix"]).view(-1, 1)
    b, col = torch.nonzero(live, as_tuple=True)
    src, dst = (base + path)[b, col], (base + i)[b, col]
    sp, dp = st["table"][b, src // ps].long(), st["table"][b, dst // ps].long()
    for pool in (st["k_pool"], st["v_pool"]):
        pool[:, dp, :, dst % ps] = pool[:, sp, :, src % ps]
    return {"k": st["k_pool"], "v": st["v_pool"]}


def run(state):
    if own:
        return _own(state)
    return {"attend": _plain_attend, "tables": _plain_tables, "write": _plain_write,
            "commit": _plain_commit}[state["case"]["kind"]](state)


# ------------------------------------------------------------------ what a pass cannot do without
def _mean(c):
    """Expected new rows and private cached rows of a sequence."""
    return (c["rows_min"] + c["rows"]) / 2, (c["len_min"] + c["len"]) / 2


def work(case):
    c = case
    if c["kind"] == "tables":
        t, p = _mean(c)
        full = math.ceil((p + t) / c["page"])
        new = full if c["admit"] else t / c["page"]
        return {"bytes": c["batch"] * (4 + 8 + 8 + 8 * new + 8 * t), "flops": 0}
    nh, nkv, hd = HEADS[c["heads"]]
    row = 2 * nkv * hd * SIZE[c["dtype"]]  # a token's K and V in one layer
    if c["kind"] == "write":
        return {"bytes": 2 * c["layers"] * c["rows"] * row + 8 * c["rows"], "flops": 0}
    t, p = _mean(c)
    if c["kind"] == "commit":
        return {"bytes": 2 * c["layers"] * c["batch"] * min(4, t / 4) * row, "flops": 0}
    m, s0, w = c["batch"] * t, c["prefix"], c["window"]
    own_keys = p + (t if c["mask"] == "tree" else t / 2)
    seen = min(s0 + own_keys, w) if w else s0 + own_keys
    shared = max(0.0, min(s0, w - c["len_min"])) if w else s0
    private = min(p + t, w) if w else p + t
    return {"bytes": (shared + c["batch"] * private) * row + 2 * m * nh * hd * SIZE[c["dtype"]],
            "flops": 4 * m * nh * hd * seen}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    """Attention row by row of its definition, one KV head at a time, on float64 keys laid out by token; the other
    kinds move or count whole values and have nothing to compute."""
    c = case
    if c["kind"] != "attend":
        return None
    st = prepare(c, seed)
    nh, nkv, hd = HEADS[c["heads"]]
    g, ps, s0 = nh // nkv, c["page"], c["prefix"]
    out = torch.zeros((st["m"], nh, hd), dtype=torch.float64, device=DEV)
    for b in range(c["batch"]):
        a, z = int(st["row0"][b]), int(st["row0"][b + 1])
        t, p = z - a, int(st["priv"][b])
        j = torch.arange(p + t, device=DEV)
        pre = torch.arange(s0, device=DEV)
        page = torch.cat([st["prefix_table"][pre // ps], st["table"][b][j // ps]]).long()
        at = torch.cat([pre % ps, j % ps])
        where = torch.cat([pre, s0 + j[:p], st["positions"][a:z]]).double()
        away = st["positions"][a:z].double()[:, None] - where[None, :]
        hide = torch.zeros((t, s0 + p + t), dtype=torch.bool, device=DEV)
        for u in range(t):
            if c["mask"] == "tree":
                word = st["bits"][a:z, u >> 6]
                hide[:, s0 + p + u] = torch.bitwise_and(torch.bitwise_right_shift(word, u & 63), 1) == 0
            else:
                hide[:u, s0 + p + u] = True
        if c["window"]:
            hide |= away >= c["window"]
        for h in range(nkv):
            k = st["k_pool"][page, h, at].double()
            v = st["v_pool"][page, h, at].double()
            kt = k.t().contiguous()
            for e in range(h * g, (h + 1) * g):
                s = (st["q"][a:z, e].double() @ kt) * float(st["scale"])
                if c["cap"]:
                    s = c["cap"] * torch.tanh(s / c["cap"])
                if c["bias"]:
                    s = s - float(st["slopes"][e]) * away
                s[hide] = -math.inf
                w = torch.exp(s - torch.logsumexp(s, 1, keepdim=True))
                w[hide.all(1)] = 0.0
                out[a:z, e] = w @ v
    return out.view(st["m"], nh * hd)
