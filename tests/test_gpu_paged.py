"""The paged KV cache and the attention that reads it, against plain
implementations in float64 (attention) or on host integers (tables, copies)."""

import math
import random

import pytest
import torch

from parallel_eagle_amd import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
TREE, CAUSAL = _lib.PE_MASK_TREE, _lib.PE_MASK_CAUSAL


def status_word():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


def random_tree(t, rng):
    """Parents of a tree of t nodes: each hangs off the prefix or an earlier node."""
    return [-1 if i == 0 or rng.random() < 0.2 else rng.randrange(max(0, i - 6), i) for i in range(t)]


def ancestor_bits(parents, words):
    rows, depth = [], []
    for t, p in enumerate(parents):
        rows.append((rows[p] if p >= 0 else 0) | (1 << t))
        depth.append(depth[p] + 1 if p >= 0 else 0)
    out = torch.zeros((len(parents), words), dtype=torch.int64)
    for t, b in enumerate(rows):
        for w in range(words):
            v = (b >> (64 * w)) & (2 ** 64 - 1)
            out[t, w] = v - 2 ** 64 if v >= 2 ** 63 else v
    return out, depth


class Case:
    """One batch: lengths, tables over shuffled pages, pools whose unused rows hold NaN."""

    def __init__(self, heads, rows, priv, prefix=0, page=16, dtype=torch.bfloat16, mask=TREE, cap=0.0, window=0,
                 bias=False, seed=0, extra_rows=0, blind=()):
        rng = random.Random(seed)
        gen = torch.Generator().manual_seed(seed)
        self.nh, self.nkv, self.hd = heads
        nh, nkv, hd = heads
        self.rows, self.priv, self.prefix, self.page, self.mask = rows, priv, prefix, page, mask
        self.cap, self.window, self.dtype = cap, window, dtype
        B = len(rows)
        self.row0 = [0]
        for r in rows:
            self.row0.append(self.row0[-1] + r)
        self.m = self.row0[-1] + extra_rows
        need = [-(-(p + r) // page) for p, r in zip(priv, rows)]
        npre = -(-prefix // page)
        pages = sum(need) + npre + 2
        perm = list(range(pages))
        rng.shuffle(perm)
        cols = max(1, max(need)) + 1
        table = torch.full((B, cols), -7, dtype=torch.int32)  # entries past a sequence's pages are no pages
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = torch.tensor(perm[at: at + n], dtype=torch.int32)
            at += n
        ptab = torch.tensor(perm[at: at + npre] + [-7], dtype=torch.int32)
        k = torch.full((pages, nkv, page, hd), math.nan)
        v = torch.full((pages, nkv, page, hd), math.nan)
        # token-major K/V of every sequence, written into the pages
        self.kpre = torch.randn((prefix, nkv, hd), generator=gen)
        self.vpre = torch.randn((prefix, nkv, hd), generator=gen)
        self.ks, self.vs = [], []

        def put(tab, ktok, vtok):
            j = torch.arange(ktok.shape[0])
            at = tab[j // page].long()
            k[at, :, j % page] = ktok
            v[at, :, j % page] = vtok

        put(ptab, self.kpre, self.vpre)
        for b in range(B):
            n = priv[b] + rows[b]
            kt, vt = torch.randn((n, nkv, hd), generator=gen), torch.randn((n, nkv, hd), generator=gen)
            self.ks.append(kt)
            self.vs.append(vt)
            put(table[b], kt, vt)
        q = 1.5 * torch.randn((self.m, nh, hd), generator=gen)
        to = lambda x: x.to(dtype).to(DEV)
        self.q, self.k_pool, self.v_pool = to(q), to(k), to(v)
        rnd = lambda x: x.to(dtype).double().to(DEV)
        self.kpre, self.vpre = rnd(self.kpre), rnd(self.vpre)
        self.ks, self.vs = [rnd(x) for x in self.ks], [rnd(x) for x in self.vs]
        self.table, self.ptab = table.to(DEV), ptab.to(DEV)
        self.seq_row0 = torch.tensor(self.row0, dtype=torch.int32, device=DEV)
        self.seq_len = torch.tensor([p + prefix for p in priv], dtype=torch.int64, device=DEV)
        self.max_rows, self.max_len = max(rows), max(priv) + prefix
        self.scale = hd ** -0.5
        words = -(-max(1, self.max_rows) // 64)
        bits = torch.zeros((self.m, words), dtype=torch.int64)
        pos = torch.zeros(self.m, dtype=torch.int64)
        for b, t in enumerate(rows):
            a = self.row0[b]
            if mask == TREE:
                bb, dep = ancestor_bits(random_tree(t, rng), words)
                bits[a: a + t] = bb
            else:
                dep = list(range(t))
            pos[a: a + t] = torch.tensor([prefix + priv[b] + d for d in dep], dtype=torch.int64)
        for r in blind:  # rows whose mask leaves them not even themselves
            bits[r] = 0
        self.bits = bits.to(DEV) if mask == TREE else None
        self.positions = pos.to(DEV)
        self.slopes = (torch.tensor([2.0 ** (-1 - 7.0 * h / nh) for h in range(nh)], dtype=torch.float32, device=DEV)
                       if bias else None)
        self.status = status_word()

    def run(self, **kw):
        args = dict(mask_mode=self.mask, bits=self.bits, positions=self.positions, prefix_table=self.ptab,
                    prefix_len=self.prefix, softcap=self.cap, slopes=self.slopes, window=self.window)
        args.update(kw)
        q = args.pop("q", self.q)
        return ops.tree_attention_paged(q, self.k_pool, self.v_pool, self.table, self.seq_row0, self.seq_len,
                                        self.scale, args.pop("max_rows", self.max_rows),
                                        args.pop("max_len", self.max_len), args.pop("status", self.status), **args)

    def expected(self):
        """(output, sum of weight * |v|) in float64 from the definition."""
        nh, nkv, hd = self.nh, self.nkv, self.hd
        out = torch.zeros((self.m, nh, hd), dtype=torch.float64, device=DEV)
        mag = torch.zeros_like(out)
        for b, t in enumerate(self.rows):
            if t == 0:
                continue
            a, p = self.row0[b], self.priv[b]
            k, v = torch.cat([self.kpre, self.ks[b]]), torch.cat([self.vpre, self.vs[b]])
            n = self.prefix + p
            pos = self.positions[a: a + t]
            dist = pos[:, None] - torch.cat([torch.arange(n, device=DEV), pos])[None, :]
            see = torch.ones((t, n + t), dtype=torch.bool, device=DEV)
            for u in range(t):
                if self.mask == TREE:
                    see[:, n + u] = ((self.bits[a: a + t, u // 64] >> (u % 64)) & 1) == 1
                else:
                    see[:u, n + u] = False
            if self.window:
                see &= dist < self.window
            for h in range(nh):
                s = self.q[a: a + t, h].double() @ k[:, h // (nh // nkv)].t().contiguous() * self.scale
                if self.cap:
                    s = self.cap * torch.tanh(s / self.cap)
                if self.slopes is not None:
                    s = s - self.slopes[h].double() * dist
                s = s.masked_fill(~see, -math.inf)
                w = torch.softmax(s, 1).nan_to_num(0.0)
                out[a: a + t, h] = w @ v[:, h // (nh // nkv)]
                mag[a: a + t, h] = w @ v[:, h // (nh // nkv)].abs()
        return out.view(self.m, nh * hd), mag.view(self.m, nh * hd)

    def check(self, got):
        """The output is rounded once (half a step of its value), 16-bit probabilities once each (half a step of every
        weight: u * sum w |v|); scores, exponentials and sums in fp32 add at most 2^-13 of sum w |v| (the longest
        product here is 256 terms of scores below 2^4: 2^8 * 2^-24 * 2^3, and as much for exp and the sums)."""
        assert int(self.status.item()) == 0
        live = self.row0[-1]
        ref, mag = self.expected()
        u = torch.finfo(self.dtype).eps / 2
        pu = 0.0 if self.dtype == torch.float32 else u
        err = (got[:live].double() - ref[:live]).abs()
        tol = u * ref[:live].abs() + (pu + 2.0 ** -13) * mag[:live]
        assert bool(torch.all(err <= tol)), ((err - tol).max().item(), err.max().item())


LAYOUTS = [((4, 2, 64), torch.float32), ((4, 4, 128), torch.bfloat16), ((10, 2, 128), torch.float16),
           ((8, 8, 64), torch.float16), ((6, 1, 64), torch.bfloat16), ((2, 1, 80), torch.bfloat16),
           ((3, 3, 36), torch.float32), ((2, 2, 256), torch.float16), ((2, 1, 7), torch.float32)]
IDS = [f"{h[0]}-{h[1]}-{h[2]}-{str(d)[6:]}" for h, d in LAYOUTS]


@pytest.mark.parametrize("heads,dtype", LAYOUTS, ids=IDS)
@pytest.mark.parametrize("prefix", [0, 1, 16, 65, 300])
def test_trees_over_a_shared_prefix(heads, dtype, prefix):
    c = Case(heads, [5, 0, 1, 26, 9], [0, 3, 17, 64, 130], prefix, dtype=dtype, seed=prefix + heads[2])
    c.check(c.run())


@pytest.mark.parametrize("heads,dtype", LAYOUTS, ids=IDS)
@pytest.mark.parametrize("prefix", [0, 77])
def test_causal_chunks(heads, dtype, prefix):
    c = Case(heads, [1, 70, 3], [200, 0, 15], prefix, page=32, dtype=dtype, mask=CAUSAL, seed=5)
    c.check(c.run())


@pytest.mark.parametrize("heads,dtype", LAYOUTS[:5], ids=IDS[:5])
@pytest.mark.parametrize("cap,window,bias", [(30.0, 0, False), (0.0, 1, False), (0.0, 50, False), (0.0, 0, True),
                                             (50.0, 100, True), (2.0, 3, True)])
@pytest.mark.parametrize("mask", [TREE, CAUSAL], ids=["tree", "causal"])
def test_capped_biased_and_windowed_scores(heads, dtype, cap, window, bias, mask):
    c = Case(heads, [26, 4, 40], [5, 150, 33], 130, dtype=dtype, mask=mask, cap=cap, window=window, bias=bias, seed=7)
    c.check(c.run())


@pytest.mark.parametrize("page", [16, 32, 128, 1024])
@pytest.mark.parametrize("heads,dtype", LAYOUTS[:4], ids=IDS[:4])
def test_page_sizes(heads, dtype, page):
    c = Case(heads, [7, 33], [100, 1], 90, page=page, dtype=dtype, seed=page)
    c.check(c.run())


@pytest.mark.parametrize("heads,dtype", LAYOUTS[:5], ids=IDS[:5])
def test_one_token_of_many_sequences(heads, dtype):
    c = Case(heads, [1] * 33, [(7 * i) % 90 for i in range(33)], 200, dtype=dtype, seed=2)
    c.check(c.run())


@pytest.mark.parametrize("heads,dtype", LAYOUTS[:4], ids=IDS[:4])
@pytest.mark.parametrize("t", [64, 65, 200, 256])
def test_wide_trees(heads, dtype, t):
    c = Case(heads, [t, 3], [40, 90], 50, dtype=dtype, seed=t)
    c.check(c.run())


@pytest.mark.parametrize("heads,dtype", LAYOUTS[:4], ids=IDS[:4])
def test_long_keys_of_few_rows(heads, dtype):
    """Few rows over many keys: the keys are split and the parts joined."""
    c = Case(heads, [2], [1500], 1100, page=64, dtype=dtype, seed=3)
    c.check(c.run())
    c = Case(heads, [1, 2], [2100, 700], 0, page=64, dtype=dtype, seed=4)
    c.check(c.run())


@pytest.mark.parametrize("heads,dtype", LAYOUTS[:4], ids=IDS[:4])
def test_many_rows_of_one_prefix(heads, dtype):
    """Row blocks of the prefix that end inside a sequence and inside a tile."""
    c = Case(heads, [26] * 11 + [31], [i for i in range(12)], 333, dtype=dtype, seed=6)
    c.check(c.run())


@pytest.mark.parametrize("cap,window,bias", [(0.0, 0, False), (40.0, 0, True), (0.0, 1500, False)])
@pytest.mark.parametrize("heads,dtype,seqs,prefix", [((40, 8, 128), torch.bfloat16, 16, 4133), ((16, 16, 64), torch.float16, 33, 5121)],
                         ids=["14b", "64"])
def test_many_rows_over_a_long_prefix(heads, dtype, seqs, prefix, cap, window, bias):
    """The prefix's own launch (row blocks of 256, two groups of waves in opposite phases)."""
    c = Case(heads, [26] * (seqs - 1) + [9], [(37 * i) % 300 for i in range(seqs)], prefix, page=64, dtype=dtype, seed=10,
             cap=cap, window=window, bias=bias)
    c.check(c.run())


@pytest.mark.parametrize("cap,window,bias", [(0.0, 0, False), (40.0, 0, True), (0.0, 300, False)])
@pytest.mark.parametrize("heads,dtype,seqs,prefix", [((40, 8, 128), torch.bfloat16, 16, 701), ((32, 32, 64), torch.float16, 20, 660)],
                         ids=["14b", "64"])
def test_prefix_shares_that_cross_row_blocks(heads, dtype, seqs, prefix, cap, window, bias):
    """136 and 160 row blocks of the prefix, fewer than the 256 workgroups that share them."""
    c = Case(heads, [26] * seqs, [(37 * i) % 90 for i in range(seqs)], prefix, page=32, dtype=dtype, seed=13, cap=cap,
             window=window, bias=bias)
    c.check(c.run())


@pytest.mark.parametrize("heads,dtype", LAYOUTS[:4], ids=IDS[:4])
@pytest.mark.parametrize("prefix", [0, 40])
def test_rows_that_see_nothing_are_zero(heads, dtype, prefix):
    # without a cache a row of no bits sees no key; with one, a window that has passed it leaves the same
    c = Case(heads, [4, 6], [0, 0], prefix, dtype=dtype, seed=8, blind=(1, 7), window=1 if prefix else 0)
    got = c.run()
    c.check(got)
    assert not got[[1, 7]].any()


@pytest.mark.parametrize("heads,dtype", LAYOUTS[:4], ids=IDS[:4])
def test_strided_rows_and_rows_behind_the_last_sequence(heads, dtype):
    c = Case(heads, [9, 20], [12, 70], 33, dtype=dtype, seed=9, extra_rows=5)
    nh, nkv, hd = heads
    wide = torch.zeros((c.m, nh + 2 * nkv, hd), dtype=dtype, device=DEV)
    wide[:, :nh] = c.q
    wide[c.row0[-1]:] = math.nan
    out = torch.full((c.m, nh * hd + 8), 7.0, dtype=dtype, device=DEV)
    got = c.run(q=wide[:, :nh], out=out[:, : nh * hd])
    assert got.data_ptr() == out.data_ptr()
    c.check(got)
    assert bool((out[:, nh * hd:] == 7.0).all()) and bool((out[c.row0[-1]:] == 7.0).all())


@pytest.mark.parametrize("heads,dtype", LAYOUTS[:4], ids=IDS[:4])
def test_unaligned_rows(heads, dtype):
    """q and out one element off a 16-byte boundary, rows an odd count apart."""
    c = Case(heads, [9, 20], [12, 70], 33, dtype=dtype, seed=9)
    nh, _, hd = heads
    n = nh * hd
    flat = torch.zeros(c.m * (n + 1) + 1, dtype=dtype, device=DEV)
    q = flat[1: 1 + c.m * (n + 1)].view(c.m, n + 1)[:, :n]
    q.copy_(c.q.view(c.m, n))
    out = torch.zeros(c.m * (n + 3) + 1, dtype=dtype, device=DEV)[1:].view(c.m, n + 3)[:, :n]
    got = c.run(q=q.as_strided((c.m, nh, hd), (n + 1, hd, 1), q.storage_offset()), out=out)
    c.check(got)


@pytest.mark.parametrize("heads,dtype", LAYOUTS[:4], ids=IDS[:4])
def test_masked_keys_may_hold_anything(heads, dtype):
    """K of nodes that no other row sees: NaN and infinities there reach no other row."""
    c = Case(heads, [6, 4], [20, 3], 17, dtype=dtype, seed=11)
    bits = torch.zeros((c.m, 1), dtype=torch.int64)
    for t in range(c.m):
        u = t - (6 if t >= 6 else 0)
        bits[t] = 1 << u  # every row sees itself alone among the new ones
    c.bits = bits.to(DEV)
    c.positions = torch.tensor([c.prefix + 20] * 6 + [c.prefix + 3] * 4, device=DEV)
    clean = c.run()
    c.check(clean)
    for b, t, val in ((0, 2, math.nan), (1, 1, math.inf)):
        j = c.priv[b] + t
        c.k_pool[int(c.table[b, j // c.page]), :, j % c.page] = val
    got = c.run()
    keep = [r for r in range(c.m) if r not in (2, 7)]
    assert torch.equal(got[keep], clean[keep])


def test_repeated_calls_are_equal_and_a_graph_replays_them():
    c = Case((10, 2, 128), [26] * 6 + [1], [200, 3, 64, 90, 17, 0, 900], 400, dtype=torch.bfloat16, seed=12)
    first = c.run()
    c.check(first)
    assert all(torch.equal(c.run(), first) for _ in range(3))
    ws = torch.empty(max(1, ops.attention_paged_workspace_bytes(c.m, 7, 10, 2, 128, c.max_rows, c.max_len, c.prefix,
                                                                c.dtype)), dtype=torch.uint8, device=DEV)
    out = torch.zeros_like(first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.run(workspace=ws, out=out)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, first)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.run(workspace=ws, out=out)
    for i in range(4):
        ws.fill_(255)  # the workspace needs no value of its own
        out.zero_()
        # shorter lengths than the launch was sized for
        c.seq_len.copy_(torch.tensor([p + c.prefix - (i if p > i else 0) for p in c.priv]))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, c.run())
    assert int(c.status.item()) == 0


@pytest.mark.parametrize("heads,dtype", [LAYOUTS[0], LAYOUTS[1]], ids=[IDS[0], IDS[1]])
def test_bad_ids_set_the_status_and_read_nothing(heads, dtype):
    def fresh(**kw):
        return Case(heads, [4, 3], [20, 40], 33, dtype=dtype, seed=13, **kw)

    c = fresh()
    good = c.run()
    c.check(good)
    for bad in (-1, c.k_pool.shape[0], 2 ** 31 - 1):
        c = fresh()
        c.table[1, 1] = bad
        got = c.run()
        assert int(c.status.item()) == _lib.PE_ERR_INDEX
        assert torch.equal(got[:4], good[:4])  # the other sequence is served
    c = fresh()
    c.ptab[1] = -3
    c.run()
    assert int(c.status.item()) == _lib.PE_ERR_INDEX
    c = fresh()
    got = c.run(max_len=c.max_len - 1, out=torch.zeros_like(good))
    assert int(c.status.item()) == _lib.PE_ERR_CAPACITY
    assert not got[4:].any() and bool((got[:4] != 0).any())
    c = fresh()
    c.seq_len[0] = c.prefix - 1
    c.run()
    assert int(c.status.item()) == _lib.PE_ERR_CAPACITY
    c = fresh()
    c.seq_row0[2] = 100
    c.run()
    assert int(c.status.item()) == _lib.PE_ERR_TREE
    c = fresh()
    c.run(max_rows=3)
    assert int(c.status.item()) == _lib.PE_ERR_TREE


def test_equals_the_contiguous_batch():
    """The same keys through tree_attention_batch: both within the rounding of the exact result."""
    c = Case((10, 2, 128), [26, 26, 5], [100, 64, 31], 0, dtype=torch.float16, seed=14)
    cap = 160
    kc = torch.zeros((3, 2, cap, 128), dtype=c.dtype, device=DEV)
    vc = torch.zeros_like(kc)
    for b in range(3):
        n = c.priv[b] + c.rows[b]
        kc[b, :, :n] = c.ks[b].to(c.dtype).transpose(0, 1)
        vc[b, :, :n] = c.vs[b].to(c.dtype).transpose(0, 1)
    c.check(ops.tree_attention_batch(c.q, kc, vc, c.seq_row0, c.seq_len, c.bits, c.scale, c.max_rows, c.max_len))
    c.check(c.run())


# ------------------------------------------------------------------ tables
def host_tables(lens, row0, table, held, free, top, ps, m, prefix):
    table, held = [list(r) for r in table], list(held)
    slots, err, off, took = [-1] * m, 0, 0, 0
    for b in range(len(lens)):
        rows, priv = row0[b + 1] - row0[b], lens[b] - prefix
        bad = priv < 0 or priv + rows > len(table[b]) * ps
        need = 0 if bad or rows == 0 else max(0, -(-(priv + rows) // ps) - held[b])
        if bad:
            err |= _lib.PE_ERR_CAPACITY
        elif off + need <= top:
            for i in range(need):
                table[b][held[b] + i] = free[top - 1 - off - i]
            held[b] += need
            took = off + need if need else took
        elif need:
            err |= _lib.PE_ERR_CAPACITY
        off += need
        for i in range(rows):
            j = priv + i
            if not bad and j // ps < held[b]:
                slots[row0[b] + i] = table[b][j // ps] * ps + j % ps
    return slots, table, held, top - took, err


@pytest.mark.parametrize("batch,rows,length,ps,prefix", [(1, 1, 0, 16, 0), (8, 26, 300, 16, 77), (3, 900, 50, 64, 0),
                                                         (300, 20, 90, 32, 5), (600, 3, 40, 16, 0)])
@pytest.mark.parametrize("short", [0, 5])
def test_page_tables(batch, rows, length, ps, prefix, short):
    rng = random.Random(batch + ps + short)
    priv = [rng.randint(0, length) for _ in range(batch)]
    n = [rng.choice([0, 1, rows, rng.randint(0, rows)]) for _ in range(batch)]
    row0 = [0]
    for r in n:
        row0.append(row0[-1] + r)
    held = [-(-p // ps) + rng.choice([0, 0, 1]) for p in priv]
    cols = max(-(-(p + r) // ps) for p, r in zip(priv, n)) + 1
    held = [min(h, cols) for h in held]
    extra = sum(max(0, -(-(p + r) // ps) - h) for p, r, h in zip(priv, n, held) if r)
    top = max(0, extra + 3 - 2 * short)  # `short`: the list runs dry
    pool = list(range(sum(held) + top))
    rng.shuffle(pool)
    table, at = [], 0
    for h in held:
        table.append(pool[at: at + h] + [-1] * (cols - h))
        at += h
    free = pool[at:] + [12345]  # an entry above the top
    m = row0[-1] + 7
    lens = [p + prefix for p in priv]
    want = host_tables(lens, row0, table, held, free, top, ps, m, prefix)
    t = lambda x, d=torch.int32: torch.tensor(x, dtype=d, device=DEV)
    for in_place in (False, True):
        tab, hd, fr, tp, st = t(table), t(held), t(free), t([top]), status_word()
        ho, to = (hd, tp) if in_place else (torch.zeros_like(hd), torch.zeros_like(tp))
        slots = ops.page_tables(t(lens, torch.int64), t(row0), tab, hd, fr, tp, ps, m, st, prefix_len=prefix,
                                held_out=None if in_place else ho, top_out=None if in_place else to)
        assert slots.tolist() == want[0] and tab.tolist() == want[1] and ho.tolist() == want[2]
        assert to.tolist() == [want[3]] and int(st.item()) == want[4] and fr.tolist() == free
        if not in_place:
            assert hd.tolist() == held and tp.tolist() == [top]


def test_page_tables_flags_what_cannot_be_served():
    t = lambda x, d=torch.int32: torch.tensor(x, dtype=d, device=DEV)
    free = t(list(range(20)))

    def call(lens, row0, held, cols=2, table=None):
        st, tab = status_word(), t([[-1] * cols] * len(lens)) if table is None else table
        slots = ops.page_tables(t(lens, torch.int64), t(row0), tab, t(held), free, t([20]), 16, row0[-1], st,
                                prefix_len=8)
        return slots.tolist(), int(st.item())

    assert call([7, 8], [0, 1, 2], [0, 0]) == ([-1, 19 * 16], _lib.PE_ERR_CAPACITY)  # shorter than the prefix
    assert call([8 + 31, 8], [0, 2, 3], [2, 0], table=t([[0, 1], [-1, -1]]))[1] == _lib.PE_ERR_CAPACITY  # table too narrow
    assert call([8, 8], [0, 1, 2], [3, 0])[1] == _lib.PE_ERR_INDEX  # holds more than its table has
    assert call([8 + 4], [0, 1], [1]) == ([-1], _lib.PE_ERR_INDEX)  # a held page that is none
    st = status_word()
    slots = torch.full((2,), 5, dtype=torch.int64, device=DEV)
    ops.page_tables(t([8, 8], torch.int64), t([0, 9, 2]), t([[-1, -1]] * 2), t([0, 0]), free, t([20]), 16, 2, st,
                    prefix_len=8, slots=slots)
    assert int(st.item()) == _lib.PE_ERR_TREE


def test_pages_return_and_are_given_out_again():
    t = lambda x, d=torch.int32: torch.tensor(x, dtype=d, device=DEV)
    table, held, st = t([[-1] * 4] * 3), t([0, 0, 0]), status_word()
    free, top = t(list(range(100, 110))), t([10])
    lens = t([0, 0, 0], torch.int64)
    ops.page_tables(lens, t([0, 40, 41, 57]), table, held, free, top, 16, 57, st)
    assert table.tolist() == [[109, 108, 107, -1], [106, -1, -1, -1], [105, -1, -1, -1]]
    assert held.tolist() == [3, 1, 1] and top.tolist() == [5]
    ops.page_release(t([2, 0]), table, held, free, top, st)
    assert held.tolist() == [0, 1, 0] and top.tolist() == [9]
    assert free.tolist()[:9] == [100, 101, 102, 103, 104, 105, 107, 108, 109]
    assert table.tolist() == [[-1] * 4, [106, -1, -1, -1], [-1] * 4] and int(st.item()) == 0
    for seqs in ([1, 1], [5], [-1]):  # listed twice, not a sequence
        ops.page_release(t(seqs), table, held, free, top, st)
        assert int(st.item()) == _lib.PE_ERR_INDEX
        st.zero_()
    assert held.tolist() == [0, 0, 0] and top.tolist() == [10] and sorted(free.tolist()) == list(range(100, 110))


# ------------------------------------------------------------------ rows into pages
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("source", ["cache", "qkv", "odd"])
@pytest.mark.parametrize("m,nkv,hd,layers", [(1, 2, 128, 1), (77, 8, 128, 2), (300, 1, 64, 3), (5, 3, 36, 1), (9, 2, 5, 2),
                                             (3, 1, 1024, 1)])
def test_write_rows_to_their_slots(dtype, source, m, nkv, hd, layers):
    gen = torch.Generator().manual_seed(m + hd)
    ps, pages = 16, -(-m // 16) + 4
    rnd = lambda *s: torch.randn(s, generator=gen).to(dtype).to(DEV)
    if source == "cache":
        k, v = (rnd(layers, nkv, m + 3, hd)[:, :, 2: m + 2].transpose(1, 2) for _ in range(2))
    elif source == "qkv":
        x = rnd(layers, m, (4 + 2) * nkv * hd)
        k, v = (x[:, :, i * nkv * hd: (i + 1) * nkv * hd].view(layers, m, nkv, hd) for i in (4, 5))
    else:  # rows an odd number of elements apart
        x = rnd(layers, m, 2 * nkv * hd + 1)
        k, v = (x[:, :, i * nkv * hd + 1: (i + 1) * nkv * hd + 1].view(layers, m, nkv, hd) for i in (0, 1))
    slots = torch.randperm(pages * ps, generator=gen)[:m]
    if m > 4:
        slots[3] = -1
    pools = [rnd(layers, pages, nkv, ps, hd) for _ in range(2)]
    want = [p.clone() for p in pools]
    for w, src in zip(want, (k, v)):
        for r, s in enumerate(slots.tolist()):
            if s >= 0:
                w[:, s // ps, :, s % ps] = src[:, r]
    st = status_word()
    ops.kv_write_paged(k, v, pools[0], pools[1], slots.to(DEV), st)
    assert torch.equal(pools[0], want[0]) and torch.equal(pools[1], want[1]) and int(st.item()) == 0


def test_write_flags_slots_outside_the_pools():
    pools = [torch.zeros((2, 3, 2, 16, 64), dtype=torch.float16, device=DEV) for _ in range(2)]
    k = torch.ones((2, 4, 2, 64), dtype=torch.float16, device=DEV)
    st = status_word()
    slots = torch.tensor([3 * 16, -2, 2 ** 40, 17], dtype=torch.int64, device=DEV)
    ops.kv_write_paged(k, k, pools[0], pools[1], slots, st)
    assert int(st.item()) == _lib.PE_ERR_INDEX
    for p in pools:
        assert bool((p[:, 1, :, 1] == 1).all()) and float(p.float().sum()) == 2 * 2 * 64


# ------------------------------------------------------------------ commit
@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 128), (torch.float32, 128), (torch.float16, 36), (torch.float16, 5),
                                      (torch.float32, 512)])
@pytest.mark.parametrize("page", [16, 64])
def test_compact_moves_the_accepted_rows(dtype, hd, page):
    rng = random.Random(hd + page)
    gen = torch.Generator().manual_seed(hd)
    B, L, nkv, prefix, T = 6, 3, 2, 9, 70
    priv = [0, 5, 60, 15, 33, 100]
    paths = [[], [0, 1, 2], sorted(rng.sample(range(T), 40)), [69], [2, 3, 9, 30], list(range(1, 65))]
    need = [-(-(p + T) // page) for p in priv]
    pages = sum(need) + 1
    perm = list(range(pages))
    rng.shuffle(perm)
    table = torch.full((B, max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(perm[at: at + n])
        at += n
    acc = torch.full((B, 2 + T), -9, dtype=torch.int32)
    for b, p in enumerate(paths):
        acc[b, 0], acc[b, 1] = len(p), 3
        acc[b, 2: 2 + len(p)] = torch.tensor(p, dtype=torch.int32)
    pools = [torch.randn((L, pages, nkv, page, hd), generator=gen).to(dtype).to(DEV) for _ in range(2)]
    want = [p.clone() for p in pools]
    for w, src in zip(want, pools):
        for b, path in enumerate(paths):
            for i, n in enumerate(path):
                s, d = priv[b] + n, priv[b] + i
                w[:, int(table[b, d // page]), :, d % page] = src[:, int(table[b, s // page]), :, s % page]
    st = status_word()
    ops.kv_compact_paged(pools[0], pools[1], table.to(DEV), torch.tensor([p + prefix for p in priv], device=DEV),
                         acc.to(DEV), st, prefix_len=prefix)
    assert torch.equal(pools[0], want[0]) and torch.equal(pools[1], want[1]) and int(st.item()) == 0


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 128), (torch.float16, 36), (torch.float32, 512)])
@pytest.mark.parametrize("step", [1, 6])
def test_compact_of_paths_longer_than_a_wave(dtype, hd, step):
    """Every row moves `step` rows down, onto rows that others are read from; 15 (layer, head) pairs."""
    L, nkv, page, T = 5, 3, 16, 200
    gen = torch.Generator().manual_seed(hd + step)
    n = T - step
    priv = [7, 0]
    pages = [-(-(p + T) // page) for p in priv]
    perm = torch.randperm(sum(pages), generator=gen).int()
    table = torch.full((2, max(pages)), -1, dtype=torch.int32)
    table[0, : pages[0]], table[1, : pages[1]] = perm[: pages[0]], perm[pages[0]:]
    acc = torch.zeros((2, 2 + T), dtype=torch.int32)
    acc[:, 0] = n
    acc[:, 2: 2 + n] = torch.arange(step, T, dtype=torch.int32)
    pools = [torch.randn((L, sum(pages), nkv, page, hd), generator=gen).to(dtype).to(DEV) for _ in range(2)]
    want = [p.clone() for p in pools]
    for w, src in zip(want, pools):
        for b in range(2):
            for i in range(n):
                s, d = priv[b] + step + i, priv[b] + i
                w[:, int(table[b, d // page]), :, d % page] = src[:, int(table[b, s // page]), :, s % page]
    st = status_word()
    ops.kv_compact_paged(pools[0], pools[1], table.to(DEV), torch.tensor(priv, device=DEV), acc.to(DEV), st)
    assert torch.equal(pools[0], want[0]) and torch.equal(pools[1], want[1]) and int(st.item()) == 0


def test_compact_flags_paths_and_pages_that_are_none():
    def call(acc, table=((0, 1),), length=4):
        pools = [torch.arange(2 * 2 * 16 * 8, dtype=torch.float32, device=DEV).view(1, 2, 2, 16, 8) for _ in range(2)]
        st = status_word()
        ops.kv_compact_paged(pools[0], pools[1], torch.tensor(table, dtype=torch.int32, device=DEV),
                             torch.tensor([length], device=DEV), torch.tensor([acc], dtype=torch.int32, device=DEV), st)
        same = torch.equal(pools[0].flatten(), torch.arange(512, dtype=torch.float32, device=DEV))
        return int(st.item()), same

    assert call([2, 0, 0, 1, -1]) == (0, True)
    assert call([1, 0, 3, 0, 0]) == (_lib.PE_ERR_INDEX, True)  # node 3 of a tree of at most 3
    assert call([2, 0, 1, 0, 0])[0] == _lib.PE_ERR_INDEX  # not increasing
    assert call([4, 0, 0, 1, 2]) == (_lib.PE_ERR_INDEX, True)  # longer than the tree
    assert call([-1, 0, 0, 0, 0]) == (_lib.PE_ERR_INDEX, True)
    assert call([1, 0, 2, 0, 0], table=((0, 2),), length=14) == (_lib.PE_ERR_INDEX, True)  # no such page
    assert call([1, 0, 2, 0, 0], length=31)[0] == _lib.PE_ERR_INDEX  # past the table
    assert call([1, 0, 2, 0, 0], length=-1) == (_lib.PE_ERR_CAPACITY, True)
    assert call([1, 0, 2, 0, 0], length=32) == (_lib.PE_ERR_CAPACITY, True)


# ------------------------------------------------------------------ together
def test_torch_ops_equal_the_wrappers():
    ops.register_torch_ops()
    c = Case((10, 2, 128), [26, 9], [40, 100], 70, dtype=torch.float16, seed=20, cap=20.0, window=90, bias=True)
    want = c.run()
    got = torch.ops.pe.tree_attention_paged(c.q, c.k_pool, c.v_pool, c.table, c.seq_row0, c.seq_len, c.scale, c.max_rows,
                                            c.max_len, c.status, TREE, c.bits, c.positions, c.ptab, c.prefix, 20.0,
                                            c.slopes, 90)
    assert torch.equal(got, want)
    t = lambda x, d=torch.int32: torch.tensor(x, dtype=d, device=DEV)
    table, held, free, top, st = t([[-1, -1]] * 2), t([0, 0]), t(list(range(6))), t([6]), status_word()
    slots = torch.ops.pe.page_tables(t([0, 0], torch.int64), t([0, 20, 23]), table, held, free, top, 16, 23, 0, st)
    assert slots.tolist() == [5 * 16 + i for i in range(16)] + [4 * 16 + i for i in range(4)] + [3 * 16 + i for i in range(3)]
    pools = [torch.zeros((2, 6, 2, 16, 64), dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    rows = torch.randn((2, 23, 2, 64), device=DEV).to(torch.bfloat16)
    torch.ops.pe.kv_write_paged(rows, rows, pools[0], pools[1], slots, st)
    acc = torch.zeros((2, 22), dtype=torch.int32, device=DEV)
    acc[0, 0], acc[0, 2], acc[0, 3] = 2, 3, 17
    torch.ops.pe.kv_compact_paged(pools[0], pools[1], table, t([0, 0], torch.int64), acc, 0, st)
    for p in pools:
        assert torch.equal(p[:, 5, :, 0], rows[:, 3]) and torch.equal(p[:, 5, :, 1], rows[:, 17])
        assert torch.equal(p[:, 5, :, 2], rows[:, 2]) and torch.equal(p[:, 3, :, 0], rows[:, 20])
    assert int(st.item()) == 0


def test_a_step_of_the_operators_in_one_graph():
    """Tables, write, attention and commit as a decode step runs them, captured once and replayed as the sequences grow,
    against the same step on host integers and float64."""
    nh, nkv, hd, ps, B, T, layers = 8, 2, 128, 16, 3, 5, 2
    gen = torch.Generator().manual_seed(30)
    t = lambda x, d=torch.int32: torch.tensor(x, dtype=d, device=DEV)
    pages = 40
    pools = [torch.zeros((layers, pages, nkv, ps, hd), dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    table, held, free, top = t([[-1] * 8] * B), t([0] * B), t(list(range(pages))), t([pages])
    seq_len, row0, st = t([0] * B, torch.int64), t([0, T, 2 * T, 3 * T]), status_word()
    bits, _ = ancestor_bits([-1, 0, 1, 0, 3], 1)
    bits = bits.repeat(B, 1).to(DEV)
    qkv = torch.zeros((layers, B * T, (nh + 2 * nkv) * hd), dtype=torch.bfloat16, device=DEV)
    acc = t([[3, 0, 0, 3, 4, 0, 0]] * B)  # the path 0, 3, 4
    out = torch.zeros((B * T, nh * hd), dtype=torch.bfloat16, device=DEV)
    slots = torch.zeros(B * T, dtype=torch.int64, device=DEV)
    ws = torch.empty(max(16, ops.attention_paged_workspace_bytes(B * T, B, nh, nkv, hd, T, 64, 0, torch.bfloat16)),
                     dtype=torch.uint8, device=DEV)
    kv = lambda i: qkv[:, :, (nh + i * nkv) * hd: (nh + (i + 1) * nkv) * hd].view(layers, B * T, nkv, hd)

    def step():
        ops.page_tables(seq_len, row0, table, held, free, top, ps, B * T, st, slots=slots)
        ops.kv_write_paged(kv(0), kv(1), pools[0], pools[1], slots, st)
        ops.tree_attention_paged(qkv[1, :, : nh * hd].view(B * T, nh, hd), pools[0][1], pools[1][1], table, row0, seq_len,
                                 hd ** -0.5, T, 64, st, bits=bits, workspace=ws, out=out)
        ops.kv_compact_paged(pools[0], pools[1], table, seq_len, acc, st)
        seq_len.add_(acc[:, 0])

    step()  # loads the kernels
    keep = [torch.zeros((B, 0, nkv, hd), dtype=torch.float64, device=DEV) for _ in range(2)]
    seq_len.zero_(), held.zero_(), top.fill_(pages), table.fill_(-1)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for rep in range(6):
        qkv.copy_(torch.randn(qkv.shape, generator=gen).to(torch.bfloat16))
        out.fill_(9.0)
        g.replay()
        torch.cuda.synchronize()
        new = [kv(i)[1].view(B, T, nkv, hd).double() for i in range(2)]
        for b in range(B):
            k, v = (torch.cat([keep[i][b], new[i][b]]) for i in range(2))
            n = keep[0].shape[1]
            see = torch.cat([torch.ones((T, n), dtype=torch.bool, device=DEV),
                             ((bits[b * T: (b + 1) * T] >> torch.arange(T, device=DEV)) & 1) == 1], 1)
            for h in range(nh):
                q = qkv[1, b * T: (b + 1) * T, h * hd: (h + 1) * hd].double()
                s = (q @ k[:, h // 4].t().contiguous() * hd ** -0.5).masked_fill(~see, -math.inf)
                w = torch.softmax(s, 1)
                ref, mag = w @ v[:, h // 4], w @ v[:, h // 4].abs()
                got = out[b * T: (b + 1) * T, h * hd: (h + 1) * hd].double()
                u = torch.finfo(torch.bfloat16).eps / 2
                assert bool(((got - ref).abs() <= u * ref.abs() + (u + 2.0 ** -13) * mag).all()), (rep, b, h)
        keep = [torch.cat([keep[i], new[i][:, [0, 3, 4]]], 1) for i in range(2)]
        assert seq_len.tolist() == [3 * (rep + 1)] * B and int(st.item()) == 0
