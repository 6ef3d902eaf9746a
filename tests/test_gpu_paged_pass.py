"""The batched pass over a paged cache behind a shared prefix, used as a server
uses it: prefix set, prompts appended in chunks, trees verified, walked and
committed, sequences released and their pages given out again. Every sequence is
checked against the oracle's batch-1 restatement (src/pe/target.py:203-224) on
its own tokens, within the pass's parity rule."""

import random

import pytest
import torch

from oracle import masks as om
from oracle import verify as ov
from oracle.model import OracleTarget
from parallel_eagle_amd import _lib
from parallel_eagle_amd import batch as pb
from parallel_eagle_amd import paged as pp
from parallel_eagle_amd.config import ModelShape
from parallel_eagle_amd.target import TargetModel
from tests.test_gpu_target import _check_acceptance, _close, _fp32_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
TOL = 2e-2


def small(weights, dtype, heads=(8, 2)):
    return ModelShape(name=f"small-{weights}", num_layers=2, hidden=512, num_heads=heads[0], num_kv_heads=heads[1],
                      head_dim=128, intermediate=1024, vocab=1024, weight_format=weights, dtype=dtype,
                      feature_layers=(1, 2, 2), qkv_bias=heads[1] == 2)


def tree(t, rng, vocab):
    parents = [-1 if i == 0 or rng.random() < 0.2 else rng.randrange(max(0, i - 5), i) for i in range(t)]
    return [rng.randrange(vocab) for _ in range(t)], parents


def rows_of(cache, b, lo, hi):
    """K rows [lo, hi) (positions) of sequence b, [L][nkv][n][hd], read through its pages."""
    s0, ps = cache.prefix_len, cache.page_size
    out = []
    for j in range(lo, hi):
        page = cache.prefix_table[j // ps] if j < s0 else cache.block_table[b, (j - s0) // ps]
        at = j % ps if j < s0 else (j - s0) % ps
        out.append(cache.k[:, int(page), :, at])
    return torch.stack(out, 2) if out else cache.k[:, 0, :, :0]


class Server:
    def __init__(self, shape, seed, batch, prefix, page_size=16, num_pages=64):
        self.shape, self.rng = shape, random.Random(seed)
        self.tm = TargetModel.synthetic(shape, seed=seed, device=DEV, keep_logical=True, norm_noise=0.1, cache_capacity=256)
        hw = self.tm.model.host_weights()
        self.orc = OracleTarget(shape, hw)
        self.orc.cache_dequant = True
        self.o32 = _fp32_oracle(shape, hw, self.orc)
        self.cache = pp.PagedKVCache(self.tm, batch, num_pages, page_size, max_len=256)
        self.tokens = [[self.rng.randrange(shape.vocab) for _ in range(prefix)] for _ in range(1)] * batch
        self.tokens = [list(t) for t in self.tokens]
        if prefix:
            c = self.tm.make_cache()
            _, _, c = self.tm.forward_cached(torch.tensor([self.tokens[0]]), c, torch.arange(prefix).unsqueeze(0))
            self.cache.set_prefix(c)

    def oracle(self, b, extra, pos, bias_of, orc):
        """The oracle's logits of `extra` rows behind sequence b's tokens."""
        n = len(self.tokens[b])
        cache = None
        if n:
            _, _, cache = orc.forward(self.tokens[b], list(range(n)), None, None)
        lg, fu, _ = orc.forward(extra, pos, cache, bias_of(orc.dtype))
        return lg[0], fu[0]

    def check(self, b, lg, fu, extra, pos, bias_of):
        o_lg, o_fu = self.oracle(b, extra, pos, bias_of, self.orc)
        r_lg, r_fu = self.oracle(b, extra, pos, bias_of, self.o32)
        ok_l, e_l = _close(lg, o_lg, TOL, r_lg)
        ok_f, e_f = _close(fu, o_fu, TOL, r_fu)
        assert ok_l and ok_f, (b, e_l, e_f)
        return o_lg

    def append(self, counts):
        new = [[self.rng.randrange(self.shape.vocab) for _ in range(n)] for n in counts]
        lg, fu, row0 = pp.forward_causal_paged(self.tm, new, self.cache)
        for b, t in enumerate(new):
            if t:
                n = len(self.tokens[b])

                def causal(dtype, n=n, t=t):
                    allow = torch.ones(len(t), n + len(t), dtype=torch.bool).tril(n)
                    return om.to_additive_bias(allow, dtype)

                self.check(b, lg[row0[b]: row0[b + 1]], fu[row0[b]: row0[b + 1]], t, list(range(n, n + len(t))), causal)
                self.tokens[b] += t
        assert self.cache.seq_lens == [len(t) for t in self.tokens]

    def step(self, sizes, plant):
        """One verification step; `plant[b]` nodes of a chain agree with the target."""
        V, B = self.shape.vocab, len(sizes)
        trees = [tree(t, self.rng, V) for t in sizes]
        g = torch.Generator().manual_seed(sum(sizes))
        roots = torch.randn(B, V, generator=g).to(self.tm.dtype)
        node_tokens, parents = [list(t[0]) for t in trees], [t[1] for t in trees]
        for b in range(B):
            if plant[b]:
                for i, p in enumerate(parents[b]):  # the first root child: the walk's lowest index among equals
                    if p == -1:
                        node_tokens[b][i] = ov.first_argmax(roots[b])
                        break
        lg, fu, tr = pp.forward_tree_paged(self.tm, node_tokens, parents, self.cache)
        out = pb.accept_batch_device(roots.to(DEV), lg, tr)
        res = [(r[2: 2 + r[0]], r[1]) for r in out.cpu().tolist()]
        want_rows = []
        for b in range(B):
            n, T = len(self.tokens[b]), sizes[b]
            pos = [n + d for d in om.tree_depths(parents[b])]
            r0 = tr.row0[b]

            def bias(dtype, b=b, n=n):
                return om.to_additive_bias(om.tree_allow_mask(parents[b], n)[n:, :], dtype)

            o_lg = self.check(b, lg[r0: r0 + T], fu[r0: r0 + T], node_tokens[b], pos, bias)
            ref = ov.accept_tree_cached(roots[b], o_lg, node_tokens[b], parents[b])
            _check_acceptance(res[b], ref, roots[b], o_lg, roots[b], lg[r0: r0 + T])
            before = rows_of(self.cache, b, n, n + T)
            want_rows.append(before[:, :, res[b][0]].clone())
        kept = [rows_of(self.cache, b, 0, len(self.tokens[b])).clone() for b in range(B)]
        pp.commit_paged(self.tm, self.cache, tr, out)
        for b in range(B):
            n, k = len(self.tokens[b]), len(res[b][0])
            assert torch.equal(rows_of(self.cache, b, 0, n), kept[b])
            assert torch.equal(rows_of(self.cache, b, n, n + k), want_rows[b])
            self.tokens[b] += [node_tokens[b][i] for i in res[b][0]]
        assert self.cache.seq_lens == [len(t) for t in self.tokens]
        return res


@pytest.mark.parametrize("weights,dtype,heads", [("nf4", "bfloat16", (8, 2)), ("dense", "float16", (4, 4))])
@pytest.mark.parametrize("prefix", [0, 37])
def test_a_server_over_pages(weights, dtype, heads, prefix):
    s = Server(small(weights, dtype, heads), 3, 3, prefix)
    s.append([20, 0, 1] if prefix else [20, 9, 1])  # up to 64 rows
    s.append([30, 40, 16])  # more than 64
    first = s.step([9, 20, 5], [1, 1, 0])
    assert len(first[0][0]) >= 1 and len(first[1][0]) >= 1
    s.step([26, 33, 26], [1, 0, 1])
    # a finished sequence's pages come back and serve the next one
    free = s.cache.pages_free()
    held = int(s.cache.held[1])
    s.cache.release(1)
    assert s.cache.pages_free() == free + held
    s.tokens[1] = s.tokens[1][:prefix]
    s.append([0, 50, 3])
    s.step([12, 12, 12], [1, 1, 1])


@pytest.mark.parametrize("weights,dtype", [("nf4", "bfloat16"), ("dense", "float16")])
def test_prompts_of_more_than_256_rows(weights, dtype):
    """Chunks of several prompts in one pass of more rows than one row block of the linears."""
    s = Server(small(weights, dtype), 6, 3, 37)
    s.append([200, 120, 7])
    s.append([1, 1, 1])
    s.append([20, 100, 200])
    s.step([12, 26, 1], [1, 0, 1])


def test_loading_a_prefilled_cache():
    """Rows moved from contiguous caches give the pass the same values: the next pass equals one over the rows that the
    paged cache appended itself, bit for bit."""
    shape = small("nf4", "bfloat16")
    a, b = Server(shape, 4, 2, 21), Server(shape, 4, 2, 21)
    a.append([40, 17])
    for i in range(2):
        c = a.tm.make_cache()
        for lyr in range(shape.num_layers):
            c.k[lyr, :, : a.cache.seq_lens[i]] = rows_of(a.cache, i, 0, a.cache.seq_lens[i])[lyr]
        c.v.zero_()
        ps, s0 = a.cache.page_size, a.cache.prefix_len
        for j in range(a.cache.seq_lens[i]):
            page = a.cache.prefix_table[j // ps] if j < s0 else a.cache.block_table[i, (j - s0) // ps]
            c.v[:, :, j] = a.cache.v[:, int(page), :, (j if j < s0 else j - s0) % ps]
        c.seq_len = a.cache.seq_lens[i]
        b.cache.load(i, c)
    assert a.cache.seq_lens == b.cache.seq_lens
    rng = random.Random(1)
    trees = [tree(t, rng, shape.vocab) for t in (11, 30)]
    args = [t[0] for t in trees], [t[1] for t in trees]
    la, fa, _ = pp.forward_tree_paged(a.tm, *args, a.cache)
    lb, fb, _ = pp.forward_tree_paged(b.tm, *args, b.cache)
    assert torch.equal(la, lb) and torch.equal(fa, fb)


def test_running_out_of_pages_raises_and_keeps_the_lengths():
    shape = small("dense", "bfloat16")
    s = Server(shape, 5, 2, 16, num_pages=5)  # one page of prefix, four left
    s.append([30, 10])  # two and one
    with pytest.raises(_lib.PEError) as e:
        pp.forward_tree_paged(s.tm, [[1] * 20, [1] * 10], [[-1] * 20, [-1] * 10], s.cache)
    assert e.value.status & _lib.PE_ERR_CAPACITY
    assert s.cache.seq_lens == [46, 26]
    s.cache.release(0)
    s.tokens[0] = s.tokens[0][:16]
    s.append([2, 9])
    with pytest.raises(ValueError):
        s.cache.release(0, 0)
    with pytest.raises(ValueError):
        s.cache.load(1, s.tm.make_cache())
    with pytest.raises(ValueError):
        s.cache.set_prefix(s.tm.make_cache())
    with pytest.raises(ValueError):
        pp.forward_causal_paged(s.tm, [[], []], s.cache)
    with pytest.raises(ValueError):
        pp.PagedKVCache(s.tm, 2, 8, page_size=48)
