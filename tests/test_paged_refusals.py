"""What the paged cache's entry points refuse on the host (no kernel is
launched: the pointers are never read) and what their wrappers raise."""

import ctypes as C
import random
import re

import pytest
import torch

from parallel_eagle_amd import _lib, ops

P = C.c_void_p(64)  # an aligned address that nothing reads


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        pytest.skip("libpe_hip.so not built")
    return _lib.load()


def attention(**kw):
    a = _lib.PagedAttentionArgs()
    for f in ("q", "k_pool", "v_pool", "out", "block_table", "prefix_table", "seq_row0", "seq_len", "bits", "positions",
              "workspace", "status"):
        setattr(a, f, 64)
    a.workspace_bytes, a.ld_q, a.ld_out, a.ld_table, a.table_cols = 1 << 40, 1024, 1024, 4, 4
    a.num_pages, a.prefix_pages, a.prefix_len, a.max_len, a.M = 100, 2, 20, 50, 10
    a.batch, a.max_rows, a.nh, a.nkv, a.hd, a.page_size = 2, 8, 8, 2, 128, 16
    a.dtype, a.mask_mode, a.words, a.scale = _lib.PE_DTYPE_BF16, _lib.PE_MASK_TREE, 1, 0.1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


REFUSED = [dict(q=None), dict(k_pool=None), dict(v_pool=None), dict(out=None), dict(block_table=None), dict(seq_row0=None),
           dict(seq_len=None), dict(status=None), dict(bits=None), dict(dtype=7), dict(page_size=48), dict(page_size=8),
           dict(page_size=2048), dict(batch=0), dict(nkv=3), dict(nkv=0), dict(hd=0), dict(hd=264), dict(M=-1),
           dict(max_rows=-1), dict(prefix_len=-1), dict(max_len=19), dict(max_len=1 << 30), dict(num_pages=0),
           dict(table_cols=0), dict(ld_table=3), dict(ld_q=1023), dict(ld_out=1016), dict(window=-1), dict(softcap=-1.0),
           dict(softcap=float("nan")), dict(softcap=float("inf")), dict(scale=float("inf")),
           dict(nkv=1 << 14, nh=1 << 14, page_size=1024, ld_q=1 << 21, ld_out=1 << 21), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(mask_mode=2),
           dict(words=0), dict(prefix_table=None), dict(prefix_pages=1), dict(window=4, positions=None),
           dict(slopes=64, positions=None), dict(workspace=72)]


@pytest.mark.parametrize("kw", REFUSED, ids=[",".join(f"{k}={v}" for k, v in r.items()) for r in REFUSED])
def test_attention_refuses(lib, kw):
    assert lib.pe_tree_attention_paged(C.byref(attention(**kw)), None) == _lib.PE_ERR_ARG


def test_attention_refuses_wide_trees_and_small_workspaces(lib):
    call = lambda **kw: lib.pe_tree_attention_paged(C.byref(attention(**kw)), None)
    assert lib.pe_tree_attention_paged(None, None) == _lib.PE_ERR_ARG
    assert call(max_rows=65) == _lib.PE_ERR_TREE
    assert call(words=5, max_rows=300) == _lib.PE_ERR_TREE
    assert call(M=0, q=None, out=None, bits=None) == _lib.PE_OK
    big = dict(M=400, max_rows=40, batch=10, prefix_len=4000, prefix_pages=250, max_len=5000, table_cols=100, ld_table=100)
    need = lib.pe_attention_paged_workspace_bytes(400, 10, 8, 2, 128, 40, 5000, 4000, _lib.PE_DTYPE_BF16)
    assert need > 0
    assert call(workspace_bytes=0, **big) == _lib.PE_ERR_WORKSPACE
    assert call(workspace=None, workspace_bytes=0, **big) == _lib.PE_ERR_WORKSPACE


def test_workspace_bytes_of_calls_that_are_refused_or_need_none(lib):
    f = lib.pe_attention_paged_workspace_bytes
    assert f(0, 2, 8, 2, 128, 8, 50, 20, 1) == 0 and f(10, 2, 8, 3, 128, 8, 50, 20, 1) == 0
    assert f(10, 2, 8, 2, 80, 8, 50, 20, 1) == 0 and f(10, 2, 8, 2, 128, 8, 50, 20, 0) == 0
    assert f(10, 2, 8, 2, 128, 8, 10, 20, 1) == 0


@pytest.mark.parametrize("heads", [(32, 32), (40, 8), (16, 16), (8, 1)])
@pytest.mark.parametrize("hd", [64, 128])
def test_a_reserve_holds_every_smaller_call(lib, heads, hd):
    rng = random.Random(hd + heads[0])
    nh, nkv = heads
    for _ in range(400):
        top = round(2 ** rng.uniform(0, 14))
        room = lib.pe_attention_paged_reserve_bytes(top, nh, nkv, hd, _lib.PE_DTYPE_BF16)
        m = rng.randint(1, top)
        batch = rng.randint(1, min(m, 65535))
        rows = rng.choice([-(-m // batch), rng.randint(1, m)])
        prefix = rng.choice([0, rng.randint(1, 100), round(2 ** rng.uniform(0, 17))])
        length = prefix + rng.choice([0, round(2 ** rng.uniform(0, 17))])
        need = lib.pe_attention_paged_workspace_bytes(m, batch, nh, nkv, hd, min(rows, 65535), length, prefix,
                                                      _lib.PE_DTYPE_BF16)
        assert need <= room, (top, m, batch, rows, length, prefix)


def tables(lib, **kw):
    d = dict(seq_len=P, seq_row0=P, batch=2, M=10, prefix=0, ps=16, table=P, ld=4, cols=4, held=P, free=P, n_free=9, top=P,
             held_out=C.c_void_p(128), top_out=C.c_void_p(192), scratch=None, slots=P, status=P)
    d.update(kw)
    return lib.pe_page_tables(*d.values(), None)


@pytest.mark.parametrize("kw", [dict(seq_len=None), dict(seq_row0=None), dict(batch=0), dict(batch=70000), dict(M=-1),
                                dict(M=1 << 31), dict(prefix=-1), dict(ps=24), dict(table=None), dict(ld=3), dict(cols=0),
                                dict(held=None), dict(free=None), dict(n_free=-1), dict(top=None), dict(held_out=None),
                                dict(top_out=None), dict(slots=None), dict(status=None)],
                         ids=lambda d: next(iter(d)))
def test_page_tables_refuses(lib, kw):
    assert tables(lib, **kw) == _lib.PE_ERR_ARG


def test_page_tables_in_place_needs_scratch(lib):
    assert tables(lib, held_out=P) == _lib.PE_ERR_WORKSPACE
    assert lib.pe_page_tables_scratch_bytes(7) == 32


def test_release_write_and_compact_refuse(lib):
    rel = lambda **kw: lib.pe_page_release(*dict(dict(seqs=P, n=1, batch=2, table=P, ld=4, cols=4, held=P, free=P, n_free=9,
                                                     top=P, status=P), **kw).values(), None)
    for kw in (dict(seqs=None), dict(n=-1), dict(batch=0), dict(table=None), dict(ld=3), dict(held=None), dict(free=None),
               dict(top=None), dict(status=None)):
        assert rel(**kw) == _lib.PE_ERR_ARG, kw
    assert rel(n=0, seqs=None) == _lib.PE_OK
    s3 = (C.c_int64 * 3)(0, 256, 128)
    wr = lambda **kw: lib.pe_kv_write_paged(*dict(dict(k=P, v=P, ks=s3, vs=s3, L=1, M=4, nkv=2, hd=128, dtype=1, kp=P, vp=P,
                                                      pages=9, ps=16, slots=P, status=P), **kw).values(), None)
    for kw in (dict(k=None), dict(v=None), dict(ks=None), dict(L=0), dict(M=-1), dict(nkv=0), dict(hd=0), dict(dtype=9),
               dict(kp=None), dict(pages=0), dict(ps=20), dict(slots=None), dict(status=None), dict(M=1 << 30, nkv=64)):
        assert wr(**kw) == _lib.PE_ERR_ARG, kw
    assert wr(M=0) == _lib.PE_OK
    co = lambda **kw: lib.pe_kv_compact_paged(*dict(dict(kp=P, vp=P, L=1, nkv=2, hd=128, dtype=1, pages=9, ps=16, table=P,
                                                        ld=4, cols=4, batch=2, lens=P, prefix=0, acc=P, rows=8, status=P),
                                                   **kw).values(), None)
    for kw in (dict(kp=None), dict(L=0), dict(nkv=0), dict(hd=0), dict(dtype=9), dict(pages=0), dict(ps=20),
               dict(table=None), dict(ld=3), dict(batch=0), dict(lens=None), dict(prefix=-1), dict(acc=None), dict(rows=0),
               dict(status=None)):
        assert co(**kw) == _lib.PE_ERR_ARG, kw


def test_the_pass_refuses_bad_paged_arguments(lib):
    d = _lib.ModelDesc()
    d.num_layers, d.hidden, d.num_heads, d.num_kv_heads, d.head_dim = 1, 512, 4, 4, 128
    d.intermediate, d.intermediate_padded, d.vocab = 1024, 1024, 1024
    d.dtype, d.weight_format, d.qkv_layout = _lib.PE_DTYPE_BF16, _lib.PE_WFMT_DENSE, _lib.PE_QKV_ROPE_PAIRED

    def call(**kw):
        a = _lib.PassArgs()
        for f in ("input_ids", "positions", "tree_bits", "k_cache", "v_cache", "workspace", "status", "seq_row0",
                  "seq_prefix", "slots", "block_table", "prefix_table"):
            setattr(a, f, 64)
        a.M, a.mask_mode, a.prefix_len, a.bits_words, a.batch, a.max_seq_rows = 8, 0, 40, 1, 2, 8
        a.ld_table = a.table_cols = 4
        a.num_pages, a.prefix_pages, a.shared_len, a.page_size = 9, 2, 20, 16
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.pe_forward(C.byref(d), C.byref(a), None)

    for kw in (dict(batch=0), dict(seq_row0=None), dict(seq_prefix=None), dict(slots=None), dict(block_table=None),
               dict(status=None), dict(node_keys=64), dict(num_pages=0), dict(shared_len=-1), dict(shared_len=41),
               dict(page_size=-16)):
        assert call(**kw) == _lib.PE_ERR_ARG, kw
    assert call(max_seq_rows=9) == _lib.PE_ERR_TREE
    assert call() == _lib.PE_ERR_WORKSPACE
    need = lib.pe_forward_paged_workspace_bytes(C.byref(d), 8, 8, 40, 2, 20)
    assert need > 0 and lib.pe_forward_paged_workspace_bytes(C.byref(d), 8, 8, 10, 2, 20) == 0
    d.head_dim = 64
    assert call(workspace_bytes=1 << 40) == _lib.PE_ERR_ARG


def test_wrappers_want_device_tensors():
    z = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.page_tables(torch.zeros(1, dtype=torch.int64), z, z.view(1, 2), z, z, z, 16, 1, z)
    with pytest.raises(ValueError):
        ops.page_release(z, z.view(1, 2), z, z, z, z)
    with pytest.raises(ValueError):
        ops.kv_write_paged(torch.zeros(1, 1, 1, 8), torch.zeros(1, 1, 1, 8), torch.zeros(1, 1, 1, 16, 8),
                           torch.zeros(1, 1, 1, 16, 8), torch.zeros(1, dtype=torch.int64), z)
    with pytest.raises(ValueError):
        ops.kv_compact_paged(torch.zeros(1, 1, 1, 16, 8), torch.zeros(1, 1, 1, 16, 8), z.view(1, 2),
                             torch.zeros(1, dtype=torch.int64), torch.zeros(1, 4, dtype=torch.int32), z)
    with pytest.raises(ValueError):
        ops.tree_attention_paged(torch.zeros(1, 1, 64), torch.zeros(1, 1, 16, 64), torch.zeros(1, 1, 16, 64), z.view(1, 2),
                                 z, torch.zeros(1, dtype=torch.int64), 1.0, 1, 1, z)


def test_the_packed_arguments_are_the_structs_fields():
    """Every field a different value, through the wrapper's format and through the struct's constructor."""
    fields = _lib.PagedAttentionArgs._fields_
    codes = {C.c_void_p: "Q", C.c_int64: "q", C.c_int32: "i", C.c_float: "f"}
    runs = re.findall(r"(\d*)([a-zA-Z])", ops._PAGED_ARGS.format)
    assert "".join(c * int(n or 1) for n, c in runs) == "".join(codes[t] for _, t in fields)
    want = [float(i) if t is C.c_float else i for i, (_, t) in enumerate(fields, 1)]
    assert ops._PAGED_ARGS.pack(*want) == bytes(_lib.PagedAttentionArgs(*want))
