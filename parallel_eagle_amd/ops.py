"""Thin torch-tensor wrappers over the C ABI of libpe_hip.so.

Every function takes device tensors, validates shapes and dtypes on the host,
launches on torch's current HIP stream and raises ``PEError`` on a non-zero
status. They are registered as torch custom ops under the ``pe`` namespace
(``torch.ops.pe.*``) where a functional form exists; in-place cache updates
stay plain functions. There is no CPU implementation behind any of them.
"""

from __future__ import annotations

import ctypes as C
import struct

import torch

from . import _lib
from ._lib import check

DTYPE_CODE = {torch.float32: _lib.PE_DTYPE_F32, torch.bfloat16: _lib.PE_DTYPE_BF16, torch.float16: _lib.PE_DTYPE_F16}


def lib():
    return _lib.load()


def stream_ptr() -> int:
    """The current stream's handle (0.3 us; building a torch.cuda.Stream object for it takes 2.9 us of every call)."""
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


def ptr(t: torch.Tensor | None) -> int | None:
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("parallel_eagle_amd kernels take HIP device tensors")
    return t.data_ptr()


def dcode(dtype: torch.dtype) -> int:
    try:
        return DTYPE_CODE[dtype]
    except KeyError as e:
        raise TypeError(f"unsupported dtype {dtype}") from e


def _req(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


# ------------------------------------------------------------------ synthetic / formats
def fill_normal(out: torch.Tensor, seed: int, stream_id: int, std: float) -> torch.Tensor:
    _req(out.is_contiguous(), "out must be contiguous")
    check(lib().pe_fill_normal(ptr(out), out.numel(), dcode(out.dtype), seed, stream_id, std, stream_ptr()),
          "pe_fill_normal")
    return out


def fill_uniform_int(out: torch.Tensor, hi: int, seed: int, stream_id: int) -> torch.Tensor:
    _req(out.dtype == torch.int64 and out.is_contiguous(), "out must be contiguous int64")
    check(lib().pe_fill_uniform_int(ptr(out), out.numel(), hi, seed, stream_id, stream_ptr()), "pe_fill_uniform_int")
    return out


def nf4_quantize(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    _req(w.dtype == torch.float32 and w.dim() == 2 and w.is_contiguous(), "w must be contiguous fp32 [N][K]")
    n, k = w.shape
    _req(k % 64 == 0, "K must be a multiple of 64")
    packed = torch.empty((n, k // 2), dtype=torch.uint8, device=w.device)
    absmax = torch.empty((n, k // 64), dtype=torch.float16, device=w.device)
    check(lib().pe_nf4_quantize(ptr(w), n, k, ptr(packed), ptr(absmax), stream_ptr()), "pe_nf4_quantize")
    return packed, absmax


def nf4_repack(packed: torch.Tensor, absmax: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Logical NF4 (packed uint8 [N][K/2], absmax fp16 or fp32 [N][K/64]) -> tiled;
    the tiled absmax keeps the absmax dtype."""
    n, kh = packed.shape
    k = kh * 2
    _req(packed.dtype == torch.uint8 and packed.is_contiguous(), "packed must be contiguous uint8 [N][K/2]")
    _req(absmax.dtype in (torch.float16, torch.float32) and absmax.shape == (n, k // 64) and absmax.is_contiguous(),
         "absmax must be contiguous fp16 or fp32 [N][K/64]")
    _req(n % 32 == 0 and k % 128 == 0, "N % 32 == 0 and K % 128 == 0 required")
    tiled = torch.empty(n * k // 2, dtype=torch.uint8, device=packed.device)
    tabs = torch.empty(n * k // 64, dtype=absmax.dtype, device=packed.device)
    fn = "pe_nf4_repack_f32abs" if absmax.dtype == torch.float32 else "pe_nf4_repack"
    check(getattr(lib(), fn)(ptr(packed), ptr(absmax), n, k, ptr(tiled), ptr(tabs), stream_ptr()), fn)
    return tiled, tabs


def nf4_dequant(tiled: torch.Tensor, tabs: torch.Tensor, n: int, k: int) -> torch.Tensor:
    _req(tabs.dtype in (torch.float16, torch.float32), "tiled absmax must be fp16 or fp32")
    out = torch.empty((n, k), dtype=torch.bfloat16, device=tiled.device)
    fn = "pe_nf4_dequant_f32abs" if tabs.dtype == torch.float32 else "pe_nf4_dequant"
    check(getattr(lib(), fn)(ptr(tiled), ptr(tabs), n, k, ptr(out), stream_ptr()), fn)
    return out


def nf4_absmax_dequant(q: torch.Tensor, code: torch.Tensor, nested_absmax: torch.Tensor, nested_blocksize: int,
                       offset: float) -> torch.Tensor:
    """bitsandbytes double-quantised absmax -> fp32: code[q[i]] * nested_absmax[i // bs] + offset."""
    _req(q.dtype == torch.uint8 and q.is_contiguous(), "q must be contiguous uint8")
    _req(code.dtype == torch.float32 and code.numel() == 256 and code.is_contiguous(), "code must be 256 fp32")
    n = q.numel()
    _req(nested_absmax.dtype == torch.float32 and nested_absmax.is_contiguous()
         and nested_absmax.numel() * nested_blocksize >= n, "nested_absmax must cover every block")
    out = torch.empty(n, dtype=torch.float32, device=q.device)
    check(lib().pe_nf4_absmax_dequant(ptr(q), n, ptr(code), ptr(nested_absmax), nested_blocksize, float(offset),
                                      ptr(out), stream_ptr()), "pe_nf4_absmax_dequant")
    return out


def dense_repack(w: torch.Tensor) -> torch.Tensor:
    _req(w.dim() == 2 and w.is_contiguous(), "w must be contiguous [N][K]")
    n, k = w.shape
    out = torch.empty(n * k, dtype=w.dtype, device=w.device)
    check(lib().pe_dense_repack(ptr(w), n, k, dcode(w.dtype), ptr(out), stream_ptr()), "pe_dense_repack")
    return out


# ------------------------------------------------------------------ GEMMs
def gemm_workspace_bytes(m: int, n: int, k: int, nf4: bool, dtype: torch.dtype, epilogue: int) -> int:
    return int(lib().pe_gemm_workspace_bytes(m, n, k, _lib.PE_WFMT_NF4 if nf4 else _lib.PE_WFMT_DENSE,
                                             dcode(dtype), epilogue))


COUNTER_BYTES = 32768  # the arrival counters at the head of a workspace, zero before its first use
# Up to this size one torch.zeros is the cheaper call: 4.9 us of host time at any size up to 16 MiB, where an allocation
# and a fill of the counters alone take 6.1 us. Calls with larger workspaces are mostly bound by the GPU's own time, in
# which filling the counters alone is shorter: attention of one node over 16000 keys (2.2 MB) takes 24.1 us and 24.9
# with all of it cleared, of 26 nodes over 4096 keys (4 MB) 19.9 and 21.4.
ZEROED_BYTES = 2 << 20


def _workspace(nbytes: int, device) -> torch.Tensor:
    """A workspace for one call: only its counters need a value (the rest is written before it is read)."""
    if nbytes <= ZEROED_BYTES:
        return torch.zeros(max(nbytes, 256), dtype=torch.uint8, device=device)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    ws[:COUNTER_BYTES].zero_()
    return ws


def linear(x: torch.Tensor, n: int, *, nf4: tuple | None = None, dense: torch.Tensor | None = None,
           epilogue: int = _lib.PE_EPI_STORE, bias: torch.Tensor | None = None, resid: torch.Tensor | None = None,
           out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Y = X . W^T with W given as nf4=(tiled, tabs) or dense (tiled/row-major)."""
    _req(x.dim() == 2 and x.stride(1) == 1, "x must be [M][K] with unit column stride")
    m, k = x.shape
    n_out = n // 2 if epilogue == _lib.PE_EPI_SWIGLU else n
    if out is None:
        out = torch.empty((m, n_out), dtype=x.dtype, device=x.device)
    _req(out.shape == (m, n_out) and out.stride(1) == 1 and out.dtype == x.dtype, "bad out")
    if resid is not None:
        _req(resid.shape == (m, n_out) and resid.dtype == x.dtype, "bad resid")
    if workspace is None:
        workspace = _workspace(gemm_workspace_bytes(m, n, k, nf4 is not None, x.dtype, epilogue), x.device)
    L = lib()
    if nf4 is not None:
        _req(x.dtype == torch.bfloat16, "NF4 linears compute in bf16")
        fn = L.pe_nf4_gemm_f32abs if nf4[1].dtype == torch.float32 else L.pe_nf4_gemm
        rc = fn(ptr(x), x.stride(0), m, k, ptr(nf4[0]), ptr(nf4[1]), n, epilogue, ptr(bias), ptr(resid),
                resid.stride(0) if resid is not None else 0, ptr(out), out.stride(0), ptr(workspace),
                workspace.numel(), stream_ptr())
    else:
        rc = L.pe_dense_gemm(ptr(x), x.stride(0), m, k, ptr(dense), dcode(x.dtype), n, epilogue, ptr(bias),
                             ptr(resid), resid.stride(0) if resid is not None else 0, ptr(out), out.stride(0),
                             ptr(workspace), workspace.numel(), stream_ptr())
    check(rc, "linear")
    return out


def xtile_index(m: int, k: int, device=None) -> torch.Tensor:
    """[m][k] -> flat position of each element in the A-tiled activation layout
    (the order the NF4 GEMM reads X as its MFMA A operand; k % 128 == 0)."""
    _req(k % 128 == 0, "A-tiled activations need K % 128 == 0")
    row = torch.arange(m, device=device).view(m, 1)
    col = torch.arange(k, device=device).view(1, k)
    units = k // 128
    mt, ln = row // 32, row % 32
    p, c = col // 128, col % 128
    return ((((mt * units + p) * 8 + (c % 64) // 8) * 64 + ln + 32 * (c // 64)) * 8 + c % 8)


def to_xtile(x: torch.Tensor) -> torch.Tensor:
    """Row-major [M][K] -> A-tiled flat buffer (rows past M of the last 32-row
    tile are zero)."""
    m, k = x.shape
    out = torch.zeros(((m + 31) // 32) * 32 * k, dtype=x.dtype, device=x.device)
    out[xtile_index(m, k, x.device).flatten()] = x.flatten()
    return out


def from_xtile(t: torch.Tensor, m: int, k: int) -> torch.Tensor:
    return t[xtile_index(m, k, t.device).flatten()].view(m, k)


def linear_tiled(xt: torch.Tensor, m: int, k: int, n: int, nf4: tuple, *, epilogue: int = _lib.PE_EPI_STORE,
                 resid: torch.Tensor | None = None, out: torch.Tensor | None = None, out_tiled: bool = False,
                 workspace: torch.Tensor | None = None) -> torch.Tensor:
    """pe_nf4_gemm_tiled: X given A-tiled (to_xtile); the output row-major, or
    A-tiled when out_tiled."""
    n_out = n // 2 if epilogue == _lib.PE_EPI_SWIGLU else n
    if out is None:
        out = (torch.zeros(((m + 31) // 32) * 32 * n_out, dtype=xt.dtype, device=xt.device) if out_tiled
               else torch.empty((m, n_out), dtype=xt.dtype, device=xt.device))
    if workspace is None:
        workspace = _workspace(gemm_workspace_bytes(m, n, k, True, xt.dtype, epilogue), xt.device)
    _req(nf4[1].dtype == torch.float16, "the A-tiled and split-partial NF4 entry points take fp16 absmax")
    check(lib().pe_nf4_gemm_tiled(ptr(xt), m, k, ptr(nf4[0]), ptr(nf4[1]), n, epilogue, None, ptr(resid),
                                  resid.stride(0) if resid is not None else 0, ptr(out),
                                  0 if out_tiled else out.stride(0), n_out // 128 if out_tiled else 0,
                                  ptr(workspace), workspace.numel(), stream_ptr()), "linear_tiled")
    return out


# ------------------------------------------------------------------ elementwise
def nf4_linear_partials(x: torch.Tensor, m: int, k: int, n: int, nf4: tuple, *, x_tiled: bool = False,
                        partials: torch.Tensor | None = None) -> tuple[torch.Tensor, int]:
    """pe_nf4_gemm_partials: fp32 split partials [S][m][n] of X . deq(W)^T (X
    row-major [m][k] or A-tiled); returns (partials, S)."""
    nbytes = int(lib().pe_nf4_gemm_partials_bytes(m, n, k))
    _req(nbytes > 0, "unsupported shape for split partials")
    if partials is None:
        partials = torch.empty(nbytes // 4, dtype=torch.float32, device=x.device)
    s = C.c_int(0)
    _req(nf4[1].dtype == torch.float16, "the A-tiled and split-partial NF4 entry points take fp16 absmax")
    check(lib().pe_nf4_gemm_partials(ptr(x), k if x_tiled else x.stride(0), int(x_tiled), m, k, ptr(nf4[0]),
                                     ptr(nf4[1]), n, ptr(partials), partials.numel() * 4, C.byref(s), stream_ptr()),
          "nf4_linear_partials")
    return partials[: s.value * m * n].view(s.value, m, n), s.value


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float, mode: int = _lib.PE_NORM_HF) -> torch.Tensor:
    """RMSNorm of the rows of x [M][H]; ``mode`` PE_NORM_HF (HF LlamaRMSNorm) or
    PE_NORM_FP32_WEIGHT (the drafter's RMSNorm, one rounding)."""
    _req(x.dim() == 2 and x.stride(1) == 1 and w.dtype == x.dtype, "bad rmsnorm args")
    out = torch.empty_like(x)
    check(lib().pe_rmsnorm_ex(ptr(x), x.stride(0), x.shape[0], x.shape[1], ptr(w), eps, dcode(x.dtype), int(mode),
                              ptr(out), out.stride(0), stream_ptr()), "pe_rmsnorm_ex")
    return out


def embed(ids: torch.Tensor, table: torch.Tensor, status: torch.Tensor) -> torch.Tensor:
    m = ids.numel()
    v, h = table.shape
    out = torch.empty((m, h), dtype=table.dtype, device=table.device)
    check(lib().pe_embed(ptr(ids), m, ptr(table), v, h, dcode(table.dtype), ptr(out), h, ptr(status),
                         stream_ptr()), "pe_embed")
    return out


def rope_qkv(qkv, nh, nkv, hd, positions, cos_sin, k_cache, v_cache, row0, status):
    m = qkv.shape[0]
    q = torch.empty((m, nh, hd), dtype=qkv.dtype, device=qkv.device)
    check(lib().pe_rope_qkv(ptr(qkv), qkv.stride(0), m, nh, nkv, hd, ptr(positions), ptr(cos_sin),
                            cos_sin.shape[1], dcode(qkv.dtype), ptr(q), ptr(k_cache), ptr(v_cache), k_cache.shape[1],
                            row0, ptr(status), stream_ptr()), "pe_rope_qkv")
    return q


# ------------------------------------------------------------------ masks
def tree_masks(parents: torch.Tensor, prefix_len: int, words: int, status: torch.Tensor):
    """parents int32 device [T] -> (bits u64 [T][words] as int64, positions int64 [T], depths int32 [T])."""
    t = parents.numel()
    bits = torch.empty((t, words), dtype=torch.int64, device=parents.device)
    pos = torch.empty(t, dtype=torch.int64, device=parents.device)
    dep = torch.empty(t, dtype=torch.int32, device=parents.device)
    check(lib().pe_tree_masks(ptr(parents), t, prefix_len, ptr(bits), words, ptr(pos), ptr(dep), ptr(status),
                              stream_ptr()), "pe_tree_masks")
    return bits, pos, dep


def tree_allow_dense(bits: torch.Tensor, prefix_len: int) -> torch.Tensor:
    t, words = bits.shape
    n = prefix_len + t
    allow = torch.empty((n, n), dtype=torch.bool, device=bits.device)
    check(lib().pe_tree_allow_dense(ptr(bits), t, words, prefix_len, ptr(allow), stream_ptr()), "pe_tree_allow_dense")
    return allow


def bias_to_bits(bias: torch.Tensor, prefix_len: int, words: int, status: torch.Tensor) -> torch.Tensor:
    _req(bias.dim() == 2 and bias.stride(1) == 1, "bias must be [T][P+T] with unit column stride")
    t = bias.shape[0]
    bits = torch.empty((t, words), dtype=torch.int64, device=bias.device)
    check(lib().pe_bias_to_bits(ptr(bias), bias.stride(0), dcode(bias.dtype), t, prefix_len, ptr(bits), words,
                                ptr(status), stream_ptr()), "pe_bias_to_bits")
    return bits


# ------------------------------------------------------------------ attention
def tree_attention(q, k_cache, v_cache, prefix_len, mask_mode, bits, scale, workspace=None):
    """q [T][nh][hd]; caches [nkv][cap][hd] (one layer)."""
    t, nh, hd = q.shape
    nkv, cap, _ = k_cache.shape
    words = bits.shape[1] if bits is not None else 0
    need = int(lib().pe_attention_workspace_bytes(t, nh, nkv, hd, prefix_len + t, dcode(q.dtype)))
    if workspace is None:
        workspace = _workspace(need, q.device)
    out = torch.empty((t, nh * hd), dtype=q.dtype, device=q.device)
    check(lib().pe_tree_attention(ptr(q), ptr(k_cache), ptr(v_cache), cap, nh, nkv, hd, t, prefix_len, mask_mode,
                                  ptr(bits), words, scale, dcode(q.dtype), ptr(out), out.stride(0), ptr(workspace),
                                  workspace.numel(), stream_ptr()), "pe_tree_attention")
    return out


def tree_attention_batch(q, k_cache, v_cache, seq_row0, seq_prefix, bits, scale, max_rows, max_prefix,
                         workspace=None):
    """q [M][nh][128]; caches [B][nkv][cap][128] (one layer per sequence);
    seq_row0 int32 [B + 1], seq_prefix int64 [B] and bits int64 [M][words] on
    the device."""
    m, nh, hd = q.shape
    b, nkv, cap, _ = k_cache.shape
    _req(hd == 128 and q.is_contiguous() and k_cache.is_contiguous() and v_cache.is_contiguous(),
         "q and the caches must be contiguous with 128-dim heads")
    need = int(lib().pe_attention_batch_workspace_bytes(max_rows, nh, nkv, max_prefix + max_rows, b))
    if workspace is None:
        workspace = _workspace(need, q.device)
    out = torch.empty((m, nh * hd), dtype=q.dtype, device=q.device)
    check(lib().pe_tree_attention_batch(ptr(q), ptr(k_cache), ptr(v_cache), cap, nkv * cap * hd, nh, nkv, max_rows,
                                        max_prefix, b, ptr(seq_row0), ptr(seq_prefix), ptr(bits), bits.shape[1],
                                        scale, dcode(q.dtype), ptr(out), out.stride(0), ptr(workspace),
                                        workspace.numel(), stream_ptr()), "pe_tree_attention_batch")
    return out


# ------------------------------------------------------------------ acceptance / cache
def argmax_rows(x: torch.Tensor) -> torch.Tensor:
    _req(x.dim() == 2 and x.stride(1) == 1, "x must be [rows][V]")
    out = torch.empty(x.shape[0], dtype=torch.int32, device=x.device)
    check(lib().pe_argmax_rows(ptr(x), x.stride(0), x.shape[0], x.shape[1], dcode(x.dtype), ptr(out), stream_ptr()),
          "pe_argmax_rows")
    return out


def accept_tree(root_logit: torch.Tensor, node_logits: torch.Tensor, node_tokens: torch.Tensor,
                parents: torch.Tensor, out: torch.Tensor | None = None, scratch: torch.Tensor | None = None):
    """Device result int32 [2 + T]: (|path|, bonus, path...)."""
    t = node_tokens.numel()
    v = root_logit.shape[-1]
    _req(root_logit.stride(-1) == 1 and (t == 0 or node_logits.stride(1) == 1), "logit rows must be contiguous")
    if out is None:
        out = torch.empty(2 + max(t, 1), dtype=torch.int32, device=root_logit.device)
    if scratch is None:
        scratch = torch.zeros(t + 2, dtype=torch.int32, device=root_logit.device)
    _req(scratch.dtype == torch.int32 and scratch.numel() >= t + 2, "scratch must hold T + 2 int32")
    ld = node_logits.stride(0) if t > 0 else v
    check(lib().pe_accept_tree(ptr(root_logit), ptr(node_logits) if t > 0 else None, ld, t, v,
                               dcode(root_logit.dtype), ptr(node_tokens) if t > 0 else None,
                               ptr(parents) if t > 0 else None, ptr(out), ptr(scratch), stream_ptr()), "pe_accept_tree")
    return out


def propose_tree(logits: torch.Tensor, widths, top_k: int, status: torch.Tensor | None = None,
                 scratch: torch.Tensor | None = None):
    """Beam tree proposal over k draft-logit rows [k][V] on the device.

    Returns (node_tokens int64 [n], parents int32 [n], status int32 [1]) as device
    tensors; n is known on the host, so nothing here waits for the GPU.
    PE_ERR_VALUE in ``status`` marks a row with a NaN or no finite value.
    ``scratch`` (k * PE_PROPOSE_SCRATCH_PER_DEPTH bytes) receives, per depth, 64
    fp32 log-probabilities and then (after all k of those) 64 int32 tokens."""
    _req(logits.dim() == 2 and logits.stride(1) == 1, "logits must be [k][V] with contiguous rows")
    k, v = logits.shape
    widths = [int(w) for w in widths]
    _req(len(widths) == k, "one width per depth row")
    dev = logits.device
    cap = k * _lib.PE_PROPOSE_MAX_WIDTH
    tokens = torch.empty(cap, dtype=torch.int64, device=dev)
    parents = torch.empty(cap, dtype=torch.int32, device=dev)
    if scratch is None:
        scratch = torch.empty(k * _lib.PE_PROPOSE_SCRATCH_PER_DEPTH, dtype=torch.uint8, device=dev)
    _req(scratch.numel() * scratch.element_size() >= k * _lib.PE_PROPOSE_SCRATCH_PER_DEPTH and scratch.is_contiguous(),
         "scratch must hold k * PE_PROPOSE_SCRATCH_PER_DEPTH bytes")
    if status is None:
        status = torch.zeros(1, dtype=torch.int32, device=dev)
    w = (C.c_int32 * k)(*widths)
    n = C.c_int32(0)
    check(lib().pe_propose_tree(ptr(logits), logits.stride(0), k, v, dcode(logits.dtype), w, int(top_k), ptr(tokens),
                                ptr(parents), C.byref(n), ptr(scratch), ptr(status), stream_ptr()), "pe_propose_tree")
    return tokens[: n.value], parents[: n.value], status


def kv_compact(k_cache, v_cache, prefix_len: int, accept_out: torch.Tensor) -> None:
    """Caches [L][nkv][cap][hd]."""
    L, nkv, cap, hd = k_cache.shape
    check(lib().pe_kv_compact(ptr(k_cache), ptr(v_cache), L, nkv, cap, hd, dcode(k_cache.dtype), prefix_len,
                              ptr(accept_out), stream_ptr()), "pe_kv_compact")


def kv_gather(k_cache, v_cache, keep: torch.Tensor, status4: torch.Tensor) -> None:
    L, nkv, cap, hd = k_cache.shape
    _req(keep.dtype == torch.int64 and keep.is_contiguous(), "keep must be contiguous int64")
    _req(status4.dtype == torch.int32 and status4.numel() >= 4, "status must be int32[4]")
    check(lib().pe_kv_gather(ptr(k_cache), ptr(v_cache), L, nkv, cap, hd, dcode(k_cache.dtype), ptr(keep),
                             keep.numel(), ptr(status4), stream_ptr()), "pe_kv_gather")


# ------------------------------------------------------------------ paged cache
def _call_on(index: int, fn, *args) -> int:
    """fn(*args, stream) on the current stream of device ``index``, whatever the current device is."""
    if index == torch._C._cuda_getDevice():
        return fn(*args, torch._C._cuda_getCurrentRawStream(index))
    with torch.cuda.device(index):
        return fn(*args, torch._C._cuda_getCurrentRawStream(index))


def _device_index(t: torch.Tensor) -> int:
    if not t.is_cuda:
        raise ValueError("parallel_eagle_amd kernels take HIP device tensors")
    return t.get_device()


def _vec(t: torch.Tensor, dtype: torch.dtype, n: int, dev: int, name: str) -> int:
    """The pointer of a contiguous vector of at least n elements on device ``dev``."""
    if (t.dtype is not dtype or t.get_device() != dev or t.numel() < n
            or (t.stride() != (1,) and (t.dim() != 1 or not t.is_contiguous()))):
        raise ValueError(f"{name} must be contiguous {dtype} with at least {n} elements, on the device of the call's "
                         "other tensors")
    return t.data_ptr()


def _table(t: torch.Tensor, batch: int, dev: int) -> tuple[int, int, int]:
    """Pointer, entries between two rows and entries of a row of a block table."""
    if t.dtype is not torch.int32 or t.get_device() != dev or t.dim() != 2:
        raise ValueError("block_table must be int32 [batch][pages] on the device of the call's other tensors")
    rows, cols = t.shape
    ld, unit = t.stride()
    if rows < batch or cols < 1 or (unit != 1 and cols > 1) or (rows > 1 and ld < cols):
        raise ValueError("block_table must have contiguous rows, one per sequence")
    return t.data_ptr(), ld if rows > 1 else cols, cols


def page_tables(seq_len: torch.Tensor, seq_row0: torch.Tensor, block_table: torch.Tensor, held: torch.Tensor,
                free_pages: torch.Tensor, free_top: torch.Tensor, page_size: int, rows: int, status: torch.Tensor, *,
                prefix_len: int = 0, held_out: torch.Tensor | None = None, top_out: torch.Tensor | None = None,
                slots: torch.Tensor | None = None) -> torch.Tensor:
    """Pages for each sequence's new rows and the rows' slots (pe_page_tables), int64 [rows].

    ``seq_len`` int64 [B] counts cached tokens (the ``prefix_len`` shared ones
    included), ``seq_row0`` int32 [B + 1] the row ranges, ``held`` int32 [B] the
    pages each sequence has; missing pages come off the end of
    ``free_pages[:free_top]`` into ``block_table`` (written in place). ``held``
    and ``free_top`` are updated in place unless ``held_out`` / ``top_out``
    receive the new counts. Slot -1: a row behind the last sequence, or without a
    page (PE_ERR_CAPACITY in ``status``)."""
    dev = _device_index(seq_row0)
    b = seq_row0.numel() - 1
    if b < 1 or not 0 <= rows < 2 ** 31:
        raise ValueError("seq_row0 must hold batch + 1 offsets, rows must be a count")
    i32 = torch.int32
    p_row0, p_len = _vec(seq_row0, i32, b + 1, dev, "seq_row0"), _vec(seq_len, torch.int64, b, dev, "seq_len")
    p_tab, ld, cols = _table(block_table, b, dev)
    p_held, p_top = _vec(held, i32, b, dev, "held"), _vec(free_top, i32, 1, dev, "free_top")
    p_free, p_status = _vec(free_pages, i32, 0, dev, "free_pages"), _vec(status, i32, 1, dev, "status")
    o_held = p_held if held_out is None else _vec(held_out, i32, b, dev, "held_out")
    o_top = p_top if top_out is None else _vec(top_out, i32, 1, dev, "top_out")
    if slots is None:
        slots = torch.empty(rows, dtype=torch.int64, device=seq_row0.device)
    p_slots = _vec(slots, torch.int64, rows, dev, "slots")
    scratch = None
    if o_held == p_held or o_top == p_top:
        scratch = torch.empty(b + 1, dtype=i32, device=seq_row0.device)
    check(_call_on(dev, lib().pe_page_tables, p_len, p_row0, b, rows, prefix_len, page_size, p_tab, ld, cols, p_held,
                   p_free, free_pages.numel(), p_top, o_held, o_top, None if scratch is None else scratch.data_ptr(),
                   p_slots, p_status), "pe_page_tables")
    return slots if slots.numel() == rows else slots[:rows]


def page_release(seqs: torch.Tensor, block_table: torch.Tensor, held: torch.Tensor, free_pages: torch.Tensor,
                 free_top: torch.Tensor, status: torch.Tensor) -> None:
    """Return the pages of the listed sequences (int32, each once) to the free list (pe_page_release)."""
    dev = _device_index(held)
    b = held.numel()
    if b < 1:
        raise ValueError("held must name the sequences")
    i32 = torch.int32
    p_tab, ld, cols = _table(block_table, b, dev)
    check(_call_on(dev, lib().pe_page_release, _vec(seqs, i32, 0, dev, "seqs"), seqs.numel(), b, p_tab, ld, cols,
                   _vec(held, i32, b, dev, "held"), _vec(free_pages, i32, 1, dev, "free_pages"), free_pages.numel(),
                   _vec(free_top, i32, 1, dev, "free_top"), _vec(status, i32, 1, dev, "status")), "pe_page_release")


def _pools(k_pool: torch.Tensor, v_pool: torch.Tensor, dim: int, dev: int) -> tuple:
    """The shape of a pair of pools."""
    shape = k_pool.shape
    if (len(shape) != dim or v_pool.shape != shape or k_pool.dtype is not v_pool.dtype or k_pool.get_device() != dev
            or v_pool.get_device() != dev or not k_pool.is_contiguous() or not v_pool.is_contiguous()
            or k_pool.numel() == 0):
        raise ValueError(f"pools must be contiguous {'[L]' if dim == 5 else ''}[pages][nkv][page_size][hd], K and V "
                         "alike, on the device of the call's other tensors")
    return shape


_I64x3 = C.c_int64 * 3


def kv_write_paged(k: torch.Tensor, v: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, slots: torch.Tensor,
                   status: torch.Tensor) -> None:
    """K/V rows [L][M][nkv][hd] (any strides over contiguous head rows: a contiguous
    cache's rows, or columns of a fused q/k/v block) to their slots of the pools
    [L][pages][nkv][page_size][hd] (pe_kv_write_paged). Rows of slot -1 are
    skipped; slots are distinct."""
    dev = _device_index(slots)
    L, pages, nkv, ps, hd = _pools(k_pool, v_pool, 5, dev)
    dt = k_pool.dtype
    shape, ks, vs = k.shape, k.stride(), v.stride()
    if (len(shape) != 4 or v.shape != shape or shape[0] != L or shape[2] != nkv or shape[3] != hd or k.dtype is not dt
            or v.dtype is not dt or (hd > 1 and (ks[3] != 1 or vs[3] != 1)) or k.get_device() != dev
            or v.get_device() != dev):
        raise ValueError("k and v must be [L][M][nkv][hd] in the pools' layers, heads, dtype and device with contiguous "
                         "head rows")
    m = shape[1]
    p_slots = _vec(slots, torch.int64, m, dev, "slots")
    if slots.numel() != m:
        raise ValueError("one slot per row")
    check(_call_on(dev, lib().pe_kv_write_paged, k.data_ptr(), v.data_ptr(), _I64x3(*ks[:3]), _I64x3(*vs[:3]), L, m, nkv,
                   hd, dcode(dt), k_pool.data_ptr(), v_pool.data_ptr(), pages, ps, p_slots,
                   _vec(status, torch.int32, 1, dev, "status")), "pe_kv_write_paged")


def kv_compact_paged(k_pool: torch.Tensor, v_pool: torch.Tensor, block_table: torch.Tensor, seq_len: torch.Tensor,
                     accept_out: torch.Tensor, status: torch.Tensor, *, prefix_len: int = 0) -> None:
    """Every sequence's accepted rows moved together in the pools [L][pages][nkv][page_size][hd], the paths from
    ``accept_out`` int32 [B][2 + max_rows] (pe_kv_compact_paged)."""
    dev = _device_index(accept_out)
    L, pages, nkv, ps, hd = _pools(k_pool, v_pool, 5, dev)
    if (accept_out.dtype is not torch.int32 or accept_out.dim() != 2 or not accept_out.is_contiguous()
            or accept_out.shape[1] < 3 or accept_out.shape[0] < 1):
        raise ValueError("accept_out must be contiguous int32 [B][2 + max_rows]")
    b, width = accept_out.shape
    p_tab, ld, cols = _table(block_table, b, dev)
    check(_call_on(dev, lib().pe_kv_compact_paged, k_pool.data_ptr(), v_pool.data_ptr(), L, nkv, hd,
                   dcode(k_pool.dtype), pages, ps, p_tab, ld, cols, b, _vec(seq_len, torch.int64, b, dev, "seq_len"),
                   prefix_len, accept_out.data_ptr(), width - 2, _vec(status, torch.int32, 1, dev, "status")),
          "pe_kv_compact_paged")


def attention_paged_workspace_bytes(m: int, batch: int, nh: int, nkv: int, hd: int, max_rows: int, max_len: int,
                                    prefix_len: int, dtype: torch.dtype) -> int:
    """Bytes of workspace a ``tree_attention_paged`` call of exactly these sizes needs (no initial value; a smaller
    call may need more, see ``attention_paged_reserve_bytes``)."""
    return int(lib().pe_attention_paged_workspace_bytes(m, batch, nh, nkv, hd, max_rows, max_len, prefix_len,
                                                        dcode(dtype)))


def attention_paged_reserve_bytes(m: int, nh: int, nkv: int, hd: int, dtype: torch.dtype) -> int:
    """Bytes of workspace that hold every ``tree_attention_paged`` call of up to m rows with these heads."""
    return int(lib().pe_attention_paged_reserve_bytes(m, nh, nkv, hd, dcode(dtype)))


# The fields of _lib.PagedAttentionArgs in order: packing them at once takes half the time of its constructor
# (0.8 against 1.6 us a call).
_PAGED_ARGS = struct.Struct("@13Q11q9i2fi")


def tree_attention_paged(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, block_table: torch.Tensor,
                         seq_row0: torch.Tensor, seq_len: torch.Tensor, scale: float, max_rows: int, max_len: int,
                         status: torch.Tensor, *, mask_mode: int = _lib.PE_MASK_TREE,
                         bits: torch.Tensor | None = None, positions: torch.Tensor | None = None,
                         prefix_table: torch.Tensor | None = None, prefix_len: int = 0, softcap: float = 0.0,
                         slopes: torch.Tensor | None = None, window: int = 0, workspace: torch.Tensor | None = None,
                         out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a batch's rows q [M][nh][hd] over a shared prefix and each
    sequence's own pages (pe_tree_attention_paged); returns [M][nh * hd].

    Pools [pages][nkv][page_size][hd] (one layer); ``seq_row0`` int32 [B + 1] and
    ``seq_len`` int64 [B] (cached tokens, the ``prefix_len`` shared ones of
    ``prefix_table`` included) on the device; ``max_rows`` and ``max_len`` bound
    them on the host. ``bits`` int64 [M][words] (tree masks); ``softcap`` caps the
    scores by a tanh, ``slopes`` fp32 [nh] subtracts slope * distance, ``window``
    hides keys that far back: the last two need ``positions`` int64 [M]. Rows of
    no sequence are left as they are in ``out``."""
    dev = _device_index(q)
    shape, dt = q.shape, q.dtype
    if len(shape) != 3 or k_pool.dtype is not dt:
        raise ValueError("q must be [M][nh][hd] in the pools' dtype")
    m, nh, hd = shape
    pages, nkv, ps, phd = _pools(k_pool, v_pool, 4, dev)
    ld_q, s_head, s_dim = q.stride()
    if phd != hd or (hd > 1 and s_dim != 1) or (nh > 1 and s_head != hd) or (m > 1 and ld_q < nh * hd):
        raise ValueError("q rows must hold their heads one after another, as wide as the pools'")
    b = seq_row0.numel() - 1
    if b < 1:
        raise ValueError("seq_row0 must hold batch + 1 offsets")
    p_row0, p_len = _vec(seq_row0, torch.int32, b + 1, dev, "seq_row0"), _vec(seq_len, torch.int64, b, dev, "seq_len")
    p_tab, ld, cols = _table(block_table, b, dev)
    p_status = _vec(status, torch.int32, 1, dev, "status")
    p_bits = p_pos = p_slopes = p_pre = words = n_pre = 0
    if mask_mode == _lib.PE_MASK_TREE:
        if (bits is None or bits.dtype is not torch.int64 or bits.dim() != 2 or bits.shape[0] < m
                or not bits.is_contiguous() or bits.get_device() != dev):
            raise ValueError("tree masks need contiguous int64 bits [M][words] on the device of the call's other tensors")
        p_bits, words = bits.data_ptr(), bits.shape[1]
    if window or slopes is not None:
        if positions is None:
            raise ValueError("a window or slopes need positions")
        p_pos = _vec(positions, torch.int64, m, dev, "positions")
    if slopes is not None:
        p_slopes = _vec(slopes, torch.float32, nh, dev, "slopes")
    if prefix_len:
        if prefix_table is None:
            raise ValueError("a prefix needs its pages")
        p_pre, n_pre = _vec(prefix_table, torch.int32, 1, dev, "prefix_table"), prefix_table.numel()
    if out is None:
        out = torch.empty((m, nh * hd), dtype=dt, device=q.device)
    elif (out.shape != (m, nh * hd) or out.dtype is not dt or out.get_device() != dev
          or (nh * hd > 1 and out.stride(1) != 1) or (m > 1 and out.stride(0) < nh * hd)):
        raise ValueError("out must be [M][nh * hd] in q's dtype and device with contiguous rows")
    if workspace is None:
        need = attention_paged_workspace_bytes(m, b, nh, nkv, hd, max_rows, max_len, prefix_len, dt)
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    p_ws = ws_bytes = 0
    if workspace is not None:
        if not workspace.is_contiguous() or workspace.get_device() != dev:
            raise ValueError("workspace must be contiguous, on the device of the call's other tensors")
        p_ws, ws_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    try:
        packed = _PAGED_ARGS.pack(
            q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), out.data_ptr(), p_tab, p_pre, p_row0, p_len, p_bits, p_pos,
            p_slopes, p_ws, p_status, ws_bytes, ld_q if m > 1 else nh * hd, out.stride(0) if m > 1 else nh * hd, ld, cols,
            pages, n_pre, prefix_len, max_len, window, m, b, max_rows, nh, nkv, hd, ps, dcode(dt), mask_mode, words, scale,
            softcap, 0)
    except (struct.error, OverflowError) as e:
        raise ValueError(f"tree_attention_paged: a count or scale that its field does not hold ({e})") from e
    a = _lib.PagedAttentionArgs.from_buffer_copy(packed)
    check(_call_on(dev, lib().pe_tree_attention_paged, C.byref(a)), "pe_tree_attention_paged")
    return out


def read_status(status: torch.Tensor, where: str) -> None:
    s = int(status[0].item())
    if s:
        status.zero_()
        raise _lib.PEError(s, where)


# ------------------------------------------------------------------ torch custom ops
# A target registered here is named by an integer handle in torch.ops.pe.verify_pass
# (a torch op takes tensors and scalars only; the pass reads the model's weights
# through its pe_model_desc).
_MODELS: dict[int, object] = {}


def register_model(target) -> int:
    """Handle of ``target`` (a TargetModel) for ``torch.ops.pe.verify_pass``; the same
    target gets the same handle."""
    for h, t in _MODELS.items():
        if t is target:
            return h
    h = len(_MODELS) + 1
    _MODELS[h] = target
    return h


def _model(handle: int):
    try:
        return _MODELS[handle]
    except KeyError as e:
        raise ValueError(f"no target registered under handle {handle} (ops.register_model)") from e


def verify_pass(target, input_ids: torch.Tensor, positions: torch.Tensor, tree_bits: torch.Tensor,
                k_cache: torch.Tensor, v_cache: torch.Tensor, prefix_len: int, workspace: torch.Tensor,
                status: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """TargetModel.forward_cached (src/pe/target.py:203-224) as one pe_forward over
    preallocated caches [L][nkv][cap][hd]: rows input_ids at positions, their K/V
    appended at [prefix_len, prefix_len + M), attention over the prefix plus the
    tree rows of tree_bits [M][words] (empty: a causal continuation). Returns
    (logits [M][V], fused [M][F]) in the model dtype; device errors go to status."""
    s = target.shape
    m = input_ids.numel()
    _req(positions.numel() == m and input_ids.dtype == torch.int64 and positions.dtype == torch.int64,
         "input_ids and positions: int64, one position per id")
    _req(k_cache.shape == v_cache.shape and k_cache.dim() == 4 and k_cache.dtype == target.dtype
         and k_cache.is_contiguous() and v_cache.is_contiguous(), "caches [L][nkv][cap][hd] in the model dtype")
    _req(status.dtype == torch.int32 and workspace.dtype == torch.uint8, "status int32, workspace uint8")
    tree = tree_bits.numel() > 0
    logits = torch.empty((m, s.vocab), dtype=target.dtype, device=input_ids.device)
    fused = torch.empty((m, target.feature_dim), dtype=target.dtype, device=input_ids.device)
    a = _lib.PassArgs()
    a.input_ids, a.positions, a.M, a.prefix_len = ptr(input_ids), ptr(positions), m, prefix_len
    a.mask_mode = _lib.PE_MASK_TREE if tree else _lib.PE_MASK_CAUSAL
    a.tree_bits, a.bits_words = (ptr(tree_bits), tree_bits.shape[1]) if tree else (None, 0)
    fl = target.feature_layers
    a.num_features = len(fl)
    for i, f in enumerate(fl[:4]):
        a.feature_layers[i] = f
    a.k_cache, a.v_cache, a.cache_capacity = ptr(k_cache), ptr(v_cache), k_cache.shape[2]
    a.logits, a.fused = ptr(logits), ptr(fused)
    a.workspace, a.workspace_bytes = ptr(workspace), workspace.numel()
    a.status = ptr(status)
    check(lib().pe_forward(C.byref(target.model.desc()), C.byref(a), stream_ptr()), "pe_forward")
    return logits, fused


_REGISTERED = False


def register_torch_ops() -> None:
    """Register the pass and its steps as torch custom ops (``torch.ops.pe.*``),
    each with a fake (meta) implementation for tracing and the cache / scratch /
    status mutations declared in its schema:

    - ``verify_pass(model, input_ids, positions, tree_bits, k_cache!, v_cache!,
      prefix_len, workspace!, status!) -> (logits, fused)``: the masked
      verification forward (src/pe/target.py:203-224), ``model`` from
      ``register_model``;
    - ``tree_masks(parents, prefix_len, words, status!) -> (bits, positions,
      depths)``: src/pe/masks.py:118-156;
    - ``accept_tree(root, node_logits, node_tokens, parents, scratch!) -> out``:
      src/pe/decode/verify.py:104-125, out = [|path|, bonus, path...];
    - ``kv_compact(k_cache!, v_cache!, prefix_len, accept_out)`` and
      ``kv_gather(k_cache!, v_cache!, keep, status!)``: gather_cache
      (src/pe/target.py:194-201);
    - ``page_tables(seq_len, seq_row0, block_table!, held!, free_pages, free_top!,
      page_size, rows, prefix_len, status!) -> slots``, ``kv_write_paged(k, v,
      k_pool!, v_pool!, slots, status!)``, ``kv_compact_paged(k_pool!, v_pool!,
      block_table, seq_len, accept_out, prefix_len, status!)`` and
      ``tree_attention_paged(q, k_pool, v_pool, block_table, seq_row0, seq_len,
      scale, max_rows, max_len, status!, mask_mode, bits?, positions?,
      prefix_table?, prefix_len, softcap, slopes?, window) -> out``: the paged
      cache and the attention that reads it;
    - ``rmsnorm``, ``argmax_rows``, ``nf4_linear``, ``dense_linear``: the pass's
      building blocks.
    """
    global _REGISTERED
    if _REGISTERED:
        return
    lib_def = torch.library.custom_op

    def op(name, schema, mutates=()):
        return lambda fn: lib_def(f"pe::{name}", fn, mutates_args=mutates, schema=schema)

    @op("verify_pass", "(int model, Tensor input_ids, Tensor positions, Tensor tree_bits, Tensor(a!) k_cache, "
        "Tensor(b!) v_cache, int prefix_len, Tensor(c!) workspace, Tensor(d!) status) -> (Tensor, Tensor)",
        ("k_cache", "v_cache", "workspace", "status"))
    def _verify_pass(model, input_ids, positions, tree_bits, k_cache, v_cache, prefix_len, workspace, status):
        return verify_pass(_model(model), input_ids, positions, tree_bits, k_cache, v_cache, prefix_len, workspace,
                           status)

    @_verify_pass.register_fake
    def _(model, input_ids, positions, tree_bits, k_cache, v_cache, prefix_len, workspace, status):
        t = _model(model)
        m = input_ids.numel()
        return (input_ids.new_empty((m, t.shape.vocab), dtype=t.dtype),
                input_ids.new_empty((m, t.feature_dim), dtype=t.dtype))

    @op("tree_masks", "(Tensor parents, int prefix_len, int words, Tensor(a!) status) -> (Tensor, Tensor, Tensor)",
        ("status",))
    def _tree_masks(parents, prefix_len, words, status):
        return tree_masks(parents, prefix_len, words, status)

    @_tree_masks.register_fake
    def _(parents, prefix_len, words, status):
        t = parents.numel()
        return (parents.new_empty((t, words), dtype=torch.int64), parents.new_empty(t, dtype=torch.int64),
                parents.new_empty(t, dtype=torch.int32))

    @op("accept_tree", "(Tensor root, Tensor node_logits, Tensor node_tokens, Tensor parents, Tensor(a!) scratch) "
        "-> Tensor", ("scratch",))
    def _accept(root, node_logits, node_tokens, parents, scratch):
        return accept_tree(root, node_logits, node_tokens, parents, scratch=scratch)

    @_accept.register_fake
    def _(root, node_logits, node_tokens, parents, scratch):
        return root.new_empty(2 + max(node_tokens.numel(), 1), dtype=torch.int32)

    @op("kv_compact", "(Tensor(a!) k_cache, Tensor(b!) v_cache, int prefix_len, Tensor accept_out) -> ()",
        ("k_cache", "v_cache"))
    def _kv_compact(k_cache, v_cache, prefix_len, accept_out):
        kv_compact(k_cache, v_cache, prefix_len, accept_out)

    @_kv_compact.register_fake
    def _(k_cache, v_cache, prefix_len, accept_out):
        return None

    @op("kv_gather", "(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor keep, Tensor(c!) status) -> ()",
        ("k_cache", "v_cache", "status"))
    def _kv_gather(k_cache, v_cache, keep, status):
        kv_gather(k_cache, v_cache, keep, status)

    @_kv_gather.register_fake
    def _(k_cache, v_cache, keep, status):
        return None

    @op("page_tables", "(Tensor seq_len, Tensor seq_row0, Tensor(a!) block_table, Tensor(b!) held, Tensor free_pages, "
        "Tensor(c!) free_top, int page_size, int rows, int prefix_len, Tensor(d!) status) -> Tensor",
        ("block_table", "held", "free_top", "status"))
    def _page_tables(seq_len, seq_row0, block_table, held, free_pages, free_top, page_size, rows, prefix_len, status):
        return page_tables(seq_len, seq_row0, block_table, held, free_pages, free_top, page_size, rows, status,
                           prefix_len=prefix_len)

    @_page_tables.register_fake
    def _(seq_len, seq_row0, block_table, held, free_pages, free_top, page_size, rows, prefix_len, status):
        return seq_len.new_empty(rows)

    @op("kv_write_paged", "(Tensor k, Tensor v, Tensor(a!) k_pool, Tensor(b!) v_pool, Tensor slots, Tensor(c!) status) "
        "-> ()", ("k_pool", "v_pool", "status"))
    def _kv_write_paged(k, v, k_pool, v_pool, slots, status):
        kv_write_paged(k, v, k_pool, v_pool, slots, status)

    @_kv_write_paged.register_fake
    def _(k, v, k_pool, v_pool, slots, status):
        return None

    @op("kv_compact_paged", "(Tensor(a!) k_pool, Tensor(b!) v_pool, Tensor block_table, Tensor seq_len, "
        "Tensor accept_out, int prefix_len, Tensor(c!) status) -> ()", ("k_pool", "v_pool", "status"))
    def _kv_compact_paged(k_pool, v_pool, block_table, seq_len, accept_out, prefix_len, status):
        kv_compact_paged(k_pool, v_pool, block_table, seq_len, accept_out, status, prefix_len=prefix_len)

    @_kv_compact_paged.register_fake
    def _(k_pool, v_pool, block_table, seq_len, accept_out, prefix_len, status):
        return None

    @op("tree_attention_paged", "(Tensor q, Tensor k_pool, Tensor v_pool, Tensor block_table, Tensor seq_row0, "
        "Tensor seq_len, float scale, int max_rows, int max_len, Tensor(a!) status, int mask_mode, Tensor? bits, "
        "Tensor? positions, Tensor? prefix_table, int prefix_len, float softcap, Tensor? slopes, int window) -> Tensor",
        ("status",))
    def _tree_attention_paged(q, k_pool, v_pool, block_table, seq_row0, seq_len, scale, max_rows, max_len, status,
                              mask_mode, bits, positions, prefix_table, prefix_len, softcap, slopes, window):
        return tree_attention_paged(q, k_pool, v_pool, block_table, seq_row0, seq_len, scale, max_rows, max_len, status,
                                    mask_mode=mask_mode, bits=bits, positions=positions, prefix_table=prefix_table,
                                    prefix_len=prefix_len, softcap=softcap, slopes=slopes, window=window)

    @_tree_attention_paged.register_fake
    def _(q, k_pool, v_pool, block_table, seq_row0, seq_len, scale, max_rows, max_len, status, mask_mode, bits, positions,
          prefix_table, prefix_len, softcap, slopes, window):
        return q.new_empty((q.shape[0], q.shape[1] * q.shape[2]))

    @op("rmsnorm", "(Tensor x, Tensor w, float eps) -> Tensor")
    def _rmsnorm(x, w, eps):
        return rmsnorm(x, w, eps)

    @_rmsnorm.register_fake
    def _(x, w, eps):
        return torch.empty_like(x)

    @op("argmax_rows", "(Tensor x) -> Tensor")
    def _argmax(x):
        return argmax_rows(x)

    @_argmax.register_fake
    def _(x):
        return x.new_empty(x.shape[0], dtype=torch.int32)

    @op("nf4_linear", "(Tensor x, Tensor tiled, Tensor tabs, int n) -> Tensor")
    def _nf4_linear(x, tiled, tabs, n):
        return linear(x, n, nf4=(tiled, tabs))

    @_nf4_linear.register_fake
    def _(x, tiled, tabs, n):
        return x.new_empty((x.shape[0], n))

    @op("dense_linear", "(Tensor x, Tensor w, int n) -> Tensor")
    def _dense_linear(x, w, n):
        return linear(x, n, dense=w)

    @_dense_linear.register_fake
    def _(x, w, n):
        return x.new_empty((x.shape[0], n))

    _REGISTERED = True
