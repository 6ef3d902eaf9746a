// What the paged attention's kernels share (not part of the C ABI).
#pragma once

#include "pe_common.h"
#include "pe_internal.h"

// A call's arguments as the kernels take them (by value).
struct PagedAttn {
  const void* q;  // [M][nh][hd], rows ld_q elements apart
  const void* k_pool;  // [num_pages][nkv][1 << ps_log2][hd]
  const void* v_pool;
  void* out;  // [M][nh * hd], rows ld_out elements apart
  const int32_t* block_table;  // [batch][cols], rows ld_table apart
  const int32_t* prefix_table;
  const int32_t* seq_row0;
  const int64_t* seq_len;
  const uint64_t* bits;  // [M][words], tree masks only
  const int64_t* positions;  // [M], only where distances count
  const float* slopes;  // [nh] or null
  int32_t* status;
  int64_t ld_q, ld_out, ld_table, cols, num_pages, prefix_len, max_len, window, M;
  int batch, max_rows, nh, nkv, hd, ps_log2, mask_mode, words;
  float scale, softcap;
  int out_units;  // > 0: out is A-tiled over all rows (nh * hd = 128 * out_units; matrix-core kernels only)
};

// the running maximum of a row that has seen nothing (its sum is 0)
constexpr float kPagedInitMax = -2.0e38f;

// Sequence b's rows and private length. A sequence whose row range, length or
// row count is outside what the call was sized for, or whose tokens do not fit
// its table, is skipped by every workgroup alike (ok false, err the status bit;
// err 0 for a sequence without rows).
struct PagedSeq {
  int row0, rows;
  int64_t priv;
  bool ok;
  int err;
};

__device__ __forceinline__ PagedSeq paged_seq(const PagedAttn& a, int b) {
  PagedSeq s;
  s.row0 = a.seq_row0[b];
  const int r1 = a.seq_row0[b + 1];
  s.rows = r1 - s.row0;
  s.priv = a.seq_len[b] - a.prefix_len;
  s.err = 0;
  if (s.row0 < 0 || s.rows < 0 || r1 > a.M || s.rows > a.max_rows)
    s.err = PE_ERR_TREE;
  else if (s.priv < 0 || s.priv > a.max_len - a.prefix_len || s.priv + s.rows > (a.cols << a.ps_log2))
    s.err = PE_ERR_CAPACITY;
  s.ok = s.err == 0 && s.rows > 0;
  return s;
}

// Four consecutive columns of a token's output row.
template <int DT>
__device__ __forceinline__ void paged_out4(const PagedAttn& a, int64_t tok, int col, const float (&v)[4]) {
  typedef typename Elem<DT>::T Te;
  Vec4<DT>::store((Te*)a.out + (a.out_units ? xtile_index((int)tok, col, a.out_units) : tok * a.ld_out + col), v);
}

// pe_paged.hip: the call on the VALU (fp32, any head size up to 256).
PE_INTERNAL int pe_internal_paged_valu(const PagedAttn& a, int dtype, hipStream_t st);

// Partial results (O, running maximum in base 2, sum) of one KV head's rows,
// kept in the order in which the matrix cores leave them: of every 32-row tile
// the hd / 8 pieces [64 lanes][4 floats] (piece 4 h + c of lane ln + 32 g: dims
// 32 h + 8 c + 4 g .. + 3 of row ln), so that writing and reading a tile are
// whole KiB. Row r of a KV head is (token r / G, query head r % G), tokens
// counted over the whole batch. Part p of KV head kvh: tiles from
// (p * nkv + kvh) * tiles on.
struct PagedParts {
  float* o;
  float* ml;  // [parts][nkv][tiles * 32][2]
  int64_t tiles;
  int pre_parts;  // parts of the prefix come first, then the private splits'
};

// The prefix's work: nkv * nblk row blocks of `block_rows` rows, each `steps`
// key steps; workgroup w takes the units [w * per, (w + 1) * per) of that
// sequence, so all workgroups do the same amount and a block is covered by a
// few of them, its parts.
struct PagedPrefix {
  uint32_t total, per, steps, nblk, block_rows;
};

__device__ __forceinline__ uint32_t prefix_first_wg(const PagedPrefix& p, uint32_t block) { return block * p.steps / p.per; }
__device__ __forceinline__ int prefix_parts_of(const PagedPrefix& p, uint32_t block) {
  return (int)((block * p.steps + p.steps - 1) / p.per - prefix_first_wg(p, block)) + 1;
}

// pe_paged_attn.hip: the call on the matrix cores (bf16 / fp16, hd 64 or 128).
PE_INTERNAL int64_t pe_internal_paged_mfma_bytes(int64_t M, int batch, int nh, int nkv, int hd, int max_rows,
                                                 int64_t max_len, int64_t prefix_len);
PE_INTERNAL int64_t pe_internal_paged_mfma_reserve(int64_t M, int nh, int nkv, int hd);
PE_INTERNAL int pe_internal_paged_mfma(const PagedAttn& a, int dtype, void* workspace, int64_t workspace_bytes,
                                       hipStream_t st);
