// The paged KV cache of a batch of sequences: pages given out and block tables
// and slot maps built from the sequences' lengths, pages returned, K/V rows
// written to their slots, accepted rows moved together, and the attention for
// the types and head sizes that the matrix cores' kernels do not take.
//
// A pool holds pages of `ps` tokens (a power of two, 16 .. 1024), one layer as
// [num_pages][nkv][ps][hd], so that one KV head's rows of a page are one
// contiguous run. A sequence's tokens are a prefix of `prefix_len` tokens that
// the whole batch shares (its own list of pages) and the sequence's private
// tokens: token prefix_len + j lies at row j % ps of page block_table[b][j / ps].
// seq_len[b] counts the cached tokens, the shared ones included.
//
// Every id that comes from device memory (page, slot, row range, path node) is
// checked before it becomes an address; what fails sets a bit of the status
// word and is skipped.

#include "pe_common.h"
#include "pe_internal.h"
#include "pe_paged.h"

namespace {

// ---------------------------------------------------------------------------
// Pages and slots
// ---------------------------------------------------------------------------
// What sequence b needs: rows, its private length, pages held and pages to add
// (0 with an error bit for a sequence that cannot be served).
struct SeqNeed {
  int row0, rows, held, need, err;
  int64_t priv;
};

__device__ __forceinline__ SeqNeed seq_need(const int64_t* seq_len, const int32_t* seq_row0, const int32_t* held,
                                            int b, int64_t M, int64_t prefix_len, int ps_log2, int64_t cols) {
  SeqNeed s;
  s.row0 = seq_row0[b];
  const int r1 = seq_row0[b + 1];
  s.rows = r1 - s.row0;
  s.priv = seq_len[b] - prefix_len;
  s.held = held[b];
  s.need = 0;
  s.err = 0;
  if (s.row0 < 0 || s.rows < 0 || r1 > M) s.err = PE_ERR_TREE;
  else if (s.held < 0 || s.held > cols) s.err = PE_ERR_INDEX;
  else if (s.priv < 0 || s.priv > (cols << ps_log2) || s.priv + s.rows > (cols << ps_log2)) s.err = PE_ERR_CAPACITY;
  if (s.err == 0 && s.rows > 0) {
    const int64_t full = (s.priv + s.rows + (int64_t(1) << ps_log2) - 1) >> ps_log2;
    s.need = full > s.held ? (int)(full - s.held) : 0;
  }
  return s;
}

// Sum over the block of a value per thread, in every thread.
template <int THREADS>
__device__ __forceinline__ int64_t block_sum(int64_t v, int64_t* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += (int64_t)shfl_xor_u64((uint64_t)v, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  int64_t t = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) t += red[w];
  __syncthreads();
  return t;
}

// Block (x, b) serves sequence b: the pages it adds are the `need` ones below
// free_pages[top - off_b], off_b the pages the sequences before it add, so
// every block finds its own from the lengths alone (B loads and one sum) and
// no block waits for another. A sequence whose pages are not all there gets
// none (then no later one that needs any does either, off_b only grows).
// held_out and top_out must not be the inputs here: tables_commit_kernel
// writes them afterwards when they are. Block x of a sequence writes the slots
// of every gridDim.x-th run of 256 rows and x == 0 its table entries; the last
// column of blocks (b == batch) marks the rows behind the last sequence.
// Bound by the launch and a chain of three dependent loads (lengths, free
// page, slot store): 3.2 us for eight trees of 26 rows, 4.4 for 256 prompts of
// 1000 rows on average (2 MB of slots and 66 KB of table entries, 0.4 us at the
// rate of a copy), the second launch of an update in place included.
constexpr int kTabThreads = 256;

__global__ __launch_bounds__(kTabThreads) void page_tables_kernel(
    const int64_t* __restrict__ seq_len, const int32_t* __restrict__ seq_row0, int batch, int64_t M,
    int64_t prefix_len, int ps_log2, int32_t* __restrict__ table, int64_t ld_table, int64_t cols,
    const int32_t* __restrict__ held, const int32_t* __restrict__ free_pages, const int32_t* __restrict__ free_top,
    int64_t n_free, int32_t* __restrict__ held_out, int32_t* __restrict__ top_out, int64_t* __restrict__ slots,
    int32_t* status) {
  __shared__ int64_t red[kTabThreads / 64];
  const int b = blockIdx.y;
  if (b == batch) {  // rows behind the last sequence (and none before the first)
    const int64_t end = min(max((int64_t)seq_row0[batch], (int64_t)0), M);
    for (int64_t r = end + blockIdx.x * kTabThreads + threadIdx.x; r < M; r += (int64_t)gridDim.x * kTabThreads)
      slots[r] = -1;
    if (blockIdx.x == 0 && threadIdx.x == 0 && seq_row0[0] != 0) atomicOr(status, PE_ERR_TREE);
    return;
  }
  const int64_t top = min(max((int64_t)free_top[0], (int64_t)0), n_free);
  int64_t part = 0;
  for (int c = threadIdx.x; c < b; c += kTabThreads)
    part += seq_need(seq_len, seq_row0, held, c, M, prefix_len, ps_log2, cols).need;
  const SeqNeed s = seq_need(seq_len, seq_row0, held, b, M, prefix_len, ps_log2, cols);
  const int64_t off = block_sum<kTabThreads>(part, red);
  const bool given = off + s.need <= top;
  if (s.err == PE_ERR_TREE) {  // its row range is not one: nothing of it can be written
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      atomicOr(status, s.err);
      held_out[b] = s.held;
    }
  } else {
    const int64_t last = given ? s.held + s.need : s.held;  // pages the sequence has
    if (blockIdx.x == 0) {
      for (int i = threadIdx.x; given && i < s.need; i += kTabThreads)
        table[b * ld_table + s.held + i] = free_pages[top - 1 - off - i];
      if (threadIdx.x == 0) {
        held_out[b] = s.err ? s.held : (int)last;
        if (s.err || !given) atomicOr(status, s.err ? s.err : PE_ERR_CAPACITY);
      }
    }
    for (int i = blockIdx.x * kTabThreads + threadIdx.x; i < s.rows; i += gridDim.x * kTabThreads) {
      const int64_t j = s.priv + i, pi = j >> ps_log2;
      int64_t slot = -1;
      if (s.err == 0 && pi < last) {
        const int page = pi < s.held ? table[b * ld_table + pi] : free_pages[top - 1 - off - (pi - s.held)];
        if (page >= 0)
          slot = ((int64_t)page << ps_log2) + (j & ((1 << ps_log2) - 1));
        else
          atomicOr(status, PE_ERR_INDEX);
      }
      slots[s.row0 + i] = slot;
    }
  }
  if (b == batch - 1 && blockIdx.x == 0) {
    // pages taken: the needs in order as long as the pool holds them
    int64_t all = off + s.need, took = all;
    if (all > top) {
      // the last sum that fits (off + need of the sequences before the first that does not)
      __shared__ unsigned long long best;
      if (threadIdx.x == 0) best = 0;
      __syncthreads();
      for (int64_t c0 = 0, run = 0; c0 < batch; c0 += kTabThreads) {
        const int c = (int)c0 + threadIdx.x;
        const int64_t n = c < batch ? seq_need(seq_len, seq_row0, held, c, M, prefix_len, ps_log2, cols).need : 0;
        int64_t incl = n;  // inclusive sum of the block's needs
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const int64_t up = (int64_t)(((uint64_t)__shfl_up((uint32_t)(incl >> 32), o, 64) << 32) |
                                       (uint64_t)__shfl_up((uint32_t)incl, o, 64));
          if ((int)(threadIdx.x & 63) >= o) incl += up;
        }
        if ((threadIdx.x & 63) == 63) red[threadIdx.x >> 6] = incl;
        __syncthreads();
        int64_t before = run, total = run;
        for (int w = 0; w < kTabThreads / 64; ++w) {
          if (w < (int)(threadIdx.x >> 6)) before += red[w];
          total += red[w];
        }
        if (n > 0 && before + incl <= top) atomicMax(&best, (unsigned long long)(before + incl));
        run = total;
        __syncthreads();
      }
      took = (int64_t)best;
    }
    if (threadIdx.x == 0) top_out[0] = (int32_t)(top - took);
  }
}

// held and free_top in place: written after every block of page_tables_kernel
// has read them (it wrote the new values to the scratch words given).
__global__ __launch_bounds__(kTabThreads) void tables_commit_kernel(const int32_t* __restrict__ src, int32_t* held,
                                                                    int batch, int32_t* top) {
  const int i = blockIdx.x * kTabThreads + threadIdx.x;
  if (held && i < batch) held[i] = src[i];
  if (top && i == 0) top[0] = src[batch];
}

// Pages of the listed sequences back onto the free list, in the order listed
// (each sequence's last page first, so that giving them out again restores the
// order). One block; a sequence that is out of range, listed before or whose
// count of pages is not one is flagged and skipped, and nothing is returned
// past the end of the list.
__global__ __launch_bounds__(kTabThreads) void page_release_kernel(const int32_t* __restrict__ seqs, int n, int batch,
                                                                   int32_t* __restrict__ table, int64_t ld_table,
                                                                   int64_t cols, int32_t* __restrict__ held,
                                                                   int32_t* __restrict__ free_pages,
                                                                   int32_t* __restrict__ free_top, int64_t n_free,
                                                                   int32_t* status) {
  __shared__ int dup;
  int64_t top = min(max((int64_t)free_top[0], (int64_t)0), n_free);
  for (int i = 0; i < n; ++i) {
    const int s = seqs[i];
    if (threadIdx.x == 0) dup = 0;
    __syncthreads();
    int mine = 0;
    for (int j = threadIdx.x; j < i; j += kTabThreads) mine |= seqs[j] == s;
    if (mine) dup = 1;
    __syncthreads();
    const bool bad = dup || s < 0 || s >= batch;
    const int cnt = bad ? 0 : held[s];
    const bool off = bad || cnt < 0 || cnt > cols || top + cnt > n_free;
    __syncthreads();  // dup and held[s] are read
    if (off) {
      if (threadIdx.x == 0) atomicOr(status, PE_ERR_INDEX);
      continue;
    }
    for (int k = threadIdx.x; k < cnt; k += kTabThreads) {
      free_pages[top + k] = table[s * ld_table + cnt - 1 - k];
      table[s * ld_table + cnt - 1 - k] = -1;
    }
    if (threadIdx.x == 0) held[s] = 0;
    top += cnt;
  }
  if (threadIdx.x == 0) free_top[0] = (int32_t)top;
}

// ---------------------------------------------------------------------------
// Rows into pages
// ---------------------------------------------------------------------------
// A copy of rows x nkv pieces of one head's row each (K and V, every layer):
// the piece of V-byte vectors, `vpr` of them, moved by `vpr` neighbouring
// lanes, one vector a thread. Pieces run over the rows of one head first: those
// are neighbours both in a page and in a contiguous cache, so a wave's stores
// fill whole KiB of a page. A row's slot and its values are asked for together.
// Bound by HBM: 2000 rows of 32 heads of 256 bytes in 8 layers, 524 MB read and
// written, 91 us (5.8 TB/s; a large copy reaches 4.97); four vectors a thread: 95.
// 208 rows of 8 heads in one layer take 2.5 us, a launch and one load's latency.
template <typename V>
__global__ __launch_bounds__(256) void kv_write_kernel(
    const uint8_t* __restrict__ ks, const uint8_t* __restrict__ vs, int64_t sl_k, int64_t sr_k, int64_t sh_k,
    int64_t sl_v, int64_t sr_v, int64_t sh_v, uint8_t* __restrict__ kp, uint8_t* __restrict__ vp, int64_t layer_bytes,
    const int64_t* __restrict__ slots, int M, int nkv, int vpr, int ps_log2, int64_t num_slots, int32_t* status) {
  const int layer = blockIdx.y;
  const bool is_v = blockIdx.z != 0;
  const uint8_t* src = (is_v ? vs : ks) + layer * (is_v ? sl_v : sl_k);
  const int64_t sr = is_v ? sr_v : sr_k, sh = is_v ? sh_v : sh_k;
  uint8_t* dst = (is_v ? vp : kp) + layer * layer_bytes;
  const uint32_t total = (uint32_t)M * (uint32_t)nkv * (uint32_t)vpr;  // vectors (below 2^31)
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  const uint32_t piece = i / (uint32_t)vpr, col = i - piece * vpr;
  const uint32_t head = piece / (uint32_t)M, r = piece - head * M;
  const int64_t slot = slots[r];
  const V v = *(const V*)(src + r * sr + head * sh + col * sizeof(V));
  if (slot >= 0 && slot < num_slots) {
    const int64_t page = slot >> ps_log2, at = slot & ((1 << ps_log2) - 1);
    *(V*)(dst + ((((page * nkv + head) << ps_log2) + at) * vpr + col) * (int64_t)sizeof(V)) = v;
  } else if (slot != -1 && !is_v && layer == 0 && head == 0 && col == 0) {
    atomicOr(status, PE_ERR_INDEX);
  }
}

// Element offset of each row's slot in head 0 of a layer's pool, -1 for a row
// without one: what the q/k/v epilogues of a pass take (head h adds h *
// page_size * hd there).
__global__ __launch_bounds__(256) void slot_offsets_kernel(const int64_t* __restrict__ slots, int M, int nkv, int hd,
                                                           int ps_log2, int64_t num_slots, int64_t* __restrict__ off,
                                                           int32_t* status) {
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r >= M) return;
  const int64_t s = slots[r];
  const bool ok = s >= 0 && s < num_slots;
  if (!ok && s != -1 && status) atomicOr(status, PE_ERR_INDEX);
  off[r] = ok ? ((((s >> ps_log2) * nkv) << ps_log2) + (s & ((1 << ps_log2) - 1))) * hd : -1;
}

// ---------------------------------------------------------------------------
// Accepted rows together
// ---------------------------------------------------------------------------
// Sequence b's private rows p + path[i] move to p + i, i < len, in every layer
// and KV head of K and V. path[i] >= i, so rows read before a later one is written
// hold what they held before the call: a wave (a workgroup of its own) moves one
// run of rows (four of 256 bytes) of kCompactHeads (layer, head) pairs at a time,
// all loads before the first store. Where the rows lie is worked out by a lane per
// row, once for all those pairs, which leaves one chain of length and path, table
// entries, rows. 32 trees of 40 to 64 nodes, 8 layers of 32 heads (33 MB, partly
// still in the caches): 6.1 us, 6.2 with 4 pairs to a wave, 6.8 with 16; eight
// trees of 26 nodes, 48 layers of 8 heads: 3.8. With one pair to a wave each
// worked the 64-bit places out again, 18 us.
constexpr int kCompactHeads = 8;

template <typename V>
__global__ __launch_bounds__(64) void kv_compact_paged_kernel(
    uint8_t* __restrict__ kp, uint8_t* __restrict__ vp, int64_t layer_bytes, int LH, int nkv, int vpr, int ps_log2,
    const int32_t* __restrict__ table, int64_t ld_table, int64_t cols, int64_t num_pages,
    const int64_t* __restrict__ seq_len, int64_t prefix_len, const int32_t* __restrict__ acc, int64_t ld_acc,
    int max_rows, int32_t* status) {
  const int b = blockIdx.z, lane = threadIdx.x;
  const int32_t* res = acc + b * ld_acc;
  int node = res[2 + min(lane, max_rows - 1)];  // asked for beside the length
  const int len = res[0];
  const int64_t p = seq_len[b] - prefix_len;
  const bool first = blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0;
  if (len <= 0) {
    if (first && len < 0) atomicOr(status, PE_ERR_INDEX);
    return;
  }
  if (len > max_rows || p < 0 || p >= (cols << ps_log2)) {
    if (first) atomicOr(status, len > max_rows ? PE_ERR_INDEX : PE_ERR_CAPACITY);
    return;
  }
  const int lh0 = blockIdx.x * kCompactHeads;
  uint8_t* pool = blockIdx.y == 0 ? kp : vp;
  const int32_t* tab = table + b * ld_table;
  const int64_t row_bytes = vpr * (int64_t)sizeof(V), head_bytes = row_bytes << ps_log2;
  int64_t head_at[kCompactHeads];  // of the wave's pairs (the last one again past the end)
  {
    int layer = lh0 / nkv, h = lh0 - layer * nkv;
#pragma unroll
    for (int k = 0; k < kCompactHeads; ++k) {
      head_at[k] = layer * layer_bytes + h * head_bytes;
      const bool more = lh0 + k + 1 < LH, wrap = h + 1 == nkv;
      layer += more && wrap ? 1 : 0;
      h = more ? (wrap ? 0 : h + 1) : h;
    }
  }
  // byte offset of private row j in KV head 0 of layer 0, -1 where no such row exists
  auto row_at = [&](int64_t j) -> int64_t {
    if (j >= (cols << ps_log2)) return -1;
    const int page = tab[j >> ps_log2];
    if (page < 0 || page >= num_pages) return -1;
    return (int64_t)page * nkv * head_bytes + (j & ((1 << ps_log2) - 1)) * row_bytes;
  };
  const int lanes = min(64, vpr);  // lanes on one row
  const int per = 64 / lanes;      // rows a load instruction moves
  const int sub = lane / lanes, c0 = lane - sub * lanes;
  bool bad = false;
  for (int i0 = 0; i0 < len; i0 += 64) {
    const int i = i0 + lane;  // this lane's row
    if (i0 > 0) node = res[2 + min(i, max_rows - 1)];
    int64_t from = -1, dst = -1;
    if (i < len) {
      if (node < i || node >= max_rows) {
        bad = true;
      } else if (node != i) {
        from = row_at(p + node);
        dst = row_at(p + i);
        if (from < 0 || dst < 0) {
          bad = true;
          dst = -1;
        }
      }
    }
    const int n = min(64, len - i0);
    for (int r0 = 0; r0 < n; r0 += per) {
      const int at = r0 + sub;
      const int64_t rf = __shfl(from, at & 63, 64), rd = __shfl(dst, at & 63, 64);
      if (sub >= per || at >= n || rd < 0) continue;
      for (int c = c0; c < vpr; c += lanes) {
        V v[kCompactHeads];
#pragma unroll
        for (int k = 0; k < kCompactHeads; ++k)  // (past the last pair: its row again)
          v[k] = *(const V*)(pool + head_at[k] + rf + c * (int64_t)sizeof(V));
#pragma unroll
        for (int k = 0; k < kCompactHeads; ++k)
          *(V*)(pool + head_at[k] + rd + c * (int64_t)sizeof(V)) = v[k];
      }
    }
  }
  if (bad && lh0 == 0 && blockIdx.y == 0) atomicOr(status, PE_ERR_INDEX);
}

// ---------------------------------------------------------------------------
// Attention on the VALU
// ---------------------------------------------------------------------------
// fp32, and the head sizes and alignments that the matrix-core kernels do not
// take: one block per (row, query head), LPK lanes (four dims each) on one key,
// 256 / LPK keys in step. Each key slot keeps its own running maximum, sum and
// weighted V (one pass, any length); the slots are joined in LDS in slot order.
// Scores, weights and sums are fp32 throughout. Bound by the latency of a slot's
// loads (kValuKeys keys in flight): 5.4 us for two fp32 trees of up to 8 nodes
// over up to 104 keys, 4 heads of 64; eight of 26 nodes over up to 1900: 96.
constexpr int kValuKeys = 4;

template <int DT, int LPK, bool VEC>
__global__ __launch_bounds__(256) void attn_paged_valu_kernel(PagedAttn a) {
  typedef Elem<DT> E;
  typedef typename E::T Te;
  constexpr int kSlots = 256 / LPK;
  const int hq = blockIdx.x, b = blockIdx.z;
  const PagedSeq s = paged_seq(a, b);
  if (!s.ok) {
    if (threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0 && s.err) atomicOr(a.status, s.err);
    return;
  }
  const int t = blockIdx.y;
  if (t >= s.rows) return;
  const int64_t m = s.row0 + t;
  const int nkv = a.nkv, hd = a.hd, kvh = hq / (a.nh / nkv), psl = a.ps_log2;
  const int sl = threadIdx.x / LPK, li = threadIdx.x % LPK, d0 = 4 * li;
  const int64_t cached = a.prefix_len + s.priv;
  const int64_t pos = a.positions ? a.positions[m] : cached + t;
  const float slope = a.slopes ? a.slopes[hq] : 0.f;
  const bool tree = a.mask_mode == PE_MASK_TREE;
  uint64_t nb[PE_TREE_MAX_WORDS];
#pragma unroll
  for (int w = 0; w < PE_TREE_MAX_WORDS; ++w) nb[w] = tree && w < a.words ? a.bits[m * a.words + w] : 0ull;
  auto load4 = [&](const Te* p, float (&v)[4]) {
    if constexpr (VEC) {
      if (d0 < hd) {
        Vec4<DT>::load(p + d0, v);
        return;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = 0.f;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = d0 + i < hd ? E::load(p, d0 + i) : 0.f;
    }
  };
  float qv[4];
  load4((const Te*)a.q + m * a.ld_q + (int64_t)hq * hd, qv);
  // keys [lo, cached) of the cache, then the row's own sequence's new rows
  const int64_t lo = a.window > 0 ? min(max(pos - a.window + 1, (int64_t)0), cached) : 0;
  const int64_t end = cached + (tree ? s.rows : t + 1);
  float mx = kPagedInitMax, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  bool bad = false;
  for (int64_t j0 = lo; j0 < end; j0 += kSlots * kValuKeys) {
    float kv[kValuKeys][4], vv[kValuKeys][4], sc[kValuKeys];
    bool see[kValuKeys];
#pragma unroll
    for (int k = 0; k < kValuKeys; ++k) {
      const int64_t j = j0 + k * kSlots + sl;
      see[k] = j < end;
      int64_t dist = pos - j;
      if (see[k] && j >= cached) {
        const int u = (int)(j - cached);
        if (tree) {
          const uint64_t w = u < 64 ? nb[0] : u < 128 ? nb[1] : u < 192 ? nb[2] : nb[3];
          see[k] = (w >> (u & 63)) & 1ull;
          if (a.positions) dist = pos - a.positions[s.row0 + u];
        }
        if (a.window > 0) see[k] = see[k] && dist < a.window;
      }
      // loads of a key that is not seen go to one that is there, so that none waits behind a branch
      const int64_t jj = min(j, end - 1);
      const bool pre = jj < a.prefix_len;
      const int64_t i = pre ? jj : jj - a.prefix_len;
      const int page = (pre ? a.prefix_table : a.block_table + b * a.ld_table)[i >> psl];
      const bool ok = page >= 0 && page < a.num_pages;
      bad = bad || (see[k] && !ok);
      see[k] = see[k] && ok;
      const int64_t at = see[k] ? ((((int64_t)page * nkv + kvh) << psl) + (i & ((1 << psl) - 1))) * hd : 0;
      sc[k] = slope * (float)dist;
      load4((const Te*)a.k_pool + at, kv[k]);
      load4((const Te*)a.v_pool + at, vv[k]);
    }
#pragma unroll
    for (int k = 0; k < kValuKeys; ++k) {
      float d = see[k] ? fmaf(qv[3], kv[k][3], fmaf(qv[2], kv[k][2], fmaf(qv[1], kv[k][1], qv[0] * kv[k][0]))) : 0.f;
#pragma unroll
      for (int o = LPK / 2; o > 0; o >>= 1) d += __shfl_xor(d, o, 64);
      if (!see[k]) continue;  // the same for every lane of the slot
      d *= a.scale;
      if (a.softcap > 0.f) d = a.softcap * tanhf(d / a.softcap);
      d -= sc[k];
      const float mn = fmaxf(mx, d);
      const float al = expf(mx - mn), p = expf(d - mn);
      mx = mn;
      l = fmaf(l, al, p);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = fmaf(acc[i], al, p * vv[k][i]);
    }
  }
  if (bad) atomicOr(a.status, PE_ERR_INDEX);
  __shared__ float s_o[kSlots][4 * LPK];
  __shared__ float s_m[kSlots], s_l[kSlots];
#pragma unroll
  for (int i = 0; i < 4; ++i) s_o[sl][d0 + i] = acc[i];
  if (li == 0) {
    s_m[sl] = mx;
    s_l[sl] = l;
  }
  __syncthreads();
  float top = kPagedInitMax;
#pragma unroll
  for (int w = 0; w < kSlots; ++w) top = fmaxf(top, s_m[w]);
  float den = 0.f;
#pragma unroll
  for (int w = 0; w < kSlots; ++w) den = fmaf(s_l[w], expf(s_m[w] - top), den);
  for (int d = threadIdx.x; d < hd; d += 256) {
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < kSlots; ++w) o = fmaf(s_o[w][d], expf(s_m[w] - top), o);
    E::store((Te*)a.out, m * a.ld_out + (int64_t)hq * hd + d, den == 0.f ? 0.f : o / den);
  }
}

int esize(int dtype) { return dtype == PE_DTYPE_F32 ? 4 : dtype == PE_DTYPE_BF16 || dtype == PE_DTYPE_F16 ? 2 : 0; }

// log2 of a page size (a power of two, 16 .. 1024), -1 for any other
int page_log2(int ps) {
  for (int k = 4; k <= 10; ++k)
    if (ps == (1 << k)) return k;
  return -1;
}

template <int DT>
void launch_valu(const PagedAttn& a, bool vec, hipStream_t st) {
  const dim3 grid(a.nh, a.max_rows, a.batch);
#define PE_VALU(LPK)                                                          \
  do {                                                                        \
    if (vec)                                                                  \
      attn_paged_valu_kernel<DT, LPK, true><<<grid, 256, 0, st>>>(a);         \
    else                                                                      \
      attn_paged_valu_kernel<DT, LPK, false><<<grid, 256, 0, st>>>(a);        \
  } while (0)
  if (a.hd <= 64) PE_VALU(16);
  else if (a.hd <= 128) PE_VALU(32);
  else PE_VALU(64);
#undef PE_VALU
}

}  // namespace

int pe_internal_paged_valu(const PagedAttn& a, int dtype, hipStream_t st) {
  const int es = esize(dtype);
  const bool vec = a.hd % 4 == 0 && a.ld_q % 4 == 0 && (((uintptr_t)a.q | (uintptr_t)a.k_pool | (uintptr_t)a.v_pool) & (4 * es - 1)) == 0;
  switch (dtype) {
    case PE_DTYPE_F32: launch_valu<PE_DTYPE_F32>(a, vec, st); break;
    case PE_DTYPE_BF16: launch_valu<PE_DTYPE_BF16>(a, vec, st); break;
    default: launch_valu<PE_DTYPE_F16>(a, vec, st); break;
  }
  PE_CHECK_LAUNCH();
  return PE_OK;
}

int pe_internal_slot_offsets(const int64_t* slots, int M, int nkv, int hd, int page_size, int64_t num_pages,
                             int64_t* off, int32_t* status, hipStream_t st) {
  const int psl = page_log2(page_size);
  if (!slots || !off || M <= 0 || psl < 0 || num_pages <= 0) return PE_ERR_ARG;
  slot_offsets_kernel<<<pe_cdiv(M, 256), 256, 0, st>>>(slots, M, nkv, hd, psl, num_pages * page_size, off, status);
  PE_CHECK_LAUNCH();
  return PE_OK;
}

extern "C" int64_t pe_page_tables_scratch_bytes(int batch) { return batch < 0 ? 0 : 4 * ((int64_t)batch + 1); }

extern "C" int pe_page_tables(const int64_t* seq_len, const int32_t* seq_row0, int batch, int64_t M,
                              int64_t prefix_len, int page_size, int32_t* block_table, int64_t ld_table, int64_t cols,
                              int32_t* held, const int32_t* free_pages, int64_t n_free, int32_t* free_top,
                              int32_t* held_out, int32_t* top_out, int32_t* scratch, int64_t* slots, int32_t* status,
                              void* stream) {
  const int psl = page_log2(page_size);
  if (!seq_len || !seq_row0 || !block_table || !held || !free_top || !held_out || !top_out || !status || batch <= 0 ||
      batch > 65534 || M < 0 || M >= (int64_t(1) << 31) || (M > 0 && !slots) || prefix_len < 0 || psl < 0 || cols <= 0 ||
      cols > (int64_t(1) << 31) || ld_table < cols || n_free < 0 || n_free >= (int64_t(1) << 31) ||
      (n_free > 0 && !free_pages))
    return PE_ERR_ARG;
  const bool in_place = held_out == held || top_out == free_top;
  if (in_place && !scratch) return PE_ERR_WORKSPACE;
  hipStream_t st = (hipStream_t)stream;
  int64_t x = (M / batch + kTabThreads - 1) / kTabThreads;  // the average sequence's rows in one step
  x = x < 1 ? 1 : x > 64 ? 64 : x;
  page_tables_kernel<<<dim3((unsigned)x, batch + 1), kTabThreads, 0, st>>>(
      seq_len, seq_row0, batch, M, prefix_len, psl, block_table, ld_table, cols, held, free_pages, free_top, n_free,
      in_place ? scratch : held_out, in_place ? scratch + batch : top_out, slots, status);
  PE_CHECK_LAUNCH();
  if (in_place) {
    tables_commit_kernel<<<pe_cdiv(batch, kTabThreads), kTabThreads, 0, st>>>(scratch, held_out, batch, top_out);
    PE_CHECK_LAUNCH();
  }
  return PE_OK;
}

extern "C" int pe_page_release(const int32_t* seqs, int n, int batch, int32_t* block_table, int64_t ld_table,
                               int64_t cols, int32_t* held, int32_t* free_pages, int64_t n_free, int32_t* free_top,
                               int32_t* status, void* stream) {
  if (n < 0 || (n > 0 && !seqs) || batch <= 0 || !block_table || cols <= 0 || ld_table < cols || !held ||
      !free_pages || n_free < 0 || n_free >= (int64_t(1) << 31) || !free_top || !status)
    return PE_ERR_ARG;
  if (n == 0) return PE_OK;
  page_release_kernel<<<1, kTabThreads, 0, (hipStream_t)stream>>>(seqs, n, batch, block_table, ld_table, cols, held,
                                                                  free_pages, free_top, n_free, status);
  PE_CHECK_LAUNCH();
  return PE_OK;
}

extern "C" int pe_kv_write_paged(const void* k, const void* v, const int64_t* k_strides, const int64_t* v_strides,
                                 int L, int64_t M, int nkv, int hd, int dtype, void* k_pool, void* v_pool,
                                 int64_t num_pages, int page_size, const int64_t* slots, int32_t* status,
                                 void* stream) {
  const int es = esize(dtype), psl = page_log2(page_size);
  if (!k || !v || !k_strides || !v_strides || !k_pool || !v_pool || !status || L <= 0 || L > 65535 || M < 0 ||
      M >= (int64_t(1) << 31) || nkv <= 0 || hd <= 0 || hd > 65536 || es == 0 || psl < 0 || num_pages <= 0 ||
      num_pages >= (int64_t(1) << 31) || (M > 0 && !slots) || M * nkv >= (int64_t(1) << 31))
    return PE_ERR_ARG;
  if (M == 0) return PE_OK;
  const int64_t row = (int64_t)hd * es;
  uint64_t any = (uint64_t)(uintptr_t)k | (uint64_t)(uintptr_t)v | (uint64_t)(uintptr_t)k_pool |
                 (uint64_t)(uintptr_t)v_pool | (uint64_t)row;
  for (int i = 0; i < 3; ++i) any |= (uint64_t)(k_strides[i] * es) | (uint64_t)(v_strides[i] * es);
  const int64_t layer_bytes = num_pages * nkv * page_size * row;
  hipStream_t st = (hipStream_t)stream;
#define PE_WRITE(V)                                                                                               \
  do {                                                                                                            \
    const int vpr = (int)(row / (int64_t)sizeof(V));                                                              \
    const int64_t blocks = (M * nkv * vpr + 255) / 256;                                                           \
    if (M * nkv * vpr >= (int64_t(1) << 31)) return PE_ERR_ARG;                                                   \
    kv_write_kernel<V><<<dim3((unsigned)blocks, L, 2), 256, 0, st>>>(                                             \
        (const uint8_t*)k, (const uint8_t*)v, k_strides[0] * es, k_strides[1] * es, k_strides[2] * es,            \
        v_strides[0] * es, v_strides[1] * es, v_strides[2] * es, (uint8_t*)k_pool, (uint8_t*)v_pool, layer_bytes, \
        slots, (int)M, nkv, vpr, psl, num_pages * page_size, status);                                             \
  } while (0)
  if (any % 16 == 0) PE_WRITE(u32x4_t);
  else if (any % 4 == 0) PE_WRITE(uint32_t);
  else PE_WRITE(uint16_t);
#undef PE_WRITE
  PE_CHECK_LAUNCH();
  return PE_OK;
}

extern "C" int pe_kv_compact_paged(void* k_pool, void* v_pool, int L, int nkv, int hd, int dtype, int64_t num_pages,
                                   int page_size, const int32_t* block_table, int64_t ld_table, int64_t cols,
                                   int batch, const int64_t* seq_len, int64_t prefix_len, const int32_t* accept_out,
                                   int max_rows, int32_t* status, void* stream) {
  const int es = esize(dtype), psl = page_log2(page_size);
  if (!k_pool || !v_pool || !block_table || !seq_len || !accept_out || !status || L <= 0 || nkv <= 0 || hd <= 0 ||
      hd > 65536 || es == 0 || psl < 0 || num_pages <= 0 || num_pages >= (int64_t(1) << 31) || cols <= 0 ||
      cols > (int64_t(1) << 31) || ld_table < cols || batch <= 0 || batch > 65535 || prefix_len < 0 || max_rows <= 0 ||
      (int64_t)L * nkv >= (int64_t(1) << 31))
    return PE_ERR_ARG;
  const int64_t row = (int64_t)hd * es;
  const uint64_t any = (uint64_t)(uintptr_t)k_pool | (uint64_t)(uintptr_t)v_pool | (uint64_t)row;
  const int64_t layer_bytes = num_pages * nkv * page_size * row;
  const dim3 grid(pe_cdiv((int64_t)L * nkv, kCompactHeads), 2, batch);
  hipStream_t st = (hipStream_t)stream;
#define PE_COMPACT(V)                                                                                             \
  kv_compact_paged_kernel<V><<<grid, 64, 0, st>>>((uint8_t*)k_pool, (uint8_t*)v_pool, layer_bytes, L * nkv, nkv, \
                                                   (int)(row / (int64_t)sizeof(V)), psl, block_table, ld_table,   \
                                                   cols, num_pages, seq_len, prefix_len, accept_out,              \
                                                   2 + (int64_t)max_rows, max_rows, status)
  if (any % 16 == 0) PE_COMPACT(u32x4_t);
  else if (any % 4 == 0) PE_COMPACT(uint32_t);
  else PE_COMPACT(uint16_t);
#undef PE_COMPACT
  PE_CHECK_LAUNCH();
  return PE_OK;
}

// ------------------------------------------------------------------ attention
static bool mfma_fits(int hd, int dtype) {
  return (hd == 64 || hd == 128) && (dtype == PE_DTYPE_BF16 || dtype == PE_DTYPE_F16);
}

extern "C" int64_t pe_attention_paged_workspace_bytes(int64_t M, int batch, int nh, int nkv, int hd, int max_rows,
                                                      int64_t max_len, int64_t prefix_len, int dtype) {
  if (M <= 0 || batch <= 0 || nh <= 0 || nkv <= 0 || nh % nkv || max_rows <= 0 || prefix_len < 0 ||
      max_len < prefix_len || !mfma_fits(hd, dtype))
    return 0;
  return pe_internal_paged_mfma_bytes(M, batch, nh, nkv, hd, max_rows, max_len, prefix_len);
}

extern "C" int pe_tree_attention_paged(const pe_paged_attention_args* p, void* stream) {
  return pe_internal_tree_attention_paged(p, 0, (hipStream_t)stream);
}

extern "C" int64_t pe_attention_paged_reserve_bytes(int64_t M, int nh, int nkv, int hd, int dtype) {
  if (M <= 0 || nh <= 0 || nkv <= 0 || nh % nkv || !mfma_fits(hd, dtype)) return 0;
  return pe_internal_paged_mfma_reserve(M, nh, nkv, hd);
}

int pe_internal_tree_attention_paged(const pe_paged_attention_args* p, int out_units, hipStream_t st) {
  if (!p) return PE_ERR_ARG;
  const int es = esize(p->dtype), psl = page_log2(p->page_size);
  const bool none = p->M == 0 || p->max_rows == 0;  // no rows: their buffers may be absent
  if (!p->k_pool || !p->v_pool || !p->block_table || !p->seq_row0 || !p->seq_len || !p->status || es == 0 || psl < 0 ||
      (!none && (!p->q || !p->out)))
    return PE_ERR_ARG;
  if (p->M < 0 || p->M >= (int64_t(1) << 31) || p->batch <= 0 || p->batch > 65535 || p->nh <= 0 || p->nkv <= 0 ||
      p->nh % p->nkv || p->hd <= 0 || p->hd > 256 || p->max_rows < 0 || p->max_rows > 65535 || p->prefix_len < 0 ||
      p->max_len < p->prefix_len || p->max_len >= (int64_t(1) << 30) || p->num_pages <= 0 ||
      p->num_pages >= (int64_t(1) << 31) || p->ld_table <= 0 || p->table_cols <= 0 || p->ld_table < p->table_cols ||
      p->table_cols >= (int64_t(1) << 31) || p->ld_q < (int64_t)p->nh * p->hd || p->ld_out < (int64_t)p->nh * p->hd ||
      p->window < 0 || !(p->softcap >= 0.f && p->softcap < INFINITY) || !(p->scale > 0.f && p->scale < INFINITY) ||
      (int64_t)p->nkv * p->page_size * p->hd * es >= (int64_t(1) << 32))
    return PE_ERR_ARG;
  if (p->prefix_len > 0 && (!p->prefix_table || p->prefix_pages < ((p->prefix_len - 1) >> psl) + 1)) return PE_ERR_ARG;
  if (p->mask_mode == PE_MASK_TREE) {
    if ((!p->bits && !none) || p->words <= 0) return PE_ERR_ARG;
    if (p->words > PE_TREE_MAX_WORDS || p->max_rows > 64 * p->words) return PE_ERR_TREE;
  } else if (p->mask_mode != PE_MASK_CAUSAL) {
    return PE_ERR_ARG;
  }
  if ((p->window > 0 || p->slopes) && !p->positions && !none) return PE_ERR_ARG;
  if (none) return PE_OK;
  PagedAttn a;
  a.q = p->q;
  a.k_pool = p->k_pool;
  a.v_pool = p->v_pool;
  a.out = p->out;
  a.block_table = p->block_table;
  a.prefix_table = p->prefix_table;
  a.seq_row0 = p->seq_row0;
  a.seq_len = p->seq_len;
  a.bits = p->mask_mode == PE_MASK_TREE ? p->bits : nullptr;
  a.positions = p->window > 0 || p->slopes ? p->positions : nullptr;
  a.slopes = p->slopes;
  a.status = p->status;
  a.ld_q = p->ld_q;
  a.ld_out = p->ld_out;
  a.ld_table = p->ld_table;
  a.cols = p->table_cols;
  a.num_pages = p->num_pages;
  a.prefix_len = p->prefix_len;
  a.max_len = p->max_len;
  a.window = p->window;
  a.M = p->M;
  a.batch = p->batch;
  a.max_rows = p->max_rows;
  a.nh = p->nh;
  a.nkv = p->nkv;
  a.hd = p->hd;
  a.ps_log2 = psl;
  a.mask_mode = p->mask_mode;
  a.words = p->words;
  a.scale = p->scale;
  a.softcap = p->softcap;
  const bool aligned = (((uintptr_t)p->q | (uintptr_t)p->k_pool | (uintptr_t)p->v_pool | (uintptr_t)p->out) & 15) == 0 &&
                       p->ld_q % 8 == 0 && p->ld_out % 8 == 0;
  a.out_units = out_units;
  if (mfma_fits(p->hd, p->dtype) && aligned)
    return pe_internal_paged_mfma(a, p->dtype, p->workspace, p->workspace_bytes, st);
  if (out_units) return PE_ERR_ARG;
  return pe_internal_paged_valu(a, p->dtype, st);
}
