// Attention over a shared prefix and paged keys on the matrix cores (bf16 /
// fp16, heads of 64 or 128).
//
//   out_r = sum_j 2^(s_rj - M) v_j / sum_j 2^(s_rj - M),  s in base 2
//
// splits over any partition of the keys into parts with their own maximum m_p,
// sum l_p and weighted sum O_p, joined by weights 2^(m_p - M). The keys of the
// prefix are the same for every row of the batch, so one KV head's rows of all
// sequences (R = M G of them) meet them as one matrix product: each K / V byte
// read serves a block of up to 256 rows, and the prefix is bound by the matrix
// cores (and the exponentials beside them) where a per-sequence pass would read
// it once per sequence. A sequence's own keys serve its own rows only.
//
// The prefix's and the sequences' own keys are shares of one launch, whose parts
// a second one joins; a large prefix (many rows over many keys) gets a launch of
// its own with wider row blocks first, and the sequences' workgroups join its
// parts to theirs and write the output themselves.
//
// Products as in the contiguous kernels: S^T = K Q^T (A = 32 keys, B = the
// wave's 32 rows, held in registers), so that a lane owns one row and 16 of 32
// keys; O^T += V^T P^T with P^T straight from the S^T registers, rounded to the
// type (half a step per weight; its sum l is of the unrounded ones, so the
// error is that of the weights alone), V^T by transposed LDS reads.

#include "pe_paged.h"

#include <algorithm>

namespace {

constexpr float kLog2e = 1.44269504088896341f;

// Physical 16-byte chunk of logical chunk c of row `row` is c ^ swizzle(row).
// 256-byte rows: (2i ^ 4i ^ j), i = row % 4, j = row / 4 % 4; 128-byte rows (two
// to a bank line): the bits of row / 2 % 8 reversed. Both are bijections on 16
// rows, so a K fragment's 16 rows fall on distinct banks, and move the upper
// bits of the chunk among four neighbouring rows, so the transposed V reads do.
template <int HD>
__device__ __forceinline__ int swizzle(int row) {
  if constexpr (HD == 128) {
    const int i = row & 3, j = (row >> 2) & 3;
    return ((i << 1) ^ (i << 2) ^ j) & 15;
  } else {
    const int i = (row >> 1) & 7;
    return ((i & 1) << 2) | (i & 2) | (i >> 2);
  }
}
template <int HD>
__device__ __forceinline__ uint32_t lds_at(int row, int chunk) {
  return (uint32_t)(row * (HD * 2) + ((chunk ^ swizzle<HD>(row)) << 4));
}

template <int DT>
__device__ __forceinline__ f32x16_t mfma32(u32x4_t a, u32x4_t b, f32x16_t c) {
  if constexpr (DT == PE_DTYPE_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0,
                                                  0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
}

// s_waitcnt with vmcnt = N, the other counters at their maxima
template <int N>
__device__ __forceinline__ void wait_vm() {
  __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));
}

// One list of pages as the key source of a KV head.
struct Pages {
  const int32_t* table;
  int lo, hi;  // keys read (counted in 32 bits: a sequence is shorter than 2^30), [lo, hi), the others of a step as the nearest
};

// What a lane's row needs besides its Q.
struct RowInfo {
  int node;       // causal: its token's index among the sequence's new rows; tree: unused
  int rel;        // its position - the position of key 0 of the list (MOD)
  float slope2;   // slope * log2 e (MOD)
  int lo, tile_lo;  // first cached key its window holds; the largest of the tile's (MOD)
  uint64_t nb0, nb1, nb2, nb3;  // ancestor bits (named: an indexed array would live in scratch memory)
};
static_assert(PE_TREE_MAX_WORDS == 4, "one field per word");

// The configuration of a workgroup: W waves, DS of them on one 32-row tile (each
// forms the tile's scores and keeps hd / DS dims of its O; with few tiles a
// workgroup waits for keys, and this needs no exchange between its waves), SB
// 32-key blocks in a step, a ring of ST steps in LDS filled straight from global
// memory (ST - 1 of them in flight while one is multiplied).
template <int HD_, int W_, int DS_, int SB_, int ST_>
struct Cfg {
  static constexpr int HD = HD_, W = W_, DS = DS_, SB = SB_, ST = ST_;
  static constexpr int NT = W / DS;                     // row tiles
  static constexpr int OB = HD / 32 / DS;               // 32-dim blocks of O a wave holds
  static constexpr int SK = 32 * SB;                    // keys of a step
  static constexpr int kHalf = SK * HD * 2;             // bytes of a step's K (and of its V)
  static constexpr int kStep = 2 * kHalf;
  static constexpr int kChunks = 2 * SK / 16 / W;       // 16-key pieces of K or V a wave loads per step
  static constexpr int kPerChunk = 16 * HD * 2 / 1024;  // load instructions of one
  static constexpr int kLoads = kChunks * kPerChunk;
  static constexpr int kSmem = ST * kStep;
  static_assert(2 * SK / 16 % W == 0, "whole pieces per wave");
};

// One 64-bit-masked step's visibility, bit j: key kb0 + j. Tree rows see keys
// below P and the nodes of their bits; causal rows those up to P + node.
__device__ __forceinline__ uint64_t node_window(int kb0, int P, uint64_t n0, uint64_t n1, uint64_t n2,
                                                uint64_t n3) {
  const int off = kb0 - P;  // node index of key kb0
  if (off <= -64) return ~0ull;
  if (off < 0) {
    const int j0 = -off;
    return ((1ull << j0) - 1) | (n0 << j0);
  }
  if (off >= 64 * PE_TREE_MAX_WORDS) return 0ull;
  const int wi = off >> 6, sh = off & 63;
  const uint64_t a = wi == 0 ? n0 : wi == 1 ? n1 : wi == 2 ? n2 : n3;
  const uint64_t b = wi == 0 ? n1 : wi == 1 ? n2 : wi == 2 ? n3 : 0ull;
  return sh ? (a >> sh) | (b << (64 - sh)) : a;
}
__device__ __forceinline__ uint64_t below(int n) {  // bits 0 .. n - 1
  return n >= 64 ? ~0ull : (n <= 0 ? 0ull : (1ull << n) - 1);
}

// The keys [s0 SK, s1 SK) of a list for the workgroup's row tiles: O^T, m, l of
// the wave's tile. `P`: the list's cached keys, new rows follow (PRE: no new rows).
// Keys outside [pg.lo, pg.hi) are masked, steps past last_key (the last that a
// row of the tile sees) skipped. npos (LDS): positions of the new rows relative
// to key 0 (MOD, where distances count).
template <int DT, typename C, bool MOD, bool PRE>
__device__ __forceinline__ void attend(const PagedAttn& a, uint8_t* smem, const Pages& pg, int kvh, int s0, int s1,
                                       int P, int new_rows, bool live, int last_key, RowInfo ri,
                                       const u32x4_t (&qf)[C::HD / 16], const int* npos, bool& bad,
                                       f32x16_t (&o)[C::OB], float& m, float& l) {
  constexpr int HD = C::HD, SB = C::SB, OB = C::OB;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int ln = lane & 31, g = lane >> 5, hb = (wave % C::DS) * OB;
  const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;
  typedef const __attribute__((address_space(4))) int32_t* const_i32;  // read through the scalar cache
  const const_i32 tab = (const_i32)(uintptr_t)uniform_ptr((const uint16_t*)pg.table);
  const int psl = a.ps_log2;
  const int clo = pg.lo >> 4, chi = (pg.hi - 1) >> 4;
  // the pages of this wave's pieces of a step, asked for a step ahead
  int page[C::kChunks];
  auto piece_of = [&](int step, int c) {
    const int ch = (wave * C::kChunks + c) % (C::SK / 16);
    const int k = step * (C::SK / 16) + ch;
    return k < clo ? clo : k > chi ? chi : k;
  };
  auto ask = [&](int step) {
#pragma unroll
    for (int c = 0; c < C::kChunks; ++c) page[c] = tab[(piece_of(step, c) << 4) >> psl];
  };
  auto issue = [&](int step) {
    const uint32_t buf = lds_base + (step % C::ST) * C::kStep;
#pragma unroll
    for (int c = 0; c < C::kChunks; ++c) {
      const int piece = wave * C::kChunks + c, ch = piece % (C::SK / 16);
      const bool is_v = piece >= C::SK / 16;
      const int k16 = piece_of(step, c);
      int pgid = page[c];
      if (pgid < 0 || pgid >= a.num_pages) {
        bad = true;
        pgid = 0;
      }
      const int64_t row = ((((int64_t)pgid * a.nkv + kvh) << psl) + ((k16 << 4) & ((1 << psl) - 1)));
      const uint16_t* src = uniform_ptr((const uint16_t*)(is_v ? a.v_pool : a.k_pool) + row * HD);
      const uint32_t dst =
          __builtin_amdgcn_readfirstlane(buf + (is_v ? C::kHalf : 0) + ch * 16 * HD * 2);
      const int rlo = max(pg.lo - (k16 << 4), 0), rhi = min(pg.hi - 1 - (k16 << 4), 15);
#pragma unroll
      for (int i = 0; i < C::kPerChunk; ++i) {
        constexpr int kLanes = HD / 8;  // lanes on a row
        const int r = i * (64 / kLanes) + lane / kLanes;
        const int rr = min(max(r, rlo), rhi);
        lds_dma16(src, (uint32_t)(rr * (HD * 2) + (((lane % kLanes) ^ swizzle<HD>(r)) << 4)), dst + i * 1024);
      }
    }
  };

#pragma unroll
  for (int h = 0; h < OB; ++h)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[h][i] = 0.f;
  m = kPagedInitMax;
  l = 0.f;
  const float scale2 = a.scale * kLog2e;
  const bool tree = a.mask_mode == PE_MASK_TREE;
  const float cap_in = MOD && a.softcap > 0.f ? 2.f * scale2 / a.softcap : 0.f, cap_out = a.softcap * kLog2e;

  if (s0 < s1) ask(s0);
  __syncthreads();  // the buffers' and hand-over's last readers are done
#pragma unroll
  for (int i = 0; i < C::ST - 1; ++i)
    if (s0 + i < s1) {
      issue(s0 + i);
      if (s0 + i + 1 < s1) ask(s0 + i + 1);
    }
  __builtin_amdgcn_s_waitcnt(0);  // Q has landed: no later wait of the compiler's covers the ring's loads
  for (int s = s0; s < s1; ++s) {
    if (s1 - 1 - s >= C::ST - 2) wait_vm<(C::ST - 2) * C::kLoads>();
    else wait_vm<0>();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();  // everyone's loads of step s have landed, and step s - 1's buffer is free
    asm volatile("" ::: "memory");
    if (s + C::ST - 1 < s1) {
      issue(s + C::ST - 1);
      if (s + C::ST < s1) ask(s + C::ST);
    }
    const int kb0 = s * C::SK;
    if (!live || kb0 > last_key) continue;  // wave-uniform: the tile sees no key of this step
    const uint8_t* kbp = smem + (s % C::ST) * C::kStep;
    const uint8_t* vbp = kbp + C::kHalf;
    f32x16_t sc[SB];
#pragma unroll
    for (int sb = 0; sb < SB; ++sb)
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[sb][i] = 0.f;
#pragma unroll
    for (int j = 0; j < HD / 16; ++j)
#pragma unroll
      for (int sb = 0; sb < SB; ++sb)
        sc[sb] = mfma32<DT>(*(const u32x4_t*)(kbp + lds_at<HD>(32 * sb + ln, 2 * j + g)), qf[j], sc[sb]);
    // sc[sb][i] is key kb0 + 32 sb + 8 (i / 4) + 4 g + i % 4 of the lane's row
    bool node_step = false;
    if constexpr (!PRE) node_step = kb0 + 32 * SB > P;
    if constexpr (MOD) {
      if (cap_in != 0.f) {
        // cap tanh(s / cap) = cap (1 - 2 / (1 + e^(2 s / cap))): both ends exact
#pragma unroll
        for (int sb = 0; sb < SB; ++sb)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float e = __builtin_amdgcn_exp2f(sc[sb][i] * cap_in);
            sc[sb][i] = fmaf(-2.f * cap_out, __builtin_amdgcn_rcpf(1.f + e), cap_out);
          }
      } else {
#pragma unroll
        for (int sb = 0; sb < SB; ++sb)
#pragma unroll
          for (int i = 0; i < 16; ++i) sc[sb][i] *= scale2;
      }
      const int d0 = ri.rel - kb0 - 4 * g;  // distance of key kb0 + 4 g
      if (node_step && tree && npos) {  // new rows lie where their positions say
#pragma unroll
        for (int sb = 0; sb < SB; ++sb)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int off = 32 * sb + 8 * (i >> 2) + (i & 3);
            const int u = kb0 - P + off + 4 * g;
            const int np = npos[max(0, min(u, new_rows - 1))];
            const int dist = u < 0 ? d0 - off : ri.rel - np;
            sc[sb][i] = fmaf(-ri.slope2, (float)dist, sc[sb][i]);
            if (a.window > 0) sc[sb][i] = dist < a.window ? sc[sb][i] : -INFINITY;
          }
      } else if (a.slopes) {
#pragma unroll
        for (int sb = 0; sb < SB; ++sb)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            sc[sb][i] = fmaf(-ri.slope2, (float)(d0 - (32 * sb + 8 * (i >> 2) + (i & 3))), sc[sb][i]);
      }
    }
    bool edge = node_step || kb0 + 32 * SB > pg.hi || kb0 < pg.lo;
    if constexpr (MOD) edge = edge || kb0 < ri.tile_lo;
    if (edge) {
      uint64_t win = ~0ull;
      if constexpr (!PRE) win = tree ? node_window(kb0, P, ri.nb0, ri.nb1, ri.nb2, ri.nb3) : below(P + ri.node + 1 - kb0);
      int lo = pg.lo;
      if constexpr (MOD) lo = max(lo, ri.lo);
      win &= below(pg.hi - kb0) & ~below(lo - kb0);
      win >>= 4 * g;
#pragma unroll
      for (int sb = 0; sb < SB; ++sb)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          sc[sb][i] = ((win >> (32 * sb + 8 * (i >> 2) + (i & 3))) & 1ull) ? sc[sb][i] : -INFINITY;
    }
    float bmax = -INFINITY;
#pragma unroll
    for (int sb = 0; sb < SB; ++sb)
#pragma unroll
      for (int i = 0; i < 16; ++i) bmax = fmaxf(bmax, sc[sb][i]);
    bmax = fmaxf(bmax, __shfl_xor(bmax, 32, 64));
    if constexpr (!MOD) bmax *= scale2;
    const float mnew = fmaxf(m, bmax);
    const float alpha = __builtin_amdgcn_exp2f(m - mnew);
    float psum = 0.f;
    uint32_t pb[SB][8];
#pragma unroll
    for (int sb = 0; sb < SB; ++sb)
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float p0 = __builtin_amdgcn_exp2f(MOD ? sc[sb][i] - mnew : fmaf(sc[sb][i], scale2, -mnew));
        const float p1 = __builtin_amdgcn_exp2f(MOD ? sc[sb][i + 1] - mnew : fmaf(sc[sb][i + 1], scale2, -mnew));
        psum += p0 + p1;
        pb[sb][i >> 1] = pack2_16<DT>(p0, p1);
      }
    psum += __shfl_xor(psum, 32, 64);
    l = l * alpha + psum;
    if (__builtin_amdgcn_ballot_w64(mnew != m) != 0ull) {
#pragma unroll
      for (int h = 0; h < OB; ++h)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[h][i] *= alpha;
    }
    m = mnew;
    // O^T += V^T P^T over the 16-key quarters of the step
    const int qg = lane >> 4, jl = lane & 15;
#pragma unroll
    for (int c = 0; c < 2 * SB; ++c) {
      const int sb = c >> 1, cq = c & 1;
      const u32x4_t bp = {pb[sb][4 * cq], pb[sb][4 * cq + 1], pb[sb][4 * cq + 2], pb[sb][4 * cq + 3]};
      const int kb = 16 * c + 4 * (qg >> 1) + (jl >> 2);
#pragma unroll
      for (int h = 0; h < OB; ++h) {
        const int db = 32 * (hb + h) + 16 * (qg & 1) + 4 * (jl & 3);
        typedef short s4v_t __attribute__((__vector_size__(4 * sizeof(short))));
        typedef __attribute__((address_space(3))) s4v_t lds_s4v_t;
        const uint2 lo = __builtin_bit_cast(
            uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4v_t*)(vbp + lds_at<HD>(kb, db >> 3) + (db & 7) * 2)));
        const uint2 hi = __builtin_bit_cast(
            uint2,
            __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4v_t*)(vbp + lds_at<HD>(kb + 8, db >> 3) + (db & 7) * 2)));
        const u32x4_t av = {lo.x, lo.y, hi.x, hi.y};
        o[h] = mfma32<DT>(av, bp, o[h]);
      }
    }
  }
}

// Work item of workgroup `b` of `n`: neighbours in the sequence of items (which
// share a KV head's keys) on one XCD (workgroup b starts on XCD b % 8).
__device__ __forceinline__ uint32_t xcd_item(uint32_t b, uint32_t n) {
  return n & 7 ? b : (b & 7) * (n >> 3) + (b >> 3);
}

template <int HD>
__device__ __forceinline__ int64_t part_tile(const PagedParts& p, int nkv, int part, int kvh, uint32_t tile) {
  return (((int64_t)part * nkv + kvh) * p.tiles + tile) * (32 * HD);
}

// `hb`: the first 32-dim block of O held.
template <int HD, int OB>
__device__ __forceinline__ void store_part(const PagedParts& p, int nkv, int part, int kvh, uint32_t row, int g, int hb,
                                           const f32x16_t (&o)[OB], float m, float l) {
  float* dst = p.o + part_tile<HD>(p, nkv, part, kvh, row >> 5) + ((row & 31) + 32 * g) * 4 + hb * 1024;
#pragma unroll
  for (int h = 0; h < OB; ++h)
#pragma unroll
    for (int c = 0; c < 4; ++c)
      *(f32x4_t*)(dst + (4 * h + c) * 256) = f32x4_t{o[h][4 * c], o[h][4 * c + 1], o[h][4 * c + 2], o[h][4 * c + 3]};
  if (g == 0 && hb == 0) {
    float2* ml = (float2*)p.ml + ((int64_t)part * nkv + kvh) * p.tiles * 32 + row;
    *ml = make_float2(m, l);
  }
}

// The lane's row's first cached key inside its window (ri.lo), the last of the
// tile's (ri.tile_lo) and the first of the workgroup's (returned); `cached` keys.
template <int W>
__device__ __forceinline__ int window_lo(const PagedAttn& a, RowInfo& ri, int cached, bool live, int* s_lo) {
  ri.lo = ri.tile_lo = 0;
  if (a.window == 0) return 0;
  ri.lo = (int)min(max((int64_t)ri.rel - a.window + 1, (int64_t)0), (int64_t)cached);
  int lo = live ? ri.lo : cached, hi = ri.lo;
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) {
    lo = min(lo, __shfl_xor(lo, d, 64));
    hi = max(hi, __shfl_xor(hi, d, 64));
  }
  ri.tile_lo = __builtin_amdgcn_readfirstlane(hi);
  if constexpr (W > 1) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s_lo[threadIdx.x >> 6] = lo;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) lo = min(lo, s_lo[i]);
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// ---------------------------------------------------------------------------
// The prefix: workgroup `w`'s share of the row blocks' key steps
// ---------------------------------------------------------------------------
template <int DT, typename C, bool MOD>
__device__ __forceinline__ void prefix_share(const PagedAttn& a, const PagedPrefix& pp, const PagedParts& parts,
                                             uint32_t w, uint8_t* smem, int* s_lo) {
  constexpr int HD = C::HD;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int ln = lane & 31, g = lane >> 5, tile = wave / C::DS, hb = (wave % C::DS) * C::OB;
  const uint32_t G = (uint32_t)(a.nh / a.nkv), R = (uint32_t)a.M * G;
  const uint32_t uend = min(pp.total, (w + 1) * pp.per);
  bool bad = false;
  for (uint32_t u = w * pp.per; u < uend;) {
    const uint32_t x = u / pp.steps;
    const int s0 = (int)(u - x * pp.steps);
    const int s1 = (int)min(pp.steps, s0 + (uend - u));
    u += s1 - s0;
    const int kvh = (int)(x / pp.nblk);
    const uint32_t blk0 = (x - kvh * pp.nblk) * pp.block_rows, row0 = blk0 + 32 * tile;
    const bool live = row0 < min(blk0 + pp.block_rows, R);
    const uint32_t row = min(row0 + ln, R - 1), tok = row / G;
    const int hq = (int)(kvh * G + (row - tok * G));
    u32x4_t qf[HD / 16];
    const uint16_t* qr = (const uint16_t*)a.q + tok * a.ld_q + (int64_t)hq * HD + 8 * g;
#pragma unroll
    for (int j = 0; j < HD / 16; ++j) qf[j] = *(const u32x4_t*)(qr + 16 * j);
    RowInfo ri;
    const int S0 = (int)a.prefix_len;
    Pages pg{a.prefix_table, 0, S0};
    int first = s0;
    if constexpr (MOD) {
      ri.rel = a.positions ? (int)a.positions[tok] : 0;
      ri.slope2 = a.slopes ? a.slopes[hq] * kLog2e : 0.f;
      const int lo = window_lo<C::W>(a, ri, S0, live, s_lo);
      pg.lo = min(lo, S0 - 1);
      if (lo > 0) first = lo >= S0 ? s1 : max(s0, lo / C::SK);  // steps behind every row's window
    }
    f32x16_t o[C::OB];
    float m, l;
    attend<DT, C, MOD, true>(a, smem, pg, kvh, first, max(first, s1), S0, 0, live, S0 - 1, ri, qf, nullptr, bad, o, m, l);
    if (live)
      store_part<HD, C::OB>(parts, a.nkv, (int)(w - prefix_first_wg(pp, x)), kvh, row0 + ln, g, hb, o, m, l);
  }
  if (bad && lane == 0) atomicOr(a.status, PE_ERR_INDEX);
}

// ---------------------------------------------------------------------------
// The sequences' own keys: item = (key split of kps keys, sequence, KV head,
// block of row tiles)
// ---------------------------------------------------------------------------
// The launch's shares of it. `direct`: a sequence of one split joins the
// prefix's parts of its rows to its own (an earlier launch wrote them, and they
// are few) and writes the output; otherwise its result is a part as well and
// paged_join_kernel writes the output.
struct PagedSeqs {
  uint32_t items, kps, nblk, block_rows;
  int nsplit, kind, direct;
};

template <int DT, int OB>
__device__ __forceinline__ void write_out(const PagedAttn& a, int64_t tok, int64_t col, const f32x16_t (&o)[OB],
                                          float l) {
  typedef typename Elem<DT>::T Te;
  Te* dst = (Te*)a.out + tok * a.ld_out + col;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int h = 0; h < OB; ++h)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float v[4] = {o[h][4 * c] * inv, o[h][4 * c + 1] * inv, o[h][4 * c + 2] * inv, o[h][4 * c + 3] * inv};
      Vec4<DT>::store(dst + 32 * h + 8 * c, v);
    }
}

template <int DT, typename C, bool MOD>
__device__ __forceinline__ void seq_item(const PagedAttn& a, const PagedPrefix& pp, const PagedParts& parts,
                                         const PagedSeqs& sq, uint32_t item, uint8_t* smem, int* s_npos, int* s_lo) {
  constexpr int HD = C::HD;
  // blocks of one (split, sequence, KV head) on one XCD, neighbours in time;
  // otherwise KV heads over the XCDs (workgroup i starts on XCD i % 8), so that
  // sequences of different lengths load them alike, and the last splits, which
  // short sequences leave empty, at the end
  uint32_t blk = 0;
  if (sq.nblk > 1) {
    const uint32_t per = sq.items / sq.nblk & 7 ? 1 : 8, q = item / (per * sq.nblk), r = item - q * per * sq.nblk;
    blk = r / per;
    item = q * per + (r - blk * per);
  }
  const uint32_t sb = item / (uint32_t)a.nkv;
  const int kvh = (int)(item - sb * a.nkv), split = (int)(sb / (uint32_t)a.batch), b = (int)(sb - split * a.batch);
  const PagedSeq s = paged_seq(a, b);
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  if (!s.ok) {
    if (s.err && tid == 0 && kvh == 0 && split == 0 && blk == 0) atomicOr(a.status, s.err);
    return;
  }
  const int T = s.rows;
  const uint32_t G = (uint32_t)(a.nh / a.nkv), R = T * G;
  const int P = (int)s.priv, S = P + T;
  const uint32_t blk0 = blk * sq.block_rows;
  const int my_splits = (int)(((uint32_t)S + sq.kps - 1) / sq.kps);
  if (blk0 >= R || split >= my_splits) return;
  const int ln = lane & 31, g = lane >> 5, tile = wave / C::DS, hb = (wave % C::DS) * C::OB;
  const bool tree = a.mask_mode == PE_MASK_TREE;
  const uint32_t row0 = blk0 + 32 * tile, row_end = min(blk0 + sq.block_rows, R);
  const bool live = row0 < row_end;
  const uint32_t row = min(row0 + ln, R - 1);
  const int t = (int)(row / G);
  const int hq = kvh * (int)G + (int)(row - t * G);
  const int64_t tok = s.row0 + t;
  u32x4_t qf[HD / 16];
  const uint16_t* qr = (const uint16_t*)a.q + tok * a.ld_q + (int64_t)hq * HD + 8 * g;
#pragma unroll
  for (int j = 0; j < HD / 16; ++j) qf[j] = *(const u32x4_t*)(qr + 16 * j);
  RowInfo ri;
  ri.node = t;
  ri.nb0 = ri.nb1 = ri.nb2 = ri.nb3 = 0ull;
  if (tree) {
    const uint64_t* bt = a.bits + tok * a.words;
    ri.nb0 = bt[0];
    if (a.words > 1) ri.nb1 = bt[1];
    if (a.words > 2) ri.nb2 = bt[2];
    if (a.words > 3) ri.nb3 = bt[3];
  }
  // the keys some row of the block sees end at hi; of this wave's tile, at last_key
  const int t_blk = min(T - 1, (int)((blk0 + sq.block_rows - 1) / G));
  const int t_tile = min(T - 1, (int)((row0 + 31) / G));
  Pages pg{a.block_table + b * a.ld_table, 0, tree ? S : P + t_blk + 1};
  const int last_key = tree ? S - 1 : P + t_tile;
  if constexpr (MOD) {
    ri.rel = a.positions ? (int)(a.positions[tok] - a.prefix_len) : 0;
    ri.slope2 = a.slopes ? a.slopes[hq] * kLog2e : 0.f;
    if (a.positions && tree)
      for (int u = tid; u < T; u += 64 * C::W) s_npos[u] = (int)(a.positions[s.row0 + u] - a.prefix_len);
    pg.lo = window_lo<C::W>(a, ri, tree ? P : pg.hi - 1, live, s_lo);
  }
  const int k0 = split * (int)sq.kps, k1 = min(pg.hi, k0 + (int)sq.kps);
  const int s1 = (k1 + C::SK - 1) / C::SK, s0 = max(k0, pg.lo) / C::SK;
  bool bad = false;
  f32x16_t o[C::OB];
  float m, l;
  attend<DT, C, MOD, false>(a, smem, pg, kvh, s0, max(s0, s1), P, T, live, last_key, ri, qf,
                            MOD && a.positions ? s_npos : nullptr, bad, o, m, l);
  if (bad && lane == 0) atomicOr(a.status, PE_ERR_INDEX);
  if (row0 + ln >= row_end) return;
  const uint32_t grow = (uint32_t)s.row0 * G + row;  // the row among the whole batch's
  if (my_splits > 1 || !sq.direct) {
    store_part<HD, C::OB>(parts, a.nkv, parts.pre_parts + split, kvh, grow, g, hb, o, m, l);
    return;
  }
  if (parts.pre_parts > 0) {
    const int n = prefix_parts_of(pp, kvh * pp.nblk + grow / pp.block_rows);
    for (int p = 0; p < n; ++p) {
      const float2 ml = ((const float2*)parts.ml)[((int64_t)p * a.nkv + kvh) * parts.tiles * 32 + grow];
      const float mx = fmaxf(m, ml.x);
      const float a0 = __builtin_amdgcn_exp2f(m - mx), a1 = __builtin_amdgcn_exp2f(ml.x - mx);
      m = mx;
      l = a0 * l + a1 * ml.y;
      const float* src = parts.o + part_tile<HD>(parts, a.nkv, p, kvh, grow >> 5) + ((grow & 31) + 32 * g) * 4 + hb * 1024;
#pragma unroll
      for (int h = 0; h < C::OB; ++h)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const f32x4_t o1 = *(const f32x4_t*)(src + (4 * h + c) * 256);
#pragma unroll
          for (int i = 0; i < 4; ++i) o[h][4 * c + i] = a0 * o[h][4 * c + i] + a1 * o1[i];
        }
    }
  }
  write_out<DT, C::OB>(a, tok, (int64_t)hq * HD + 32 * hb + 4 * g, o, l);
}

// ---------------------------------------------------------------------------
// Kernels
// ---------------------------------------------------------------------------
// Many rows over a long prefix: eight tiles (256 rows) on every K / V byte, one
// workgroup per CU.
template <int HD> using Wide = Cfg<HD, 8, 1, 2, 4>;
// Four waves, 64 KiB of LDS (32 KiB for heads of 64), two workgroups per CU.
template <int HD> using Four = Cfg<HD, 4, 1, 2, 2>;
template <int HD> using Two = Cfg<HD, 4, 2, HD == 128 ? 1 : 2, 4>;
template <int HD> using One = Cfg<HD, 4, HD == 128 ? 4 : 2, HD == 128 ? 1 : 2, 4>;

template <int DT, int HD, bool MOD>
__global__ __launch_bounds__(512, 2) void paged_prefix_kernel(PagedAttn a, PagedPrefix pp, PagedParts parts) {
  __shared__ __align__(1024) uint8_t smem[Wide<HD>::kSmem];
  __shared__ int s_lo[8];
  prefix_share<DT, Wide<HD>, MOD>(a, pp, parts, xcd_item(blockIdx.x, gridDim.x), smem, s_lo);
}

// Workgroups [0, n_pre) take the prefix, the rest the sequences' own keys: on
// the two places of a CU the one waits for the matrix cores while the other
// waits for memory.
template <int DT, int HD, bool MOD>
__global__ __launch_bounds__(256, 2) void paged_attn_kernel(PagedAttn a, PagedPrefix pp, PagedParts parts, PagedSeqs sq,
                                                            uint32_t n_pre, int pre_kind) {
  constexpr int kSmem = Two<HD>::kSmem > Four<HD>::kSmem ? Two<HD>::kSmem : Four<HD>::kSmem;
  static_assert(One<HD>::kSmem <= kSmem, "one ring for every kind");
  __shared__ __align__(1024) uint8_t smem[kSmem];
  __shared__ int s_npos[MOD ? 64 * PE_TREE_MAX_WORDS : 1];
  __shared__ int s_lo[4];
  if (blockIdx.x < n_pre) {
    const uint32_t w = xcd_item(blockIdx.x, n_pre);
    if (pre_kind == 4) prefix_share<DT, Four<HD>, MOD>(a, pp, parts, w, smem, s_lo);
    else if (pre_kind == 2) prefix_share<DT, Two<HD>, MOD>(a, pp, parts, w, smem, s_lo);
    else prefix_share<DT, One<HD>, MOD>(a, pp, parts, w, smem, s_lo);
  } else {
    const uint32_t item = blockIdx.x - n_pre;
    if (sq.kind == 4) seq_item<DT, Four<HD>, MOD>(a, pp, parts, sq, item, smem, s_npos, s_lo);
    else if (sq.kind == 2) seq_item<DT, Two<HD>, MOD>(a, pp, parts, sq, item, smem, s_npos, s_lo);
    else seq_item<DT, One<HD>, MOD>(a, pp, parts, sq, item, smem, s_npos, s_lo);
  }
}

// Joins the parts: one thread per (row, four dims), 32 rows x 32 dims a block
// (512 contiguous bytes of a part per load), the prefix's parts first, then the
// splits in key order.
template <int DT, int HD>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttn a, PagedPrefix pp, PagedParts parts, PagedSeqs sq) {
  const int b = blockIdx.z, kvh = blockIdx.y;
  const PagedSeq s = paged_seq(a, b);
  if (!s.ok) return;
  const int my_splits = (int)(((uint32_t)(s.priv + s.rows) + sq.kps - 1) / sq.kps);
  const uint32_t G = (uint32_t)(a.nh / a.nkv), R = s.rows * G;
  const uint32_t row = blockIdx.x / (HD / 32) * 32 + (threadIdx.x & 31);
  const int piece = (int)(blockIdx.x % (HD / 32)) * 8 + (int)(threadIdx.x >> 5);  // dims 4 piece .. + 3
  if ((my_splits <= 1 && sq.direct) || row >= R) return;
  const uint32_t grow = (uint32_t)s.row0 * G + row;
  const int npre = parts.pre_parts > 0 ? prefix_parts_of(pp, kvh * pp.nblk + grow / pp.block_rows) : 0;
  const float* src = parts.o + part_tile<HD>(parts, a.nkv, 0, kvh, grow >> 5) + (piece >> 1) * 256 +
                     ((int)(grow & 31) + 32 * (piece & 1)) * 4;
  const float2* sml = (const float2*)parts.ml + (int64_t)kvh * parts.tiles * 32 + grow;
  const int64_t o_part = (int64_t)a.nkv * parts.tiles * (32 * HD), ml_part = (int64_t)a.nkv * parts.tiles * 32;
  float m = kPagedInitMax, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  constexpr int kAhead = 4;  // parts asked for before the first is joined
  const int n = npre + my_splits;
  for (int i0 = 0; i0 < n; i0 += kAhead) {
    float2 ml[kAhead];
    f32x4_t v[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = min(i0 + k, n - 1), p = i < npre ? i : parts.pre_parts + i - npre;
      ml[k] = sml[p * ml_part];
      v[k] = *(const f32x4_t*)(src + p * o_part);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (i0 + k >= n) break;
      const float mx = fmaxf(m, ml[k].x);
      const float a0 = __builtin_amdgcn_exp2f(m - mx), a1 = __builtin_amdgcn_exp2f(ml[k].x - mx);
      m = mx;
      l = a0 * l + a1 * ml[k].y;
#pragma unroll
      for (int d = 0; d < 4; ++d) o[d] = a0 * o[d] + a1 * v[k][d];
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const float v[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
  typedef typename Elem<DT>::T Te;
  const uint32_t tok = grow / G;
  const int hq = (int)(kvh * G + (grow - tok * G));
  Vec4<DT>::store((Te*)a.out + tok * a.ld_out + (int64_t)hq * HD + 4 * piece, v);
}

// ------------------------------------------------------------------ plans
constexpr int kCus = 256;
constexpr int kSeqWgs = 2048, kMinSplit = 256, kSplitRows = 8, kPrefixSteps = 4, kFusedPre = 256;
constexpr int64_t kWideUnits = 4096;

// A launch's workgroups: which configuration, row tiles per block and how many
// blocks hold `tiles` row tiles in equal shares.
struct Shape {
  int kind, tiles;
  int64_t blocks;
};
Shape shape_of(int64_t tiles, int most) {
  const int64_t blocks = (tiles + most - 1) / most;
  const int each = (int)((tiles + blocks - 1) / blocks);
  return {most == 8 ? 8 : each > 2 ? 4 : each, each, blocks};
}
// Keys of a step: 32 for 128-dim heads with one or two tiles, else 64.
int step_keys(const Shape& s, int hd) { return hd == 64 || s.kind >= 4 ? 64 : 32; }

struct Plan {
  PagedPrefix pp;
  PagedSeqs sq;
  PagedParts pt;
  bool wide, join;
  int pre_kind;
  int64_t units, items, pre_wgs, o_bytes, ml_bytes;
};

Plan make_plan(int64_t M, int batch, int nh, int nkv, int hd, int max_rows, int64_t max_len, int64_t prefix_len) {
  Plan p;
  const int G = nh / nkv;
  const int64_t tiles = (M * G + 31) / 32;
  p.pt.tiles = tiles;
  p.pp = PagedPrefix{0, 1, 1, 1, 32};
  p.pre_wgs = p.units = 0;
  p.pt.pre_parts = p.pre_kind = 0;
  p.wide = false;
  if (prefix_len > 0) {
    const int64_t s64 = (prefix_len - 1) / 64 + 1;
    // many rows over many keys: the wide blocks' own launch
    p.wide = tiles > 4 && tiles * s64 * nkv >= kWideUnits * 8;
    const Shape pre = shape_of(tiles, p.wide ? 8 : 4);
    p.pre_kind = pre.kind;
    const int64_t steps = (prefix_len - 1) / step_keys(pre, hd) + 1, blocks = nkv * pre.blocks;
    p.units = blocks * steps;
    const int64_t want = std::min<int64_t>(p.wide ? kCus : kFusedPre, std::max(blocks, p.units / kPrefixSteps));
    const int64_t per = (p.units + want - 1) / want;
    p.pp = PagedPrefix{(uint32_t)p.units, (uint32_t)per, (uint32_t)steps, (uint32_t)pre.blocks, (uint32_t)(32 * pre.tiles)};
    p.pre_wgs = (p.units + per - 1) / per;
    p.pt.pre_parts = (int)((steps - 1) / per) + 2;
  }
  const Shape seq = shape_of(((int64_t)max_rows * G + 31) / 32, 4);
  const int64_t keys = max_len - prefix_len + max_rows;
  const int64_t wgs = batch * nkv * seq.blocks;
  const int64_t least = std::max<int64_t>(kMinSplit, kSplitRows * std::min<int64_t>(32 * seq.tiles, max_rows * G));
  int64_t ns = std::max(std::min<int64_t>(2 * kCus / wgs, keys / kMinSplit), std::min<int64_t>(kSeqWgs / wgs, keys / least));
  ns = std::max<int64_t>(1, ns);
  const int64_t kps = (((keys + ns - 1) / ns + 63) / 64) * 64;
  const int64_t nsplit = (keys + kps - 1) / kps;
  p.items = wgs * nsplit;
  const bool direct = prefix_len == 0 || (p.wide && p.pt.pre_parts <= 3);
  p.sq = PagedSeqs{(uint32_t)p.items, (uint32_t)kps, (uint32_t)seq.blocks, (uint32_t)(32 * seq.tiles), (int)nsplit, seq.kind,
                   direct};
  p.join = nsplit > 1 || !direct;
  const int64_t parts = p.pt.pre_parts + (p.join ? nsplit : 0);
  p.o_bytes = parts * nkv * tiles * 32 * hd * 4;
  p.ml_bytes = parts * nkv * tiles * 32 * 8;
  return p;
}

template <int DT, int HD, bool MOD>
int launch_all(const Plan& p, const PagedAttn& a, hipStream_t st) {
  if (p.wide) {
    paged_prefix_kernel<DT, HD, MOD><<<(unsigned)p.pre_wgs, 512, 0, st>>>(a, p.pp, p.pt);
    PE_CHECK_LAUNCH();
  }
  const uint32_t n_pre = p.wide ? 0 : (uint32_t)p.pre_wgs;
  paged_attn_kernel<DT, HD, MOD><<<n_pre + (unsigned)p.items, 256, 0, st>>>(a, p.pp, p.pt, p.sq, n_pre, p.pre_kind);
  PE_CHECK_LAUNCH();
  if (p.join) {
    const int64_t tiles = ((int64_t)a.max_rows * (a.nh / a.nkv) + 31) / 32;
    paged_join_kernel<DT, HD><<<dim3((unsigned)(tiles * (HD / 32)), a.nkv, a.batch), 256, 0, st>>>(a, p.pp, p.pt, p.sq);
    PE_CHECK_LAUNCH();
  }
  return PE_OK;
}

}  // namespace

int64_t pe_internal_paged_mfma_bytes(int64_t M, int batch, int nh, int nkv, int hd, int max_rows, int64_t max_len,
                                     int64_t prefix_len) {
  const Plan p = make_plan(M, batch, nh, nkv, hd, max_rows, max_len, prefix_len);
  return p.o_bytes + p.ml_bytes;
}

int pe_internal_paged_mfma(const PagedAttn& a, int dtype, void* workspace, int64_t workspace_bytes, hipStream_t st) {
  Plan p = make_plan(a.M, a.batch, a.nh, a.nkv, a.hd, a.max_rows, a.max_len, a.prefix_len);
  if (p.o_bytes > 0 && (!workspace || workspace_bytes < p.o_bytes + p.ml_bytes)) return PE_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 15) return PE_ERR_ARG;
  // rows and work units are counted in 32 bits
  if (a.M * a.nh >= (int64_t(1) << 31) || p.units >= (int64_t(1) << 31) ||
      p.items >= (int64_t(1) << 30) || a.nkv > 65535)
    return PE_ERR_ARG;
  p.pt.o = (float*)workspace;
  p.pt.ml = (float*)((char*)workspace + p.o_bytes);
  const bool mod = a.softcap > 0.f || a.slopes || a.window > 0;
#define PE_GO(DT, HD) return mod ? launch_all<DT, HD, true>(p, a, st) : launch_all<DT, HD, false>(p, a, st)
  if (dtype == PE_DTYPE_BF16) {
    if (a.hd == 128) PE_GO(PE_DTYPE_BF16, 128);
    PE_GO(PE_DTYPE_BF16, 64);
  }
  if (a.hd == 128) PE_GO(PE_DTYPE_F16, 128);
  PE_GO(PE_DTYPE_F16, 64);
#undef PE_GO
}
