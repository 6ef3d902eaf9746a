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
#include <type_traits>

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

// A row's two lanes (l and l ^ 32) joined: both get the larger value, or the sum.
__device__ __forceinline__ float max_halves(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_halves(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// s_waitcnt with vmcnt = N, the other counters at their maxima
template <int N>
__device__ __forceinline__ void wait_vm() {
  __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));
}

typedef short s4v_t __attribute__((__vector_size__(4 * sizeof(short))));
typedef __attribute__((address_space(3))) s4v_t lds_s4v_t;

// Loads of 16 keys of one KV head (one page holds them: page sizes are
// multiples of 16) straight into LDS, their 16-byte chunks swizzled by row.
template <int HD>
struct PageLoads {
  static constexpr int kLanes = HD / 8;             // lanes on a row
  static constexpr int kN = 16 * HD * 2 / 1024;     // load instructions
  const uint8_t *k, *v;                             // the head's first row in page 0
  uint32_t page_bytes, pages, mask;
  uint32_t off[kN];                                 // the lane's byte offsets among the 16 rows

  __device__ __forceinline__ PageLoads(const PagedAttn& a, int kvh, int lane) {
    const uint32_t head = (uint32_t)(HD * 2) << a.ps_log2;  // bytes of a head's rows of a page
    page_bytes = head * (uint32_t)a.nkv;
    pages = (uint32_t)a.num_pages;
    mask = (1u << a.ps_log2) - 1;
    k = (const uint8_t*)a.k_pool + (uint64_t)head * (uint32_t)kvh;
    v = (const uint8_t*)a.v_pool + (uint64_t)head * (uint32_t)kvh;
#pragma unroll
    for (int i = 0; i < kN; ++i) off[i] = (uint32_t)((i * (64 / kLanes) + lane / kLanes) * (HD * 2)) + chunk(lane, i);
  }
  __device__ __forceinline__ static uint32_t chunk(int lane, int i) {
    return (uint32_t)(((lane % kLanes) ^ swizzle<HD>(i * (64 / kLanes) + lane / kLanes)) << 4);
  }
  // keys key .. key + 15 (those outside [lo, hi) as the nearest inside) to LDS at dst
  __device__ __forceinline__ void issue(const uint8_t* base, int page, int key, int lo, int hi, uint32_t dst, int lane,
                                        bool& bad) const {
    const bool ok = (uint32_t)page < pages;
    bad = bad || !ok;
    const uint8_t* src = base + (uint64_t)(ok ? (uint32_t)page : 0u) * page_bytes + ((uint32_t)key & mask) * (HD * 2);
    if (key >= lo && key + 16 <= hi) {
#pragma unroll
      for (int i = 0; i < kN; ++i) lds_dma16(src, off[i], dst + i * 1024);
    } else {
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int r = min(max(i * (64 / kLanes) + lane / kLanes, lo - key), hi - 1 - key);
        lds_dma16(src, (uint32_t)(r * (HD * 2)) + chunk(lane, i), dst + i * 1024);
      }
    }
  }
};

// The keys of an item: `pre_steps` steps of the prefix's `pre` keys (none: 0),
// then the steps of a sequence's own keys [0, hi), P of them cached and new rows
// after those. Keys are counted in 32 bits: a sequence is shorter than 2^30.
struct Keys {
  const int32_t* pre_table;
  const int32_t* table;
  int pre_steps, pre;
  int P, hi;
  int base;      // position of key 0 of the sequence's own
  int lo;        // first position that a row of the workgroup sees (0 without a window)
  int new_rows;
  int last;      // last own key that a row of the wave's tile sees
};

// What a lane's row needs besides its Q.
struct RowInfo {
  int node;         // causal: its token's index among the sequence's new rows
  int pos;          // its position (MOD)
  float slope2;     // slope * log2 e (MOD)
  int lo, tile_lo;  // first position its window holds; the largest of the tile's (MOD)
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

// The steps [s0, s1) of the keys for the workgroup's row tiles: O^T, m, l of the
// wave's tile. Keys before k.lo and past a list's end are masked (their loads go
// to the nearest key of the list that is read, so that no page outside it is
// touched), steps past k.last skipped. npos (LDS): positions of the new rows of
// a tree (MOD, where distances count).
template <int DT, typename C, bool MOD>
__device__ __forceinline__ void attend(const PagedAttn& a, uint8_t* smem, const Keys& k, int kvh, int s0, int s1,
                                       bool live, const RowInfo& ri, const u32x4_t (&qf)[C::HD / 16], const int* npos,
                                       bool& bad, f32x16_t (&o)[C::OB], float& m, float& l) {
  constexpr int HD = C::HD, SB = C::SB, OB = C::OB;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int ln = lane & 31, g = lane >> 5, hb = (wave % C::DS) * OB;
  const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;
  typedef const __attribute__((address_space(4))) int32_t* const_i32;  // read through the scalar cache
  const const_i32 tab_pre = (const_i32)(uintptr_t)uniform_ptr((const uint16_t*)k.pre_table);
  const const_i32 tab_own = (const_i32)(uintptr_t)uniform_ptr((const uint16_t*)k.table);
  const int psl = a.ps_log2;
  const int lo_pre = min(k.lo, max(k.pre - 1, 0)), lo_own = min(max(k.lo - k.base, 0), max(k.hi - 1, 0));
  const PageLoads<HD> ld(a, kvh, lane);
  // this wave's pieces (16 keys of K or V) of a step: the keys and their page, asked for a step ahead
  int page[C::kChunks], key[C::kChunks];
  auto ask = [&](int step) {
    const bool pre = step < k.pre_steps;
    const const_i32 tab = pre ? tab_pre : tab_own;
    const int at = (pre ? step : step - k.pre_steps) * C::SK;
    const int first = (pre ? lo_pre : lo_own) & ~15, last = ((pre ? k.pre : k.hi) - 1) & ~15;
#pragma unroll
    for (int c = 0; c < C::kChunks; ++c) {
      key[c] = max(first, min(at + 16 * ((wave * C::kChunks + c) % (C::SK / 16)), last));
      page[c] = tab[key[c] >> psl];
    }
  };
  auto issue = [&](int step) {
    const bool pre = step < k.pre_steps;
    const uint32_t buf = lds_base + (step % C::ST) * C::kStep;
#pragma unroll
    for (int c = 0; c < C::kChunks; ++c) {
      const int piece = wave * C::kChunks + c;
      const bool is_v = piece >= C::SK / 16;
      ld.issue(is_v ? ld.v : ld.k, page[c], key[c], pre ? lo_pre : lo_own, pre ? k.pre : k.hi,
               buf + (is_v ? C::kHalf : 0) + (piece % (C::SK / 16)) * 16 * HD * 2, lane, bad);
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

  // the lane's LDS offsets: K row ln of a 32-key block, and V's transposed reads
  const int qg = lane >> 4, jl = lane & 15, vrow = 4 * (qg >> 1) + (jl >> 2), vcol = 16 * (qg & 1) + 4 * (jl & 3);
  // (the chunk's upper bits, 2 j of K and 4 h of V, meet only zeros of the rest: one exclusive or each)
  const uint32_t k_at = lds_at<HD>(ln, g);
  const uint32_t v_at[2] = {(lds_at<HD>(vrow, vcol >> 3) ^ (hb << 6)) + (vcol & 7) * 2,
                            (lds_at<HD>(vrow + 8, vcol >> 3) ^ (hb << 6)) + (vcol & 7) * 2};

  if (s0 < s1) ask(s0);
  __syncthreads();  // the buffers' last readers are done
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
    const bool pre = s < k.pre_steps;
    const int kb0 = (pre ? s : s - k.pre_steps) * C::SK, kpos = kb0 + (pre ? 0 : k.base);  // key 0 of the step
    if (!live || (!pre && kb0 > k.last)) continue;  // wave-uniform: the tile sees no key of this step
    const uint32_t stage = (s % C::ST) * C::kStep;
    const uint32_t ks = stage + k_at, vs[2] = {stage + v_at[0], stage + v_at[1]};
    // products on two chains of accumulators at least (a chain alone waits for each product)
    constexpr int kChains = SB > 1 ? SB : 2;
    f32x16_t sc[kChains];
    // Fragments in groups of LDS reads, kAhead groups ahead of the products that
    // use them: kS groups of four products of S, then 2 SB groups (16 keys each)
    // of V, whose first kAhead are read before the softmax. (One group ahead
    // where other scores leave 64 keys of 128 dims no registers.)
    constexpr int kS = SB * HD / 64, kAll = kS + 2 * SB, kAhead = MOD && HD == 128 && SB == 2 ? 1 : 2, kF = kAhead + 1;
    u32x4_t f[kF][4];
    auto read = [&](int gr) {
      if (gr < kS) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = 4 * gr + i;  // product SB j + sb
          f[gr % kF][i] = *(const u32x4_t*)(smem + (ks ^ ((at / SB) << 5)) + (at % SB) * 32 * HD * 2);
        }
      } else if (gr < kAll) {
#pragma unroll
        for (int h = 0; h < OB; ++h) {
          const uint8_t* vq = smem + C::kHalf + (gr - kS) * 16 * HD * 2;
          const uint2 x = __builtin_bit_cast(
              uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4v_t*)(vq + (vs[0] ^ (h << 6)))));
          const uint2 y = __builtin_bit_cast(
              uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4v_t*)(vq + (vs[1] ^ (h << 6)))));
          f[gr % kF][h] = u32x4_t{x.x, x.y, y.x, y.y};
        }
      }
    };
#pragma unroll
    for (int gr = 0; gr < kAhead; ++gr) read(gr);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int gr = 0; gr < kS; ++gr) {
      read(gr + kAhead);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = 4 * gr + i;
        sc[at % kChains] =
            mfma32<DT>(f[gr % kF][i], qf[at / SB], at < kChains ? f32x16_t{} : sc[at % kChains]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (SB == 1) {
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[0][i] += sc[1][i];
    }
    // sc[sb][i] is key kb0 + 32 sb + 8 (i / 4) + 4 g + i % 4 of the lane's row
    const bool node_step = !pre && kb0 + 32 * SB > k.P;
    if constexpr (MOD) {
      const bool capped = cap_in != 0.f, sloped = a.slopes != nullptr;
      if (capped) {
        // cap tanh(s / cap) = cap (1 - 2 / (1 + e^(2 s / cap))): both ends exact
#pragma unroll
        for (int sb = 0; sb < SB; ++sb)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float e = __builtin_amdgcn_exp2f(sc[sb][i] * cap_in);
            sc[sb][i] = fmaf(-2.f * cap_out, __builtin_amdgcn_rcpf(1.f + e), cap_out);
          }
      }
      const int d0 = ri.pos - kpos - 4 * g;  // distance of key kb0 + 4 g
      const float mul = capped ? 1.f : scale2;
      if (node_step && npos) {  // a tree's new rows lie where their positions say
#pragma unroll
        for (int sb = 0; sb < SB; ++sb)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int off = 32 * sb + 8 * (i >> 2) + (i & 3);
            const int u = kb0 - k.P + off + 4 * g;
            const int np = npos[max(0, min(u, k.new_rows - 1))];
            const int dist = u < 0 ? d0 - off : ri.pos - np;
            sc[sb][i] = fmaf(sc[sb][i], mul, -ri.slope2 * (float)dist);
            if (a.window > 0) sc[sb][i] = dist < a.window ? sc[sb][i] : -INFINITY;
            if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // few positions in registers at a time
          }
      } else if (sloped) {
        const float c0 = -ri.slope2 * (float)d0;
#pragma unroll
        for (int sb = 0; sb < SB; ++sb)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            sc[sb][i] = fmaf(sc[sb][i], mul, fmaf(ri.slope2, (float)(32 * sb + 8 * (i >> 2) + (i & 3)), c0));
      } else if (!capped) {
#pragma unroll
        for (int sb = 0; sb < SB; ++sb)
#pragma unroll
          for (int i = 0; i < 16; ++i) sc[sb][i] *= scale2;
      }
    }
    const int hi = pre ? k.pre : k.hi;
    bool edge = node_step || kb0 + 32 * SB > hi;
    if constexpr (MOD) edge = edge || kpos < ri.tile_lo;
    if (edge) {
      uint64_t win = ~0ull;
      if (node_step)
        win = tree ? node_window(kb0, k.P, ri.nb0, ri.nb1, ri.nb2, ri.nb3) : below(k.P + ri.node + 1 - kb0);
      win &= below(hi - kb0);
      if constexpr (MOD) win &= ~below(ri.lo - kpos);
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
    bmax = max_halves(bmax);
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
    l = l * alpha + psum;  // of the lane's half of the keys: the halves are joined at the end
    if (__builtin_amdgcn_ballot_w64(mnew != m) != 0ull) {
#pragma unroll
      for (int h = 0; h < OB; ++h)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[h][i] *= alpha;
    }
    m = mnew;
    // O^T += V^T P^T over the 16-key quarters of the step
#pragma unroll
    for (int c = 0; c < 2 * SB; ++c) {
      const int q = c & 1;
      const u32x4_t bp = {pb[c >> 1][4 * q], pb[c >> 1][4 * q + 1], pb[c >> 1][4 * q + 2], pb[c >> 1][4 * q + 3]};
      read(kS + c + kAhead);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int h = 0; h < OB; ++h) o[h] = mfma32<DT>(f[(kS + c) % kF][h], bp, o[h]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  l = sum_halves(l);
}

// ---------------------------------------------------------------------------
// The prefix's wide blocks: eight waves, two to a SIMD, in opposite phases
// ---------------------------------------------------------------------------
// A step of a wave is 32 matrix instructions (1024 cycles of the matrix core)
// and about as many cycles of exponentials and other vector work. In step with
// each other, the two waves of a SIMD would compete for the one and then for the
// other: the same kernel with one barrier a step ran at 37% of the matrix
// core's rate. So waves 0 - 3 and 4 - 7 work in turns. Phase X of a step: O^T +=
// V^T P^T of the step before, then S^T = K Q^T; phase Y: softmax of S, O's
// rescaling. A barrier ends each phase; group 0 is in X when group 1 is in Y.
//
// In phases counted from the start of the item, group e does X of step i in
// phase 2 i + e and Y in the next. Group 0 loads the steps' K, group 1 their V,
// each in its phases Y (X is the longer one): in Y of step i what step i + 2
// needs, into the ring's buffer of step i - 2. K(i - 2) was last read in phase
// 2 i - 3 and V(i - 2) in 2 i - 1, both before those phases (2 i + 1 and 2 i + 2).
// K(i + 1) has to be there at the end of phase 2 i + 1 and V(i) as well: the
// loads issued after those are one step's, so two steps are in flight.
//
// LDS reads run two groups of four matrix instructions ahead of their use.
// 14b, 64 trees of 26 nodes over 8192 shared keys (279 GFLOP of products with the
// prefix): 249 us, 1.12 PFLOP/s, where a large matrix product of the library
// reaches 1.21 on the same card; one barrier a step took 19 us more on the whole
// call, phases without s_setprio 4 us more, without the slack below 9 us.
// A row's running maximum follows its block's only when it is passed by more
// than 2^8 (kSlack): O and l are sums of the same 2^(s - m), whichever m, and the
// weights, at most 2^8, lose nothing in fp32 nor when rounded (fp16's largest
// value is 2^16); O's 64 products a step are mostly saved.
constexpr float kSlack = 8.f;

template <int DT, typename C, bool MOD>
__device__ __forceinline__ void attend_wide(const PagedAttn& a, uint8_t* smem, const int32_t* table, int n, int lo,
                                            int kvh, int s0, int s1, bool live, const RowInfo& ri,
                                            const u32x4_t (&qf)[C::HD / 16], bool& bad, f32x16_t (&o)[C::HD / 32],
                                            float& m, float& l) {
  constexpr int HD = C::HD, NJ = HD / 16, NH = HD / 32;
  static_assert(C::W == 8 && C::SB == 2 && C::ST == 4 && C::kChunks == 1, "the schedule above");
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int ln = lane & 31, g = lane >> 5, grp = wave >> 2;
  const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;
  typedef const __attribute__((address_space(4))) int32_t* const_i32;
  const const_i32 tab = (const_i32)(uintptr_t)uniform_ptr((const uint16_t*)table);
  const int psl = a.ps_log2, lo_k = min(lo, n - 1);
  const PageLoads<HD> ld(a, kvh, lane);
  const int ch = wave & 3;  // this wave's 16 keys of K (waves 0 - 3) or V of a step
  int page = 0, key = 0;
  auto ask = [&](int step) {
    key = max(lo_k & ~15, min(step * 64 + 16 * ch, (n - 1) & ~15));
    page = tab[key >> psl];
  };
  auto issue = [&](int step) {
    ld.issue(grp ? ld.v : ld.k, page, key, lo_k, n, lds_base + (step & 3) * C::kStep + grp * C::kHalf + ch * 16 * HD * 2,
             lane, bad);
  };

#pragma unroll
  for (int h = 0; h < NH; ++h)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[h][i] = 0.f;
  m = kPagedInitMax;
  l = 0.f;
  const float scale2 = a.scale * kLog2e;
  const float cap_in = MOD && a.softcap > 0.f ? 2.f * scale2 / a.softcap : 0.f, cap_out = a.softcap * kLog2e;
  f32x16_t sc[2];
  uint32_t pb[2][8];
#pragma unroll
  for (int sb = 0; sb < 2; ++sb) {
#pragma unroll
    for (int i = 0; i < 8; ++i) pb[sb][i] = 0u;
#pragma unroll
    for (int i = 0; i < 16; ++i) sc[sb][i] = 0.f;
  }
  // the lane's LDS offsets: K row ln of a 32-key half, and V's transposed reads
  const int qg = lane >> 4, jl = lane & 15, vrow = 4 * (qg >> 1) + (jl >> 2), vcol = 16 * (qg & 1) + 4 * (jl & 3);
  uint32_t k_at[NJ], v_at[2][NH];
#pragma unroll
  for (int j = 0; j < NJ; ++j) k_at[j] = lds_at<HD>(ln, 2 * j + g);
#pragma unroll
  for (int h = 0; h < NH; ++h) {
    v_at[0][h] = lds_at<HD>(vrow, (32 * h + vcol) >> 3) + (vcol & 7) * 2;
    v_at[1][h] = lds_at<HD>(vrow + 8, (32 * h + vcol) >> 3) + (vcol & 7) * 2;
  }

  // Phase X: `pv`: step s - 1's P V, `qk`: step s's scores. Groups of LDS reads
  // 0 .. 3: V of a 16-key quarter (4 products of hd 128, 2 of 64), then K, as
  // many products a group.
  auto phase_x = [&](int s, bool pv, bool qk) {
    const uint8_t* vbp = smem + ((s - 1) & 3) * C::kStep + C::kHalf;
    const uint8_t* kbp = smem + (s & 3) * C::kStep;
    constexpr int kG = 4 + 4;  // groups
    u32x4_t f[3][NH];
    auto read = [&](int gr) {
      if (gr < 4) {
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                        (lds_s4v_t*)(vbp + v_at[0][h] + gr * 16 * HD * 2)));
          const uint2 y = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                        (lds_s4v_t*)(vbp + v_at[1][h] + gr * 16 * HD * 2)));
          f[gr % 3][h] = u32x4_t{x.x, x.y, y.x, y.y};
        }
      } else if (gr < kG) {
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          const int at = (gr - 4) * NH + h;  // product 2 j + sb
          f[gr % 3][h] = *(const u32x4_t*)(kbp + k_at[at >> 1] + (at & 1) * 32 * HD * 2);
        }
      }
    };
    auto mul = [&](int gr) {
      if (gr < 4) {
        const int sb = gr >> 1, q = gr & 1;
        const u32x4_t bp = {pb[sb][4 * q], pb[sb][4 * q + 1], pb[sb][4 * q + 2], pb[sb][4 * q + 3]};
#pragma unroll
        for (int h = 0; h < NH; ++h) o[h] = mfma32<DT>(f[gr % 3][h], bp, o[h]);
      } else {
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          const int at = (gr - 4) * NH + h;
          if (at < 2)
            sc[at] = mfma32<DT>(f[gr % 3][h], qf[0], f32x16_t{});
          else
            sc[at & 1] = mfma32<DT>(f[gr % 3][h], qf[at >> 1], sc[at & 1]);
        }
      }
    };
    static_assert(4 * NH == 2 * NJ, "four groups of K");
    const int g0 = pv ? 0 : 4, g1 = qk ? kG : 4;
    // three bodies, so that each is straight code
    auto run = [&](auto from, auto to) {
      constexpr int F = decltype(from)::value, T = decltype(to)::value;
      read(F);
      if constexpr (F + 1 < T) read(F + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int gr = F; gr < T; ++gr) {
        if (gr + 2 < T) read(gr + 2);
        __builtin_amdgcn_sched_barrier(0);
        mul(gr);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    if (g0 == 0 && g1 == kG) run(std::integral_constant<int, 0>{}, std::integral_constant<int, kG>{});
    else if (g0 == 0) run(std::integral_constant<int, 0>{}, std::integral_constant<int, 4>{});
    else run(std::integral_constant<int, 4>{}, std::integral_constant<int, kG>{});
  };

  auto phase_y = [&](int s) {
    const int kb0 = s * 64;
    if constexpr (MOD) {
      const bool capped = cap_in != 0.f;
      if (capped) {
#pragma unroll
        for (int sb = 0; sb < 2; ++sb)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float e = __builtin_amdgcn_exp2f(sc[sb][i] * cap_in);
            sc[sb][i] = fmaf(-2.f * cap_out, __builtin_amdgcn_rcpf(1.f + e), cap_out);
          }
      }
      const float mul = capped ? 1.f : scale2;
      if (a.slopes) {
        const float c0 = -ri.slope2 * (float)(ri.pos - kb0 - 4 * g);
#pragma unroll
        for (int sb = 0; sb < 2; ++sb)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            sc[sb][i] = fmaf(sc[sb][i], mul, fmaf(ri.slope2, (float)(32 * sb + 8 * (i >> 2) + (i & 3)), c0));
      } else if (!capped) {
#pragma unroll
        for (int sb = 0; sb < 2; ++sb)
#pragma unroll
          for (int i = 0; i < 16; ++i) sc[sb][i] *= scale2;
      }
    }
    bool edge = kb0 + 64 > n;
    if constexpr (MOD) edge = edge || kb0 < ri.tile_lo;
    if (edge) {
      uint64_t win = below(n - kb0);
      if constexpr (MOD) win &= ~below(ri.lo - kb0);
      win >>= 4 * g;
#pragma unroll
      for (int sb = 0; sb < 2; ++sb)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          sc[sb][i] = ((win >> (32 * sb + 8 * (i >> 2) + (i & 3))) & 1ull) ? sc[sb][i] : -INFINITY;
    }
    float bmax = -INFINITY;
#pragma unroll
    for (int sb = 0; sb < 2; ++sb)
#pragma unroll
      for (int i = 0; i < 16; ++i) bmax = fmaxf(bmax, sc[sb][i]);
    bmax = max_halves(bmax);
    if constexpr (!MOD) bmax *= scale2;
    if (__builtin_amdgcn_ballot_w64(bmax > m + kSlack) != 0ull) {
      const float mnew = fmaxf(m, bmax);
      const float alpha = __builtin_amdgcn_exp2f(m - mnew);
      l *= alpha;
      m = mnew;
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[h][i] *= alpha;
    }
    float psum[2] = {0.f, 0.f};
#pragma unroll
    for (int sb = 0; sb < 2; ++sb)
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float p0 = __builtin_amdgcn_exp2f(MOD ? sc[sb][i] - m : fmaf(sc[sb][i], scale2, -m));
        const float p1 = __builtin_amdgcn_exp2f(MOD ? sc[sb][i + 1] - m : fmaf(sc[sb][i + 1], scale2, -m));
        psum[0] += p0;
        psum[1] += p1;
        pb[sb][i >> 1] = pack2_16<DT>(p0, p1);
      }
    l += psum[0] + psum[1];  // of the lane's half of the keys: the halves are joined at the end
  };

  // the end of a phase; `landed`: this wave's loads but the last step's have to be there
  const int steps = s1 - s0;
  auto leave = [&](bool landed, bool later) {
    if (landed) {
      if (later) wait_vm<C::kLoads>();
      else wait_vm<0>();
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  if (steps <= 0) return;
  ask(s0);
  __syncthreads();  // the buffers' last readers are done
  issue(s0);
  if (s0 + 1 < s1) {
    ask(s0 + 1);
    issue(s0 + 1);
    if (s0 + 2 < s1) ask(s0 + 2);
  }
  __builtin_amdgcn_s_waitcnt(0);  // Q has landed: no later wait of the compiler's covers the ring's loads
  leave(false, false);
  if (grp) leave(false, false);
  for (int i = 0; i < steps; ++i) {
    if (live) {
      __builtin_amdgcn_s_setprio(1);
      phase_x(s0 + i, i > 0, true);
      __builtin_amdgcn_s_setprio(0);
    }
    leave(grp, i + 1 < steps);  // group 1: V of step i
    const int st = s0 + i + 2;
    if (st < s1) {
      issue(st);
      if (st + 1 < s1) ask(st + 1);
    }
    if (live) phase_y(s0 + i);
    leave(!grp, st < s1);  // group 0: K of step i + 1
  }
  if (live) phase_x(s1, true, false);
  if (!grp) leave(false, false);  // the other group's last phase but one
  l = sum_halves(l);
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

// The first position that the lane's row sees (ri.lo, at most `end`), the last
// of the tile's (ri.tile_lo) and the first of the workgroup's (returned).
template <int W>
__device__ __forceinline__ int window_lo(const PagedAttn& a, RowInfo& ri, int end, bool live, int* s_lo) {
  ri.lo = ri.tile_lo = 0;
  if (a.window == 0) return 0;
  ri.lo = (int)min(max((int64_t)ri.pos - a.window + 1, (int64_t)0), (int64_t)end);
  int lo = live ? ri.lo : end, hi = ri.lo;
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) {
    lo = min(lo, __shfl_xor(lo, d, 64));
    hi = max(hi, __shfl_xor(hi, d, 64));
  }
  ri.tile_lo = __builtin_amdgcn_readfirstlane(hi);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s_lo[threadIdx.x >> 6] = lo;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < W; ++i) lo = min(lo, s_lo[i]);
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
  // its pieces of blocks from the last to the first: a piece that ends its share
  // starts at key 0 and one that starts it ends at the last key, so workgroups
  // walk the keys at the same time, from one copy in their XCD's L2
  const uint32_t u0 = w * pp.per;
  bool bad = false;
  for (uint32_t u = min(pp.total, u0 + pp.per); u > u0;) {
    const uint32_t x = (u - 1) / pp.steps, first_u = max(u0, x * pp.steps);
    const int s0 = (int)(first_u - x * pp.steps);
    const uint32_t past = u - x * pp.steps;  // a block's last steps may be beyond its keys
    u = first_u;
    const int s1 = min((int)past, ((int)a.prefix_len - 1) / C::SK + 1);
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
    Keys k{a.prefix_table, a.prefix_table, 1 << 30, S0, 0, 0, S0, 0, 0, 0};
    int first = s0;
    if constexpr (MOD) {
      ri.pos = a.positions ? (int)a.positions[tok] : 0;
      ri.slope2 = a.slopes ? a.slopes[hq] * kLog2e : 0.f;
      k.lo = window_lo<C::W>(a, ri, S0, live, s_lo);
      if (k.lo > 0) first = k.lo >= S0 ? s1 : max(s0, k.lo / C::SK);  // steps behind every row's window
    }
    f32x16_t o[C::OB];
    float m, l;
    if constexpr (C::W == 8)
      attend_wide<DT, C, MOD>(a, smem, a.prefix_table, S0, k.lo, kvh, first, s1, live, ri, qf, bad, o, m, l);
    else
      attend<DT, C, MOD>(a, smem, k, kvh, first, max(first, s1), live, ri, qf, nullptr, bad, o, m, l);
    if (live)
      store_part<HD, C::OB>(parts, a.nkv, (int)(w - prefix_first_wg(pp, x)), kvh, row0 + ln, g, hb, o, m, l);
  }
  if (bad && lane == 0) atomicOr(a.status, PE_ERR_INDEX);
}

// ---------------------------------------------------------------------------
// The sequences' own keys: item = (key split, sequence, KV head, block of row
// tiles)
// ---------------------------------------------------------------------------
// The launch's shares of it, in key steps of `step` keys: the prefix's
// `pre_steps` first where the items take it themselves (a prefix that is short
// beside a sequence's rows: its parts would cost more than reading it again),
// then the sequence's own. `direct`: a sequence of one split joins the
// prefix's parts of its rows to its own (an earlier launch wrote them, and they
// are few) and writes the output; otherwise its result is a part as well and
// paged_join_kernel writes the output.
// The most parts of the prefix that a sequence's workgroup joins itself (14b,
// trees of 26 nodes: 64 over 8192 keys, 3 parts, 326, and 345 with the join's
// launch; 16 over 8192, 6 parts, 94 / 104; 16 over 16384, 8 parts, 165 / 170).
constexpr int kDirectParts = 8;
struct PagedSeqs {
  uint32_t items, nblk, block_rows;
  int split_steps, pre_steps, step, nsplit, kind, direct;
};
__device__ __forceinline__ int splits_of(const PagedSeqs& sq, const PagedSeq& s) {
  return (sq.pre_steps + ((int)s.priv + s.rows - 1) / sq.step) / sq.split_steps + 1;
}

template <int DT, int OB>
__device__ __forceinline__ void write_out(const PagedAttn& a, int64_t tok, int col, const f32x16_t (&o)[OB],
                                          float l) {
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int h = 0; h < OB; ++h)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float v[4] = {o[h][4 * c] * inv, o[h][4 * c + 1] * inv, o[h][4 * c + 2] * inv, o[h][4 * c + 3] * inv};
      paged_out4<DT>(a, tok, col + 32 * h + 8 * c, v);
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
  const int my_splits = splits_of(sq, s);
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
  const int S0 = (int)a.prefix_len;
  Keys k{a.prefix_table, a.block_table + b * a.ld_table, sq.pre_steps, sq.pre_steps ? S0 : 0, P,
         tree ? S : P + t_blk + 1, S0, 0, T, tree ? S - 1 : P + t_tile};
  const int s_end = sq.pre_steps + (k.hi + C::SK - 1) / C::SK;
  int s0 = split * sq.split_steps;
  const int s1 = min(s_end, s0 + sq.split_steps);
  if constexpr (MOD) {
    ri.pos = a.positions ? (int)a.positions[tok] : 0;
    ri.slope2 = a.slopes ? a.slopes[hq] * kLog2e : 0.f;
    if (a.positions && tree)
      for (int u = tid; u < T; u += 64 * C::W) s_npos[u] = (int)a.positions[s.row0 + u];
    k.lo = window_lo<C::W>(a, ri, S0 + (tree ? P : k.hi - 1), live, s_lo);
    if (k.lo >= S0) s0 = max(s0, sq.pre_steps + (k.lo - S0) / C::SK);  // steps behind every row's window
    else if (sq.pre_steps) s0 = max(s0, k.lo / C::SK);
  }
  bool bad = false;
  f32x16_t o[C::OB];
  float m, l;
  attend<DT, C, MOD>(a, smem, k, kvh, s0, max(s0, s1), live, ri, qf, MOD && a.positions && tree ? s_npos : nullptr, bad, o,
                     m, l);
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
  write_out<DT, C::OB>(a, tok, hq * HD + 32 * hb + 4 * g, o, l);
}

// ---------------------------------------------------------------------------
// Kernels
// ---------------------------------------------------------------------------
// Many rows over a long prefix: eight tiles (256 rows) on every K / V byte, one
// workgroup per CU.
template <int HD> using Wide = Cfg<HD, 8, 1, 2, 4>;
// Four waves, 64 KiB of LDS, two workgroups per CU. (Steps of 32 keys instead of
// 64 for 128-dim heads: level for plain scores, 12% slower for capped ones.)
template <int HD> using Four = Cfg<HD, 4, 1, 2, HD == 128 ? 2 : 4>;
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
// splits in key order. Bound by latency (7 - 10 us at 10 - 60 MB of parts, the
// launch included), so kAhead parts are asked for at once; eight at once were
// level at best and cost registers.
template <int DT, int HD>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttn a, PagedPrefix pp, PagedParts parts, PagedSeqs sq) {
  const int b = blockIdx.z, kvh = blockIdx.y;
  const PagedSeq s = paged_seq(a, b);
  if (!s.ok) return;
  const int my_splits = splits_of(sq, s);
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
    float mx = m;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) mx = fmaxf(mx, ml[k].x);  // past the end: the last one again
    const float a0 = __builtin_amdgcn_exp2f(m - mx);
    m = mx;
    l *= a0;
#pragma unroll
    for (int d = 0; d < 4; ++d) o[d] *= a0;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const float a1 = i0 + k < n ? __builtin_amdgcn_exp2f(ml[k].x - mx) : 0.f;
      l = fmaf(a1, ml[k].y, l);
#pragma unroll
      for (int d = 0; d < 4; ++d) o[d] = fmaf(a1, v[k][d], o[d]);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const float v[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
  const uint32_t tok = grow / G;
  const int hq = (int)(kvh * G + (grow - tok * G));
  paged_out4<DT>(a, tok, hq * HD + 4 * piece, v);
}

// ------------------------------------------------------------------ plans
// The rules below choose among forms that compute the same thing, by counts of
// rows, keys and workgroups. Both sides of each were measured (us a call, all
// launches; "14b": 40 query heads on 8 KV heads of 128 dims, "7b": 32 on 32).
constexpr int kCus = 256;
// A prefix of up to this many keys, or of as many as a sequence has rows, is
// read with each sequence's own keys: its parts would cost more than that.
// 7b, 12 sequences of up to 18 rows, 10 shared keys: 10.8, as a share of its own
// 15.8; 14b, 7 of 270 rows, 12 keys: 44.2 / 67.3; 59 of 6 rows, 23 keys: 35.2 /
// 45.7. Past the rule it loses: four times as many keys as rows, 14b, 43
// sequences, 279 keys: 73.6 folded / 68.5; up to 128 keys, 2 sequences, 93: 15.2 / 13.4.
constexpr int64_t kFoldKeys = 64;
// Wide blocks in a launch of their own from this many (32-row tile, 64-key step,
// KV head) units on: 14b, trees of 26 nodes, 64 over 8192 shared keys (266 240
// units): 326 with the wide launch, 449 without; 16 over 8192 (66 560): 94 / 185;
// 32 over 3000 (48 880): 101 / 107. Below, the shared launch, where the
// sequences' loads fill the prefix's waits: 32 over 1500 (24 960) 73.6 / 66.0; 7b,
// 16 over 3000 (19 552) 68.1 / 54.9, over 2048 (13 312) 71.7 / 63.5.
constexpr int64_t kWideUnits = 32768;
// Workgroups of the prefix in the shared launch, one of the two places of each
// CU. 7b, 16 trees over 2048 keys: 63.2; 128 of them 65.2, 384 69.6, 512 66.5;
// four chunks of 128 rows with slopes: 53.0, 57.4 (128), 63.5 (512).
constexpr int64_t kFusedPre = 256;
// The least steps of a prefix share. 27 sequences of one token: 16.4; 2 steps
// 21.1 (more parts to join); 8 steps lose on short prefixes, 26.2 / 19.3.
constexpr int64_t kPrefixSteps = 4;
// Workgroups that the splits of the sequences' keys are to reach: 1024 where a
// workgroup has more than 64 rows (14b, 8 capped sequences with a window: 62;
// 512: 81; 1536: 66), 2048 where it has fewer, whose parts are smaller (14b, 64
// one-token sequences: 52.3; 1024: 55.1; 4096: 57.7).
constexpr int64_t kSeqWgs = 1024, kSlimWgs = 2048;
// The least keys of a split, and the least per row of its block: 64 (one 14b
// sequence of 428 keys: 12.0; 128: 13.2) and 2 (the capped sequences above:
// 57.4; 8: 78.8; chunks with slopes 45.2 / 52.0).
constexpr int64_t kMinSplit = 64, kSplitRows = 2;
// Row tiles x KV heads x splits at most: bounds the parts of a batch that is
// mostly padding.
constexpr int64_t kSplitTiles = 10240;

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
// Keys of a step (the configurations above).
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
  const Shape seq = shape_of(((int64_t)max_rows * G + 31) / 32, 4);
  const int step = step_keys(seq, hd);
  const int64_t own_keys = max_len - prefix_len + max_rows;
  const bool fold = prefix_len <= std::max<int64_t>(kFoldKeys, max_rows * G);
  const int64_t pre_steps = fold ? (prefix_len + step - 1) / step : 0;
  if (!fold) {
    const int64_t s64 = (prefix_len - 1) / 64 + 1;
    // many rows over many keys: the wide blocks' own launch
    p.wide = tiles > 4 && tiles * s64 * nkv >= kWideUnits;
    const Shape pre = shape_of(tiles, p.wide ? 8 : 4);
    p.pre_kind = pre.kind;
    const int64_t steps = (prefix_len - 1) / step_keys(pre, hd) + 1, blocks = nkv * pre.blocks;
    if (p.wide) {
      p.units = blocks * steps;
      const int64_t per = (p.units + kCus - 1) / kCus;
      p.pp = PagedPrefix{(uint32_t)p.units, (uint32_t)per, (uint32_t)steps, (uint32_t)pre.blocks, (uint32_t)(32 * pre.tiles)};
      p.pt.pre_parts = (int)((steps - 1) / per) + 2;
    } else {
      // the sequences' steps of 64 keys per place, half of the longest on average: the
      // prefix's shares run beside them, and fewer parts are cheaper to join
      const int64_t beside = batch * nkv * seq.blocks * own_keys / (64 * 2 * 2 * kCus);
      const int64_t least = std::max<int64_t>(kPrefixSteps, beside * 64 / step_keys(pre, hd));
      const int64_t k = std::max<int64_t>(1, std::min<int64_t>(kFusedPre / blocks, steps / least));
      const int64_t per = (steps + k - 1) / k, parts = (steps + per - 1) / per;
      if (2 * blocks > kFusedPre && 4 * blocks * parts < 3 * kFusedPre) {
        // a share per block would leave over a quarter of the places empty: shares that cross
        // blocks (14b, 16 trees of 26 nodes over 2048 keys, 136 blocks: 46.1, 60.8 with a share
        // each; where whole shares fill the places they are as good or better, 61.3 / 65.6)
        const int64_t even = std::max(least, (blocks * steps + kFusedPre - 1) / kFusedPre);
        p.units = blocks * steps;
        p.pp = PagedPrefix{(uint32_t)p.units, (uint32_t)even, (uint32_t)steps, (uint32_t)pre.blocks,
                           (uint32_t)(32 * pre.tiles)};
        p.pt.pre_parts = (int)((steps - 1) / even) + 2;
      } else {
        p.units = blocks * per * parts;
        p.pp = PagedPrefix{(uint32_t)p.units, (uint32_t)per, (uint32_t)(per * parts), (uint32_t)pre.blocks,
                           (uint32_t)(32 * pre.tiles)};
        p.pt.pre_parts = (int)parts;
      }
    }
    p.pre_wgs = (p.units + p.pp.per - 1) / p.pp.per;
  }
  const int64_t steps = pre_steps + (own_keys - 1) / step + 1;
  const int64_t wgs = batch * nkv * seq.blocks;
  const int64_t blk_rows = std::min<int64_t>(32 * seq.tiles, (int64_t)max_rows * G);
  // splits fill the machine about twice (few rows: four times, their parts are
  // small), each no shorter than kMinSplit keys or kSplitRows keys a row; a batch
  // of many padding rows has its parts limited
  const int64_t ns = std::max<int64_t>(
      1, std::min({(blk_rows > 64 ? kSeqWgs : kSlimWgs) / wgs,
                   steps * step / std::max<int64_t>(kMinSplit, kSplitRows * blk_rows), kSplitTiles / (nkv * tiles)}));
  const int64_t split_steps = (steps + ns - 1) / ns, nsplit = (steps + split_steps - 1) / split_steps;
  p.items = wgs * nsplit;
  const bool direct = fold || (p.wide && p.pt.pre_parts <= kDirectParts);
  p.sq = PagedSeqs{(uint32_t)p.items, (uint32_t)seq.blocks, (uint32_t)(32 * seq.tiles), (int)split_steps, (int)pre_steps,
                   step, (int)nsplit, seq.kind, direct};
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

// Row tiles x KV heads x parts that no plan of up to M rows passes: the wide
// launch's parts, of at most 256 / (nkv blocks) + 2 per block of eight tiles, or
// the shared launch's, of which there are as many as workgroups (four tiles
// each), one, or up to three of fewer than 768 tiles; and the splits (make_plan's
// limit).
int64_t pe_internal_paged_mfma_reserve(int64_t M, int nh, int nkv, int hd) {
  const int64_t tiles = nkv * ((M * (nh / nkv) + 31) / 32);
  return (2 * tiles + 8 * kCus + std::max(tiles, kSplitTiles)) * (32 * hd * 4 + 32 * 8);
}

int pe_internal_paged_mfma(const PagedAttn& a, int dtype, void* workspace, int64_t workspace_bytes, hipStream_t st) {
  const bool mod = a.softcap > 0.f || a.slopes || a.window > 0;
  Plan p = make_plan(a.M, a.batch, a.nh, a.nkv, a.hd, a.max_rows, a.max_len, a.prefix_len);
  if (p.o_bytes > 0 && (!workspace || workspace_bytes < p.o_bytes + p.ml_bytes)) return PE_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 15) return PE_ERR_ARG;
  // rows and work units are counted in 32 bits
  if (a.M * a.nh >= (int64_t(1) << 31) || p.units >= (int64_t(1) << 31) ||
      p.items >= (int64_t(1) << 30) || a.nkv > 65535)
    return PE_ERR_ARG;
  p.pt.o = (float*)workspace;
  p.pt.ml = (float*)((char*)workspace + p.o_bytes);
#define PE_GO(DT, HD) return mod ? launch_all<DT, HD, true>(p, a, st) : launch_all<DT, HD, false>(p, a, st)
  if (dtype == PE_DTYPE_BF16) {
    if (a.hd == 128) PE_GO(PE_DTYPE_BF16, 128);
    PE_GO(PE_DTYPE_BF16, 64);
  }
  if (a.hd == 128) PE_GO(PE_DTYPE_F16, 128);
  PE_GO(PE_DTYPE_F16, 64);
#undef PE_GO
}
