// Local branch on a paged cache (page = chunk = 64 tokens), for the last T tokens of every sequence: one token of a decode
// step, a slice of a prompt, or T drafted tokens that form a tree.
//
//   o_t = sum_j softmax_j(scale q_t . k_j) v_j,   lse_t = log sum_j exp(scale q_t . k_j)
//
// over the slots j that token t sees.  With base = length - T and p = base + depth(t) (depth = t in a chain) these are the
// committed slots left(p) <= j < base, left(p) = p - window + 1, moved to its chunk's first token with `expand`, and the new
// tokens u that are t itself or its ancestors and sit at left(p) or later; with mask_lmk no token at a chunk's last position.
//
// A row is a (token, query head of the KV head's group) pair.  Two kernels, both with the rows as the columns of the matrix
// products S^T = K q^T and O^T += V^T P (a row's scores, maximum and sum stay in the lanes that hold its column):
//   paged_attn_rows   16 or 32 rows a workgroup, its wavefronts share the keys (bound by the memory system),
//   paged_attn_tiles  64, 128 or 256 rows a workgroup, 32 a wavefront, pages staged in LDS (bound by the matrix and vector units).
// A long range of keys is split over workgroups; paged_attn_join adds their shares up, in a fixed order.
// Scores, maxima, sums and outputs are fp32; probabilities are rounded to bf16 for the second product, their sum is taken
// before the rounding.  Each is off by up to 2^-8 of itself, of random sign, which adds as much to an output's error as its own
// rounding: 1.9e-3 to 2.4e-3 of the output's norm against 64 bits, 1.6e-3 where the output alone is rounded.  (Two products with a
// probability's leading and next bits would keep the latter, for half as many matrix instructions again.)
//
// Values at slots that a row does not see meet a probability of exactly 0, which an infinity or a NaN there would turn into a
// NaN.  Behind the last token, where a page holds what its last user left, and in place of a page that is not mapped values
// are read as zeros.  Elsewhere (a token before the window, a landmark, another branch's draft) a row whose result is no finite
// number is computed once more, token by token over the slots that it sees alone (paged_redo_row): the common call pays a
// comparison, a call all of whose rows take that way 12 times its time (one token) to 190 times (trees: 88 us become 17 ms).
#include <string.h>

#include "common.h"
#include "lds_dma.h"
#include "../../include/hils_amd.h"

#define PA_PAGE 64
#define PA_MAX_TREE 256                       // drafted tokens of a tree
#define PA_WORDS (PA_MAX_TREE / 32 + 3)       // mask words of a token: one of zeros before, two behind
typedef unsigned pa_u4 __attribute__((ext_vector_type(4)));
typedef short pa_s4 __attribute__((ext_vector_type(4)));
typedef short pa_s8 __attribute__((ext_vector_type(8)));

struct PagedDims {
  int B, T, HQ, H, G, window, expand, mask_lmk, max_pages, num_pages, seq_len, n_blk, n_split, ragged, parents_stride;
  uint32_t g_magic;
  float c2;                     // scale * log2(e)
  long q_sb, q_st, q_sh;        // elements between sequences, tokens and heads of q
  const int32_t* table;         // (B, max_pages)
  const int32_t* lengths;       // (B) or null: seq_len
  const int32_t* parents;       // (B, T) or (T), or null: a chain
};

// Where a workgroup's keys lie and where its results go.
struct PagedSpan {
  int base, lo, hi, p0, p1;  // committed tokens, first slot and end of what any row sees, pages of this workgroup's share
  bool alive;
};

__device__ __forceinline__ int paged_left(int p, const PagedDims& dm) {
  const int left = p - dm.window + 1;
  return dm.expand ? left & -PA_PAGE : left;
}

// Slots [lo, hi) that the tokens t0 .. t1 of a sequence of `len` see, and their pages from lo / PA_PAGE on.
__device__ __forceinline__ int paged_pages(const PagedDims& dm, int len, int t0, int t1, int& lo, int& hi) {
  const int base = len - dm.T, left = paged_left(base + t0, dm);
  lo = left > 0 ? left : 0;
  const long end = (long)dm.max_pages * PA_PAGE;
  hi = base + t1 + 1 < end ? base + t1 + 1 : (int)end;
  const int n = len >= dm.T ? (hi + PA_PAGE - 1) / PA_PAGE - lo / PA_PAGE : 0;
  return n > 0 ? n : 0;
}

// Sums over the lanes up to this one.
__device__ __forceinline__ int paged_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);  // from 1, 2, 4, 8 lanes before, in rows of 16
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // a row's last sum to the row behind it,
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // that of two rows to the two behind them
  return x;
}

// Shares of a ragged batch, up to 64 sequences, lane b's of sequence b: n_split a sequence on average, as many as make the
// longest share shortest.  With c pages a share a sequence of n pages needs ceil(n / c); c lies between all / (n_split B) and
// all / ((n_split - 1) B), where sum (1 + (n - 1) / c) < B + (n_split - 1) B fits in any case; five halvings come within 4 % of
// the best c.  Equal numbers of shares leave the longest sequence's workgroups alone at the end: trees of 64 tokens for four
// sequences of 8K to 16K (8 shares on average), see the tile kernel's figures.
__device__ __forceinline__ int paged_ragged(const PagedDims& dm, int lane, int len) {
  int lo, hi;
  const int n = lane < dm.B ? paged_pages(dm, len, 0, dm.T - 1, lo, hi) : 0;
  const int slots = dm.n_split * dm.B;
  const int sum = __builtin_amdgcn_readlane(paged_scan(n), 63);
  const float all = (float)(sum > 1 ? sum : 1), rest = n > 1 ? (float)(n - 1) : 0.f;
  const auto shares = [&](float c) __attribute__((always_inline)) {
    return lane < dm.B ? 1 + (int)fminf(rest * __builtin_amdgcn_rcpf(c), 63.f) : 0;
  };
  float few = all / (float)slots, fit = all / (float)(slots - dm.B) * (1.f + 0x1p-18f);
  for (int i = 0; i < 5; ++i) {
    const float c = 0.5f * (few + fit);
    if (__builtin_amdgcn_readlane(paged_scan(shares(c)), 63) <= slots) fit = c;
    else few = c;
  }
  return shares(fit);
}

// What a workgroup works on: share `share` of `of` of a sequence's pages.  The row blocks of a (share, KV head) read the same
// pages: neighbours on one XCD (the hardware hands consecutive workgroups to the eight XCDs in turn); so do the VS workgroups
// that have a part of the values' features each.  `slot` numbers the
// shares of all sequences (it is the sequence where none is split).  False for what is left over at the end.
struct PagedUnit {
  int blk, vs, hk, slot, b, share, of, len;
};
template <int VS>
__device__ __forceinline__ bool paged_unit(const PagedDims& dm, int lane, PagedUnit& u) {
  const int total = dm.n_blk * VS * dm.n_split * dm.H * dm.B, per_xcd = (total + 7) / 8;
  const int id = (int)(blockIdx.x % 8) * per_xcd + (int)(blockIdx.x / 8);
  if (id >= total) return false;
  const int part = id / VS, rest = part / dm.n_blk;
  u.vs = id - part * VS;
  u.blk = part - rest * dm.n_blk;
  u.slot = rest / dm.H;
  u.hk = rest - u.slot * dm.H;
  if (dm.ragged) {
    const int len = lane < dm.B ? dm.lengths[lane] : 0;
    const int n = paged_ragged(dm, lane, len), behind = paged_scan(n);
    if (u.slot >= __builtin_amdgcn_readlane(behind, 63)) return false;
    u.b = 63 - __builtin_clzll(__ballot(lane < dm.B && behind - n <= u.slot));
    u.of = __builtin_amdgcn_readlane(n, u.b);
    u.share = u.slot - __builtin_amdgcn_readlane(behind, u.b) + u.of;
    u.len = __builtin_amdgcn_readlane(len, u.b);
    return true;
  }
  u.b = u.slot / dm.n_split;
  u.of = dm.n_split;
  u.share = u.slot - u.b * dm.n_split;
  u.len = dm.lengths ? dm.lengths[u.b] : dm.seq_len;
  return true;
}

__device__ __forceinline__ PagedSpan paged_span(const PagedDims& dm, const PagedUnit& u, int r0, int r1) {
  PagedSpan sp;
  sp.base = u.len - dm.T;
  sp.alive = u.len >= dm.T;
  const int t0 = dm.parents ? 0 : (int)hils_udiv(r0, dm.G, dm.g_magic);
  const int t1 = dm.parents ? dm.T - 1 : (int)hils_udiv(r1 - 1, dm.G, dm.g_magic);
  const int n = paged_pages(dm, u.len, t0, t1, sp.lo, sp.hi), first = sp.lo / PA_PAGE;
  const int per = (n + u.of - 1) / u.of;
  const int a = u.share * per < n ? u.share * per : n;
  sp.p0 = first + a;
  sp.p1 = first + (a + per < n ? a + per : n);
  return sp;
}

// Ancestors of the tokens t0 .. t0 + nt - 1 as bits of slots base + u, and the first committed slot each sees.  A token whose
// way to the root passes a parent that is neither -1 nor an earlier token takes no part: it sees nothing.
// par: this thread's parents as paged_parents() read them (before loads that are not to be waited for here).
// par_s: T words, mask_s: nt rows of PA_WORDS, left_s: nt words.  Ends without a barrier.
template <int NT>
__device__ __forceinline__ void paged_parents(const PagedDims& dm, int b, int tid, int (&par)[(PA_MAX_TREE + NT - 1) / NT]) {
  const int32_t* from = dm.parents + (long)b * dm.parents_stride;
#pragma unroll
  for (int i = 0; i < (PA_MAX_TREE + NT - 1) / NT; ++i) par[i] = tid + i * NT < dm.T ? from[tid + i * NT] : -2;
}
template <int NT>
__device__ __forceinline__ void paged_tree(const PagedDims& dm, int base, int t0, int nt, int tid,
                                           const int (&par)[(PA_MAX_TREE + NT - 1) / NT], int* par_s, unsigned* mask_s, int* left_s) {
#pragma unroll
  for (int i = 0; i < (PA_MAX_TREE + NT - 1) / NT; ++i)
    if (tid + i * NT < dm.T) par_s[tid + i * NT] = par[i];
  for (int i = tid; i < nt * PA_WORDS; i += NT) mask_s[i] = 0;
  lds_barrier();
  if (tid >= nt || t0 + tid >= dm.T) {
    if (tid < nt) left_s[tid] = 0x7fffffff;
    return;
  }
  unsigned* row = mask_s + tid * PA_WORDS + 1;
  int depth = -1, node = t0 + tid, word = node >> 5;
  unsigned bits = 0;
  bool ok = true;
  while (node >= 0) {  // (every step goes to an earlier token)
    ++depth;
    if ((node >> 5) != word) {
      row[word] = bits;
      bits = 0;
      word = node >> 5;
    }
    bits |= 1u << (node & 31);
    const int up = par_s[node];
    ok = ok && up >= -1 && up < node;
    node = ok ? up : -1;
  }
  row[word] = bits;
  const int p = base + depth;
  const int left = paged_left(p, dm);
  const bool landmark = dm.mask_lmk && ((base & (PA_PAGE - 1)) + depth >= PA_PAGE - 1);
  if (ok && (left > base || landmark)) {  // some of the ancestors lie before the window or are landmarks
    node = t0 + tid;
    for (int at = p; node >= 0; --at) {
      if (at < left || (dm.mask_lmk && (at & (PA_PAGE - 1)) == PA_PAGE - 1)) row[node >> 5] &= ~(1u << (node & 31));
      node = par_s[node];
    }
  }
  if (!ok)
    for (int w = 0; w < PA_WORDS - 1; ++w) row[w] = 0;
  left_s[tid] = ok ? left : 0x7fffffff;
}

// 32 bits of a mask row from bit `off` on, off > -32
__device__ __forceinline__ unsigned paged_bits(const unsigned* row, int off) {
  const int w = (off >> 5) + 1, s = off & 31;
  const uint64_t two = (uint64_t)row[w + 1] << 32 | row[w];
  return (unsigned)(two >> s);
}

// Where a row's results go: o and lse, or the share of the range that the workgroup had.
struct PagedOut {
  bf16_t* o;
  float* lse;
  float* part;   // (shares of all sequences, T, HQ, D) fp32, then (.., 2): maximum (score units) and sum
  long n_rows;
};

template <int D>
__device__ __forceinline__ void paged_store4(const PagedDims& dm, const PagedOut& out, long row, int d4, f32x4_t x, float M,
                                             float L) {
  if (dm.n_split > 1) {
    float* p = out.part + row * D + d4 * 4;
    *(f32x4_t*)p = x;
    if (d4 == 0) {
      float* ml = out.part + out.n_rows * dm.n_split * D + row * 2;
      ml[0] = M;
      ml[1] = L;
    }
    return;
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  uint2 pk;
  pk.x = pack_bf2(x[0] * inv, x[1] * inv);
  pk.y = pack_bf2(x[2] * inv, x[3] * inv);
  *(uint2*)(out.o + row * D + d4 * 4) = pk;
  if (d4 == 0) out.lse[row] = L == 0.f ? HILS_NEG_INF : (M * dm.c2 + __builtin_amdgcn_logf(L)) * HILS_LN2;
}

// One row over the pages p0 .. p1 - 1, by one wavefront, looking at no token that the row does not see.
template <int D, int VS>
__device__ __forceinline__ void paged_redo_row(const PagedDims& dm, const PagedOut& out, const bf16_t* qr, const bf16_t* k,
                                            const bf16_t* v, const int32_t* table, int hk, int base, int p0, int p1, int t,
                                            int left, const unsigned* mask_row, long row, int vs, int lane) {
  constexpr int DV = D / VS, NF = DV > 64 ? DV / 64 : 1;
  const bool mine = DV >= 64 || lane < DV;  // lanes that have features of the DV from f0 on
  const int f0 = vs * DV + (mine ? lane : 0);
  float m = HILS_NEG_INF, l = 0.f, x[NF];
#pragma unroll
  for (int f = 0; f < NF; ++f) x[f] = 0.f;
  for (int p = p0; p < p1; ++p) {
    const int page = table[p];
    if ((unsigned)page >= (unsigned)dm.num_pages) continue;
    const int slot = p * PA_PAGE + lane;
    bool see;
    if (mask_row) {
      const int u = slot - base;
      see = u < 0 ? slot >= left && !(dm.mask_lmk && lane == PA_PAGE - 1)
                  : u < dm.T && (mask_row[(u >> 5) + 1] >> (u & 31) & 1);
    } else {
      see = slot >= left && slot <= base + t && !(dm.mask_lmk && lane == PA_PAGE - 1);
    }
    const long at = ((long)page * dm.H + hk) * PA_PAGE * D;
    float s = HILS_NEG_INF;
    if (see) {
      s = 0.f;
      for (int d = 0; d < D; d += 8) {
        float a[8], c[8];
        unpack8(*(const uint4*)(qr + d), a);
        unpack8(*(const uint4*)(k + at + (long)lane * D + d), c);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(a[e], c[e], s);
      }
    }
    const float m_new = fmaxf(m, wave_max(s));
    const float mc = m_new > HILS_NEG_INF ? m_new * dm.c2 : 0.f;
    const float corr = m_new > HILS_NEG_INF ? __builtin_amdgcn_exp2f(fmaf(m, dm.c2, -mc)) : 1.f;
    const float e = see ? __builtin_amdgcn_exp2f(fmaf(s, dm.c2, -mc)) : 0.f;
    m = m_new;
    l = l * corr + wave_sum(e);
#pragma unroll
    for (int f = 0; f < NF; ++f) x[f] *= corr;
    uint64_t who = __ballot(see);
    while (who) {
      const int i = __builtin_ctzll(who);
      who &= who - 1;
      const float pe = __shfl(e, i, 64);
#pragma unroll
      for (int f = 0; f < NF; ++f) x[f] = fmaf(pe, bf2f(v[at + (long)i * D + f * 64 + f0]), x[f]);
    }
  }
  if (dm.n_split > 1) {
    float* part = out.part + row * D;
#pragma unroll
    for (int f = 0; f < NF; ++f)
      if (mine) part[f * 64 + f0] = x[f];
    if (lane == 0 && vs == 0) {
      float* ml = out.part + out.n_rows * dm.n_split * D + row * 2;
      ml[0] = m;
      ml[1] = l;
    }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int f = 0; f < NF; ++f)
    if (mine) out.o[row * D + f * 64 + f0] = f2bf(x[f] * inv);
  if (lane == 0 && vs == 0) out.lse[row] = l == 0.f ? HILS_NEG_INF : (m * dm.c2 + __builtin_amdgcn_logf(l)) * HILS_LN2;
}

// ---- few rows ----------------------------------------------------------------------------------
// 16 NR rows a workgroup; units of 32 tokens (half a page) go to its wavefronts in turn, the next unit's keys and values
// under way while one is worked on; the wavefronts' results meet in LDS.  K rows are read straight into A operands (a lane 16
// bytes of its token's row), V goes through the wavefront's own LDS area and is read by the transposing load.  Bound by HBM:
// a token of 16 sequences of 16K to 32K, 8 KV heads of 128, 237 us (1.54 GB: 6.5 TB/s, a plain read reaches 6.9), and with a
// window of 512 by the latencies around it: 32 such sequences 14.3 us (74 MB), one of 2 KV heads of 64 5.6 us.  Where there
// are few of them a workgroup is bound by what its compute unit takes in (some 65 GB/s): then VS of them have a part of the
// values' features each and all keys (1 to 8 sequences, 8 KV heads of 128, window 512: 8.7 us alone, 7.8 by two, 7.5 by four).
template <int D, int NR, int NWV, bool TREE, bool PAST, int VS>
__global__ void __launch_bounds__(NWV * 64) __attribute__((amdgpu_waves_per_eu(NR == 2 && D == 128 ? 1 : 2)))
paged_attn_rows(const bf16_t* __restrict__ q, const bf16_t* __restrict__ k, const bf16_t* __restrict__ v, PagedDims dm,
                PagedOut out) {
  constexpr int DV = D / VS, KS = D / 32, MT = DV / 16, ROWS = 16 * NR;
  constexpr int VL = DV / 8, TPI = 64 / VL, VI = 32 / TPI;  // lanes per V row, rows per load, loads per unit
  constexpr int VP = 2 * DV + 16, OP = DV + 4;
  constexpr int AREA = 32 * VP > ROWS * OP * 4 ? 32 * VP : ROWS * OP * 4;
  __shared__ __align__(16) unsigned char area_s[NWV * AREA];
  __shared__ float m_s[NWV][ROWS], l_s[NWV][ROWS];
  __shared__ int par_s[TREE ? PA_MAX_TREE : 1], left_s[ROWS];
  __shared__ unsigned mask_s[TREE ? ROWS * PA_WORDS : 1], odd_s;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, j = lane >> 4;
  PagedUnit at;
  if (!paged_unit<VS>(dm, lane, at)) return;
  const int blk = at.blk, hk = at.hk, b = at.b;
  const int n_rows = dm.T * dm.G, r0 = blk * ROWS;
  const int r1 = r0 + ROWS < n_rows ? r0 + ROWS : n_rows;
  const PagedSpan sp = paged_span(dm, at, r0, r1);
  const int32_t* table = dm.table + (long)b * dm.max_pages;
  const int t0 = hils_udiv(r0, dm.G, dm.g_magic);

  const int u0 = sp.p0 * 2, u1 = sp.p1 * 2, len = __builtin_amdgcn_readfirstlane(at.len);
  // page of the units that this wavefront takes: lane i holds that of its i-th one
  int pages_of = -1;
  auto ask_pages = [&](int first) __attribute__((always_inline)) {
    const int u = first + lane * NWV;
    pages_of = u < u1 ? table[u >> 1] : -1;
  };
  ask_pages(u0 + wave);
  int par[TREE ? (PA_MAX_TREE + NWV * 64 - 1) / (NWV * 64) : 1];
  if constexpr (TREE) paged_parents<NWV * 64>(dm, b, tid, par);
  bf16x8_t qb[NR][KS];
  int row_t[NR];
#pragma unroll
  for (int rt = 0; rt < NR; ++rt) {
    const int r = r0 + rt * 16 + col;
    const int rc = r < r1 ? r : r1 - 1;
    const int t = hils_udiv(rc, dm.G, dm.g_magic), g = rc - t * dm.G;
    row_t[rt] = r < r1 ? t : -1;
    const bf16_t* qp = q + b * dm.q_sb + t * dm.q_st + (hk * dm.G + g) * dm.q_sh + j * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qb[rt][ks] = *(const bf16x8_t*)(qp + ks * 32);
  }
  const bf16_t* kb = k + (long)hk * PA_PAGE * D + col * D + j * 8;
  const bf16_t* vb = v + (long)hk * PA_PAGE * D + lane / VL * D + lane % VL * 8 + at.vs * DV;
  const long page_el = (long)dm.H * PA_PAGE * D;
  auto issue = [&](pa_u4 (&kd)[2][KS], pa_u4 (&vd)[VI], int page, int half) __attribute__((always_inline)) {
    const long at = (unsigned)page < (unsigned)dm.num_pages ? page * page_el : 0;  // (not mapped: not worked on)
    const bf16_t* kp = kb + at + half * 32 * D;
    const bf16_t* vp = vb + at + half * 32 * D;
#pragma unroll
    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) kd[tt][ks] = *(const pa_u4*)(kp + tt * 16 * D + ks * 32);
#pragma unroll
    for (int i = 0; i < VI; ++i) vd[i] = PAST ? __builtin_nontemporal_load((const pa_u4*)(vp + i * TPI * D)) : *(const pa_u4*)(vp + i * TPI * D);
  };

  unsigned char* area = area_s + wave * AREA;
  unsigned char* const w_addr = area + (lane / VL) * VP + (lane % VL) * 16;
  const unsigned char* const t_addr = area + (4 * j + (col >> 2)) * VP + (col & 3) * 8;
  f32x4_t O[NR][MT];
  float m_run[NR], l_run[NR];  // of this lane's rows over the units seen (l_run: this lane's tokens)
#pragma unroll
  for (int rt = 0; rt < NR; ++rt) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) O[rt][mt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    m_run[rt] = HILS_NEG_INF;
    l_run[rt] = 0.f;
  }
  // visible slots of the rows: [vlo, vlo + vspan], and in a tree the mask's bits behind the committed tokens
  int vlo[NR];
  unsigned vspan[NR];
  const unsigned* mrow[NR];

  auto unit = [&](const pa_u4 (&kd)[2][KS], const pa_u4 (&vd)[VI], int u) __attribute__((always_inline)) {
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < VI; ++i) *(pa_u4*)(w_addr + i * TPI * VP) = vd[i];
    if (u * 32 + 32 > len) {  // (the same for the whole wavefront) values behind the last token: zeros
#pragma unroll
      for (int i = 0; i < VI; ++i)
        if (u * 32 + lane / VL + i * TPI >= len) *(pa_u4*)(w_addr + i * TPI * VP) = pa_u4{0, 0, 0, 0};
    }
    __builtin_amdgcn_wave_barrier();
    f32x4_t S[NR][2];
#pragma unroll
    for (int rt = 0; rt < NR; ++rt)
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        S[rt][tt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          S[rt][tt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, kd[tt][ks]), qb[rt][ks], S[rt][tt], 0, 0, 0);
      }
    const int slot0 = u * 32 + 4 * j;
    float corr[NR];
    bf16x8_t pb[NR];
#pragma unroll
    for (int rt = 0; rt < NR; ++rt) {
      const unsigned from = (unsigned)(slot0 - vlo[rt]);
      unsigned extra = 0;
      if (TREE && u * 32 + 32 > sp.base) {  // (the same for the whole wavefront)
        const int off = u * 32 - sp.base;
        extra = off < dm.T ? paged_bits(mrow[rt], off) >> (4 * j) : 0u;
      }
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          bool see = from + (unsigned)(tt * 16 + i) <= vspan[rt];
          if (dm.mask_lmk && tt == 1 && i == 3) see = see && !((u & 1) && j == 3);
          if (TREE) see = see || (extra >> (tt * 16 + i) & 1);
          S[rt][tt][i] = see ? S[rt][tt][i] : HILS_NEG_INF;
        }
      float mx = HILS_NEG_INF;
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, S[rt][tt][i]);
      mx = rows_max(mx);
      const float m_new = fmaxf(m_run[rt], mx);
      const bool any = m_new > HILS_NEG_INF;
      const float mc = any ? m_new * dm.c2 : 0.f;
      corr[rt] = any ? __builtin_amdgcn_exp2f(fmaf(m_run[rt], dm.c2, -mc)) : 1.f;  // exp2(-inf) = 0: nothing yet
      m_run[rt] = m_new;
      float sum = 0.f;
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = __builtin_amdgcn_exp2f(fmaf(S[rt][tt][i], dm.c2, -mc));
          S[rt][tt][i] = e;
          sum += e;
        }
      l_run[rt] = l_run[rt] * corr[rt] + sum;
      pa_u4 pk;
      pk.x = pack_bf2(S[rt][0][0], S[rt][0][1]);
      pk.y = pack_bf2(S[rt][0][2], S[rt][0][3]);
      pk.z = pack_bf2(S[rt][1][0], S[rt][1][1]);
      pk.w = pack_bf2(S[rt][1][2], S[rt][1][3]);
      pb[rt] = __builtin_bit_cast(bf16x8_t, pk);
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const pa_s4 a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) pa_s4*)(t_addr + mt * 32));
      const pa_s4 a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) pa_s4*)(t_addr + mt * 32 + 16 * VP));
      const bf16x8_t a = __builtin_bit_cast(bf16x8_t, (pa_s8)__builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
      for (int rt = 0; rt < NR; ++rt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) O[rt][mt][i] *= corr[rt];
        O[rt][mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pb[rt], O[rt][mt], 0, 0, 0);
      }
    }
  };

  {
    // two units' loads in flight (and none that are not worked on: a window's wavefronts have two or three units)
    pa_u4 ka[2][KS], va[VI], kc[2][KS], vc[VI];
    int n_mine = u1 > u0 + wave ? (u1 - u0 - wave + NWV - 1) / NWV : 0;
    auto page_at = [&](int i) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(pages_of, i & 63); };
    int pg_a = page_at(0), pg_c;
    if (n_mine > 0) issue(ka, va, pg_a, (u0 + wave) & 1);
    if constexpr (TREE) paged_tree<NWV * 64>(dm, sp.base, t0, ROWS, tid, par, par_s, mask_s, left_s);
    if (tid == 0) odd_s = 0;
    lds_barrier();
#pragma unroll
    for (int rt = 0; rt < NR; ++rt) {
      const bool live = row_t[rt] >= 0 && sp.alive;
      const int i = live ? row_t[rt] - t0 : 0;
      int lo = TREE ? left_s[i] : paged_left(sp.base + row_t[rt], dm);
      lo = lo > 0 ? lo : 0;
      const int last = TREE ? sp.base - 1 : sp.base + row_t[rt];
      const bool some = live && last >= lo;
      vlo[rt] = some ? lo : 0x7fffffff;
      vspan[rt] = some ? (unsigned)(last - lo) : 0u;
      if (TREE) mrow[rt] = mask_s + (live ? i : 0) * PA_WORDS;
    }
    // (the queries are here from now on: waited for inside the loop, the unit under way would be waited for with them)
#pragma unroll
    for (int rt = 0; rt < NR; ++rt)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qb[rt][ks]));
    auto next_page = [&](int i) __attribute__((always_inline)) {  // page of this wavefront's unit i, asked for 64 at a time
      if ((i & 63) == 0) {
        ask_pages(u0 + wave + i * NWV);
        asm volatile("" : "+v"(pages_of));  // (waited for here: behind the branch, every unit would wait for all loads)
      }
      return page_at(i);
    };
    int u = u0 + wave, i = 0;
    for (; i + 2 < n_mine; i += 2, u += 2 * NWV) {
      pg_c = next_page(i + 1);
      issue(kc, vc, pg_c, (u + NWV) & 1);
      if ((unsigned)pg_a < (unsigned)dm.num_pages) unit(ka, va, u);
      pg_a = next_page(i + 2);
      issue(ka, va, pg_a, u & 1);
      if ((unsigned)pg_c < (unsigned)dm.num_pages) unit(kc, vc, u + NWV);
    }
    if (i + 1 < n_mine) {
      pg_c = next_page(i + 1);
      issue(kc, vc, pg_c, (u + NWV) & 1);
      if ((unsigned)pg_a < (unsigned)dm.num_pages) unit(ka, va, u);
      if ((unsigned)pg_c < (unsigned)dm.num_pages) unit(kc, vc, u + NWV);
    } else if (i < n_mine && (unsigned)pg_a < (unsigned)dm.num_pages) {
      unit(ka, va, u);
    }
  }
  // park the partial results: accumulator register i of tile mt in lane (row = col, j) is feature mt*16 + 4j + i
  __builtin_amdgcn_wave_barrier();
  float* o_s = (float*)area;
#pragma unroll
  for (int rt = 0; rt < NR; ++rt) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) *(f32x4_t*)&o_s[(rt * 16 + col) * OP + mt * 16 + 4 * j] = O[rt][mt];
    const float l_row = rows_sum(l_run[rt]);
    if (j == 0) {
      m_s[wave][rt * 16 + col] = m_run[rt];
      l_s[wave][rt * 16 + col] = l_row;
    }
  }
  __syncthreads();
  for (int p = tid; p < ROWS * (DV / 4); p += NWV * 64) {
    const int rr = p / (DV / 4), d4 = p % (DV / 4), r = r0 + rr;
    if (r >= r1) continue;
    float M = HILS_NEG_INF;
#pragma unroll
    for (int w = 0; w < NWV; ++w) M = fmaxf(M, m_s[w][rr]);
    float L = 0.f;
    f32x4_t x = {0.f, 0.f, 0.f, 0.f};
    // (no maximum: nothing was seen, and the sums are zero, or scores that are not numbers, which the sums keep)
#pragma unroll
    for (int w = 0; w < NWV; ++w) {
      const float f = M > HILS_NEG_INF ? __builtin_amdgcn_exp2f((m_s[w][rr] - M) * dm.c2) : 1.f;
      const f32x4_t ow = *(const f32x4_t*)((const float*)(area_s + w * AREA) + rr * OP + d4 * 4);
      L = fmaf(f, l_s[w][rr], L);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = fmaf(f, ow[i], x[i]);
    }
    const int t = hils_udiv(r, dm.G, dm.g_magic), g = r - t * dm.G;
    const long row = ((long)at.slot * dm.T + t) * dm.HQ + hk * dm.G + g;
    paged_store4<D>(dm, out, row, at.vs * (DV / 4) + d4, x, M, L);
    const float all = (x[0] + x[1]) + (x[2] + x[3]);  // (no finite number if one of them is none)
    if (!(fabsf(all) < INFINITY)) atomicOr(&odd_s, 1u << rr);
  }
  __syncthreads();
  if (const unsigned odd = odd_s; odd != 0) {
    for (int rr = wave; rr < r1 - r0; rr += NWV) {
      if (!(odd >> rr & 1)) continue;
      const int r = r0 + rr, t = hils_udiv(r, dm.G, dm.g_magic), g = r - t * dm.G;
      const long row = ((long)at.slot * dm.T + t) * dm.HQ + hk * dm.G + g;
      int left = TREE ? left_s[t - t0] : paged_left(sp.base + t, dm);
      paged_redo_row<D, VS>(dm, out, q + b * dm.q_sb + t * dm.q_st + (hk * dm.G + g) * dm.q_sh, k, v, table, hk, sp.base, sp.p0,
                        sp.p1, t, left, TREE ? mask_s + (t - t0) * PA_WORDS : nullptr, row, at.vs, lane);
    }
  }
}

// ---- many rows ---------------------------------------------------------------------------------
// 32 rows a wavefront, or two wavefronts that have half of every page each and add up at the end (KW == 2: where the rows fill
// less than half of a compute unit's wavefronts; trees of 64 tokens for 4 sequences, 8 KV heads of 128, window 512: 64 rows by
// 4 wavefronts 15.9 us, by 2 17.9); pages go straight into LDS, keys into one of four buffers, values into one of four others,
// asked for two or three steps before they are used.  32x32x16 products: a row's scores of half a page (32 tokens) are 16 registers of two
// lanes, which are the second product's operand as they are.  A step issues, half by half, the products of page p's output
// and of page p + 1's scores between the exponentials of the half page behind (the matrix and vector instructions of one
// wavefront overlap, those of two that run in step hardly do).  The exponentials' reference point follows a row's maximum
// only when a score is more than 2^6 above it: the others need no reduction over lanes and no rescaling, and probabilities
// of up to 2^6 enter sum and output alike.
// Bound by latencies where a window has ten pages (18 us for trees of 63 tokens for 8 sequences, 8 KV heads of 128: 7.6 in the
// steps), else by the vector and matrix units together.  A page of 256 rows takes 1.6 us where 32 workgroups have the chip to
// themselves, 0.85 of it matrix products, and 2.25 with one on every compute unit (four trees of 64 tokens, 4 KV heads of 128,
// everything seen: 89 us for 32 pages a workgroup, 312 for 128: 0.95 PFLOP/s in the steps, 1.41 in a large product).
// Sequences of 8K to 16K: 72 to 78 us with the join (51 GFLOP): 25 to 28 pages of the longest share, 7 us of start and end,
// the join's 10.
// The buffers come first: their places are then plain offsets, and a buffer's number is two bits of them.
template <int D, int NW, int KW, bool TREE>
static constexpr size_t paged_tiles_smem() {
  return 2 * 4 * (size_t)PA_PAGE * 2 * D + (TREE ? (NW / KW * 32 * (PA_WORDS + 1) + PA_MAX_TREE) * sizeof(int) : 0);
}

template <int D, int NW, int KW, bool TREE>
__global__ void __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(2)))
paged_attn_tiles(const bf16_t* __restrict__ q, const bf16_t* __restrict__ k, const bf16_t* __restrict__ v, PagedDims dm,
                 PagedOut out) {
  constexpr int NT = NW * 64, RW = NW / KW, ROWS = RW * 32, KS = D / 16, FT = D / 32, RP = 2 * D, SEG = D / 8;
  constexpr int NB = 4, PAGE = PA_PAGE * RP, NP = PAGE / 1024 / NW;  // loads of a page's keys per wavefront
  static_assert(NP >= 1 && NP * NW * 1024 == PAGE, "every wavefront loads whole rows");
  constexpr float LAZY = 6.f;
  extern __shared__ __align__(16) unsigned char pa_dyn[];
  unsigned* const mask_s = (unsigned*)(pa_dyn + 2 * NB * PAGE);
  int* const left_s = (int*)(mask_s + ROWS * PA_WORDS);
  int* const par_s = left_s + ROWS;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, h = lane >> 5;
  const int rg = wave % RW, kg = wave / RW;  // rows and half of every page (KW == 2) that are this wavefront's
  PagedUnit at;
  if (!paged_unit<1>(dm, lane, at)) return;
  const int blk = at.blk, hk = at.hk, b = at.b;
  const int n_rows = dm.T * dm.G, r0 = blk * ROWS;
  const int r1 = r0 + ROWS < n_rows ? r0 + ROWS : n_rows;
  const PagedSpan sp = paged_span(dm, at, r0, r1);
  const int32_t* table = dm.table + (long)b * dm.max_pages;
  const int t0 = hils_udiv(r0, dm.G, dm.g_magic);

  const int p0 = __builtin_amdgcn_readfirstlane(sp.p0);
  const int n = __builtin_amdgcn_readfirstlane(sp.p1 - sp.p0);
  int pages_of = -1, pages_at = p0;  // lane i holds the page of chunk pages_at + i
  auto ask_pages = [&]() __attribute__((always_inline)) {
    pages_of = pages_at + lane < sp.p1 ? table[pages_at + lane] : -1;
  };
  auto page_at = [&](int p) __attribute__((always_inline)) {
    if (p - pages_at >= 64) {
      pages_at += 64;
      ask_pages();
      asm volatile("" : "+v"(pages_of));  // (waited for here: behind the branch, every step would wait for all its loads)
    }
    return __builtin_amdgcn_readlane(pages_of, p - pages_at);
  };
  unsigned d_off[NP < 4 ? NP : 4];  // (the fifth load's places are the first one's, 4 KiB further)
#pragma unroll
  for (int i = 0; i < (NP < 4 ? NP : 4); ++i) {
    const int x = (wave * NP + i) * 64 + lane, row = x / SEG, pc = x % SEG;
    d_off[i] = (unsigned)(row * RP + (pc ^ lz_swz<D>(row)) * 16);
  }
  const unsigned lds0 = __builtin_amdgcn_readfirstlane(lz_lds_addr(pa_dyn) + wave * (NP * 1024));
  const unsigned long long head_b = (unsigned long long)hk * PAGE, page_b = (unsigned long long)dm.H * PAGE;
  // Page x's keys lie in buffer gray(x % 4), its values in that buffer of the four behind: from one page to the next one bit
  // of the buffer's number changes, the lower and the higher in turn.
  unsigned known = 0;  // bit i: the page i fetches back is mapped
  auto k_buffer = [&](int x) __attribute__((always_inline)) { return lds0 + (unsigned)((x & 3) ^ (x >> 1 & 1)) * PAGE; };
  auto v_buffer = [&](int x) __attribute__((always_inline)) { return k_buffer(x) + NB * PAGE; };
  auto page_place = [&](int x) __attribute__((always_inline)) {  // where in the pools page x lies (past the end: anywhere)
    const int page = x < n ? page_at(p0 + x) : -1;
    const bool mapped = (unsigned)page < (unsigned)dm.num_pages;
    known = known << 1 | (unsigned)mapped;
    return lz_uniform((mapped ? page * page_b : 0) + head_b);
  };
  const unsigned long long k_pool = lz_uniform((unsigned long long)k), v_pool = lz_uniform((unsigned long long)v);
  auto fetch = [&](unsigned long long from, unsigned to) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NP; ++i) lz_dma16(to + i * 1024, d_off[i & 3], from + (i >> 2) * 4096);
  };

  const int r = r0 + rg * 32 + col;
  const int rc = r < r1 ? r : r1 - 1;
  const int my_t = hils_udiv(rc, dm.G, dm.g_magic), my_g = rc - my_t * dm.G;
  const bool live = r < r1 && sp.alive;
  bf16x8_t qa[KS];
  {
    const bf16_t* qp = q + b * dm.q_sb + my_t * dm.q_st + (hk * dm.G + my_g) * dm.q_sh + h * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qa[ks] = *(const bf16x8_t*)(qp + ks * 16);
  }
  int par[TREE ? (PA_MAX_TREE + NT - 1) / NT : 1];
  if constexpr (TREE) paged_parents<NT>(dm, b, tid, par);
  ask_pages();
  // (the queries and pages are here from now on: the compiler's waits know nothing of the loads into LDS and would wait for
  // them too)
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qa[ks]));
  asm volatile("" : "+v"(pages_of));
  if constexpr (TREE) asm volatile("" : "+v"(par[0]), "+v"(par[(PA_MAX_TREE - 1) / NT]));
  const unsigned long long place0 = page_place(0), place1 = page_place(1), place2 = page_place(2);
  unsigned long long place = page_place(3);  // of page x + 3 before step x
  unsigned long long place_k = KW == 2 ? page_place(4) : 0;  // of page x + 4
  if (n > 0) {
    fetch(k_pool + place0, k_buffer(0));
    fetch(k_pool + place1, k_buffer(1));
    fetch(v_pool + place0, v_buffer(0));
  }
  if constexpr (TREE) paged_tree<NT>(dm, sp.base, t0, ROWS, tid, par, par_s, mask_s, left_s);
  if (n > 0) {
    fetch(k_pool + place2, k_buffer(2));
    fetch(v_pool + place1, v_buffer(1));
    fetch(k_pool + place, k_buffer(3));
    fetch(v_pool + place2, v_buffer(2));
  }
  if constexpr (TREE) lds_barrier();
  // visible slots of the row: [vlo, vlo + vspan], and in a tree the mask's bits behind the committed tokens
  int vlo;
  unsigned vspan;
  int all_lo = 0, all_hi = 0x7fffffff;  // slots that all rows of the wavefront see
  const unsigned* mrow = TREE ? mask_s + (live ? my_t - t0 : 0) * PA_WORDS : nullptr;
  {
    int lo = TREE ? left_s[live ? my_t - t0 : 0] : paged_left(sp.base + my_t, dm);
    lo = lo > 0 ? lo : 0;
    const int last = TREE ? sp.base - 1 : sp.base + my_t;
    const bool some = live && last >= lo;
    vlo = some ? lo : 0x7fffffff;
    vspan = some ? (unsigned)(last - lo) : 0u;
    if (live) {
      all_lo = lo;
      all_hi = last + 1;
    }
  }
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) {
    all_lo = max(all_lo, __shfl_xor(all_lo, x, 64));
    all_hi = min(all_hi, __shfl_xor(all_hi, x, 64));
  }
  all_lo = __builtin_amdgcn_readfirstlane(all_lo);
  all_hi = __builtin_amdgcn_readfirstlane(all_hi);

  f32x16_t acc[FT];
#pragma unroll
  for (int ft = 0; ft < FT; ++ft)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[ft][i] = 0.f;
  float ref = HILS_NEG_INF, l_run = 0.f;  // reference point (log2 units) and this lane's share of the sum
  unsigned k_off[KS], v_off[FT][2];       // this lane's places in a half page, in the buffers of this step
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) k_off[ks] = (unsigned)((col + 32 * kg) * RP + ((2 * ks + h) ^ lz_swz<D>(col)) * 16);
#pragma unroll
  for (int ft = 0; ft < FT; ++ft)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = 4 * h + 8 * e + ((lane & 15) >> 2), pc = ft * 4 + (lane >> 4 & 1) * 2 + (lane >> 1 & 1);
      v_off[ft][e] = (unsigned)(NB * PAGE + (row + 32 * kg) * RP + (pc ^ lz_swz<D>(row)) * 16 + (lane & 1) * 8);
    }

  auto products = [&](f32x16_t& st, int half) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 16; ++i) st[i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      st = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8_t*)(pa_dyn + (k_off[ks] + half * 32 * RP)), qa[ks], st, 0, 0, 0);
  };
  // scores of a half of page x: -inf where the row does not see a token (token (i >> 2) * 8 + 4 h + (i & 3) in register i)
  auto hide = [&](f32x16_t& st, int x, int half, int back) __attribute__((always_inline)) {  // back: fetches of keys since
    const int first = (p0 + x) * PA_PAGE + half * 32;
    const bool mapped = known >> back & 1;
    if (first < all_lo || first + 32 > all_hi || !mapped) {
      unsigned seen = 0;  // bit i: the row sees token first + i
      if (mapped) {
        const int lo = vlo - first, hi = (int)((unsigned)vlo + vspan - (unsigned)first);
        if (lo < 32 && hi >= 0) seen = ~0u << (lo > 0 ? lo : 0) & ~0u >> (hi < 31 ? 31 - hi : 0);
        if (TREE) {
          if (dm.mask_lmk && half) seen &= 0x7fffffffu;
          const int off = first - sp.base;
          if (off > -32 && off < dm.T) seen |= paged_bits(mrow, off);
        }
      }
      seen >>= 4 * h;
#pragma unroll
      for (int i = 0; i < 16; ++i) st[i] = seen >> ((i >> 2) * 8 + (i & 3)) & 1 ? st[i] : HILS_NEG_INF;
    }
    // a committed landmark is its page's last token (a drafted one has been left out of the masks)
    if (half && dm.mask_lmk && (!TREE || first + 32 <= sp.base)) st[15] = h == 1 ? HILS_NEG_INF : st[15];
  };
  // Probabilities e[i0 .. i0 + N) of scores about the reference point, into the sums and, in pairs, into the second product's
  // operand.
  float ref0 = 0.f;  // (the reference point, 0 where nothing has been seen)
  auto weigh = [&](const f32x16_t& st, pa_u4 (&p)[2], float (&sum)[2], auto i0, auto count) __attribute__((always_inline)) {
    constexpr int I0 = decltype(i0)::value, N = decltype(count)::value;
#pragma unroll
    for (int i = I0; i < I0 + N; i += 2) {
      const float e0 = __builtin_amdgcn_exp2f(fmaf(st[i], dm.c2, -ref0)), e1 = __builtin_amdgcn_exp2f(fmaf(st[i + 1], dm.c2, -ref0));
      sum[0] += e0;
      sum[1] += e1;
      p[i >> 3][i >> 1 & 3] = pack_bf2(e0, e1);
    }
  };
  typedef std::integral_constant<int, 0> Zero;
  // The same for all 16 with the reference point moved to the maximum where a row has a score (mx: of this lane) far above it.
  // Returns the factor that the accumulators are due.
  auto settle = [&](const f32x16_t& st, pa_u4 (&p)[2], float mx) __attribute__((always_inline)) {
    mx = lz_halves_max(mx) * dm.c2;
    const float to = mx > ref + LAZY ? mx : ref;
    const float corr = to > ref ? __builtin_amdgcn_exp2f(ref - to) : 1.f;  // exp2(-inf) = 0: nothing yet
    ref = to;
    ref0 = to > HILS_NEG_INF ? to : 0.f;
    float sum[2] = {0.f, 0.f};
    weigh(st, p, sum, Zero{}, std::integral_constant<int, 16>{});
    l_run = fmaf(l_run, corr, sum[0] + sum[1]);
    return corr;
  };
  auto highest = [](const f32x16_t& st) __attribute__((always_inline)) {
    float mx = fmaxf(st[0], st[1]);
#pragma unroll
    for (int i = 2; i < 16; ++i) mx = fmaxf(mx, st[i]);
    return mx;
  };
  f32x16_t sa, sb;  // scores of first halves, of second halves
  pa_u4 pa[2], pb[2];
  static_assert(KW * NP <= KS, "a half page's products issue the loads of a page's keys or values, or both");
  constexpr int AH = 3;  // products of each kind that operands are read ahead of
  // Step x, both halves of a page a wavefront's: the products of page x's output and of page x + 1's scores, a pair of them at
  // a time (D / 16 pairs a half), and between them the probabilities of the half page behind, from the scores that the half
  // step before has left; the loads of page x + 3's values and x + 4's keys.  One half a wavefront's (KW == 2): the products of
  // page x's output and of page x + 2's scores, between them the probabilities of page x + 1; the loads of page x + 3's values
  // and x + 5's keys.
  auto step = [&](int x, unsigned long long v_from, unsigned v_to, unsigned long long k_from, unsigned k_to, f32x16_t& s1,
                  f32x16_t& s2, pa_u4 (&p1)[2], pa_u4 (&p2)[2]) __attribute__((always_inline)) {
    bf16x8_t va[AH + 1], ka[AH + 1];
    auto operands = [&](int y) __attribute__((always_inline)) {
      const int half = y / KS, s = y % KS / FT, ft = y % FT;  // (KW == 2: the half is in the offsets)
      const unsigned char* a0p = pa_dyn + (v_off[ft][0] + (half * 32 + s * 16) * RP);
      const unsigned char* a1p = pa_dyn + (v_off[ft][1] + (half * 32 + s * 16) * RP);
      const pa_s4 a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) pa_s4*)a0p);
      const pa_s4 a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) pa_s4*)a1p);
      va[y % (AH + 1)] = __builtin_bit_cast(bf16x8_t, (pa_s8)__builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7));
      ka[y % (AH + 1)] = *(const bf16x8_t*)(pa_dyn + (k_off[y % KS] + half * 32 * RP));
    };
    float sum[2], mx;
    // the y-th pair; probabilities of `now` into pn
    auto pair = [&](auto yc, f32x16_t& now, f32x16_t& nx, const pa_u4 (&p)[2], pa_u4 (&pn)[2]) __attribute__((always_inline)) {
      constexpr int y = decltype(yc)::value, z = y % KS;
      if constexpr (y + AH < 2 / KW * KS) operands(y + AH);
      acc[y % FT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va[y % (AH + 1)], __builtin_bit_cast(bf16x8_t, p[z / FT]), acc[y % FT], 0, 0, 0);
      nx = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[y % (AH + 1)], qa[z], nx, 0, 0, 0);
      if constexpr (KW == 2 && z >= NP && z < 2 * NP) lz_dma16(k_to + (z - NP) * 1024, d_off[(z - NP) & 3], k_from + ((z - NP) >> 2) * 4096);
      else if constexpr (z < NP) lz_dma16((y < KS ? v_to : k_to) + z * 1024, d_off[z & 3], (y < KS ? v_from : k_from) + (z >> 2) * 4096);
      if (z > 0) {  // (none beside the first pair: its scores are not there yet)
        constexpr int per = KS == 8 ? 2 : 4, first = (z - 1) * per;
        weigh(now, pn, sum, std::integral_constant<int, first>{}, std::integral_constant<int, z == KS - 1 ? 16 - first : per>{});
        if (z == KS - 1) mx = highest(now);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    auto finish = [&](f32x16_t& now, pa_u4 (&pn)[2]) __attribute__((always_inline)) {
      float l_new = l_run + (sum[0] + sum[1]);
      asm volatile("" : "+v"(pn[0]), "+v"(pn[1]), "+v"(l_new), "+v"(mx));  // (taken between the products, not behind them)
      __builtin_amdgcn_sched_barrier(0);
      const bool moves = __any(mx * dm.c2 > ref + LAZY);
      float corr = 1.f;
      if (moves) corr = settle(now, pn, mx);
      else l_run = l_new;
      if (moves) {
#pragma unroll
        for (int ft = 0; ft < FT; ++ft)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[ft][i] *= corr;
      }
    };
#define PA_PAIR(Y_, NOW_, NX_, P_, PN_) pair(std::integral_constant<int, Y_>{}, NOW_, NX_, P_, PN_)
#define PA_HALF(Y_, NOW_, NX_, P_, PN_)                                                                             \
  PA_PAIR(Y_ + 1, NOW_, NX_, P_, PN_);                                                                              \
  PA_PAIR(Y_ + 2, NOW_, NX_, P_, PN_);                                                                              \
  PA_PAIR(Y_ + 3, NOW_, NX_, P_, PN_);                                                                              \
  if constexpr (KS == 8) {                                                                                          \
    PA_PAIR(Y_ + 4, NOW_, NX_, P_, PN_);                                                                            \
    PA_PAIR(Y_ + 5, NOW_, NX_, P_, PN_);                                                                            \
    PA_PAIR(Y_ + 6, NOW_, NX_, P_, PN_);                                                                            \
    PA_PAIR(Y_ + 7, NOW_, NX_, P_, PN_);                                                                            \
  }
#pragma unroll
    for (int y = 0; y < AH; ++y) operands(y);
#pragma unroll
    for (int i = 0; i < 16; ++i) s2[i] = 0.f;
    sum[0] = sum[1] = 0.f;
    __builtin_amdgcn_sched_barrier(0);
    PA_PAIR(0, s1, s2, p1, p2);
    if (KW == 2) hide(s1, x + 1, kg, 4);
    else hide(s1, x, 1, 4);
    asm volatile("" : "+v"(s1));  // (the exponentials stay behind this point, between the products)
    __builtin_amdgcn_sched_barrier(0);
    PA_HALF(0, s1, s2, p1, p2)
    finish(s1, p2);
    if constexpr (KW == 1) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s1[i] = 0.f;
      sum[0] = sum[1] = 0.f;
      __builtin_amdgcn_sched_barrier(0);
      PA_PAIR(KS, s2, s1, p2, p1);
      hide(s2, x + 1, 0, 3);
      asm volatile("" : "+v"(s2));
      __builtin_amdgcn_sched_barrier(0);
      PA_HALF(KS, s2, s1, p2, p1)
      finish(s2, p1);
    }
#undef PA_HALF
#undef PA_PAIR
  };
  // Values behind the last token, and of a page that is not mapped: zeros, as soon as this wavefront's loads of them have
  // landed (and before the barrier behind which the others read them).
  const int rows_in = at.len - (p0 + n - 1) * PA_PAGE;  // of the last page
  auto clear_stale = [&](int x, int back) __attribute__((always_inline)) {  // back: fetches of keys since page x
    const int rows = !(known >> back & 1) ? 0 : x < n - 1 ? PA_PAGE : rows_in;
    if (rows >= PA_PAGE) return;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int piece = (wave * NP + i) * 64 + lane;
      if (piece / SEG >= rows) *(uint4*)(pa_dyn + (NB + ((x & 3) ^ (x >> 1 & 1))) * PAGE + piece * 16) = make_uint4(0, 0, 0, 0);
    }
  };
  auto turn_k = [&](int x) __attribute__((always_inline)) {  // the bit in which the buffers of pages x and x + 1 differ
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) k_off[ks] ^= x & 1 ? 2 * PAGE : PAGE;
  };
  auto turn_v = [&](int x) __attribute__((always_inline)) {
#pragma unroll
    for (int ft = 0; ft < FT; ++ft)
#pragma unroll
      for (int e = 0; e < 2; ++e) v_off[ft][e] ^= x & 1 ? 2 * PAGE : PAGE;
  };
  if (KW == 1 && n > 0) {
    lz_landed<6 * NP>();  // keys of page 0
    lds_barrier();
    products(sa, 0);
    products(sb, 1);
    hide(sa, 0, 0, 3);
    (void)settle(sa, pa, highest(sa));
    for (int x = 0; x < n; ++x) {
      lz_landed<4 * NP>();  // keys of x + 1, values of x
      clear_stale(x, 3);
      lds_barrier();        // ... of all wavefronts; keys of x and values of x - 1 have been read
      const unsigned long long v_from = v_pool + place;
      place = page_place(x + 4);
      turn_k(x);
      step(x, v_from, v_buffer(x + 3), k_pool + place, k_buffer(x + 4), sb, sa, pa, pb);
      turn_v(x);
    }
    lz_landed<0>();
  }
  if (KW == 2 && n > 0) {
    lz_landed<5 * NP>();  // keys of pages 0 and 1
    lds_barrier();
    products(sa, 0);
    turn_k(0);
    products(sb, 0);
    hide(sa, 0, kg, 4);
    (void)settle(sa, pa, highest(sa));
    lz_landed<3 * NP>();
    lds_barrier();  // (the keys of page 0 have been read)
    fetch(k_pool + place_k, k_buffer(4));
    auto one = [&](int x, f32x16_t& s1, f32x16_t& s2, pa_u4 (&p1)[2], pa_u4 (&p2)[2]) __attribute__((always_inline)) {
      lz_landed<4 * NP>();  // keys of x + 2, values of x
      clear_stale(x, 4);
      lds_barrier();        // ... of all wavefronts; keys of x + 1 and values of x - 1 have been read
      const unsigned long long v_from = v_pool + place;
      place = place_k;
      place_k = page_place(x + 5);
      turn_k(x + 1);
      step(x, v_from, v_buffer(x + 3), k_pool + place_k, k_buffer(x + 5), s1, s2, p1, p2);
      turn_v(x);
    };
    for (int x = 0; x < n; x += 2) {
      one(x, sb, sa, pa, pb);
      if (x + 1 < n) one(x + 1, sa, sb, pb, pa);
    }
    lz_landed<0>();
  }
  if constexpr (KW == 2) {  // the halves' results meet in the buffers
    float* const mine = (float*)pa_dyn + rg * (FT * 16 + 2) * 64 + lane * 4;
    float* const mine_l = (float*)pa_dyn + rg * (FT * 16 + 2) * 64 + FT * 16 * 64 + lane;
    lds_barrier();
    if (kg == 1) {
#pragma unroll
      for (int ft = 0; ft < FT; ++ft)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4)
          *(f32x4_t*)(mine + (ft * 4 + i4) * 256) = f32x4_t{acc[ft][4 * i4], acc[ft][4 * i4 + 1], acc[ft][4 * i4 + 2], acc[ft][4 * i4 + 3]};
      mine_l[0] = ref;
      mine_l[64] = l_run;
    }
    lds_barrier();
    if (kg == 1) return;
    const float ref1 = mine_l[0], to = fmaxf(ref, ref1);
    // (neither has a finite score: the sums are zero, or scores that are not numbers, which the sums keep)
    const float f0 = to > HILS_NEG_INF ? __builtin_amdgcn_exp2f(ref - to) : 1.f, f1 = to > HILS_NEG_INF ? __builtin_amdgcn_exp2f(ref1 - to) : 1.f;
#pragma unroll
    for (int ft = 0; ft < FT; ++ft)
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        const f32x4_t x = *(const f32x4_t*)(mine + (ft * 4 + i4) * 256);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[ft][4 * i4 + i] = fmaf(acc[ft][4 * i4 + i], f0, x[i] * f1);
      }
    l_run = fmaf(l_run, f0, mine_l[64] * f1);
    ref = to;
  }

  // accumulator register i of tile ft is feature ft*32 + (i >> 2)*8 + 4h + (i & 3) of row `col`
  const hils_uint2v two = __builtin_amdgcn_permlane32_swap(__float_as_uint(l_run), __float_as_uint(l_run), false, false);
  const float l = __uint_as_float(two.x) + __uint_as_float(two.y);
  const float m = ref / dm.c2;  // (score units, as the joined shares have it)
  const long row = ((long)at.slot * dm.T + my_t) * dm.HQ + hk * dm.G + my_g;
  float all = 0.f;
#pragma unroll
  for (int ft = 0; ft < FT; ++ft)
#pragma unroll
    for (int i = 0; i < 16; ++i) all += acc[ft][i];
  if (r < r1) {
#pragma unroll
    for (int ft = 0; ft < FT; ++ft)
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        const f32x4_t x = {acc[ft][4 * i4], acc[ft][4 * i4 + 1], acc[ft][4 * i4 + 2], acc[ft][4 * i4 + 3]};
        paged_store4<D>(dm, out, row, ft * 8 + i4 * 2 + h, x, m, l);
      }
  }
  uint64_t odd = __ballot(r < r1 && !(fabsf(all) < INFINITY));
  odd = (odd | odd >> 32) & 0xffffffffu;
  if (odd) {
    __builtin_amdgcn_s_waitcnt(0);  // (the stores above are in memory before the same wavefront writes there again)
    while (odd) {
      const int i = __builtin_ctzll(odd);
      odd &= odd - 1;
      const int rr = r0 + rg * 32 + i, tr = hils_udiv(rr, dm.G, dm.g_magic), gr = rr - tr * dm.G;
      const int left = TREE ? left_s[tr - t0] : paged_left(sp.base + tr, dm);
      paged_redo_row<D, 1>(dm, out, q + b * dm.q_sb + tr * dm.q_st + (hk * dm.G + gr) * dm.q_sh, k, v, table, hk, sp.base, sp.p0,
                        sp.p1, tr, left, TREE ? mask_s + (tr - t0) * PA_WORDS : nullptr,
                        ((long)at.slot * dm.T + tr) * dm.HQ + hk * dm.G + gr, 0, lane);
    }
  }
}

// ---- shares of a range added up ------------------------------------------------------------------
// A wavefront a row: lane i weighs share i (there are up to 64), then groups of D / 4 lanes take every GR-th share, four loads
// under way, and add up across the groups.  Bound by HBM or the launch: 8192 rows of 8 shares (34 MB) in 7.5 to 10 us, 512 in 5.
template <int D>
__global__ void __launch_bounds__(256) paged_attn_join(PagedDims dm, PagedOut out) {
  constexpr int LPR = D / 4, GR = 64 / LPR;  // lanes per row of features, groups
  const int rows = dm.T * dm.HQ, at = blockIdx.x * 4 + (threadIdx.x >> 6), b = blockIdx.y;
  const int lane = threadIdx.x & 63, d4 = lane % LPR, gr = lane / LPR;
  if (at >= rows) return;  // (a whole wavefront)
  int n_split = dm.n_split, slot = b * n_split;
  if (dm.ragged) {
    const int n = paged_ragged(dm, lane, lane < dm.B ? dm.lengths[lane] : 0), behind = paged_scan(n);
    n_split = __builtin_amdgcn_readlane(n, b);
    slot = __builtin_amdgcn_readlane(behind, b) - n_split;
  }
  const long row = (long)b * rows + at, first = (long)slot * rows + at;
  const float* ml = out.part + out.n_rows * dm.n_split * D + first * 2;
  const float* part = out.part + first * D + d4 * 4;
  float m = HILS_NEG_INF, l = 0.f;
  if (lane < n_split) {
    m = ml[2l * lane * rows];
    l = ml[2l * lane * rows + 1];
  }
  const float M = wave_max(m);
  // (a share that saw nothing counts for nothing, whatever lies there)
  const float f = l == 0.f ? 0.f : M > HILS_NEG_INF ? __builtin_amdgcn_exp2f((m - M) * dm.c2) : 1.f;
  const float L = wave_sum(l == 0.f ? 0.f : f * l);
  f32x4_t x = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = gr; s0 < n_split + gr; s0 += 4 * GR) {
    f32x4_t y[4];
    float w[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int s = s0 + u * GR;
      w[u] = __shfl(f, s & 63, 64);
      w[u] = s < n_split ? w[u] : 0.f;
      y[u] = *(const f32x4_t*)(part + (long)(s < n_split ? s : 0) * rows * D);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = w[u] != 0.f ? fmaf(w[u], y[u][i], x[i]) : x[i];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (GR == 4) x[i] += __shfl_xor(x[i], 16, 64);
    x[i] += __shfl_xor(x[i], 32, 64);
  }
  if (gr) return;
  const float inv = L == 0.f ? 0.f : 1.f / L;
  uint2 pk;
  pk.x = pack_bf2(x[0] * inv, x[1] * inv);
  pk.y = pack_bf2(x[2] * inv, x[3] * inv);
  *(uint2*)(out.o + row * D + d4 * 4) = pk;
  if (d4 == 0) out.lse[row] = L == 0.f ? HILS_NEG_INF : (M * dm.c2 + __builtin_amdgcn_logf(L)) * HILS_LN2;
}

// ---- host ----------------------------------------------------------------------------------------
struct PagedPlan {
  bool past;           // values are read past the caches
  int rows, nw, kw;    // rows a workgroup; wavefronts of the tile kernel and those that share a row (0: the row kernel)
  int vs;              // workgroups of a row block that have a part of the values' features each
  int n_blk, n_split;
};

// Which kernel, and over how many workgroups a range of keys is split.
// What the variants cost, in microseconds, from sweeps of every variant and share count over 1 to 32 sequences, 1 to 128 new
// tokens, windows of 512 tokens and contexts of 512 to 32768: a launch is about
//   fixed + rounds * (start + page * pages of a share)
// or, where that is longer, the bytes read once at 7 TB/s or those that all workgroups read at 19.5 TB/s; a round is one
// workgroup on every compute unit, and where a second one fits beside it (heads of 64) the two take (1 + beside) rounds.  More
// than one share adds the join, its results written and read at 3.1 TB/s.  The choice that this predicts to be shortest was
// within 2 % of the best measured one on average and within 17 % in the worst of 187 calls; fixed
// thresholds on rows and pages were 15 % off on average and lost up to 1.7 times (1 token, 8 KV heads of 128, 4096 tokens: 8
// shares 12.9 us, 32 shares 8.5; 16 tokens, 2 KV heads of 64, window 512: 32 rows a workgroup 10.1, 16 rows 7.5).
// What this does not cover: page tables much wider than the sequences.  All pages that the table and the window allow count,
// and short sequences in a long table are cut into shares, and given row blocks, that are meant for more keys: 512 tokens, 32 / 8
// heads of 128, in tables of 8 and of 2048 pages: one token of one sequence 7.3 and 8.8 us, of 16 sequences 7.8 and 24, four
// trees of 64 (4 KV heads) 15 and 29.  And `page` of the 256-row variant is that of a chip with few workgroups.
struct PagedCost {
  int rows, vs, nw, kw;
  float fixed, start, page, beside;
};
static const PagedCost kPagedCost128[] = {{16, 1, 0, 0, 1.1f, 3.9f, 0.53f, 1.f}, {16, 2, 0, 0, 1.0f, 3.5f, 0.44f, 1.f},
                                          {16, 4, 0, 0, 1.0f, 3.1f, 0.42f, 1.f}, {32, 1, 0, 0, 3.9f, 3.8f, 0.74f, 1.f},
                                          {64, 1, 4, 2, 4.9f, 2.4f, 0.76f, 1.f}, {128, 1, 8, 2, 6.4f, 2.1f, 0.95f, 1.f},
                                          {256, 1, 8, 1, 6.9f, 0.f, 1.59f, 1.f}};
static const PagedCost kPagedCost64[] = {{16, 1, 0, 0, 2.3f, 2.2f, 0.26f, 0.81f}, {16, 2, 0, 0, 2.4f, 1.9f, 0.21f, 0.81f},
                                         {32, 1, 0, 0, 3.7f, 1.9f, 0.47f, 0.49f}, {64, 1, 4, 2, 4.3f, 2.1f, 0.56f, 0.46f},
                                         {128, 1, 4, 1, 6.3f, 0.f, 0.88f, 0.53f}};

static PagedPlan paged_choose(int B, int T, int HQ, int H, int D, int window, int max_pages) {
  PagedPlan best = {};
  const int G = HQ / H;
  const long rows = (long)T * G, cus = hils_device_cus();
  const auto pages_of = [&](long tokens) {  // pages that `tokens` new tokens and the window before them can lie on
    const long pages = ((long)window + tokens + 2 * PA_PAGE - 3) / PA_PAGE;
    return pages < max_pages ? pages : max_pages;
  };
  const float read = (float)B * H * pages_of(T) * PA_PAGE * D * 4 / 7e6f;
  // Sequences of a batch differ in length where the window does not make their ranges alike, and the last workgroups run alone:
  // smaller ones are better by about a twentieth of one's time (16 sequences of 16K to 32K, 8 KV heads of 128: 2 shares 255 us,
  // 4 shares 237; all of 8K: 81 and 85).
  const bool uneven = B > 1 && pages_of(T) == max_pages;
  float least = 0.f;
  const PagedCost* cost = D == 128 ? kPagedCost128 : kPagedCost64;
  for (int i = 0; i < (D == 128 ? 7 : 5); ++i) {
    const PagedCost& c = cost[i];
    const int per = c.rows;
    if (per > 16 && rows <= per / 2) break;  // (the variants before hold every row with fewer of them empty)
    const long n_blk = (rows + per - 1) / per, tokens = per / G + 1 > PA_MAX_TREE ? per / G + 1 : PA_MAX_TREE;
    const long pages = pages_of(T < tokens ? T : tokens);
    for (int n_split = 1; n_split <= 64 && (n_split == 1 || 2 * n_split <= pages); n_split += n_split < 4 ? 1 : n_split / 4) {
      const long wgs = n_blk * c.vs * n_split * H * B, n = (wgs + cus - 1) / cus;
      const float rounds = c.beside < 1.f ? (n / 2) * (1.f + c.beside) + n % 2 : (float)n;
      const float one = c.start + c.page * ((pages + n_split - 1) / n_split), work = rounds * one;
      const float near = (float)wgs * ((pages + n_split - 1) / n_split) * PA_PAGE * D * 2 * (1.f + 1.f / c.vs) / 19.5e6f;
      // (the fourth powers: a sweep near two bounds takes longer than either)
      const auto fourth = [](float x) { return x * x * x * x; };
      float t = c.fixed + (uneven ? 0.05f * one : 0.f) + sqrtf(sqrtf(fourth(work) + fourth(read) + fourth(near)));
      if (n_split > 1) t += 3.5f + (float)B * rows * H * n_split * (D + 2) * 8 / 3.1e6f;
      if (best.n_blk && t >= least) continue;
      least = t;
      best.rows = c.rows;
      best.vs = c.vs;
      best.nw = c.nw;
      best.kw = c.kw;
      best.n_blk = (int)n_blk;
      best.n_split = n_split;
    }
  }
  // One row block of 16 reads a key and a value once.  Where all of them do not fit the last cache, values go past it: 16 sequences
  // of 16K to 32K, 8 KV heads of 128 (1.54 GB): 277 -> 255 us; where they fit, and are there from the call before, that would lose
  // (32768 tokens, 8 heads of 128: 28 -> 33 us).  Keys are read 64 bytes of a row at a time, half a cache line, and lose by it
  // at any size.
  best.past = best.rows == 16 && best.n_blk == 1 && best.vs == 1 &&
              (double)B * H * pages_of(T) * PA_PAGE * D * 4 > HILS_LAST_CACHE;
  return best;
}

// (The choice takes 0.6 us; a thread that asks for the same sizes again, as a workspace's size and the call do, gets the same.)
static PagedPlan paged_plan(int B, int T, int HQ, int H, int D, int window, int max_pages) {
  static thread_local int sizes[8];
  static thread_local PagedPlan plan;
  const int now[8] = {B, T, HQ, H, D, window, max_pages, hils_device_cus()};
  if (memcmp(sizes, now, sizeof(now))) {
    plan = paged_choose(B, T, HQ, H, D, window, max_pages);
    memcpy(sizes, now, sizeof(now));
  }
  return plan;
}

static size_t paged_ws(const PagedPlan& pl, long rows, int D) {
  return pl.n_split > 1 ? (size_t)rows * pl.n_split * (D + 2) * sizeof(float) : 0;
}

extern "C" size_t hils_paged_attn_workspace(int B, int T, int HQ, int H, int D, int window, int max_pages) {
  if (B <= 0 || T <= 0 || H <= 0 || HQ <= 0 || HQ % H != 0 || window <= 0 || max_pages <= 0) return 0;
  return paged_ws(paged_plan(B, T, HQ, H, D, window, max_pages), (long)B * T * HQ, D);
}

template <int D, bool TREE>
static int paged_launch(const PagedPlan& pl, const bf16_t* q, const bf16_t* k, const bf16_t* v, const PagedDims& dm,
                        const PagedOut& out, hipStream_t st) {
  const dim3 grid((unsigned)(((long)dm.n_blk * pl.vs * dm.n_split * dm.H * dm.B + 7) / 8 * 8));
#define PA_TILES(NW_, KW_)                                                                           \
  do {                                                                                               \
    static HilsLdsReserve reserved;                                                                  \
    const auto kern = paged_attn_tiles<D, NW_, KW_, TREE>;                                           \
    constexpr size_t smem = paged_tiles_smem<D, NW_, KW_, TREE>();                                   \
    if (int rc = hils_reserve_lds(&reserved, (const void*)kern, smem, "hils_paged_attn")) return rc; \
    hipLaunchKernelGGL(kern, grid, dim3(NW_ * 64), smem, st, q, k, v, dm, out);                      \
  } while (0)
  constexpr int VS4 = D == 128 ? 4 : 2;  // (heads of 64 gain nothing by four)
  if (pl.vs == 4) hipLaunchKernelGGL((paged_attn_rows<D, 1, 8, TREE, false, VS4>), grid, dim3(512), 0, st, q, k, v, dm, out);
  else if (pl.vs == 2) hipLaunchKernelGGL((paged_attn_rows<D, 1, 8, TREE, false, 2>), grid, dim3(512), 0, st, q, k, v, dm, out);
  else if (pl.rows == 16 && pl.past) hipLaunchKernelGGL((paged_attn_rows<D, 1, 8, TREE, true, 1>), grid, dim3(512), 0, st, q, k, v, dm, out);
  else if (pl.rows == 16) hipLaunchKernelGGL((paged_attn_rows<D, 1, 8, TREE, false, 1>), grid, dim3(512), 0, st, q, k, v, dm, out);
  else if (pl.rows == 32) hipLaunchKernelGGL((paged_attn_rows<D, 2, 4, TREE, false, 1>), grid, dim3(256), 0, st, q, k, v, dm, out);
  else if (pl.rows == 64) PA_TILES(4, 2);
  else if constexpr (D == 64) PA_TILES(4, 1);
  else if (pl.rows == 128) PA_TILES(8, 2);
  else PA_TILES(8, 1);
#undef PA_TILES
  if (dm.n_split > 1) {
    hipLaunchKernelGGL((paged_attn_join<D>), dim3((dm.T * dm.HQ + 3) / 4, dm.B), dim3(256), 0, st, dm, out);
  }
  return HILS_OK;
}

extern "C" int hils_paged_attn(const void* q, const void* k_pages, const void* v_pages, const int32_t* page_table,
                               const int32_t* lengths, const int32_t* parents, void* o, float* lse, void* workspace,
                               size_t workspace_bytes, size_t q_batch_stride, size_t q_token_stride, size_t q_head_stride,
                               int B, int T, int HQ, int H, int D, int max_pages, int num_pages, int seq_len,
                               int parents_per_batch, int window, int mask_lmk, int expand_to_chunk, float sm_scale,
                               void* stream) {
  HILS_REQUIRE(q && k_pages && v_pages && page_table && o && lse, "hils_paged_attn: null pointer");
  HILS_REQUIRE(B > 0 && T > 0 && HQ > 0 && H > 0 && max_pages > 0 && num_pages > 0, "hils_paged_attn: sizes must be positive");
  HILS_REQUIRE(HQ % H == 0, "hils_paged_attn: HQ (%d) must be a multiple of H (%d)", HQ, H);
  HILS_REQUIRE(D == 64 || D == 128, "hils_paged_attn: head dim (%d) must be 64 or 128", D);
  HILS_REQUIRE(window >= 1, "hils_paged_attn: window must be positive");
  HILS_REQUIRE(sm_scale > 0.f && sm_scale < INFINITY, "hils_paged_attn: sm_scale must be positive and finite");
  HILS_REQUIRE(!parents || T <= PA_MAX_TREE, "hils_paged_attn: a tree has at most %d tokens (got %d)", PA_MAX_TREE, T);
  HILS_REQUIRE(max_pages <= (1 << 24), "hils_paged_attn: the page table is too wide");
  HILS_REQUIRE(lengths || (seq_len >= T && seq_len <= (long)max_pages * PA_PAGE),
               "hils_paged_attn: seq_len %d is shorter than the %d tokens or longer than the page table", seq_len, T);
  HILS_REQUIRE(B <= 65535 && H <= 65535 && (long)T * (HQ / H) * (HQ / H) < (1l << 31) && (long)T * HQ < (1l << 31) - 4, "hils_paged_attn: sizes too large for the grid");
  HILS_REQUIRE(q_batch_stride % 8 == 0 && q_token_stride % 8 == 0 && q_head_stride % 8 == 0 && (uintptr_t)q % 16 == 0,
               "hils_paged_attn: q's strides and address must be multiples of 16 bytes");
  HILS_REQUIRE((uintptr_t)k_pages % 16 == 0 && (uintptr_t)v_pages % 16 == 0 && (uintptr_t)workspace % 16 == 0,
               "hils_paged_attn: pages and workspace must lie at multiples of 16 bytes");
  HILS_REQUIRE((uintptr_t)o % 8 == 0 && (uintptr_t)lse % 4 == 0, "hils_paged_attn: o must lie at a multiple of 8 bytes, lse of 4 bytes");
  const PagedPlan pl = paged_plan(B, T, HQ, H, D, window, max_pages);
  const long rows = (long)B * T * HQ;
  HILS_REQUIRE((long)pl.n_blk * pl.vs * pl.n_split * H * B < (1l << 31) - 8, "hils_paged_attn: sizes too large for the grid");
  const size_t need = paged_ws(pl, rows, D);
  HILS_REQUIRE(need == 0 || (workspace && workspace_bytes >= need),
               "hils_paged_attn: workspace too short: %zu bytes, %zu needed", workspace_bytes, need);
  PagedDims dm{B, T, HQ, H, HQ / H, window, expand_to_chunk, mask_lmk, max_pages, num_pages, seq_len, pl.n_blk, pl.n_split,
               lengths && pl.n_split > 1 && B > 1 && B <= 64,
               parents_per_batch ? T : 0, hils_udiv_magic(HQ / H), sm_scale * HILS_LOG2E, (long)q_batch_stride,
               (long)q_token_stride, (long)q_head_stride, page_table, lengths, parents};
  PagedOut out{(bf16_t*)o, lse, (float*)workspace, rows};
  hipStream_t st = (hipStream_t)stream;
  const bf16_t *qq = (const bf16_t*)q, *kk = (const bf16_t*)k_pages, *vv = (const bf16_t*)v_pages;
  int rc;
  if (D == 64) rc = parents ? paged_launch<64, true>(pl, qq, kk, vv, dm, out, st) : paged_launch<64, false>(pl, qq, kk, vv, dm, out, st);
  else rc = parents ? paged_launch<128, true>(pl, qq, kk, vv, dm, out, st) : paged_launch<128, false>(pl, qq, kk, vv, dm, out, st);
  if (rc) return rc;
  HILS_CHECK_LAUNCH("hils_paged_attn");
  return HILS_OK;
}
