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
//   paged_attn_tiles  128 rows a workgroup, 32 a wavefront, pages staged in LDS (bound by the matrix and vector units).
// A long range of keys is split over workgroups; paged_attn_join adds their shares up, in a fixed order.
// Scores, maxima, sums and outputs are fp32; probabilities are rounded to bf16 for the second product (half a step of
// 2^-9 each, of random sign, about the size of the output's own rounding), their sum is taken before the rounding.
//
// Values at slots that a row does not see meet a probability of exactly 0, which an infinity or a NaN there (a stale slot
// behind the last token, a rejected draft) would turn into a NaN.  A row whose result is no finite number is therefore
// computed once more, token by token over the slots that it sees alone (paged_redo_row): the common call pays a comparison.
#include "common.h"
#include "../../include/hils_amd.h"

#define PA_PAGE 64
#define PA_MAX_TREE 256                       // drafted tokens of a tree
#define PA_WORDS (PA_MAX_TREE / 32 + 3)       // mask words of a token: one of zeros before, two behind
typedef unsigned pa_u4 __attribute__((ext_vector_type(4)));
typedef short pa_s4 __attribute__((ext_vector_type(4)));
typedef short pa_s8 __attribute__((ext_vector_type(8)));

struct PagedDims {
  int B, T, HQ, H, G, window, expand, mask_lmk, max_pages, num_pages, seq_len, n_blk, n_split, parents_stride;
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

__device__ __forceinline__ PagedSpan paged_span(const PagedDims& dm, int b, int r0, int r1, int share) {
  PagedSpan sp;
  const int len = dm.lengths ? dm.lengths[b] : dm.seq_len;
  sp.base = len - dm.T;
  sp.alive = len >= dm.T;
  const int t0 = dm.parents ? 0 : (int)hils_udiv(r0, dm.G, dm.g_magic);
  const int t1 = dm.parents ? dm.T - 1 : (int)hils_udiv(r1 - 1, dm.G, dm.g_magic);
  int lo = paged_left(sp.base + t0, dm);
  sp.lo = lo > 0 ? lo : 0;
  const long end = (long)dm.max_pages * PA_PAGE;
  sp.hi = sp.base + t1 + 1 < end ? sp.base + t1 + 1 : (int)end;
  const int first = sp.lo / PA_PAGE;
  int n = sp.alive ? (sp.hi + PA_PAGE - 1) / PA_PAGE - first : 0;
  n = n > 0 ? n : 0;
  const int per = (n + dm.n_split - 1) / dm.n_split;
  const int a = share * per < n ? share * per : n;
  sp.p0 = first + a;
  sp.p1 = first + (a + per < n ? a + per : n);
  return sp;
}

// Ancestors of the tokens t0 .. t0 + nt - 1 as bits of slots base + u, and the first committed slot each sees.  A token whose
// way to the root passes a parent that is neither -1 nor an earlier token takes no part: it sees nothing.
// par_s: T words, mask_s: nt rows of PA_WORDS, left_s: nt words.  Ends without a barrier.
__device__ __forceinline__ void paged_tree(const PagedDims& dm, int b, int base, int t0, int nt, int tid, int n_thr, int* par_s,
                                           unsigned* mask_s, int* left_s) {
  const int32_t* par = dm.parents + (long)b * dm.parents_stride;
  for (int i = tid; i < dm.T; i += n_thr) par_s[i] = par[i];
  for (int i = tid; i < nt * PA_WORDS; i += n_thr) mask_s[i] = 0;
  __syncthreads();
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
  float* part;   // (rows, shares, D) fp32, then (rows, shares, 2): maximum (score units) and sum
  long n_rows;
};

template <int D>
__device__ __forceinline__ void paged_store4(const PagedDims& dm, const PagedOut& out, long row, int share, int d4, f32x4_t x,
                                             float M, float L) {
  if (dm.n_split > 1) {
    float* p = out.part + (row * dm.n_split + share) * D + d4 * 4;
    *(f32x4_t*)p = x;
    if (d4 == 0) {
      float* ml = out.part + out.n_rows * dm.n_split * D + (row * dm.n_split + share) * 2;
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
template <int D>
__device__ __forceinline__ void paged_redo_row(const PagedDims& dm, const PagedOut& out, const bf16_t* qr, const bf16_t* k,
                                            const bf16_t* v, const int32_t* table, int hk, int base, int p0, int p1, int t,
                                            int left, const unsigned* mask_row, long row, int share, int lane) {
  float m = HILS_NEG_INF, l = 0.f, x[D / 64];
#pragma unroll
  for (int f = 0; f < D / 64; ++f) x[f] = 0.f;
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
    for (int f = 0; f < D / 64; ++f) x[f] *= corr;
    uint64_t who = __ballot(see);
    while (who) {
      const int i = __builtin_ctzll(who);
      who &= who - 1;
      const float pe = __shfl(e, i, 64);
#pragma unroll
      for (int f = 0; f < D / 64; ++f) x[f] = fmaf(pe, bf2f(v[at + (long)i * D + f * 64 + lane]), x[f]);
    }
  }
  if (dm.n_split > 1) {
    float* part = out.part + (row * dm.n_split + share) * D;
#pragma unroll
    for (int f = 0; f < D / 64; ++f) part[f * 64 + lane] = x[f];
    if (lane == 0) {
      float* ml = out.part + out.n_rows * dm.n_split * D + (row * dm.n_split + share) * 2;
      ml[0] = m;
      ml[1] = l;
    }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int f = 0; f < D / 64; ++f) out.o[row * D + f * 64 + lane] = f2bf(x[f] * inv);
  if (lane == 0) out.lse[row] = l == 0.f ? HILS_NEG_INF : (m * dm.c2 + __builtin_amdgcn_logf(l)) * HILS_LN2;
}

// ---- few rows ----------------------------------------------------------------------------------
// 16 NR rows a workgroup; units of 32 tokens (half a page) go to its wavefronts in turn, the next unit's keys and values
// under way while one is worked on; the wavefronts' results meet in LDS.  K rows are read straight into A operands (a lane 16
// bytes of its token's row), V goes through the wavefront's own LDS area and is read by the transposing load.
template <int D, int NR, int NWV, bool TREE>
__global__ void __launch_bounds__(NWV * 64) __attribute__((amdgpu_waves_per_eu(NR == 2 && D == 128 ? 1 : 2)))
paged_attn_rows(const bf16_t* __restrict__ q, const bf16_t* __restrict__ k, const bf16_t* __restrict__ v, PagedDims dm,
                PagedOut out) {
  constexpr int KS = D / 32, MT = D / 16, ROWS = 16 * NR;
  constexpr int VL = D / 8, TPI = 64 / VL, VI = 32 / TPI;  // lanes per V row, rows per load, loads per unit
  constexpr int VP = 2 * D + 16, OP = D + 4;
  constexpr int AREA = 32 * VP > ROWS * OP * 4 ? 32 * VP : ROWS * OP * 4;
  __shared__ __align__(16) unsigned char area_s[NWV * AREA];
  __shared__ float m_s[NWV][ROWS], l_s[NWV][ROWS];
  __shared__ int par_s[TREE ? PA_MAX_TREE : 1], left_s[ROWS];
  __shared__ unsigned mask_s[TREE ? ROWS * PA_WORDS : 1], odd_s;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, j = lane >> 4;
  const int blk = blockIdx.x / dm.n_split, share = blockIdx.x % dm.n_split, hk = blockIdx.y, b = blockIdx.z;
  const int n_rows = dm.T * dm.G, r0 = blk * ROWS;
  const int r1 = r0 + ROWS < n_rows ? r0 + ROWS : n_rows;
  const PagedSpan sp = paged_span(dm, b, r0, r1, share);
  const int32_t* table = dm.table + (long)b * dm.max_pages;
  const int t0 = hils_udiv(r0, dm.G, dm.g_magic);

  const int u0 = sp.p0 * 2, u1 = sp.p1 * 2;
  // page of the units that this wavefront takes: lane i holds that of its i-th one
  int pages_of = -1;
  auto ask_pages = [&](int first) __attribute__((always_inline)) {
    const int u = first + lane * NWV;
    pages_of = u < u1 ? table[u >> 1] : -1;
  };
  ask_pages(u0 + wave);
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
  const bf16_t* vb = v + (long)hk * PA_PAGE * D + lane * 8;
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
    for (int i = 0; i < VI; ++i) vd[i] = *(const pa_u4*)(vp + i * TPI * D);
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
    // two units' loads in flight; past the last unit the same one is asked for again and not worked on
    pa_u4 ka[2][KS], va[VI], kc[2][KS], vc[VI];
    int n_mine = u1 > u0 + wave ? (u1 - u0 - wave + NWV - 1) / NWV : 0;
    auto page_at = [&](int i) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(pages_of, i & 63); };
    int pg_a = page_at(0), pg_c;
    if (n_mine > 0) issue(ka, va, pg_a, (u0 + wave) & 1);
    if (TREE) paged_tree(dm, b, sp.base, t0, ROWS, tid, NWV * 64, par_s, mask_s, left_s);
    if (tid == 0) odd_s = 0;
    __syncthreads();
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
      if ((i & 63) == 0) ask_pages(u0 + wave + i * NWV);
      return page_at(i);
    };
    int u = u0 + wave, i = 0;
    for (; i + 1 < n_mine; i += 2, u += 2 * NWV) {
      pg_c = next_page(i + 1);
      issue(kc, vc, pg_c, (u + NWV) & 1);
      if ((unsigned)pg_a < (unsigned)dm.num_pages) unit(ka, va, u);
      const bool more = i + 2 < n_mine;  // (else the last one is asked for again and not worked on)
      pg_a = more ? next_page(i + 2) : pg_c;
      issue(ka, va, pg_a, (more ? u : u + NWV) & 1);
      if ((unsigned)pg_c < (unsigned)dm.num_pages) unit(kc, vc, u + NWV);
    }
    if (i < n_mine && (unsigned)pg_a < (unsigned)dm.num_pages) unit(ka, va, u);
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
  for (int p = tid; p < ROWS * (D / 4); p += NWV * 64) {
    const int rr = p / (D / 4), d4 = p % (D / 4), r = r0 + rr;
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
    const long row = ((long)b * dm.T + t) * dm.HQ + hk * dm.G + g;
    paged_store4<D>(dm, out, row, share, d4, x, M, L);
    const float all = (x[0] + x[1]) + (x[2] + x[3]);  // (no finite number if one of them is none)
    if (!(fabsf(all) < INFINITY)) atomicOr(&odd_s, 1u << rr);
  }
  __syncthreads();
  if (const unsigned odd = odd_s; odd != 0) {
    for (int rr = wave; rr < r1 - r0; rr += NWV) {
      if (!(odd >> rr & 1)) continue;
      const int r = r0 + rr, t = hils_udiv(r, dm.G, dm.g_magic), g = r - t * dm.G;
      const long row = ((long)b * dm.T + t) * dm.HQ + hk * dm.G + g;
      int left = TREE ? left_s[t - t0] : paged_left(sp.base + t, dm);
      paged_redo_row<D>(dm, out, q + b * dm.q_sb + t * dm.q_st + (hk * dm.G + g) * dm.q_sh, k, v, table, hk, sp.base, sp.p0,
                        sp.p1, t, left, TREE ? mask_s + (t - t0) * PA_WORDS : nullptr, row, share, lane);
    }
  }
}

// ---- many rows ---------------------------------------------------------------------------------
// 32 rows a wavefront, four wavefronts; a page's keys and values go through registers into one of two LDS buffers while the
// page before is worked on.  Both row-major, 16-byte piece p of row r at p ^ (r & pieces - 1), which no read conflicts over.
template <int D>
static constexpr size_t paged_tiles_smem() { return 2 * 2 * (size_t)PA_PAGE * 2 * D; }

template <int D, bool TREE>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))
paged_attn_tiles(const bf16_t* __restrict__ q, const bf16_t* __restrict__ k, const bf16_t* __restrict__ v, PagedDims dm,
                 PagedOut out) {
  constexpr int RT = 2, NT = 256, ROWS = 128, KS = D / 32, DT = D / 16, RP = 2 * D, SEG = D / 8;
  constexpr int PT = 64 * SEG / NT;        // 16-byte pieces per thread of a page's keys (and of its values)
  constexpr int TILE = PA_PAGE * RP;       // bytes of a page's keys
  constexpr float LAZY = 6.f;              // log2 of the growth of a row's maximum that moves its reference point
  extern __shared__ __align__(16) unsigned char pa_dyn[];
  __shared__ int par_s[TREE ? PA_MAX_TREE : 1], left_s[ROWS];
  __shared__ unsigned mask_s[TREE ? ROWS * PA_WORDS : 1];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, j = lane >> 4;
  // the row blocks of a (sequence, KV head, share) read the same pages: neighbours on one XCD
  const int total = dm.n_blk * dm.n_split * dm.H * dm.B, per_xcd = (total + 7) / 8;
  const int id = (int)(blockIdx.x % 8) * per_xcd + (int)(blockIdx.x / 8);
  if (id >= total) return;
  const int blk = id % dm.n_blk, share = id / dm.n_blk % dm.n_split, pair = id / dm.n_blk / dm.n_split;
  const int hk = pair % dm.H, b = pair / dm.H;
  const int n_rows = dm.T * dm.G, r0 = blk * ROWS;
  const int r1 = r0 + ROWS < n_rows ? r0 + ROWS : n_rows;
  const PagedSpan sp = paged_span(dm, b, r0, r1, share);
  const int32_t* table = dm.table + (long)b * dm.max_pages;
  const int t0 = hils_udiv(r0, dm.G, dm.g_magic);
  const long page_el = (long)dm.H * PA_PAGE * D, head_el = (long)hk * PA_PAGE * D;

  int pages_of = -1;
  auto ask_pages = [&](int first) __attribute__((always_inline)) {
    pages_of = first + lane < sp.p1 ? table[first + lane] : -1;
  };
  auto page_at = [&](int p) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(pages_of, (p - sp.p0) & 63); };
  pa_u4 kd[PT], vd[PT];
  auto issue = [&](int page) __attribute__((always_inline)) {
    const long at = ((unsigned)page < (unsigned)dm.num_pages ? page * page_el : 0) + head_el + tid * 8;
#pragma unroll
    for (int i = 0; i < PT; ++i) kd[i] = *(const pa_u4*)(k + at + i * NT * 8);
#pragma unroll
    for (int i = 0; i < PT; ++i) vd[i] = *(const pa_u4*)(v + at + i * NT * 8);
  };
  auto put = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PT; ++i) {
      const int pc = tid + NT * i, row = pc / SEG;
      unsigned char* to = pa_dyn + buf * 2 * TILE + row * RP + ((pc % SEG) ^ (row & (SEG - 1))) * 16;
      *(pa_u4*)to = kd[i];
      *(pa_u4*)(to + TILE) = vd[i];
    }
  };
  ask_pages(sp.p0);
  int page = page_at(sp.p0);
  if (sp.p0 < sp.p1) issue(page);

  bf16x8_t qa[RT][KS];
  int row_t[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = r0 + wave * 32 + rt * 16 + col;
    const int rc = r < r1 ? r : r1 - 1;
    const int t = hils_udiv(rc, dm.G, dm.g_magic), g = rc - t * dm.G;
    row_t[rt] = r < r1 ? t : -1;
    const bf16_t* qp = q + b * dm.q_sb + t * dm.q_st + (hk * dm.G + g) * dm.q_sh + j * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qa[rt][ks] = *(const bf16x8_t*)(qp + ks * 32);
  }
  if (TREE) paged_tree(dm, b, sp.base, t0, ROWS, tid, NT, par_s, mask_s, left_s);
  if (sp.p0 < sp.p1) put(0);
  __syncthreads();
  int vlo[RT];
  unsigned vspan[RT];
  const unsigned* mrow[RT];
  int some_lo = 0x7fffffff, all_lo = 0, some_hi = 0, all_hi = 0x7fffffff;  // slots that any row sees, that all see
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const bool live = row_t[rt] >= 0 && sp.alive;
    const int i = live ? row_t[rt] - t0 : 0;
    int lo = TREE ? left_s[i] : paged_left(sp.base + row_t[rt], dm);
    lo = lo > 0 ? lo : 0;
    const int last = TREE ? sp.base - 1 : sp.base + row_t[rt];
    const bool some = live && last >= lo;
    vlo[rt] = some ? lo : 0x7fffffff;
    vspan[rt] = some ? (unsigned)(last - lo) : 0u;
    if (TREE) mrow[rt] = mask_s + i * PA_WORDS;
    if (live) {  // (a drafted token sees itself at least, one that takes no part has its window's start out of reach)
      const int from = TREE && lo < 0x7fffffff && lo > sp.base ? sp.base : lo, to = TREE ? sp.base + dm.T : last + 1;
      some_lo = from < some_lo ? from : some_lo;
      all_lo = lo > all_lo ? lo : all_lo;
      some_hi = to > some_hi ? to : some_hi;
      all_hi = last + 1 < all_hi ? last + 1 : all_hi;
    }
  }
#pragma unroll
  for (int x = 1; x < 16; x <<= 1) {
    some_lo = min(some_lo, __shfl_xor(some_lo, x, 64));
    all_lo = max(all_lo, __shfl_xor(all_lo, x, 64));
    some_hi = max(some_hi, __shfl_xor(some_hi, x, 64));
    all_hi = min(all_hi, __shfl_xor(all_hi, x, 64));
  }
  some_lo = __builtin_amdgcn_readfirstlane(some_lo);
  all_lo = __builtin_amdgcn_readfirstlane(all_lo);
  some_hi = __builtin_amdgcn_readfirstlane(some_hi);
  all_hi = __builtin_amdgcn_readfirstlane(all_hi);

  f32x4_t acc[RT][DT];
  float m_run[RT], l_run[RT];  // reference point (score units) and sum, per row (lane & 15)
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[rt][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    m_run[rt] = HILS_NEG_INF;
    l_run[rt] = 0.f;
  }
  unsigned k_off[KS], v_off[DT];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) k_off[ks] = (unsigned)(col * RP + ((ks * 4 + j) ^ (col & (SEG - 1))) * 16);
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    const int row = 4 * j + (col >> 2);
    v_off[dt] = (unsigned)(row * RP + ((dt * 2 + (col >> 1 & 1)) ^ (row & (SEG - 1))) * 16 + (col & 1) * 8);
  }

  // (the queries are here from now on: waited for inside the loop, the page under way would be waited for with them)
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qa[rt][ks]));

  auto tile_step = [&](int p, const unsigned char* k_s) __attribute__((always_inline)) {
    const unsigned char* v_s = k_s + TILE;
    f32x4_t s[RT][4];  // scores, then probabilities: slot tt*16 + 4j + i of the page, row lane & 15
    float corr[RT];
    bool rescale = false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) s[rt][tt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const bf16x8_t a = *(const bf16x8_t*)(k_s + k_off[ks] + tt * 16 * RP);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[rt][tt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, qa[rt][ks], s[rt][tt], 0, 0, 0);
        if (ks == KS - 1 && (tt & 1)) __builtin_amdgcn_sched_barrier(0);  // (operand reads of later steps stay behind)
      }
    if (p * PA_PAGE < all_lo || p * PA_PAGE + PA_PAGE > all_hi) {  // some row does not see all of the page
      const int slot0 = p * PA_PAGE + 4 * j;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const unsigned from = (unsigned)(slot0 - vlo[rt]);
        uint64_t extra = 0;
        if (TREE && p * PA_PAGE + PA_PAGE > sp.base) {
          const int off = p * PA_PAGE - sp.base;
          const unsigned x0 = off > -32 && off < dm.T ? paged_bits(mrow[rt], off) : 0u;
          const unsigned x1 = off + 32 < dm.T ? paged_bits(mrow[rt], off + 32) : 0u;
          extra = ((uint64_t)x1 << 32 | x0) >> (4 * j);
        }
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            bool see = from + (unsigned)(tt * 16 + i) <= vspan[rt];
            if (TREE && dm.mask_lmk && tt == 3 && i == 3) see = see && j != 3;
            if (TREE) see = see || (extra >> (tt * 16 + i) & 1);
            s[rt][tt][i] = see ? s[rt][tt][i] : HILS_NEG_INF;
          }
      }
    }
    // a committed landmark is its page's last token (a drafted one has been left out of the masks)
    if (dm.mask_lmk && (!TREE || p * PA_PAGE + PA_PAGE <= sp.base)) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) s[rt][3][3] = j == 3 ? HILS_NEG_INF : s[rt][3][3];
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float mx = HILS_NEG_INF;
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[rt][tt][i]);
      mx = rows_max(mx);
      // the reference point of the exponentials follows the maximum only when that grows by more than 2^LAZY, or when
      // nothing is accumulated yet: most pages rescale no accumulators
      const bool fresh = l_run[rt] == 0.f;
      const bool move = fresh | ((mx - m_run[rt]) * dm.c2 > LAZY);
      const float m_new = move ? fmaxf(m_run[rt], mx) : m_run[rt];
      const bool any = m_new > HILS_NEG_INF;
      corr[rt] = (move & any & !fresh) ? __builtin_amdgcn_exp2f((m_run[rt] - m_new) * dm.c2) : 1.f;
      const float mc = any ? m_new * dm.c2 : 0.f;
      rescale |= corr[rt] != 1.f;
      float sum = 0.f;
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = __builtin_amdgcn_exp2f(fmaf(s[rt][tt][i], dm.c2, -mc));  // masked: exp2(-inf) = 0
          s[rt][tt][i] = e;
          sum += e;
        }
      sum = rows_sum(sum);
      l_run[rt] = l_run[rt] * corr[rt] + sum;
      m_run[rt] = m_new;
    }
    if (__any(rescale)) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[rt][dt][i] *= corr[rt];
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16x8_t pb[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        pa_u4 u;
        u.x = pack_bf2(s[rt][2 * h][0], s[rt][2 * h][1]);
        u.y = pack_bf2(s[rt][2 * h][2], s[rt][2 * h][3]);
        u.z = pack_bf2(s[rt][2 * h + 1][0], s[rt][2 * h + 1][1]);
        u.w = pack_bf2(s[rt][2 * h + 1][2], s[rt][2 * h + 1][3]);
        pb[rt] = __builtin_bit_cast(bf16x8_t, u);
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const unsigned char* at = v_s + v_off[dt] + (2 * h * 16) * RP;
        const pa_s4 b0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) pa_s4*)at);
        const pa_s4 b1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) pa_s4*)(at + 16 * RP));
        const bf16x8_t a = __builtin_bit_cast(bf16x8_t, (pa_s8)__builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) acc[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pb[rt], acc[rt][dt], 0, 0, 0);
        if ((dt & 3) == 3) __builtin_amdgcn_sched_barrier(0);
      }
    }
  };

  for (int p = sp.p0; p < sp.p1; ++p) {
    const int now = page;
    if (p + 1 < sp.p1) {
      if (((p + 1 - sp.p0) & 63) == 0) ask_pages(p + 1);
      page = page_at(p + 1);
      issue(page);
    }
    if ((unsigned)now < (unsigned)dm.num_pages && p * PA_PAGE < some_hi && p * PA_PAGE + PA_PAGE > some_lo)
      tile_step(p, pa_dyn + ((p - sp.p0) & 1) * 2 * TILE);
    if (p + 1 < sp.p1) put((p + 1 - sp.p0) & 1);
    __syncthreads();
  }

#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = r0 + wave * 32 + rt * 16 + col;
    const int rc = r < r1 ? r : r1 - 1;
    const int t = hils_udiv(rc, dm.G, dm.g_magic), g = rc - t * dm.G;
    const long row = ((long)b * dm.T + t) * dm.HQ + hk * dm.G + g;
    float all = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) all += (acc[rt][dt][0] + acc[rt][dt][1]) + (acc[rt][dt][2] + acc[rt][dt][3]);
    if (r < r1) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) paged_store4<D>(dm, out, row, share, dt * 4 + j, acc[rt][dt], m_run[rt], l_run[rt]);
    }
    uint64_t odd = __ballot(r < r1 && !(fabsf(all) < INFINITY));
    odd = (odd | odd >> 16 | odd >> 32 | odd >> 48) & 0xffff;
    if (odd) {
      __builtin_amdgcn_s_waitcnt(0);  // (the stores above are in memory before the same wavefront writes there again)
      while (odd) {
        const int i = __builtin_ctzll(odd);
        odd &= odd - 1;
        const int rr = r0 + wave * 32 + rt * 16 + i, tr = hils_udiv(rr, dm.G, dm.g_magic), gr = rr - tr * dm.G;
        const int left = TREE ? left_s[tr - t0] : paged_left(sp.base + tr, dm);
        paged_redo_row<D>(dm, out, q + b * dm.q_sb + tr * dm.q_st + (hk * dm.G + gr) * dm.q_sh, k, v, table, hk, sp.base,
                          sp.p0, sp.p1, tr, left, TREE ? mask_s + (tr - t0) * PA_WORDS : nullptr,
                          ((long)b * dm.T + tr) * dm.HQ + hk * dm.G + gr, share, lane);
      }
    }
  }
}

// ---- shares of a range added up ------------------------------------------------------------------
template <int D>
__global__ void __launch_bounds__(256) paged_attn_join(PagedOut out, int n_split, float c2) {
  constexpr int LPR = D / 4;  // lanes per row, four features each
  const long row = (long)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  const int d4 = threadIdx.x % LPR;
  if (row >= out.n_rows) return;
  const float* ml = out.part + out.n_rows * n_split * D + row * n_split * 2;
  const float* part = out.part + row * n_split * D + d4 * 4;
  float M = HILS_NEG_INF;
  for (int s = 0; s < n_split; ++s) M = fmaxf(M, ml[2 * s]);
  float L = 0.f;
  f32x4_t x = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < n_split; ++s) {
    const float l = ml[2 * s + 1];
    if (l == 0.f) continue;  // (nothing seen there)
    const float f = M > HILS_NEG_INF ? __builtin_amdgcn_exp2f((ml[2 * s] - M) * c2) : 1.f;
    const f32x4_t y = *(const f32x4_t*)(part + (long)s * D);
    L = fmaf(f, l, L);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = fmaf(f, y[i], x[i]);
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  uint2 pk;
  pk.x = pack_bf2(x[0] * inv, x[1] * inv);
  pk.y = pack_bf2(x[2] * inv, x[3] * inv);
  *(uint2*)(out.o + row * D + d4 * 4) = pk;
  if (d4 == 0) out.lse[row] = L == 0.f ? HILS_NEG_INF : (M * c2 + __builtin_amdgcn_logf(L)) * HILS_LN2;
}

// ---- host ----------------------------------------------------------------------------------------
struct PagedPlan {
  bool tiles;
  int nr, n_blk, n_split;
};

// Which kernel, and over how many workgroups a range of keys is split.
static PagedPlan paged_plan(int B, int T, int HQ, int H, int window, int max_pages) {
  PagedPlan pl;
  const int rows = T * (HQ / H);
  // pages of the longest range a workgroup can have
  const long seen = (long)window + (T < 128 ? T : 128) + 2 * PA_PAGE - 3;
  const int pages = (int)(seen / PA_PAGE < max_pages ? seen / PA_PAGE : max_pages);
  pl.tiles = rows > 64 && (long)((rows + 31) / 32) * H * B * pages > 2048;
  pl.nr = rows > 16 ? 2 : 1;
  const int per = pl.tiles ? 128 : 16 * pl.nr;
  pl.n_blk = (rows + per - 1) / per;
  const long wgs = (long)pl.n_blk * H * B;
  const long want = (2l * hils_device_cus() + wgs - 1) / wgs;  // two workgroups a compute unit
  const int least = 8;                                         // pages of a share
  int most = pages / least;
  most = most > 1 ? most : 1;
  pl.n_split = (int)(want < most ? want : most);
  pl.n_split = pl.n_split > 64 ? 64 : pl.n_split;
  return pl;
}

static size_t paged_ws(const PagedPlan& pl, long rows, int D) {
  return pl.n_split > 1 ? (size_t)rows * pl.n_split * (D + 2) * sizeof(float) : 0;
}

extern "C" size_t hils_paged_attn_workspace(int B, int T, int HQ, int H, int D, int window, int max_pages) {
  if (B <= 0 || T <= 0 || H <= 0 || HQ <= 0 || HQ % H != 0 || window <= 0 || max_pages <= 0) return 0;
  return paged_ws(paged_plan(B, T, HQ, H, window, max_pages), (long)B * T * HQ, D);
}

template <int D, bool TREE>
static int paged_launch(const PagedPlan& pl, const bf16_t* q, const bf16_t* k, const bf16_t* v, const PagedDims& dm,
                        const PagedOut& out, hipStream_t st) {
  if (pl.tiles) {
    auto kern = paged_attn_tiles<D, TREE>;
    static HilsLdsReserve reserved;
    if (int rc = hils_reserve_lds(&reserved, (const void*)kern, paged_tiles_smem<D>(), "hils_paged_attn")) return rc;
    const long total = (long)dm.n_blk * dm.n_split * dm.H * dm.B;
    hipLaunchKernelGGL(kern, dim3((unsigned)((total + 7) / 8 * 8)), dim3(256), paged_tiles_smem<D>(), st, q, k, v, dm, out);
  } else {
    const dim3 grid(dm.n_blk * dm.n_split, dm.H, dm.B);
    if (pl.nr == 1) hipLaunchKernelGGL((paged_attn_rows<D, 1, 8, TREE>), grid, dim3(512), 0, st, q, k, v, dm, out);
    else hipLaunchKernelGGL((paged_attn_rows<D, 2, 4, TREE>), grid, dim3(256), 0, st, q, k, v, dm, out);
  }
  if (dm.n_split > 1) {
    const int per = 256 / (D / 4);
    hipLaunchKernelGGL((paged_attn_join<D>), dim3((unsigned)((out.n_rows + per - 1) / per)), dim3(256), 0, st, out, dm.n_split, dm.c2);
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
  HILS_REQUIRE(B <= 65535 && H <= 65535 && (long)T * (HQ / H) * (HQ / H) < (1l << 31), "hils_paged_attn: sizes too large for the grid");
  HILS_REQUIRE(q_batch_stride % 8 == 0 && q_token_stride % 8 == 0 && q_head_stride % 8 == 0 && (uintptr_t)q % 16 == 0,
               "hils_paged_attn: q's strides and address must be multiples of 16 bytes");
  const PagedPlan pl = paged_plan(B, T, HQ, H, window, max_pages);
  const long rows = (long)B * T * HQ;
  HILS_REQUIRE((long)pl.n_blk * pl.n_split * H * B < (1l << 31) - 8, "hils_paged_attn: sizes too large for the grid");
  const size_t need = paged_ws(pl, rows, D);
  HILS_REQUIRE(need == 0 || (workspace && workspace_bytes >= need),
               "hils_paged_attn: workspace too short: %zu bytes, %zu needed", workspace_bytes, need);
  PagedDims dm{B, T, HQ, H, HQ / H, window, expand_to_chunk, mask_lmk, max_pages, num_pages, seq_len, pl.n_blk, pl.n_split,
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
