// Rotary positions by position: y = R(position) x for the queries and keys of every token, and the same fused with the
// append of keys and values to a paged cache.
//
// The first R features of a head vector are R/2 pairs (x1, x2): features i and i + R/2, or 2i and 2i + 1 (interleaved).
//   y1 = s (x1 cos a - x2 sin a),   y2 = s (x2 cos a + x1 sin a),   a = position * inv_freq[i],
// the other D - R features pass through.  The backward is the same with -a (`sign`).
//
// The angle of a far position has lost its fraction of a turn in fp32 (position 10^6, inv_freq 1: steps of 0.06), so it is
// formed in turns in fp64 and reduced to [-1/2, 1/2] there; the rotation is fp64 too (fp32's rate on this chip, and the kernel
// waits for memory), so that what is rounded to bf16 is the exact value: a key in the cache is the same whatever computed
// it.
// Bound by HBM: q and k in and out.  A workgroup owns a few tokens of all heads; their R/2 angles each are worked out
// once, into LDS, for all heads (an angle costs some 60 instructions: per head they would be most of the kernel).  A
// thread's unit is 16 features that go together: two 16-byte pieces in and out, two units' loads in flight.  q and k of 8
// sequences of 8192, 16 + 16 heads of 64: 100 us (537 MB: 5.3 TB/s); of 32768 tokens, 32 + 8 heads of 128: 135 us (5.0);
// 8191 new tokens of 4 sequences into their pages, 4 KV heads: 134 us (5.0); a copy of as much runs at 4.9 to 5.4.
#include "common.h"
#include "../../include/hils_amd.h"

struct RotaryDims {
  long n_tok;                                 // B * T
  int T, HQ, H, D, R, tpb, interleaved, append, pos_wide, pos_batch, freq_wide, pos0, max_pages, num_pages, seq_len;
  uint32_t m_unit, m_head, m_tok;             // division by D/16, by the heads of a token, by T
  float scale, sign;
  long q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh;  // elements between sequences, tokens, heads
  const void* positions;                      // (B, T) or (T) int32 / int64, or null: pos0 + t (append: the token's slot)
  const void* inv_freq;                       // R/2, fp32 or fp64
  const int32_t* table;                       // (B, max_pages)
  const int32_t* lengths;                     // (B) or null: seq_len
};

#define ROT_UN 2
#define ROT_WAVES 4

// Eight pairs of a unit.  What is exact to 2^-53 goes to bf16 by way of fp32, as a conversion from fp64 does: half a step of
// bf16 and at most 2^-24 more.
template <bool INTERLEAVED>
__device__ __forceinline__ void rotary_turn(const uint4 lo, const uint4 hi, const double* c, const double* s, uint4& out_lo,
                                            uint4& out_hi) {
  float a[8], b[8], y1[8], y2[8];
  unpack8(lo, a);
  unpack8(hi, b);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const double x1 = INTERLEAVED ? (i < 4 ? a[2 * i & 7] : b[2 * i & 7]) : a[i];
    const double x2 = INTERLEAVED ? (i < 4 ? a[(2 * i + 1) & 7] : b[(2 * i + 1) & 7]) : b[i];
    y1[i] = (float)fma(x1, c[i], -(x2 * s[i]));
    y2[i] = (float)fma(x2, c[i], x1 * s[i]);
  }
  unsigned* wl = (unsigned*)&out_lo;
  unsigned* wh = (unsigned*)&out_hi;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    wl[i] = INTERLEAVED ? pack_bf2(y1[i], y2[i]) : pack_bf2(y1[2 * i], y1[2 * i + 1]);
    wh[i] = INTERLEAVED ? pack_bf2(y1[4 + i], y2[4 + i]) : pack_bf2(y2[2 * i], y2[2 * i + 1]);
  }
}

template <bool INTERLEAVED, bool APPEND>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(ROT_WAVES)))
rotary_kernel(const bf16_t* __restrict__ q, const bf16_t* __restrict__ k, const bf16_t* __restrict__ v,
              bf16_t* __restrict__ q_out, bf16_t* __restrict__ k_out, bf16_t* __restrict__ v_out, RotaryDims dm) {
  extern __shared__ __align__(16) double rot_s[];
  __shared__ long slot_s[8];  // place of a token's key in the pages, in rows of a pool's first head; -1: none
  const int half = dm.R / 2, tid = threadIdx.x;
  double* cos_s = rot_s;
  double* sin_s = rot_s + dm.tpb * half;
  const long tok0 = (long)blockIdx.x * dm.tpb;
  const int n = dm.n_tok - tok0 < dm.tpb ? (int)(dm.n_tok - tok0) : dm.tpb;
  const int b0 = (int)((unsigned long)tok0 / (unsigned)dm.T), t0 = (int)(tok0 - (long)b0 * dm.T);
  auto token = [&](int tk, int& b, int& t) __attribute__((always_inline)) {  // (a workgroup has up to eight tokens)
    t = t0 + tk;
    const int w = dm.T >= 8 ? t >= dm.T : (int)hils_udiv(t, dm.T, dm.m_tok);
    b = b0 + w;
    t -= w * dm.T;
  };
  const int U = dm.D / 16, UR = dm.R / 16, NH = dm.HQ + dm.H + (APPEND ? dm.H : 0);
  const int total = n * NH * U;
  uint4 lo[ROT_UN], hi[ROT_UN];
  bf16_t* to[ROT_UN];
  int gap[ROT_UN], tab[ROT_UN];  // elements between a unit's pieces; its first angle, -1: not rotated
  int late[ROT_UN];              // token whose place in the pages `to` waits for, -1: none
  auto load = [&](int e0) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < ROT_UN; ++x) {
      const int e = e0 + 256 * x;
      to[x] = nullptr;
      gap[x] = 8;
      tab[x] = late[x] = -1;
      lo[x] = hi[x] = make_uint4(0, 0, 0, 0);
      if (e < total) {
        const int r = hils_udiv(e, U, dm.m_unit), u = e - r * U;
        const int tk = hils_udiv(r, NH, dm.m_head);
        int h = r - tk * NH, b, t;
        token(tk, b, t);
        const bf16_t* from;
        bool turn = u < UR;
        if (h < dm.HQ) {
          from = q + b * dm.q_sb + t * dm.q_st + h * dm.q_sh;
          to[x] = q_out + ((tok0 + tk) * dm.HQ + h) * dm.D;
        } else {
          h -= dm.HQ;
          const bool is_v = h >= dm.H;
          h = is_v ? h - dm.H : h;
          turn = turn && !is_v;
          from = is_v ? v + b * dm.v_sb + t * dm.v_st + h * dm.v_sh : k + b * dm.k_sb + t * dm.k_st + h * dm.k_sh;
          if (APPEND) {
            to[x] = (is_v ? v_out : k_out) + (long)h * 64 * dm.D;
            late[x] = tk;
          } else {
            to[x] = k_out + ((tok0 + tk) * dm.H + h) * dm.D;
          }
        }
        const int first = turn && !INTERLEAVED ? u * 8 : u * 16;
        if (turn) {
          tab[x] = tk * half + u * 8;
          gap[x] = INTERLEAVED ? 8 : half;
        }
        to[x] += first;
        lo[x] = *(const uint4*)(from + first);
        hi[x] = *(const uint4*)(from + first + gap[x]);
      }
    }
  };
  load(tid);  // (under way while the angles are worked out)
  if (APPEND && tid < n) {
    int b, t;
    token(tid, b, t);
    const int len = dm.lengths ? dm.lengths[b] : dm.seq_len, slot = len - dm.T + t, c = slot >> 6;
    // (a sequence shorter than T takes no part: the tokens that it has stay as they are)
    const int page = len >= dm.T && c < dm.max_pages ? dm.table[(long)b * dm.max_pages + c] : -1;
    slot_s[tid] = (unsigned)page < (unsigned)dm.num_pages ? (long)page * dm.H * 64 + (slot & 63) : -1;
  }
  for (int i = tid; i < n * half; i += 256) {
    const int tk = i / half, f = i - tk * half;
    int b, t;
    token(tk, b, t);
    double p;
    if (dm.positions) {
      const long at = (dm.pos_batch ? (long)b * dm.T : 0) + t;
      p = dm.pos_wide ? (double)((const int64_t*)dm.positions)[at] : (double)((const int32_t*)dm.positions)[at];
    } else {
      p = APPEND ? (double)((dm.lengths ? dm.lengths[b] : dm.seq_len) - dm.T + t) : (double)((long)dm.pos0 + t);
    }
    const double w = dm.freq_wide ? ((const double*)dm.inv_freq)[f] : (double)((const float*)dm.inv_freq)[f];
    const double turns = p * (w * 0.15915494309189533577);  // 1 / (2 pi)
    double sn, cs;
    sincospi(2.0 * (turns - rint(turns)), &sn, &cs);
    // (eight units in step read angles 64 bytes apart; of two that are 256 bytes apart one reads its second pair first: 136.7 -> 134.4
    // us for the prompts' append.  Half of the LDS unit's busy cycles, a quarter of the kernel's, still count as bank conflicts.)
    const int at = i ^ (i >> 4 & 2);
    cos_s[at] = cs * dm.scale;
    sin_s[at] = sn * dm.scale * dm.sign;
  }
  __syncthreads();
  for (int e0 = tid; e0 < total; e0 += 256 * ROT_UN) {
    if (e0 != tid) load(e0);
#pragma unroll
    for (int x = 0; x < ROT_UN; ++x) {
      if (!to[x]) continue;
      if (tab[x] >= 0) {
        double c[8], sn[8];
        const int turn = tab[x] >> 4 & 2;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          c[i] = cos_s[(tab[x] + (i & 6) ^ turn) + (i & 1)];
          sn[i] = sin_s[(tab[x] + (i & 6) ^ turn) + (i & 1)];
        }
        const uint4 l0 = lo[x], h0 = hi[x];
        rotary_turn<INTERLEAVED>(l0, h0, c, sn, lo[x], hi[x]);
      }
      if (late[x] >= 0) {
        const long at = slot_s[late[x]];
        if (at < 0) continue;
        to[x] += at * dm.D;
      }
      *(uint4*)to[x] = lo[x];
      *(uint4*)(to[x] + gap[x]) = hi[x];
    }
  }
}

static int rotary_launch(const char* who, RotaryDims& dm, const void* q, const void* k, const void* v, void* q_out, void* k_out,
                         void* v_out, hipStream_t st) {
  const int heads = dm.HQ + dm.H + (dm.append ? dm.H : 0), units = heads * (dm.D / 16);
  // tokens of a workgroup: two units a thread and more, while there are a few workgroups for every compute unit
  long tpb = dm.n_tok / (4l * hils_device_cus());
  const int most = 2048 / units;
  tpb = tpb < most ? tpb : most;
  tpb = dm.R == 0 || tpb < 4096 / dm.R ? tpb : 4096 / dm.R;  // (tables of up to 32 KiB of LDS)
  dm.tpb = tpb < 1 ? 1 : tpb > 8 ? 8 : (int)tpb;
  dm.m_unit = hils_udiv_magic(dm.D / 16);
  dm.m_head = hils_udiv_magic(heads);
  dm.m_tok = hils_udiv_magic(dm.T);
  const long blocks = (dm.n_tok + dm.tpb - 1) / dm.tpb;
  HILS_REQUIRE(blocks <= 2147483647L && (long)dm.tpb * units * heads < (1l << 31), "%s: sizes too large for the grid", who);
  auto kern = dm.append ? (dm.interleaved ? rotary_kernel<true, true> : rotary_kernel<false, true>)
                        : (dm.interleaved ? rotary_kernel<true, false> : rotary_kernel<false, false>);
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(256), (size_t)dm.tpb * dm.R * sizeof(double), st, (const bf16_t*)q,
                     (const bf16_t*)k, (const bf16_t*)v, (bf16_t*)q_out, (bf16_t*)k_out, (bf16_t*)v_out, dm);
  HILS_CHECK_LAUNCH(who);
  return HILS_OK;
}

static bool rotary_aligned(const void* p, size_t sb, size_t st, size_t sh) {
  return !p || ((uintptr_t)p % 16 == 0 && sb % 8 == 0 && st % 8 == 0 && sh % 8 == 0);
}

extern "C" int hils_rotary(const void* q, const void* k, void* q_out, void* k_out, const void* positions, const void* inv_freq,
                           size_t q_batch_stride, size_t q_token_stride, size_t q_head_stride, size_t k_batch_stride,
                           size_t k_token_stride, size_t k_head_stride, int B, int T, int HQ, int H, int D, int rotary_dim,
                           int interleaved, int positions_64, int positions_per_batch, int first_position, int inv_freq_64,
                           float scale, float sin_sign, void* stream) {
  HILS_REQUIRE(q && q_out && inv_freq && (H == 0 || (k && k_out)), "hils_rotary: null pointer");
  HILS_REQUIRE(B > 0 && T > 0 && HQ > 0 && H >= 0, "hils_rotary: sizes must be positive");
  HILS_REQUIRE(D > 0 && D % 16 == 0 && D <= 1024, "hils_rotary: D (%d) must be a multiple of 16 up to 1024", D);
  HILS_REQUIRE(rotary_dim > 0 && rotary_dim % 16 == 0 && rotary_dim <= D,
               "hils_rotary: rotary_dim (%d) must be a multiple of 16 up to D (%d)", rotary_dim, D);
  HILS_REQUIRE((long)(HQ + H) * (D / 16) <= (1 << 20), "hils_rotary: too many heads");
  HILS_REQUIRE(rotary_aligned(q, q_batch_stride, q_token_stride, q_head_stride) &&
                   rotary_aligned(k, k_batch_stride, k_token_stride, k_head_stride) && rotary_aligned(q_out, 0, 0, 0) &&
                   rotary_aligned(k_out, 0, 0, 0),
               "hils_rotary: addresses and strides must be multiples of 16 bytes");
  RotaryDims dm{};
  dm.n_tok = (long)B * T;
  dm.T = T, dm.HQ = HQ, dm.H = H, dm.D = D, dm.R = rotary_dim, dm.interleaved = interleaved;
  dm.pos_wide = positions_64, dm.pos_batch = positions_per_batch, dm.pos0 = first_position, dm.freq_wide = inv_freq_64;
  dm.scale = scale, dm.sign = sin_sign;
  dm.q_sb = q_batch_stride, dm.q_st = q_token_stride, dm.q_sh = q_head_stride;
  dm.k_sb = k_batch_stride, dm.k_st = k_token_stride, dm.k_sh = k_head_stride;
  dm.positions = positions, dm.inv_freq = inv_freq;
  return rotary_launch("hils_rotary", dm, q, k, nullptr, q_out, k_out, nullptr, (hipStream_t)stream);
}

extern "C" int hils_paged_append(const void* q, const void* k, const void* v, void* q_out, void* k_pages, void* v_pages,
                                 const int32_t* page_table, const int32_t* lengths, const void* positions,
                                 const void* inv_freq, size_t q_batch_stride, size_t q_token_stride, size_t q_head_stride,
                                 size_t k_batch_stride, size_t k_token_stride, size_t k_head_stride, size_t v_batch_stride,
                                 size_t v_token_stride, size_t v_head_stride, int B, int T, int HQ, int H, int D,
                                 int rotary_dim, int interleaved, int positions_64, int inv_freq_64, int max_pages,
                                 int num_pages, int seq_len, float scale, void* stream) {
  HILS_REQUIRE(k && v && k_pages && v_pages && page_table && (HQ == 0 || (q && q_out)) && (rotary_dim == 0 || inv_freq),
               "hils_paged_append: null pointer");
  HILS_REQUIRE(B > 0 && T > 0 && HQ >= 0 && H > 0 && max_pages > 0 && num_pages > 0, "hils_paged_append: sizes must be positive");
  HILS_REQUIRE(D > 0 && D % 16 == 0 && D <= 1024, "hils_paged_append: D (%d) must be a multiple of 16 up to 1024", D);
  HILS_REQUIRE(rotary_dim >= 0 && rotary_dim % 16 == 0 && rotary_dim <= D,
               "hils_paged_append: rotary_dim (%d) must be a multiple of 16 up to D (%d)", rotary_dim, D);
  HILS_REQUIRE(HQ == 0 || rotary_dim > 0, "hils_paged_append: q is given to be rotated: inv_freq is missing");
  HILS_REQUIRE(max_pages <= (1 << 24), "hils_paged_append: the page table is too wide");
  HILS_REQUIRE(lengths || (seq_len >= T && seq_len <= (long)max_pages * 64),
               "hils_paged_append: seq_len %d is shorter than the %d tokens or longer than the page table", seq_len, T);
  HILS_REQUIRE((long)(HQ + 2 * H) * (D / 16) <= (1 << 20), "hils_paged_append: too many heads");
  HILS_REQUIRE(rotary_aligned(q, q_batch_stride, q_token_stride, q_head_stride) &&
                   rotary_aligned(k, k_batch_stride, k_token_stride, k_head_stride) &&
                   rotary_aligned(v, v_batch_stride, v_token_stride, v_head_stride) && rotary_aligned(q_out, 0, 0, 0) &&
                   rotary_aligned(k_pages, 0, 0, 0) && rotary_aligned(v_pages, 0, 0, 0),
               "hils_paged_append: addresses and strides must be multiples of 16 bytes");
  RotaryDims dm{};
  dm.n_tok = (long)B * T;
  dm.T = T, dm.HQ = HQ, dm.H = H, dm.D = D, dm.R = rotary_dim, dm.interleaved = interleaved, dm.append = 1;
  dm.pos_wide = positions_64, dm.pos_batch = 1, dm.freq_wide = inv_freq_64;
  dm.max_pages = max_pages, dm.num_pages = num_pages, dm.seq_len = seq_len;
  dm.scale = scale, dm.sign = 1.f;
  dm.q_sb = q_batch_stride, dm.q_st = q_token_stride, dm.q_sh = q_head_stride;
  dm.k_sb = k_batch_stride, dm.k_st = k_token_stride, dm.k_sh = k_head_stride;
  dm.v_sb = v_batch_stride, dm.v_st = v_token_stride, dm.v_sh = v_head_stride;
  dm.positions = positions, dm.inv_freq = inv_freq, dm.table = page_table, dm.lengths = lengths;
  return rotary_launch("hils_paged_append", dm, q, k, v, q_out, k_pages, v_pages, (hipStream_t)stream);
}
