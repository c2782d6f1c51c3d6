// Moving what a paged cache holds: whole pages (forks of a sequence, compaction of a pool) and accepted drafts.
#include "common.h"
#include "../../include/hils_amd.h"

// ---- whole pages -------------------------------------------------------------------------------
// pool[dst[i]] = pool[src[i]] for every i and up to eight pools at once.  Bound by HBM (every byte read and written once)
// or, for a few pages, by the one launch.  A workgroup copies one piece of 32 KiB of a pair of pages, its eight 16-byte
// loads per thread in flight together.  Moves larger than the last cache go past it: 2048 pages of 2 x 128 KiB and small
// pools (1.08 GB read and written) in 208 us (5.2 TB/s), 217 through the caches; a fork of 32 pages takes 5 us either way and
// its pages are read next.
typedef unsigned pg_u4 __attribute__((ext_vector_type(4)));
#define PC_POOLS 8
#define PC_PIECE 32768

struct PageCopy {
  unsigned char* pool[PC_POOLS];
  long bytes[PC_POOLS];       // of a page
  int first[PC_POOLS + 1];    // first piece of a pool among the pieces of a pair
  int unit[PC_POOLS];         // 16, 4 or 1: what every page of the pool is a whole number of, and aligned to
  int n_pools, num_pages, wide;
  int past;                   // past the caches: what is read and written does not fit the last of them
  uint32_t m_pieces;
  const void* src;
  const void* dst;
};

template <typename V, bool PAST>
__device__ __forceinline__ void page_copy_piece(unsigned char* to, const unsigned char* from, int bytes) {
  const V* f = (const V*)from;
  V* t = (V*)to;
  const int n = bytes / (int)sizeof(V);
  for (int i0 = threadIdx.x; i0 < n; i0 += 256 * 8) {
    V x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i0 + 256 * u < n) x[u] = PAST ? __builtin_nontemporal_load(f + i0 + 256 * u) : f[i0 + 256 * u];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i0 + 256 * u < n) {
        if (PAST) __builtin_nontemporal_store(x[u], t + i0 + 256 * u);
        else t[i0 + 256 * u] = x[u];
      }
  }
}

__global__ void __launch_bounds__(256) page_copy_kernel(PageCopy pc) {
  const int pieces = pc.first[pc.n_pools];
  const int pair = hils_udiv(blockIdx.x, pieces, pc.m_pieces), piece = blockIdx.x - pair * pieces;
  const long src = pc.wide ? ((const int64_t*)pc.src)[pair] : ((const int32_t*)pc.src)[pair];
  const long dst = pc.wide ? ((const int64_t*)pc.dst)[pair] : ((const int32_t*)pc.dst)[pair];
  if (src < 0 || dst < 0 || src >= pc.num_pages || dst >= pc.num_pages || src == dst) return;
  int p = 0;
  while (p + 1 < pc.n_pools && piece >= pc.first[p + 1]) ++p;
  const long at = (long)(piece - pc.first[p]) * PC_PIECE, left = pc.bytes[p] - at;
  const int bytes = left < PC_PIECE ? (int)left : PC_PIECE;
  const unsigned char* from = pc.pool[p] + src * pc.bytes[p] + at;
  unsigned char* to = pc.pool[p] + dst * pc.bytes[p] + at;
  if (pc.unit[p] == 16 && pc.past) page_copy_piece<pg_u4, true>(to, from, bytes);
  else if (pc.unit[p] == 16) page_copy_piece<pg_u4, false>(to, from, bytes);
  else if (pc.unit[p] == 4) page_copy_piece<uint32_t, false>(to, from, bytes);
  else page_copy_piece<unsigned char, false>(to, from, bytes);
}

extern "C" int hils_copy_pages(void** pools, const size_t* page_bytes, const void* src, const void* dst, int n_pools, int n,
                               int num_pages, int indices_64, void* stream) {
  HILS_REQUIRE(pools && page_bytes && src && dst, "hils_copy_pages: null pointer");
  HILS_REQUIRE(n_pools >= 1 && n_pools <= PC_POOLS, "hils_copy_pages: 1 to %d pools (got %d)", PC_POOLS, n_pools);
  HILS_REQUIRE(n > 0 && num_pages > 0, "hils_copy_pages: sizes must be positive");
  PageCopy pc{};
  for (int i = 0; i < n_pools; ++i) {
    HILS_REQUIRE(pools[i], "hils_copy_pages: null pointer");
    HILS_REQUIRE(page_bytes[i] > 0 && page_bytes[i] < ((size_t)1 << 40), "hils_copy_pages: page size out of range");
    pc.pool[i] = (unsigned char*)pools[i];
    pc.bytes[i] = (long)page_bytes[i];
    const uintptr_t all = (uintptr_t)pools[i] | (uintptr_t)page_bytes[i];
    pc.unit[i] = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
    const long pieces = (pc.bytes[i] + PC_PIECE - 1) / PC_PIECE;
    HILS_REQUIRE(pc.first[i] + pieces < (1 << 26), "hils_copy_pages: pages too large");
    pc.first[i + 1] = pc.first[i] + (int)pieces;
  }
  double moved = 0;
  for (int i = 0; i < n_pools; ++i) moved += 2. * pc.bytes[i] * n;
  pc.past = moved > HILS_LAST_CACHE;
  const long blocks = (long)pc.first[n_pools] * n;
  HILS_REQUIRE(blocks <= 2147483647L && blocks * pc.first[n_pools] < (1l << 32), "hils_copy_pages: too much for one call");
  pc.n_pools = n_pools;
  pc.num_pages = num_pages;
  pc.wide = indices_64;
  pc.m_pieces = hils_udiv_magic(pc.first[n_pools]);
  pc.src = src;
  pc.dst = dst;
  hipLaunchKernelGGL(page_copy_kernel, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, pc);
  HILS_CHECK_LAUNCH("hils_copy_pages");
  return HILS_OK;
}

// ---- accepted drafts ---------------------------------------------------------------------------
// Token path[b][i] of the drafts behind `base` committed tokens becomes the sequence's token base + i: its key and value
// move from slot base + path[b][i] to slot base + i.  Only the longest start of a path that grows strictly counts (a
// negative entry ends it), so path[i] >= i and no move overwrites what a later one reads: a thread owns 16 bytes of
// every token and moves eight tokens at a time, all eight read before the first is written.  Bound by its latencies (path and
// table, values, stores): 3 to 5 us.
#define ACC_MAX 256

__global__ void __launch_bounds__(256)
paged_accept_kernel(bf16_t* __restrict__ k, bf16_t* __restrict__ v, const int32_t* __restrict__ table,
                    const int32_t* __restrict__ bases, const int32_t* __restrict__ path, int base0, int n, int H, int D,
                    int max_pages, int num_pages) {
  __shared__ long from_s[ACC_MAX], to_s[ACC_MAX];  // place of a token, in tokens of a pool's first head; -1: none
  __shared__ int count_s;
  const int b = blockIdx.y, tid = threadIdx.x;
  const long base = bases ? bases[b] : base0;
  if (tid == 0) count_s = n;
  __syncthreads();
  if (tid < n) {
    const int now = path[(long)b * n + tid], before = tid ? path[(long)b * n + tid - 1] : -1;
    if (now < 0 || now <= before) atomicMin(&count_s, tid);
    auto place = [&](long slot) -> long {
      if (slot < 0 || slot >= (long)max_pages * 64) return -1;
      const int page = table[(long)b * max_pages + (slot >> 6)];
      return (unsigned)page < (unsigned)num_pages ? (long)page * H * 64 + (slot & 63) : -1;
    };
    const bool moves = base >= 0 && now > tid;  // (a token already in its place stays)
    const long f = moves ? place(base + now) : -1, t = moves ? place(base + tid) : -1;
    from_s[tid] = t < 0 ? -1 : f;
    to_s[tid] = t;
  }
  __syncthreads();
  const int count = count_s, pph = D / 8, all = 2 * H * pph;
  const int e = blockIdx.x * 256 + tid;
  if (e >= all) return;
  const int pc = e % pph, hh = e / pph;
  bf16_t* pool = (hh >= H ? v : k) + (long)(hh >= H ? hh - H : hh) * 64 * D + pc * 8;
  for (int i0 = 0; i0 < count; i0 += 8) {
    pg_u4 x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i0 + u < count && from_s[i0 + u] >= 0) x[u] = *(const pg_u4*)(pool + from_s[i0 + u] * D);
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i0 + u < count && from_s[i0 + u] >= 0) *(pg_u4*)(pool + to_s[i0 + u] * D) = x[u];
  }
}

extern "C" int hils_paged_accept(void* k_pages, void* v_pages, const int32_t* page_table, const int32_t* bases,
                                 const int32_t* path, int B, int n, int H, int D, int max_pages, int num_pages, int base,
                                 void* stream) {
  HILS_REQUIRE(k_pages && v_pages && page_table && path, "hils_paged_accept: null pointer");
  HILS_REQUIRE(B > 0 && H > 0 && max_pages > 0 && num_pages > 0, "hils_paged_accept: sizes must be positive");
  HILS_REQUIRE(B <= 65535, "hils_paged_accept: too many sequences");
  HILS_REQUIRE(n >= 1 && n <= ACC_MAX, "hils_paged_accept: a path has 1 to %d tokens (got %d)", ACC_MAX, n);
  HILS_REQUIRE(D > 0 && D % 8 == 0 && (long)H * D < (1l << 28), "hils_paged_accept: D (%d) must be a multiple of 8", D);
  HILS_REQUIRE(max_pages <= (1 << 24), "hils_paged_accept: the page table is too wide");
  HILS_REQUIRE(bases || base >= 0, "hils_paged_accept: base must not be negative");
  HILS_REQUIRE((uintptr_t)k_pages % 16 == 0 && (uintptr_t)v_pages % 16 == 0, "hils_paged_accept: pages must lie at multiples of 16 bytes");
  const int all = 2 * H * (D / 8);
  hipLaunchKernelGGL(paged_accept_kernel, dim3((all + 255) / 256, B), dim3(256), 0, (hipStream_t)stream, (bf16_t*)k_pages,
                     (bf16_t*)v_pages, page_table, bases, path, base, n, H, D, max_pages, num_pages);
  HILS_CHECK_LAUNCH("hils_paged_accept");
  return HILS_OK;
}
