// Pages of the 4-bit cache shared, copied and packed: sequences that go on from others (several answers to one prompt), and the pages in use brought
// to the front of the pool.  The reference keeps one dense cache of one sequence (external/llm/layers.lisp:19-33).  Layout: kv4.h.
#include <algorithm>

#include "kv4.h"

namespace cthip {

typedef uint32_t page_dwords __attribute__((ext_vector_type(4)));

// A page of a pool by 256 threads, four loads of 16 bytes a thread at once
__device__ __forceinline__ void copy_page(unsigned char *pool, int src, int dst, int page_bytes) {
  const page_dwords *s = (const page_dwords *)(pool + (int64_t)src * page_bytes);
  page_dwords *d = (page_dwords *)(pool + (int64_t)dst * page_bytes);
  const int n = page_bytes / 16;
  for (int e = threadIdx.x; e < n; e += 4 * 256) {
    page_dwords v[4];
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (e + 256 * k < n) v[k] = s[e + 256 * k];
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (e + 256 * k < n) d[e + 256 * k] = v[k];
  }
}

// ---- sequences that go on from others ----
// Full pages are the same for parent and child and stay shared; a partly filled one is copied into a page from the free stack.  One that lies outside the pool holds no
// rows: the child's entry is then the parent's, since a page from the stack would show the child what its last owner left there.  A child is nobody's parent
// in the same call and named once, so what is read (parents' tables and lengths) is not what is written (children's), and the forks need no
// order among themselves but that of the pages they take: how many forks in front of it need one, every workgroup counts for itself.
struct ForkArgs {
  int *tables, *lens, *n_free_out, *refused;
  unsigned char *k_pages, *v_pages;
  const int *parents, *children, *at, *free_pages, *n_free;
  int table_stride, n_seqs, n_forks, n_layers, n_pages, page_bytes;
  bool rows_too, free_too;
};

__global__ __launch_bounds__(256) void k_kv_fork(ForkArgs a) {
  __shared__ int s_first[kKv4MaxSeqs];                 // the first fork that a sequence is the child of
  __shared__ unsigned s_parent[kKv4MaxSeqs / 32];      // whether it is a parent
  __shared__ int s_count[2][4];
  const int tid = threadIdx.x, mine = blockIdx.y;
  // This workgroup's own fork and a fork a thread are asked for first, and so is what lies behind them wherever that is in range: round trips beside those of the checks
  // (one after the other 6.0 us for 8 forks of one sequence in 12 layers, so 5.2)
  const bool own = mine < a.n_forks, some = tid < a.n_forks;
  const int my_parent = own ? a.parents[mine] : -1, my_child = own ? a.children[mine] : -1, my_at = own ? a.at[mine] : 0;
  const int tid_parent = some ? a.parents[tid] : -1, tid_child = some ? a.children[tid] : -1, tid_at = some ? a.at[tid] : 0;
  const int have = max(a.n_free[0], 0);
  const bool my_parent_ok = my_parent >= 0 && my_parent < a.n_seqs, reads = my_parent_ok && my_at >= 0 && my_at / kKvPageRows < a.table_stride;
  const int *from = a.tables + (int64_t)(my_parent_ok ? my_parent : 0) * a.table_stride;
  // the parent's page that a fork ends in
  auto ends_in = [&](int p, int at) { return p >= 0 && p < a.n_seqs && at >= 0 && at / kKvPageRows < a.table_stride ? a.tables[(int64_t)p * a.table_stride + at / kKvPageRows] : -1; };
  const int src = reads ? from[my_at / kKvPageRows] : -1, tid_len = tid_parent >= 0 && tid_parent < a.n_seqs ? a.lens[tid_parent] : -1, tid_src = ends_in(tid_parent, tid_at);
  for (int i = tid; i < a.n_seqs; i += 256) s_first[i] = INT_MAX;
  for (int i = tid; i < (a.n_seqs + 31) / 32; i += 256) s_parent[i] = 0;
  __syncthreads();
  for (int f = tid; f < a.n_forks; f += 256) {
    const int p = f == tid ? tid_parent : a.parents[f], c = f == tid ? tid_child : a.children[f];
    if (c >= 0 && c < a.n_seqs) atomicMin(&s_first[c], f);
    if (p >= 0 && p < a.n_seqs) atomicOr(&s_parent[p >> 5], 1u << (p & 31));
  }
  __syncthreads();
  // whether a fork can be made but for its page, and whether it needs one
  auto fine = [&](int f, int p, int c, int at, int len, int page, bool &need) {
    const bool ok = p >= 0 && p < a.n_seqs && c >= 0 && c < a.n_seqs && at >= 0 && s_first[c] == f && !((s_parent[c >> 5] >> (c & 31)) & 1u) && at <= len &&
                    at <= a.table_stride * kKvPageRows;
    need = ok && at % kKvPageRows != 0 && page >= 0 && page < a.n_pages;
    return ok;
  };
  int before = 0, all = 0;  // forks that need a page
  for (int f = tid; f < a.n_forks; f += 256) {
    bool need;
    const int p = f == tid ? tid_parent : a.parents[f];
    const int c = f == tid ? tid_child : a.children[f], at = f == tid ? tid_at : a.at[f], len = f == tid ? tid_len : p >= 0 && p < a.n_seqs ? a.lens[p] : -1;
    fine(f, p, c, at, len, f == tid ? tid_src : ends_in(p, at), need);
    all += need;
    before += need && f < mine;
  }
  for (int o = 32; o > 0; o >>= 1) before += __shfl_xor(before, o, 64), all += __shfl_xor(all, o, 64);
  if ((tid & 63) == 0) s_count[0][tid >> 6] = before, s_count[1][tid >> 6] = all;
  __syncthreads();
  before = (s_count[0][0] + s_count[0][1]) + (s_count[0][2] + s_count[0][3]);
  all = (s_count[1][0] + s_count[1][1]) + (s_count[1][2] + s_count[1][3]);
  if (a.free_too && blockIdx.x == 0 && mine == 0 && tid == 0) a.n_free_out[0] = a.n_free[0] - min(all, have);
  if (!a.rows_too) return;
  bool need, ok = fine(mine, my_parent, my_child, my_at, my_parent_ok ? a.lens[my_parent] : -1, src, need);
  ok = ok && (!need || before < have);
  if (blockIdx.x == 0 && tid == 0) a.refused[mine] = ok ? 0 : 1;
  if (!ok) return;
  const int full = my_at / kKvPageRows, page = need ? a.free_pages[have - 1 - before] : -1;
  if (blockIdx.x == 0) {
    int *to = a.tables + (int64_t)my_child * a.table_stride;
    for (int c = tid; c < full + (my_at % kKvPageRows != 0); c += 256) to[c] = c == full && need ? page : from[c];
    if (tid == 0) a.lens[my_child] = my_at;
    return;
  }
  if (!need || page < 0 || page >= a.n_pages) return;
  const int64_t layer = (int64_t)(blockIdx.x - 1) * a.n_pages * a.page_bytes;
  copy_page(a.k_pages + layer, src, page, a.page_bytes);
  copy_page(a.v_pages + layer, src, page, a.page_bytes);
}

// ---- the pages in use to the front of the pool ----
// Of u pages in use, those whose id is u or more go, in order, to the ids below u that are not in use, in order: there are as many of these, what is
// read is not what is written, and a call repeated on the same tables writes the same bytes.  map: in use (1) or not, then where each page
// goes; moves: (from, to).
constexpr int kPackThreads = 1024;
constexpr int kBitPages = 1 << 17;  // pages that there are bits for in LDS
__global__ __launch_bounds__(256) void k_kv_compact_clear(int *map, int n_pages) {
  for (int64_t i = blockIdx.x * 256 + threadIdx.x; i < n_pages; i += (int64_t)gridDim.x * 256) map[i] = 0;
}
__device__ __forceinline__ int pages_of(int len, int table_stride) { return min(max(len, 0) / kKvPageRows + (max(len, 0) % kKvPageRows != 0), table_stride); }
__global__ __launch_bounds__(256) void k_kv_compact_mark(int *map, const int *__restrict__ tables, int table_stride, const int *__restrict__ lens, int n_pages) {
  const int pages = pages_of(lens[blockIdx.x], table_stride);
  for (int c = threadIdx.x; c < pages; c += 256) {
    const int id = tables[(int64_t)blockIdx.x * table_stride + c];
    if (id >= 0 && id < n_pages) map[id] = 1;
  }
}
// exclusive sums of two counts over the workgroup, and their totals
__device__ __forceinline__ int2 pack_scan(int2 v, int2 (*part)[kPackThreads / 64], int2 &total) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  int2 s = v;
  for (int o = 1; o < 64; o <<= 1) {
    const int x = __shfl_up(s.x, o, 64), y = __shfl_up(s.y, o, 64);
    if (lane >= o) s.x += x, s.y += y;
  }
  __syncthreads();
  if (lane == 63) (*part)[wv] = s;
  __syncthreads();
  int2 before = {0, 0};
  total = {0, 0};
  for (int w = 0; w < kPackThreads / 64; w++) {
    const int2 p = (*part)[w];
    if (w < wv) before.x += p.x, before.y += p.y;
    total.x += p.x, total.y += p.y;
  }
  return {before.x + s.x - v.x, before.y + s.y - v.y};
}
// MARK: the pages in use are found here too, as bits in LDS; a thread then has the 32 pages of a word.  Otherwise another launch has marked them in map, where a bit
// for each would not fit, and a thread has eight.
template <bool MARK>
__global__ __launch_bounds__(kPackThreads) void k_kv_compact_plan(int *map, int2 *moves, int *n_moves, int *free_pages, int *n_free, int n_pages, const int *__restrict__ tables,
                                                                  int table_stride, const int *__restrict__ lens, int n_seqs) {
  constexpr int EACH = MARK ? 32 : 8;
  __shared__ int2 part[kPackThreads / 64];
  __shared__ unsigned s_bits[MARK ? kBitPages / 32 : 1];
  const int tid = threadIdx.x, groups = (n_pages + EACH - 1) / EACH;
  if (MARK) {
    for (int i = tid; i < groups; i += kPackThreads) s_bits[i] = 0;
    __syncthreads();
    const int entries = n_pages > 0 ? n_seqs * table_stride : 0;
    for (int e0 = tid; e0 < entries; e0 += 4 * kPackThreads) {  // (lengths and entries of four at once)
      int id[4], len[4];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int e = e0 + k * kPackThreads;
        if (e < entries) id[k] = tables[e], len[k] = lens[e / table_stride];
      }
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int e = e0 + k * kPackThreads;
        if (e < entries && e % table_stride < pages_of(len[k], table_stride) && id[k] >= 0 && id[k] < n_pages) atomicOr(&s_bits[id[k] >> 5], 1u << (id[k] & 31));
      }
    }
    __syncthreads();
  }
  auto in_use = [&](int i) {  // of pages EACH i and on, as bits
    if (MARK) return s_bits[i];
    unsigned w = 0;
    for (int k = 0; k < EACH; k++)
      if (EACH * i + k < n_pages && map[EACH * i + k]) w |= 1u << k;
    return w;
  };
  int used = 0;
  for (int i = tid; i < groups; i += kPackThreads) used += __popc(in_use(i));
  int2 total;
  pack_scan({used, 0}, &part, total);
  used = total.x;
  int2 done = {0, 0};
  for (int i0 = 0; i0 < groups; i0 += kPackThreads) {
    const int i = i0 + tid, first = EACH * i;
    unsigned go = 0, hole = 0;
    if (i < groups) {
      const unsigned w = in_use(i), all = EACH == 32 && n_pages - first >= 32 ? ~0u : (1u << min(EACH, n_pages - first)) - 1u;
      const unsigned front = used <= first ? 0u : used - first >= 32 ? ~0u : (1u << (used - first)) - 1u;  // those whose id is below the number in use
      go = w & ~front, hole = ~w & front & all;
    }
    int2 at = pack_scan({(int)__popc(go), (int)__popc(hole)}, &part, total);
    at.x += done.x, at.y += done.y;
    for (; go; go &= go - 1) moves[at.x++].x = first + __builtin_ctz(go);
    for (; hole; hole &= hole - 1) moves[at.y++].y = first + __builtin_ctz(hole);
    done.x += total.x, done.y += total.y;
  }
  for (int i = tid; i < n_pages; i += kPackThreads) {
    free_pages[i] = i < n_pages - used ? n_pages - 1 - i : -1;
    if (i < used) map[i] = i;
  }
  __syncthreads();
  for (int k = tid; k < done.x; k += kPackThreads) map[moves[k].x] = moves[k].y;  // (no other page from `used` on is in use)
  if (tid == 0) n_free[0] = n_pages - used, n_moves[0] = done.x;
}
struct MoveArgs {
  int *tables_out;
  unsigned char *k_pages, *v_pages;
  const int *tables, *lens, *map, *n_moves;
  const int2 *moves;
  int table_stride, n_seqs, n_layers, n_pages, page_bytes;
};
// blockIdx.y = 0: tables; otherwise the pages of layer y - 1
__global__ __launch_bounds__(256) void k_kv_compact_move(MoveArgs a) {
  if (blockIdx.y == 0) {
    for (int i = blockIdx.x; i < a.n_seqs; i += gridDim.x) {
      const int pages = pages_of(a.lens[i], a.table_stride);
      for (int c = threadIdx.x; c < a.table_stride; c += 256) {
        const int64_t at = (int64_t)i * a.table_stride + c;
        const int id = a.tables[at];
        a.tables_out[at] = c < pages && id >= 0 && id < a.n_pages ? a.map[id] : id;
      }
    }
    return;
  }
  const int n = a.n_moves[0];
  const int64_t layer = (int64_t)(blockIdx.y - 1) * a.n_pages * a.page_bytes;
  for (int m = blockIdx.x; m < n; m += gridDim.x) {
    const int2 move = a.moves[m];
    copy_page(a.k_pages + layer, move.x, move.y, a.page_bytes);
    copy_page(a.v_pages + layer, move.x, move.y, a.page_bytes);
  }
}

}  // namespace cthip

using namespace cthip;

static bool pools_ok(const void *k, const void *v) { return (((uintptr_t)k | (uintptr_t)v) & 15) == 0; }

extern "C" {

int cthip_kv_fork_paged_q4(int *tables, int table_stride, int *lens, int n_seqs, int *n_free_out, int *refused, void *k_pages, void *v_pages, int n_layers, int n_pages,
                           const int *parents, const int *children, const int *at, int n_forks, const int *free_pages, const int *n_free, int kv_heads, int head_dim) {
  CTHIP_REQUIRE_INIT();
  CTHIP_ARG(n_seqs >= 0 && n_forks >= 0 && n_layers >= 0 && n_pages >= 0 && n_pages <= INT_MAX / kKvPageRows && table_stride > 0 && table_stride <= INT_MAX / kKvPageRows);
  if (!kv4_shape_ok(kv_heads, head_dim)) return fail(CTHIP_E_UNSUPPORTED, "cthip_kv_fork_paged_q4: %d heads of %d (head sizes 32, 64, 128)", kv_heads, head_dim);
  if (n_seqs > kKv4MaxSeqs || n_forks > kKv4MaxSeqs || n_layers > (1 << 20))
    return fail(CTHIP_E_UNSUPPORTED, "cthip_kv_fork_paged_q4: %d forks of %d sequences, %d layers (at most %d, %d, 1048576)", n_forks, n_seqs, n_layers, kKv4MaxSeqs, kKv4MaxSeqs);
  CTHIP_ARG(n_free && n_free_out && (n_forks == 0 || (refused && parents && children && at && free_pages)));
  CTHIP_ARG(n_forks == 0 || n_seqs == 0 || (tables && lens));
  CTHIP_ARG(n_forks == 0 || n_layers == 0 || n_pages == 0 || (k_pages && v_pages && pools_ok(k_pages, v_pages)));
  const bool in_place = n_free_out == n_free;
  if (n_forks == 0 && in_place) return 0;
  // (several workgroups read the number of free pages while one of them would overwrite it: a launch of its own behind them then)
  ForkArgs a = {tables, lens, n_free_out, refused, (unsigned char *)k_pages, (unsigned char *)v_pages, parents, children, at, free_pages, n_free, table_stride, n_seqs, n_forks,
                n_layers, n_pages, kv_heads * kv4_head_bytes(head_dim), n_forks > 0, !in_place};
  const unsigned copies = n_pages && n_forks ? (unsigned)n_layers : 0u;
  hipLaunchKernelGGL(k_kv_fork, dim3(1 + copies, (unsigned)std::max(n_forks, 1)), dim3(256), 0, state().stream, a);
  CTHIP_LAUNCH_CHECK();
  if (in_place) {
    a.rows_too = false, a.free_too = true;
    hipLaunchKernelGGL(k_kv_fork, dim3(1), dim3(256), 0, state().stream, a);
    CTHIP_LAUNCH_CHECK();
  }
  return 0;
}

int64_t cthip_kv_compact_paged_q4_workspace(int n_pages) {
  if (n_pages < 0 || n_pages > INT_MAX / kKvPageRows) return fail(CTHIP_E_BAD_ARG, "cthip_kv_compact_paged_q4_workspace: %d pages", n_pages);
  return 64 + 8ll * n_pages;
}

int cthip_kv_compact_paged_q4(int *tables_out, int *free_pages, int *n_free, void *k_pages, void *v_pages, int n_layers, int n_pages, const int *tables, int table_stride,
                              const int *lens, int n_seqs, int kv_heads, int head_dim, void *workspace) {
  CTHIP_REQUIRE_INIT();
  CTHIP_ARG(n_seqs >= 0 && n_layers >= 0 && n_pages >= 0 && n_pages <= INT_MAX / kKvPageRows && table_stride > 0);
  if (!kv4_shape_ok(kv_heads, head_dim)) return fail(CTHIP_E_UNSUPPORTED, "cthip_kv_compact_paged_q4: %d heads of %d (head sizes 32, 64, 128)", kv_heads, head_dim);
  if (n_seqs > 65535 || n_layers >= 65535) return fail(CTHIP_E_UNSUPPORTED, "cthip_kv_compact_paged_q4: %d sequences, %d layers (at most 65535, 65534)", n_seqs, n_layers);
  CTHIP_ARG(n_free && workspace && ((uintptr_t)workspace & 15) == 0 && (n_pages == 0 || free_pages) && (n_seqs == 0 || (tables_out && tables && lens)));
  CTHIP_ARG(n_layers == 0 || n_pages == 0 || (k_pages && v_pages && pools_ok(k_pages, v_pages)));
  int *n_moves = (int *)workspace, *map = n_moves + 16;
  int2 *moves = (int2 *)(map + n_pages + (n_pages & 1));  // (half of the pages at most)
  // One launch that reads whole tables, or three of which one reads what is in use of them: full tables of 30 x 32 entries 7.4 us and 11.1, 128 x 128 16.7 and 33.9,
  // 512 x 128 49 and 110.  An entry costs one workgroup 0.45 ns, the other way a page 1.2 and the launches 3 us.
  const bool mark = n_pages == 0 || (n_pages <= kBitPages && (int64_t)n_seqs * table_stride <= 2ll * n_pages + (1 << 14));
  if (mark) {
    hipLaunchKernelGGL(k_kv_compact_plan<true>, dim3(1), dim3(kPackThreads), 0, state().stream, map, moves, n_moves, free_pages, n_free, n_pages, tables, table_stride, lens, n_seqs);
  } else {
    hipLaunchKernelGGL(k_kv_compact_clear, dim3((unsigned)std::min(1024, (n_pages + 255) / 256)), dim3(256), 0, state().stream, map, n_pages);
    CTHIP_LAUNCH_CHECK();
    if (n_seqs > 0) hipLaunchKernelGGL(k_kv_compact_mark, dim3((unsigned)n_seqs), dim3(256), 0, state().stream, map, tables, table_stride, lens, n_pages);
    CTHIP_LAUNCH_CHECK();
    hipLaunchKernelGGL(k_kv_compact_plan<false>, dim3(1), dim3(kPackThreads), 0, state().stream, map, moves, n_moves, free_pages, n_free, n_pages, nullptr, 0, nullptr, 0);
  }
  CTHIP_LAUNCH_CHECK();
  const MoveArgs a = {tables_out, (unsigned char *)k_pages, (unsigned char *)v_pages, tables, lens, map, n_moves, moves, table_stride, n_seqs, n_layers, n_pages,
                      kv_heads * kv4_head_bytes(head_dim)};
  const int most = std::max(std::max(1, n_pages / 2), std::min(n_seqs, 256));
  hipLaunchKernelGGL(k_kv_compact_move, dim3((unsigned)std::min(most, 2048), 1u + (n_pages ? (unsigned)n_layers : 0u)), dim3(256), 0, state().stream, a);
  CTHIP_LAUNCH_CHECK();
  return 0;
}

}  // extern "C"
