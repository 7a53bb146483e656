// Attention of a ragged batch of query rows over the 4-bit paged cache (layout: kv4.h).  The reference attends one sequence over
// a dense fp32 cache (external/llm/layers.lisp:3-5,19-33).
#include <type_traits>

#include "kv4.h"

namespace cthip {

struct Kv4Attn {
  float *out;
  const float *q;
  const unsigned char *k_pages, *v_pages;
  const int *tables, *lens, *starts;
  int64_t q_stride;
  int n_pages, table_stride, n_seqs, n_rows, H, Hkv;
  int unit;        // pages are counted in units of 2^unit where they are shared out
  int *tickets;    // workspace: a counter per job that is shared, zero between calls
  float *parts;    // and the shares' records: 16 rows of unnormalised outputs, their maxima, their sums
};

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kTileRows = 16;        // rows (query row, query head of the group) of a tile
constexpr int kTargetGroups = 1024;  // workgroups that the pages are shared out to
constexpr int kSplitSlots = 2048;    // records of shares in the workspace
constexpr int kMaxShares = 64;

// sum over the lanes up to this one
__device__ __forceinline__ int wave_scan_int(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
  return v;
}

// Which part of the batch a workgroup takes.  A job is a tile of rows of one key / value head of one sequence; a job with many
// pages is shared by several workgroups.  The lengths are on the device only, so every wavefront works the division out for
// itself: pages of all jobs / kTargetGroups = pages of a share, and the running sum of jobs x shares says whose share this is.
struct Share {
  int seq, head, tile;
  int len, rows, row0;    // of the sequence: keys, rows of this step and the first of them
  int first, pages, per;  // this share's first page, the job's pages, the pages of a share
  int share, shares;      // of the job
  int slot;               // of the job's first record
};
__device__ __forceinline__ bool find_share(const Kv4Attn &a, int id, Share &w) {
  const int lane = threadIdx.x & 63, G = a.H / a.Hkv;
  const int64_t most = (int64_t)a.table_stride * kKvPageRows;
  auto look = [&](int i, int &len, int &row0, int &rows, int &tiles, int &pages) {
    len = 0, row0 = 0, rows = 0;
    if (i < a.n_seqs) {
      len = a.lens[i], row0 = a.starts[i];
      const int end = min(a.starts[i + 1], a.n_rows);
      rows = row0 >= 0 && end > row0 ? end - row0 : 0;
    }
    tiles = (rows * G + kTileRows - 1) / kTileRows;
    pages = a.n_pages > 0 && len > 0 ? (int)((min((int64_t)len, most) + kKvPageRows - 1) / kKvPageRows) : 0;
  };
  int len, row0, rows, tiles, pages;
  int64_t total = 0;
  int longest = 0;
  for (int i0 = 0; i0 < a.n_seqs; i0 += 64) {
    look(i0 + lane, len, row0, rows, tiles, pages);
    // (in units of 2^unit pages, rounded up, so that 64 sequences' sum fits: the launcher chooses)
    const int sum = wave_scan_int(tiles * a.Hkv * ((pages >> a.unit) + 1));
    total += __builtin_amdgcn_readlane(sum, 63);
    int p = tiles ? pages : 0;
    for (int o = 32; o > 0; o >>= 1) p = max(p, __shfl_xor(p, o, 64));
    longest = max(longest, p);
  }
  int64_t per = ((total + kTargetGroups - 1) / kTargetGroups) << a.unit;
  per = max(per, (int64_t)(longest + kMaxShares - 1) / kMaxShares);
  w.per = (int)min((per + 3) / 4 * 4, (int64_t)1 << 30);  // four wavefronts take pages in turn
  int before = 0, slots = 0;
  for (int i0 = 0; i0 < a.n_seqs; i0 += 64) {
    if (a.n_seqs > 64) look(i0 + lane, len, row0, rows, tiles, pages);
    const int shares = max(1, (pages + w.per - 1) / w.per), jobs = tiles * a.Hkv;
    const int sum = wave_scan_int(jobs * shares), sums = wave_scan_int(shares > 1 ? jobs * shares : 0);
    const unsigned long long past = __ballot(before + sum > id);
    if (past) {
      const int l = (int)__builtin_ctzll(past);
      const int mine = __builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(jobs * shares, l);
      const int at = id - before - mine;
      w.shares = __builtin_amdgcn_readlane(shares, l);
      // (starts that overlap can sum to anything: such rows are nobody's)
      if ((unsigned)at >= (unsigned)__builtin_amdgcn_readlane(jobs * shares, l)) return false;
      const int job = at / w.shares, nt = __builtin_amdgcn_readlane(tiles, l);
      w.share = at - job * w.shares;
      w.head = job / nt;
      w.tile = job - w.head * nt;
      w.seq = i0 + l;
      w.len = __builtin_amdgcn_readlane(len, l);
      w.rows = __builtin_amdgcn_readlane(rows, l);
      w.row0 = __builtin_amdgcn_readlane(row0, l);
      w.pages = __builtin_amdgcn_readlane(pages, l);
      w.slot = slots + __builtin_amdgcn_readlane(sums, l) - __builtin_amdgcn_readlane(shares > 1 ? jobs * shares : 0, l) + job * w.shares;
      return w.shares == 1 || (unsigned)w.slot <= (unsigned)(kSplitSlots - w.shares);
    }
    before += __builtin_amdgcn_readlane(sum, 63);
    slots += __builtin_amdgcn_readlane(sums, 63);
  }
  return false;
}

// One page for one wavefront and 16 rows.  S^T = K Q^T and O^T = V^T P^T: the row is the lane's number modulo 16 throughout (scores,
// maxima, sums and outputs), lane group g = lane / 16 holds keys 16 s + 4 g + i of the page and channels 4 g + i of a result tile.
//   scores  Numbers as fp16 integers, q as two fp16 terms (22 bits of the row's largest); a block's scale is applied to its 32-wide
//           partial sum.  (The nibbles as they stand are fp16 subnormals n 2^-24 and would need no conversion, but the matrix
//           instruction adds products of subnormals with five bits less: 2.8e-6 of a score instead of 6e-8.)
//   output  2^c p d as two fp16 terms (22 bits of each), values as exact fp16 integers, fp32 accumulators.  2^c brings the largest
//           scale seen so far to 2^13: products down to 2^-27 of p = 1 at that scale keep their 22 bits, smaller ones lie on a grid
//           of 2^-38 of it.  It goes into the exponent of p, so that sums and outputs carry it alike.
template <int DH>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void k_kv4_attn(Kv4Attn a) {
  constexpr int NB = DH / 32, PITCH = DH + 4;
  __shared__ float s_o[4][kTileRows][PITCH];
  __shared__ float s_m[4][kTileRows], s_l[4][kTileRows], s_w[4][kTileRows];
  __shared__ float s_sum[kTileRows];
  __shared__ __attribute__((aligned(16))) unsigned char s_scale[4][2][kKvPageRows * NB * 2];
  __shared__ int s_ticket;
  Share w;
  if (!find_share(a, blockIdx.x, w)) return;
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, g = lane >> 4;
  const int G = a.H / a.Hkv;
  // this lane's row
  const int rho = w.tile * kTileRows + n, j = rho / G;
  const bool active = j < w.rows;
  const int head = w.head * G + rho - j * G;
  const int64_t all = (int64_t)a.table_stride * kKvPageRows;
  const int limit = active ? (int)min((int64_t)w.len - w.rows + j, all - 1) : -1;  // the last key it sees
  // pages that any row / every row of the tile sees (rows rise with n)
  const int j1 = min(w.rows - 1, (w.tile * kTileRows + kTileRows - 1) / G), j0 = w.tile * kTileRows / G;
  const int last = (int)min((int64_t)w.len - w.rows + j1, all - 1), least = (int)min((int64_t)w.len - w.rows + j0, all - 1);
  const int pages = a.n_pages > 0 && last >= 0 ? last / kKvPageRows + 1 : 0;
  const int shares = max(1, (pages + w.per - 1) / w.per);  // (at most w.shares: a row of the sequence's last tile sees the most)
  if (w.share >= shares) return;
  const int p0 = w.share * w.per, p1 = min(pages, p0 + w.per);

  half8 q_hi[NB], q_lo[NB];
  float weight;
  {
    float x[NB][8];
    const float *src = a.q + (int64_t)(w.row0 + (active ? j : 0)) * a.q_stride + head * DH;
    float top = 0.0f;
    bool odd = false;
#pragma unroll
    for (int b = 0; b < NB; b++) {
      f4_any u = *(const f4_any *)(src + b * 32 + g * 8), v = *(const f4_any *)(src + b * 32 + g * 8 + 4);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        x[b][e] = active ? u[e] : 0.0f, x[b][4 + e] = active ? v[e] : 0.0f;
        top = fmaxf(top, fmaxf(fabsf(x[b][e]), fabsf(x[b][4 + e])));
        odd = odd || !(fabsf(x[b][e]) < INFINITY) || !(fabsf(x[b][4 + e]) < INFINITY);
      }
    }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    int bad = odd;
    bad |= __shfl_xor(bad, 16, 64);
    bad |= __shfl_xor(bad, 32, 64);
    // a power of two that brings the row's largest into [2^9, 2^10): fp16's own 11 bits, and 11 below them
    int e = top > 0.0f ? ilogbf(top) : 0;
    if (bad) e = 0;
    const float up = ldexpf(1.0f, 9 - e > 126 ? 126 : 9 - e);
#pragma unroll
    for (int b = 0; b < NB; b++) {
#pragma unroll
      for (int k = 0; k < 8; k++) {
        // the order in which a dword's nibbles come apart: channels 0 2 4 6 1 3 5 7
        const int ch = k < 4 ? (k & 1) * 2 + (k >> 1) * 4 : 1 + (k & 1) * 2 + ((k - 4) >> 1) * 4;
        const float y = bad ? 0.0f : x[b][ch] * up;
        q_hi[b][k] = (_Float16)y;
        q_lo[b][k] = (_Float16)(y - (float)q_hi[b][k]);
      }
    }
    // scores as powers of two: log2(e) / sqrt(DH), and the powers of two taken off again
    weight = bad ? NAN : 1.44269504f / sqrtf((float)DH) / up;
  }

  f32x4 o[NB][2];
#pragma unroll
  for (int b = 0; b < NB; b++) o[b][0] = o[b][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, l = 0.0f;
  int c = 100;  // (no scale seen)

  // page ids of the next 64 pages of this wavefront, one a lane
  const int *table = a.tables + (int64_t)w.seq * a.table_stride;
  const int head_bytes = kv4_head_bytes(DH);
  int ids = 0, ids_from = -1;
  auto page_id = [&](int k) {  // k: this wavefront's k-th page (the same in every lane)
    if (ids_from < 0 || k >= ids_from + 64) {
      ids_from = k;
      const int p = p0 + wv + 4 * (k + lane);
      ids = p < p1 ? table[p] : -1;
    }
    return __builtin_amdgcn_readlane(ids, k - ids_from);
  };
  // A page's quants come straight to the lanes that multiply them; its scales, which 16 lanes share, come as one piece a lane
  // and go through LDS (read by the lanes from memory they were 64 registers and 16 loads a page).
  typedef uint32_t kdw __attribute__((ext_vector_type(NB)));
  typedef unsigned short sdw __attribute__((ext_vector_type(NB)));
  kdw kq[4];
  u32x4 vq[NB];
  sdw ks, vs;
  int id_k = -1, id_v = -1;
  auto ask_k = [&](int k) {
    id_k = page_id(k);
    const unsigned char *p = a.k_pages + ((int64_t)(id_k >= 0 && id_k < a.n_pages ? id_k : 0) * a.Hkv + w.head) * head_bytes;
#pragma unroll
    for (int s = 0; s < 4; s++) kq[s] = *(const kdw *)(p + kv4_key_offset(16 * s + n, g, 0, DH));
    ks = *(const sdw *)(p + 32 * DH + lane * NB * 2);
  };
  auto ask_v = [&](int id) {
    id_v = id;
    const unsigned char *p = a.v_pages + ((int64_t)(id >= 0 && id < a.n_pages ? id : 0) * a.Hkv + w.head) * head_bytes;
#pragma unroll
    for (int b = 0; b < NB; b++) vq[b] = *(const u32x4 *)(p + (b * 16 + n) * kKvPageRows + 16 * g);
    vs = *(const sdw *)(p + 32 * DH + lane * NB * 2);
  };
  // the scales of block b, rows 16 t + 4 g ..
  auto scales = [&](int which, int t, int b) {
    return *(const half4 *)(s_scale[wv][which] + ((4 * t + g) * NB + b) * 8);
  };

  const int mine = p0 + wv < p1 ? (p1 - p0 - wv + 3) / 4 : 0;
  if (mine > 0) {
    ask_k(0);
    ask_v(id_k);
  }
  // numbers that the compiler does not see through: a * half + zero and half * minus + a are then one mixed instruction each, where a product
  // or a difference is a conversion more
  float zero = 0.0f, minus = -1.0f;
  asm volatile("" : "+s"(zero), "+s"(minus));
  // Nibbles 0 and 4 of four dwords as numbers -8 .. 7: set behind 0x6400 they read 1024 + n, n the nibble with its upper bit flipped.  (The mask
  // and 0x6400 in registers of both kinds: one instruction for the and and the or.)
  uint32_t nibbles = 0x000F000Fu, thousand = 0x64006400u;
  asm volatile("" : "+s"(nibbles), "+v"(thousand));
  auto numbers = [&](uint32_t u0, uint32_t u1, uint32_t u2, uint32_t u3) {
    const u32x4 raw = {(u0 & nibbles) | thousand, (u1 & nibbles) | thousand, (u2 & nibbles) | thousand, (u3 & nibbles) | thousand};
    return __builtin_bit_cast(half8, raw) - (_Float16)1032.0f;
  };
  auto one_page = [&](auto whole, int k) {
    constexpr bool FULL = decltype(whole)::value;  // every row of the tile sees every row of the page
    const int page = p0 + wv + 4 * k;
    const int from = FULL ? 0 : id_v >= 0 && id_v < a.n_pages ? page * kKvPageRows : INT_MAX - kKvPageRows;  // (absent: behind every limit)
    *(sdw *)(s_scale[wv][0] + lane * NB * 2) = ks;
    *(sdw *)(s_scale[wv][1] + lane * NB * 2) = vs;
    const sdw vs_now = vs;
    f32x4 s[4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
      s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int b = 0; b < NB; b++) {
        const uint32_t u = kq[t][b] ^ 0x88888888u;
        const half8 kk = numbers(u, u >> 4, u >> 8, u >> 12);
        f32x4 x = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, q_lo[b], f32x4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
        x = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, q_hi[b], x, 0, 0, 0);
        const half4 d = scales(0, t, b);
#pragma unroll
        for (int i = 0; i < 4; i++) s[t][i] = fmaf(x[i], (float)d[i], s[t][i]);
      }
    }
    if (k + 1 < mine) ask_k(k + 1);
    float top = -INFINITY;
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if (!FULL && from + 16 * t + 4 * g + i > limit) s[t][i] = -INFINITY;
        top = fmaxf(top, s[t][i]);
      }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    if (__ballot(top > m)) {  // a new maximum in some row
      const float m_new = fmaxf(m, top), corr = m_new > -INFINITY ? __builtin_amdgcn_exp2f((m - m_new) * weight) : 1.0f;
      m = m_new;
      l *= corr;
#pragma unroll
      for (int b = 0; b < NB; b++) o[b][0] *= corr, o[b][1] *= corr;
    }
    {
      float d = 0.0f;  // the largest scale of the page's rows that are there (each lane has a piece of the page's scales)
#pragma unroll
      for (int x = 0; x < NB; x++) {
        const int flat = lane * NB + x, row = flat / (4 * NB) * 4 + flat % 4;
        const float dx = fabsf(half_bits_to_float(vs_now[x]));
        if (FULL || from + row <= last) d = fmaxf(d, dx);
      }
      d = fminf(wave_max(d), 65504.0f);
      const int want = 13 - ((int)(__float_as_uint(d) >> 23) - 127);
      if (d > 0.0f && want < c) {  // (uniform)
        const float f = ldexpf(1.0f, want - c);
        c = want;
        l *= f;
#pragma unroll
        for (int b = 0; b < NB; b++) o[b][0] *= f, o[b][1] *= f;
      }
    }
    const float base = (m > -INFINITY ? m * weight : 0.0f) - (float)c;
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        s[t][i] = __builtin_amdgcn_exp2f(fmaf(s[t][i], weight, -base));
        if (!FULL && from + 16 * t + 4 * g + i > limit) s[t][i] = 0.0f;
        l += s[t][i];
      }
#pragma unroll
    for (int b = 0; b < NB; b++) {
      u32x4 hi[2], lo[2];  // rows 16 t + 4 g + (0, 2, 1, 3), t = 0 1 and 2 3
#pragma unroll
      for (int t = 0; t < 4; t++) {
        const half4 d = scales(1, t, b);
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          x[i] = fmaf(s[t][i], (float)d[i], zero);
          if (!FULL && from + 16 * t + 4 * g + i > limit) x[i] = 0.0f;  // (the scale of a row that is not seen may be anything)
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const half2v h = __builtin_convertvector((f32x2){x[i], x[i + 2]}, half2v);
          const f32x2 r = {fmaf((float)h[0], minus, x[i]), fmaf((float)h[1], minus, x[i + 2])};
          hi[t >> 1][2 * (t & 1) + i] = __builtin_bit_cast(uint32_t, h);
          lo[t >> 1][2 * (t & 1) + i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, half2v));
        }
      }
#pragma unroll
      for (int part = 0; part < 2; part++) {
        const half8 ph = __builtin_bit_cast(half8, hi[part]), pl = __builtin_bit_cast(half8, lo[part]);
        const uint32_t u0 = vq[b][2 * part] ^ 0x88888888u, u1 = vq[b][2 * part + 1] ^ 0x88888888u;
#pragma unroll
        for (int half = 0; half < 2; half++) {
          const half8 vv = numbers(u0 >> (4 * half), u0 >> (4 * half + 8), u1 >> (4 * half), u1 >> (4 * half + 8));
          o[b][half] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv, pl, o[b][half], 0, 0, 0);
          o[b][half] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv, ph, o[b][half], 0, 0, 0);
        }
      }
    }
    if (k + 1 < mine) ask_v(id_k);
  };
  for (int k = 0; k < mine; k++) {
    if (id_v >= 0 && id_v < a.n_pages && (p0 + wv + 4 * k) * kKvPageRows + kKvPageRows - 1 <= least) one_page(std::true_type(), k);
    else one_page(std::false_type(), k);
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);

  // the four wavefronts' results meet
  if (g == 0) s_m[wv][n] = m * weight - (float)c, s_l[wv][n] = l;
#pragma unroll
  for (int b = 0; b < NB; b++)
#pragma unroll
    for (int half = 0; half < 2; half++) *(f32x4 *)&s_o[wv][n][b * 32 + half * 16 + 4 * g] = o[b][half];
  __syncthreads();
  float *record = a.parts + (int64_t)(w.slot + w.share) * kTileRows * (DH + 2);
  if (tid < kTileRows) {
    float M = -INFINITY, L = 0.0f;
    for (int x = 0; x < 4; x++) M = fmaxf(M, s_m[x][tid]);
    for (int x = 0; x < 4; x++) {
      const float e = s_m[x][tid] > -INFINITY ? __builtin_amdgcn_exp2f(s_m[x][tid] - M) : s_l[x][tid] == s_l[x][tid] ? 0.0f : 1.0f;
      s_w[x][tid] = e;
      L = fmaf(e, s_l[x][tid], L);
    }
    s_sum[tid] = L;
    if (shares > 1) {
      __hip_atomic_store(record + kTileRows * DH + tid, M, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(record + kTileRows * (DH + 1) + tid, L, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  __syncthreads();
  for (int e = tid; e < kTileRows * DH; e += 256) {
    const int r = e / DH, c = e % DH, rr = w.tile * kTileRows + r, jj = rr / G;
    float x = 0.0f;
    for (int k = 0; k < 4; k++) x = fmaf(s_w[k][r], s_o[k][r][c], x);
    if (shares > 1) {
      __hip_atomic_store(record + e, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    } else if (jj < w.rows) {
      const float L = s_sum[r];
      a.out[((int64_t)(w.row0 + jj) * a.H + w.head * G + rr - jj * G) * DH + c] = L != 0.0f ? x / L : 0.0f;
    }
  }
  if (shares == 1) return;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this thread's device-scope stores have reached memory
  __syncthreads();
  if (tid == 0) s_ticket = __hip_atomic_fetch_add(a.tickets + w.slot, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (s_ticket != shares - 1) return;  // (uniform)
  // the last of the job's workgroups adds the shares up, in their order
  if (tid == 0) __hip_atomic_store(a.tickets + w.slot, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // the next call counts again
  const float *records = a.parts + (int64_t)w.slot * kTileRows * (DH + 2);
  for (int e = tid; e < kTileRows * DH; e += 256) {
    const int r = e / DH, c = e % DH, rr = w.tile * kTileRows + r, jj = rr / G;
    if (jj >= w.rows) continue;
    float M = -INFINITY, L = 0.0f, x = 0.0f;
    for (int k = 0; k < shares; k++)
      M = fmaxf(M, __hip_atomic_load(records + (int64_t)k * kTileRows * (DH + 2) + kTileRows * DH + r, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    for (int k = 0; k < shares; k++) {
      const float *rec = records + (int64_t)k * kTileRows * (DH + 2);
      const float mk = __hip_atomic_load(rec + kTileRows * DH + r, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      const float lk = __hip_atomic_load(rec + kTileRows * (DH + 1) + r, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      const float xk = __hip_atomic_load(rec + e, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      const float f = mk > -INFINITY ? __builtin_amdgcn_exp2f(mk - M) : lk == lk ? 0.0f : 1.0f;
      L = fmaf(f, lk, L);
      x = fmaf(f, xk, x);
    }
    a.out[((int64_t)(w.row0 + jj) * a.H + w.head * G + rr - jj * G) * DH + c] = L != 0.0f ? x / L : 0.0f;
  }
}

}  // namespace cthip

using namespace cthip;

extern "C" {

int64_t cthip_sdpa_paged_q4_workspace(int head_dim) {
  if (!kv4_shape_ok(1, head_dim)) return fail(CTHIP_E_BAD_ARG, "cthip_sdpa_paged_q4_workspace: head size %d (32, 64, 128)", head_dim);
  return 4 * (2048ll + 2048ll * 16 * (head_dim + 2));
}

int cthip_sdpa_paged_q4(float *out, const float *q, int64_t q_stride, const void *k_pages, const void *v_pages, int n_pages, const int *tables, int table_stride,
                        const int *lens, const int *starts, int n_seqs, int n_rows, int H, int Hkv, int Dh, void *workspace) {
  CTHIP_REQUIRE_INIT();
  CTHIP_ARG(n_seqs >= 0 && n_rows >= 0 && n_pages >= 0 && n_pages <= INT_MAX / kKvPageRows && table_stride > 0 && table_stride <= INT_MAX / kKvPageRows);
  CTHIP_ARG(H > 0 && Hkv > 0 && H % Hkv == 0);
  if (!kv4_shape_ok(Hkv, Dh) || H > 65535) return fail(CTHIP_E_UNSUPPORTED, "cthip_sdpa_paged_q4: %d heads over %d of %d (at most 65535 heads, head sizes 32, 64, 128)", H, Hkv, Dh);
  if (n_seqs > kKv4MaxSeqs) return fail(CTHIP_E_UNSUPPORTED, "cthip_sdpa_paged_q4: %d sequences in one call (at most %d)", n_seqs, kKv4MaxSeqs);
  if (n_seqs == 0 || n_rows == 0) return 0;
  CTHIP_ARG(out && q && tables && lens && starts && workspace && q_stride >= (int64_t)H * Dh);
  CTHIP_ARG(n_pages == 0 || (k_pages && v_pages));
  CTHIP_ARG((((uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)workspace) & 15) == 0);
  // rows of a tile share a key / value head: at most this many tiles of all sequences, and as many jobs a head
  const int64_t tiles = (int64_t)n_rows * (H / Hkv) / kTileRows + (n_seqs < n_rows ? n_seqs : n_rows), jobs = tiles * Hkv;
  if (jobs > (1 << 28)) return fail(CTHIP_E_UNSUPPORTED, "cthip_sdpa_paged_q4: %d rows of %d heads in one call", n_rows, H);
  int unit = 0;
  while (jobs * ((table_stride >> unit) + 1) > INT_MAX) unit++;
  const Kv4Attn a = {out,   q,      (const unsigned char *)k_pages, (const unsigned char *)v_pages, tables, lens, starts, q_stride, n_pages, table_stride, n_seqs, n_rows, H, Hkv,
                     unit,  (int *)workspace, (float *)workspace + kSplitSlots};
  const dim3 grid((unsigned)(jobs + kTargetGroups)), block(256);
  switch (Dh) {
    case 32: hipLaunchKernelGGL(k_kv4_attn<32>, grid, block, 0, state().stream, a); break;
    case 64: hipLaunchKernelGGL(k_kv4_attn<64>, grid, block, 0, state().stream, a); break;
    default: hipLaunchKernelGGL(k_kv4_attn<128>, grid, block, 0, state().stream, a); break;
  }
  CTHIP_LAUNCH_CHECK();
  return 0;
}

}  // extern "C"
