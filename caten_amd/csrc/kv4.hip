// Batched serving over a paged KV cache in 4 bits: block tables and slot maps from the sequences' lengths, rows into the
// cache and back, and the reordering of a beam search's sequences.  The reference keeps one dense fp32 cache per model
// (external/llm/layers.lisp:19-33) and one sequence; a server holds many sequences of different lengths, so here all of them
// take pages from one pool, and everything a step needs to know about who owns what is worked out on the device: a step's
// launches can be captured once and replayed.  Layout of a page: kv4.h.
#include <algorithm>

#include "kv4.h"

namespace cthip {

// ---- block tables and slot maps ----
// starts = exclusive sum of the new rows, pages wanted = ceil((len + new) / 64) - ceil(len / 64), and their exclusive sum says
// which entries of the free stack a sequence gets.  Every workgroup works the two sums out for itself (n <= 4096 in LDS, at most
// four sequences a thread) and then finds the sequence of each of its rows by bisection: one launch, nothing to wait for
// between workgroups.  The row that opens a page enters it into the table.  Bound by latencies: a launch, two sums over 1024
// threads (data-parallel moves; by exchanges through LDS and 256 rows a workgroup 14.4 us instead of 7.5 for 500 sequences with room for
// 150000 rows) and a bisection.  64 sequences of a decode step: 4.8 us.
constexpr int kPlanThreads = 1024, kPlanRows = 2048;  // rows of a workgroup: most decode steps are one workgroup

template <int CTRL, int ROWS>
__device__ __forceinline__ int64_t scan_step(int64_t v) {  // plus the value a data-parallel move brings; 0 where it brings none
  const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, ROWS == 0xF), hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, ROWS, 0xF, ROWS == 0xF);
  return v + (int64_t)((uint64_t)hi << 32 | lo);
}
// exclusive, over kPlanThreads threads; part: LDS of a call's own
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t *part, int64_t &total) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  int64_t s = v;
  s = scan_step<0x111, 0xF>(s);  // row_shr 1, 2, 4, 8, then the rows' ends
  s = scan_step<0x112, 0xF>(s);
  s = scan_step<0x114, 0xF>(s);
  s = scan_step<0x118, 0xF>(s);
  s = scan_step<0x142, 0xA>(s);
  s = scan_step<0x143, 0xC>(s);
  if (lane == 63) part[wv] = s;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; w++) {
    const int64_t p = part[w];
    if (w < wv) before += p;
    total += p;
  }
  return before + s - v;
}

__global__ __launch_bounds__(kPlanThreads) void k_kv_plan(int *__restrict__ slots, int *__restrict__ positions, int *__restrict__ starts, int *tables,
                                                          int table_stride, int *lens_out, int *n_free_out, int *refused, const int *lens,
                                                          const int *__restrict__ new_lens, int n, const int *__restrict__ free_pages,
                                                          const int *n_free, int max_rows, bool rows_too, bool lens_too) {
  __shared__ int s_start[kKv4MaxSeqs + 1];  // first row; rows past max_rows are all the same to a reader: they saturate
  __shared__ int s_len[kKv4MaxSeqs];        // rows in the cache, -1 = refused
  __shared__ int s_page[kKv4MaxSeqs];       // pages handed out in front of it
  __shared__ int64_t part[4][kPlanThreads / 64];  // (two for a round, in turn: nobody waits until they have been read)
  __shared__ int s_refused, s_used;
  const int tid = threadIdx.x;
  const int64_t cap = (int64_t)table_stride * kKvPageRows, have_free = n_free[0];
  if (tid == 0) s_refused = 0, s_used = 0;
  __syncthreads();
  int64_t row0 = 0, page0 = 0;
  int bad = 0;
  for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int i = i0 + tid;
    const int64_t len = i < n ? lens[i] : 0, add = i < n ? new_lens[i] : 0;
    int64_t rows, pages;
    const int64_t start = row0 + block_scan(add > 0 ? add : 0, part[i0 / kPlanThreads % 2 * 2], rows);
    bool ok = len >= 0 && add >= 0 && len + add <= cap && start + add <= max_rows;
    const int64_t need = ok ? (len + add + kKvPageRows - 1) / kKvPageRows - (len + kKvPageRows - 1) / kKvPageRows : 0;
    const int64_t before = page0 + block_scan(need, part[i0 / kPlanThreads % 2 * 2 + 1], pages);
    ok = ok && (need == 0 || before + need <= have_free);
    if (i < n) {
      s_start[i] = (int)min(start, (int64_t)INT_MAX);
      s_len[i] = ok ? (int)len : -1;
      s_page[i] = (int)min(before, (int64_t)INT_MAX);
      if (!ok) bad++;
      else if (need) atomicMax(&s_used, (int)(before + need));  // sequences are refused from one on: the last one with pages has the sum of them all
    }
    row0 += rows;
    page0 += pages;
  }
  if (bad) atomicAdd(&s_refused, bad);
  if (tid == 0) s_start[n] = (int)min(row0, (int64_t)INT_MAX);
  __syncthreads();  // every length has been read: lens_out may be the same array where this is the only workgroup
  if (blockIdx.x == 0 && lens_too) {
    for (int i = tid; i < n; i += kPlanThreads) {
      if (s_len[i] >= 0) lens_out[i] = s_len[i] + s_start[i + 1] - s_start[i];
      else if (lens_out != lens) lens_out[i] = lens[i];
    }
    if (tid == 0) {
      n_free_out[0] = (int)have_free - s_used;
      refused[0] = s_refused;
    }
  }
  if (!rows_too) return;
  if (blockIdx.x == 0)
    for (int i = tid; i <= n; i += kPlanThreads) starts[i] = s_start[i];
  const int rows = s_start[n];
  const int r1 = min((int64_t)max_rows, (int64_t)(blockIdx.x + 1) * kPlanRows);
  for (int r = blockIdx.x * kPlanRows + tid; r < r1; r += kPlanThreads) {
    int slot = -1, at = -1;
    if (r < rows) {
      int lo = 0, hi = n;  // s_start[lo] <= r < s_start[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_start[mid] <= r) lo = mid;
        else hi = mid;
      }
      const int len = s_len[lo];
      if (len >= 0) {
        at = len + r - s_start[lo];
        const int page = at / kKvPageRows, have = (len + kKvPageRows - 1) / kKvPageRows;
        int id;
        if (page < have) {
          id = tables[(int64_t)lo * table_stride + page];
        } else {
          id = free_pages[(int)have_free - 1 - (s_page[lo] + page - have)];
          if (at % kKvPageRows == 0) tables[(int64_t)lo * table_stride + page] = id;
        }
        if (id >= 0 && id <= INT_MAX / kKvPageRows - 1) slot = id * kKvPageRows + at % kKvPageRows;
      }
    }
    slots[r] = slot;
    if (positions) positions[r] = at;
  }
}

// ---- pages back to the free stack ----
// The stack's own array is the set of pages: filled with all ids, those in use struck out (by any number of threads, with the same value), and
// what is left moved to the front, one workgroup, 8192 at a time: a chunk has been read by all threads before what is left of it is
// written, in front of the next one's place.  Three launches: 9.5 us for 144 beams and a pool of 3000 pages; 100000 pages, 71 us, wait for that one
// workgroup's round trips.
constexpr int kFreeEach = 8;
__global__ __launch_bounds__(256) void k_kv_free_all(int *free_pages, int n_pages) {
  for (int64_t i = blockIdx.x * 256 + threadIdx.x; i < n_pages; i += (int64_t)gridDim.x * 256) free_pages[i] = (int)i;
}
__global__ __launch_bounds__(256) void k_kv_free_strike(int *free_pages, const int *__restrict__ tables, int table_stride, const int *__restrict__ lens, int n_pages) {
  const int len = max(lens[blockIdx.x], 0), pages = min(len / kKvPageRows + (len % kKvPageRows != 0), table_stride);
  for (int c = threadIdx.x; c < pages; c += 256) {
    const int id = tables[(int64_t)blockIdx.x * table_stride + c];
    if (id >= 0 && id < n_pages) free_pages[id] = -1;
  }
}
__global__ __launch_bounds__(kPlanThreads) void k_kv_free_pack(int *free_pages, int *n_free, int n_pages) {
  __shared__ int64_t part[2][kPlanThreads / 64];
  int kept = 0;
  for (int i0 = 0, round = 0; i0 < n_pages; i0 += kFreeEach * kPlanThreads, round++) {
    int id[kFreeEach], mine = 0;
#pragma unroll
    for (int k = 0; k < kFreeEach; k++) {
      const int i = i0 + kFreeEach * (int)threadIdx.x + k;
      id[k] = i < n_pages ? free_pages[i] : -1;
      mine += id[k] >= 0;
    }
    int64_t all;
    int at = kept + (int)block_scan(mine, part[round & 1], all);
#pragma unroll
    for (int k = 0; k < kFreeEach; k++)
      if (id[k] >= 0) free_pages[at++] = id[k];
    kept += (int)all;
  }
  if (threadIdx.x == 0) n_free[0] = kept;
}

// ---- rows into the cache ----
// Four lanes hold a block of 32 channels, eight each.  d = m / -8 as fp16, m the value of largest magnitude (the positive one
// of two), kept finite; u = floor(x / d + 1/2) within -8 .. 7, d being the scale as it is STORED.  The quotient is taken by a
// reciprocal, and what it leaves, x - u d, is exact in fp32 (u d has 15 bits, and what is left of x where u is not 0 no more than x has):
// where that is not within half a step, u moves by one, so the number is the one of real arithmetic whatever the reciprocal's
// rounding.  A block with an infinity or a NaN has a NaN scale.  Bound by the rows that come in (8 bytes a channel of keys and values):
// 6001 rows of 8 heads of 128 in 17.2 us, 3.3 TB/s in and out of the card; back as fp32 17.6 us.
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, dpp_f<0xB1>(v));
  return fmaxf(v, dpp_f<0x4E>(v));
}

__device__ __forceinline__ uint32_t kv4_quantise8(const float *x, unsigned short &scale) {  // the eight two's complement nibbles, channel 0 lowest
  float hi = x[0], lo = x[0], odd = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    hi = fmaxf(hi, x[e]);
    lo = fminf(lo, x[e]);
    if (!(fabsf(x[e]) < INFINITY)) odd = 1.0f;
  }
  hi = quad_max(hi);
  lo = -quad_max(-lo);
  odd = quad_max(odd);
  const float m = hi >= -lo ? hi : lo;
  const _Float16 d16 = (_Float16)fminf(fmaxf(m * -0.125f, -65504.0f), 65504.0f);
  const float d = (float)d16, ds = fabsf(d);
  scale = odd != 0.0f ? (unsigned short)0x7E00 : __builtin_bit_cast(unsigned short, d16);
  if (odd != 0.0f || ds == 0.0f) return 0u;
  const float inv = 1.0f / ds, half = 0.5f * ds;
  float u[8], xs[8];
  bool off = false;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    xs[e] = d < 0.0f ? -x[e] : x[e];
    u[e] = floorf(fmaf(xs[e], inv, 0.5f));
    const float left = fmaf(-u[e], ds, xs[e]);
    off = off || left >= half || left < -half;
  }
  if (off) {  // (seldom: within 2^-20 of a border)
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const float left = fmaf(-u[e], ds, xs[e]);
      u[e] += left >= half ? 1.0f : left < -half ? -1.0f : 0.0f;
    }
  }
  // four numbers as one of base 16; with 8 added to each the digits are nibbles
  float lo4 = 0.0f, hi4 = 0.0f;
#pragma unroll
  for (int e = 3; e >= 0; e--) {
    lo4 = fmaf(lo4, 16.0f, fminf(fmaxf(u[e], -8.0f), 7.0f));
    hi4 = fmaf(hi4, 16.0f, fminf(fmaxf(u[4 + e], -8.0f), 7.0f));
  }
  return ((uint32_t)((int)lo4 + 0x8888) | (uint32_t)((int)hi4 + 0x8888) << 16) ^ 0x88888888u;
}

struct Kv4Rows {
  unsigned char *k_pages, *v_pages;
  const float *k_in, *v_in;  // into the cache
  float *k_out, *v_out;      // out of it
  int64_t k_stride, v_stride;
  const int *slots;
  int n_rows, n_pages, kv;
};
// nibbles 0 .. 3 of a dword as the low halves of its bytes
__device__ __forceinline__ uint32_t spread4(uint32_t w) { return (w & 0xF) | (w & 0xF0) << 4 | (w & 0xF00) << 8 | (w & 0xF000) << 12; }
// The quad of lanes that holds a value block: lanes 0 and 1 its channels 0 .. 15, 2 and 3 their partners.  Each lane gets the four bytes of
// four channels, the first of which is returned.
__device__ __forceinline__ int value_bytes(uint32_t w, int g, unsigned char *bytes) {
  const uint32_t other = __builtin_bit_cast(uint32_t, dpp_f<0x4E>(__builtin_bit_cast(float, w)));
  const uint32_t low = g < 2 ? w : other, high = g < 2 ? other : w;
  const int j0 = g < 2 ? 0 : 4;
#pragma unroll
  for (int j = 0; j < 4; j++) bytes[j] = (unsigned char)(((low >> 4 * (j0 + j)) & 15u) | ((high >> 4 * (j0 + j)) & 15u) << 4);
  return 8 * (g & 1) + j0;
}
__device__ __forceinline__ void load8(const float *src, float *x) {
  *(f4_any *)x = *(const f4_any *)src;
  *(f4_any *)(x + 4) = *(const f4_any *)(src + 4);
}
__device__ __forceinline__ void key_values(uint32_t w, float d, float *x) {
#pragma unroll
  for (int j = 0; j < 4; j++) {
    x[j] = d * (float)((int)(w << (28 - 8 * j)) >> 28);
    x[4 + j] = d * (float)((int)(w << (24 - 8 * j)) >> 28);
  }
}

// Few rows: one row per blockIdx.x (fewer than 2^15 of them, since a row has 32 channels at least), keys (blockIdx.z = 0) or values; a thread per eight channels
template <bool IN>
__global__ __launch_bounds__(256) void k_kv4_rows(Kv4Rows a, int dh) {
  const int e8 = blockIdx.y * 256 + threadIdx.x;  // eighth of the row
  if (e8 >= a.kv * dh / 8) return;                 // (kv * dh / 8 is a multiple of 4: whole quads leave)
  const int slot = a.slots[blockIdx.x];
  if (slot < 0 || slot >= a.n_pages * kKvPageRows) return;
  const bool values = blockIdx.z != 0;
  const int row = slot % kKvPageRows, h = 8 * e8 / dh, c8 = e8 - h * (dh / 8), b = c8 >> 2, g = c8 & 3;
  unsigned char *head = (values ? a.v_pages : a.k_pages) + ((int64_t)(slot / kKvPageRows) * a.kv + h) * kv4_head_bytes(dh);
  float x[8];
  if (IN) {
    load8((values ? a.v_in + blockIdx.x * a.v_stride : a.k_in + blockIdx.x * a.k_stride) + 8 * e8, x);
    unsigned short d;
    const uint32_t w = kv4_quantise8(x, d);
    if (g == 0) *(unsigned short *)(head + kv4_scale_offset(row, b, dh)) = d;
    if (!values) {
      *(uint32_t *)(head + kv4_key_offset(row, g, b, dh)) = spread4(w) | spread4(w >> 16) << 4;
    } else {
      unsigned char bytes[4];
      const int c = value_bytes(w, g, bytes);
#pragma unroll
      for (int j = 0; j < 4; j++) head[kv4_value_offset(row, b, c + j)] = bytes[j];
    }
  } else {
    float *out = values ? a.v_out : a.k_out;
    if (!out) return;
    const float d = half_bits_to_float(*(const unsigned short *)(head + kv4_scale_offset(row, b, dh)));
    if (!values) {
      key_values(*(const uint32_t *)(head + kv4_key_offset(row, g, b, dh)), d, x);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) x[j] = d * (float)((int)((uint32_t)head[kv4_value_offset(row, b, 8 * (g & 1) + j)] << (g < 2 ? 28 : 24)) >> 28);
    }
    float *dst = out + (int64_t)blockIdx.x * a.kv * dh + 8 * e8;
    *(f4_any *)dst = *(const f4_any *)x;
    *(f4_any *)(dst + 4) = *(const f4_any *)(x + 4);
  }
}

// Many rows: 64 consecutive ones of one head a workgroup.  Where their slots follow one another -- a piece of a prompt: the end of a page and
// the beginning of another, or a whole one -- values and scales go through LDS, where they lie as in a page, and four rows at a time
// between there and memory: row by row they are single bytes, each in a line of its own.
template <int DH, bool IN>
__global__ __launch_bounds__(256) void k_kv4_rows64(Kv4Rows a) {
  constexpr int NB = DH / 32, TPR = DH / 8, LINE = kKvPageRows + 4;  // (lines of 17 dwords: a row's bytes lie in different banks)
  __shared__ int s_slot[kKvPageRows];
  __shared__ __align__(16) unsigned char s_v[DH / 2 * LINE];
  __shared__ __align__(16) unsigned short s_d[kKvPageRows * NB];  // [row / 4][block][row % 4]
  const int tid = threadIdx.x, r0 = blockIdx.x * kKvPageRows, count = min(kKvPageRows, a.n_rows - r0), h = blockIdx.y;
  const bool values = blockIdx.z != 0;
  if (!IN && !(values ? a.v_out : a.k_out)) return;
  if (tid < kKvPageRows) s_slot[tid] = tid < count ? a.slots[r0 + tid] : -1;
  __syncthreads();
  const int first = s_slot[0], o = first & (kKvPageRows - 1), split = kKvPageRows - o;  // rows split .. lie in a second page
  const int page_a = first / kKvPageRows, page_b = split < count ? s_slot[split] / kKvPageRows : page_a;
  bool fine = true;
  if (tid < count) {
    const int slot = s_slot[tid];
    fine = slot >= 0 && slot < a.n_pages * kKvPageRows && slot / kKvPageRows == (tid < split ? page_a : page_b) && (slot & (kKvPageRows - 1)) == ((o + tid) & (kKvPageRows - 1));
  }
  const bool follow = __syncthreads_and(fine);  // every slot one behind the other
  unsigned char *pool = values ? a.v_pages : a.k_pages;
  auto head_of = [&](int page) { return pool + ((int64_t)page * a.kv + h) * kv4_head_bytes(DH); };
  auto there = [&](int row) { return ((row - o) & (kKvPageRows - 1)) < count; };  // row of a page: whether it is one of ours
  auto home = [&](int row) { return head_of(row >= o ? page_a : page_b); };
  // the pages' values (four rows of a channel pair a dword, which in a page lie one behind the other) and scales
  auto exchange = [&]() {
    for (int d = tid; values && d < DH / 2 * 16; d += 256) {
      const int line = d >> 4, q = d & 15, row = 16 * (q & 3) + 4 * (q >> 2);
      unsigned char *mine = s_v + line * LINE + 4 * q;
      if (there(row) && there(row + 3) && (row + 3 < o || row >= o)) {
        uint32_t *p = (uint32_t *)(home(row) + 4 * d);
        if (IN) *p = *(const uint32_t *)mine;
        else *(uint32_t *)mine = *p;
      } else {
        for (int i = 0; i < 4; i++)
          if (there(row + i)) {
            unsigned char *p = home(row + i) + 4 * d + i;
            if (IN) *p = mine[i];
            else mine[i] = *p;
          }
      }
    }
    for (int d = tid; d < 16 * NB; d += 256) {
      const int row = d / NB * 4;
      unsigned short *mine = s_d + 4 * d;
      if (there(row) && there(row + 3) && (row + 3 < o || row >= o)) {
        uint2 *p = (uint2 *)(home(row) + 32 * DH + 8 * d);
        if (IN) *p = *(const uint2 *)mine;
        else *(uint2 *)mine = *p;
      } else {
        for (int i = 0; i < 4; i++)
          if (there(row + i)) {
            unsigned short *p = (unsigned short *)(home(row + i) + 32 * DH + 8 * d) + i;
            if (IN) *p = mine[i];
            else mine[i] = *p;
          }
      }
    }
  };
  if (!IN && follow) {
    exchange();
    __syncthreads();
  }
  const int c8 = tid % TPR, b = c8 >> 2, g = c8 & 3;
#pragma unroll
  for (int pass = 0; pass < kKvPageRows / (256 / TPR); pass++) {
    const int r = pass * (256 / TPR) + tid / TPR;
    const int slot = r < count ? s_slot[r] : -1, row = slot & (kKvPageRows - 1);
    if (slot < 0 || slot >= a.n_pages * kKvPageRows) continue;  // (whole quads)
    unsigned char *head = head_of(slot / kKvPageRows);
    unsigned short *scale = follow ? s_d + ((row >> 2) * NB + b) * 4 + (row & 3) : (unsigned short *)(head + kv4_scale_offset(row, b, DH));
    float x[8];
    if (IN) {
      load8((values ? a.v_in + (r0 + r) * a.v_stride : a.k_in + (r0 + r) * a.k_stride) + h * DH + 8 * c8, x);
      unsigned short d;
      const uint32_t w = kv4_quantise8(x, d);
      if (g == 0) *scale = d;
      if (!values) {
        *(uint32_t *)(head + kv4_key_offset(row, g, b, DH)) = spread4(w) | spread4(w >> 16) << 4;
      } else {
        unsigned char bytes[4];
        const int c = value_bytes(w, g, bytes);
#pragma unroll
        for (int j = 0; j < 4; j++) {
          if (follow) s_v[(b * 16 + c + j) * LINE + kv4_value_place(row)] = bytes[j];
          else head[kv4_value_offset(row, b, c + j)] = bytes[j];
        }
      }
    } else {
      const float d = half_bits_to_float(*scale);
      if (!values) {
        key_values(*(const uint32_t *)(head + kv4_key_offset(row, g, b, DH)), d, x);
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const int line = b * 16 + 8 * (g & 1) + j;
          const unsigned char byte = follow ? s_v[line * LINE + kv4_value_place(row)] : head[line * kKvPageRows + kv4_value_place(row)];
          x[j] = d * (float)((int)((uint32_t)byte << (g < 2 ? 28 : 24)) >> 28);
        }
      }
      float *dst = (values ? a.v_out : a.k_out) + ((int64_t)(r0 + r) * a.kv + h) * DH + 8 * c8;
      // (more than the caches between here and the reader would keep: 39 -> 34 us for 6001 rows of 8 heads of 128 in and out)
      __builtin_nontemporal_store(*(const f4_any *)x, (f4_any *)dst);
      __builtin_nontemporal_store(*(const f4_any *)(x + 4), (f4_any *)(dst + 4));
    }
  }
  if (IN && follow) {
    __syncthreads();
    exchange();
  }
}

template <bool IN>
static int launch_kv4_rows(const Kv4Rows &a, int dh) {
  const int eighths = a.kv * dh / 8;
  // Rows of a step, a few a sequence, or long prompts.  512 rows of 8 heads of 128, one behind the other: 4.3 us row by row, 6.9 by 64 at a time;
  // 1024: 6.3 and 7.0; 2048: 10.2 and 7.8; 4096: 17.6 and 10.7 (out of the cache 3.9, 6.2; 5.2, 6.4; 9.0, 7.3; 16.3, 10.3).  Fewer and narrower
  // heads: alike at 2^20 channels in all.
  if ((int64_t)a.n_rows * a.kv * dh < (1 << 20)) {
    hipLaunchKernelGGL(k_kv4_rows<IN>, dim3((unsigned)a.n_rows, (unsigned)((eighths + 255) / 256), 2), dim3(256), 0, state().stream, a, dh);
  } else {
    const dim3 grid((unsigned)((a.n_rows + kKvPageRows - 1) / kKvPageRows), (unsigned)a.kv, 2);
#define ROWS(DH_) hipLaunchKernelGGL((k_kv4_rows64<DH_, IN>), grid, dim3(256), 0, state().stream, a)
    if (dh == 32) ROWS(32);
    else if (dh == 64) ROWS(64);
    else ROWS(128);
#undef ROWS
  }
  CTHIP_LAUNCH_CHECK();
  return 0;
}

// ---- reordering of beams ----
// Pages that are full are the same for all beams of a request and stay shared; the partly filled last page is each beam's
// own.  A parent's page goes to its first child as it is; every further child needs a copy, and there are as many pages of
// beams without a child: the further children take them in order.  A page that is copied from is kept by somebody and is not
// copied to, so the copies need no order among themselves, and a call repeated on the same tables writes the same bytes.
// Bound by a launch and three round trips (parents, table, page) where there is little to copy: 4.6 us for 4 beams; 24 x 6 beams in 22 layers,
// 33 MB: 8.7 us (a load for each parent in turn, and a workgroup for each page: 13).
struct ReorderArgs {
  int *tables_out, *history_out;
  unsigned char *k_pages, *v_pages;
  const int *tables, *lens, *parents, *history, *tokens, *step;
  int table_stride, n_layers, n_pages, beams, cols, page_bytes;
};
constexpr int kMaxBeams = 32;
typedef uint32_t dwords4 __attribute__((ext_vector_type(4)));

// blockIdx.y = beam; blockIdx.x = 0: its row of the table and its history, otherwise a page of keys and one of values in layer x - 1.  Who is
// whose child is worked out from one load of all parents.
__global__ __launch_bounds__(256) void k_beam_reorder(ReorderArgs a) {
  const int n0 = blockIdx.y / a.beams * a.beams, j = blockIdx.y - n0, tid = threadIdx.x, lane = tid & 63;
  int parent = lane;
  if (lane < a.beams) {
    const int p = a.parents[n0 + lane];
    if (p >= 0 && p < a.beams) parent = p;
  }
  const int len = a.lens[blockIdx.y / a.beams];
  int rank = 0;  // children in front of this one that need a copy
  bool further = false;
  unsigned alive = 0;
  for (int i = 0; i < a.beams; i++) {
    const int p = __builtin_amdgcn_readlane(parent, i);
    const bool again = (alive >> p) & 1u;
    alive |= 1u << p;
    if (i < j && again) rank++;
    if (i == j) further = again;
  }
  const int mine = __builtin_amdgcn_readlane(parent, j);
  const int last = len > 0 ? len / kKvPageRows : 0;
  const bool tail = len > 0 && len % kKvPageRows != 0 && last < a.table_stride;
  int owner = mine;  // whose last page this beam gets
  if (further) {
    unsigned dead = ~alive;  // (there are as many of them among the beams as further children)
    for (int k = 0; k < rank; k++) dead &= dead - 1;
    owner = __builtin_ctz(dead);
  }
  const int *from = a.tables + (int64_t)(n0 + mine) * a.table_stride;
  if (blockIdx.x == 0) {
    const int *own = a.tables + (int64_t)blockIdx.y * a.table_stride, *tail_of = a.tables + (int64_t)(n0 + owner) * a.table_stride;
    int *to = a.tables_out + (int64_t)blockIdx.y * a.table_stride;
    for (int c = tid; c < a.table_stride; c += 256) to[c] = c < last ? from[c] : c == last && tail ? tail_of[c] : own[c];
    if (a.history_out) {
      const int at = a.step[0];
      const int *old = a.history + (int64_t)(n0 + mine) * a.cols;
      int *h = a.history_out + (int64_t)blockIdx.y * a.cols;
      for (int c = tid; c < a.cols; c += 256) h[c] = c == at ? a.tokens[blockIdx.y] : old[c];
    }
    return;
  }
  if (!further || !tail) return;
  const int src = from[last], dst = a.tables[(int64_t)(n0 + owner) * a.table_stride + last];
  if (src < 0 || src >= a.n_pages || dst < 0 || dst >= a.n_pages) return;
  const int layer = blockIdx.x - 1, n = a.page_bytes / 16;
  for (int values = 0; values < 2; values++) {
    unsigned char *pool = (values ? a.v_pages : a.k_pages) + (int64_t)layer * a.n_pages * a.page_bytes;
    const dwords4 *s = (const dwords4 *)(pool + (int64_t)src * a.page_bytes);
    dwords4 *d = (dwords4 *)(pool + (int64_t)dst * a.page_bytes);
    for (int e = tid; e < n; e += 4 * 256) {
      dwords4 v[4];
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (e + 256 * k < n) v[k] = s[e + 256 * k];
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (e + 256 * k < n) d[e + 256 * k] = v[k];
    }
  }
}

}  // namespace cthip

using namespace cthip;

static bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

extern "C" {

int64_t cthip_kv_page_bytes_q4(int kv_heads, int head_dim) {
  if (!kv4_shape_ok(kv_heads, head_dim)) return fail(CTHIP_E_BAD_ARG, "cthip_kv_page_bytes_q4: %d heads of %d (head sizes 32, 64, 128)", kv_heads, head_dim);
  return (int64_t)kv_heads * kv4_head_bytes(head_dim);
}

int cthip_kv_plan_paged(int *slots, int *positions, int *starts, int *tables, int table_stride, int *lens_out, int *n_free_out, int *refused,
                        const int *lens, const int *new_lens, int n_seqs, const int *free_pages, const int *n_free, int max_rows) {
  CTHIP_REQUIRE_INIT();
  CTHIP_ARG(n_seqs >= 0 && max_rows >= 0 && max_rows <= (1 << 30) && table_stride > 0 && table_stride <= INT_MAX / kKvPageRows);
  if (n_seqs > kKv4MaxSeqs) return fail(CTHIP_E_UNSUPPORTED, "cthip_kv_plan_paged: %d sequences in one call (at most %d)", n_seqs, kKv4MaxSeqs);
  CTHIP_ARG(starts && lens_out && n_free_out && refused && n_free && (max_rows == 0 || slots));
  CTHIP_ARG(n_seqs == 0 || (tables && lens && new_lens && free_pages));
  const int blocks = max_rows > 0 ? (max_rows + kPlanRows - 1) / kPlanRows : 1;
  // several workgroups read the lengths while one of them would overwrite them: a launch of its own behind them then
  const bool apart = blocks > 1 && (lens_out == lens || n_free_out == n_free);
  hipLaunchKernelGGL(k_kv_plan, dim3((unsigned)blocks), dim3(kPlanThreads), 0, state().stream, slots, positions, starts, tables, table_stride, lens_out, n_free_out, refused,
                     lens, new_lens, n_seqs, free_pages, n_free, max_rows, true, !apart);
  CTHIP_LAUNCH_CHECK();
  if (apart) {
    hipLaunchKernelGGL(k_kv_plan, dim3(1), dim3(kPlanThreads), 0, state().stream, slots, positions, starts, tables, table_stride, lens_out, n_free_out, refused, lens,
                       new_lens, n_seqs, free_pages, n_free, max_rows, false, true);
    CTHIP_LAUNCH_CHECK();
  }
  return 0;
}

int cthip_kv_free_paged(int *free_pages, int *n_free, const int *tables, int table_stride, const int *lens, int n_seqs, int n_pages) {
  CTHIP_REQUIRE_INIT();
  CTHIP_ARG(n_seqs >= 0 && n_pages >= 0 && n_pages <= INT_MAX / kKvPageRows && table_stride > 0);
  if (n_seqs > 65535) return fail(CTHIP_E_UNSUPPORTED, "cthip_kv_free_paged: %d sequences in one call (at most 65535)", n_seqs);
  CTHIP_ARG(n_free && (n_pages == 0 || free_pages) && (n_seqs == 0 || (tables && lens)));
  if (n_pages > 0) {
    hipLaunchKernelGGL(k_kv_free_all, dim3((unsigned)std::min(1024, (n_pages + 255) / 256)), dim3(256), 0, state().stream, free_pages, n_pages);
    CTHIP_LAUNCH_CHECK();
  }
  if (n_pages > 0 && n_seqs > 0) {
    hipLaunchKernelGGL(k_kv_free_strike, dim3((unsigned)n_seqs), dim3(256), 0, state().stream, free_pages, tables, table_stride, lens, n_pages);
    CTHIP_LAUNCH_CHECK();
  }
  hipLaunchKernelGGL(k_kv_free_pack, dim3(1), dim3(kPlanThreads), 0, state().stream, free_pages, n_free, n_pages);
  CTHIP_LAUNCH_CHECK();
  return 0;
}

int cthip_kv_append_paged_q4(void *k_pages, void *v_pages, const float *k_rows, const float *v_rows, int64_t k_stride, int64_t v_stride, const int *slots,
                             int n_rows, int n_pages, int kv_heads, int head_dim) {
  CTHIP_REQUIRE_INIT();
  CTHIP_ARG(n_rows >= 0 && n_pages >= 0 && n_pages <= INT_MAX / kKvPageRows);
  if (!kv4_shape_ok(kv_heads, head_dim)) return fail(CTHIP_E_UNSUPPORTED, "cthip_kv_append_paged_q4: %d heads of %d (head sizes 32, 64, 128)", kv_heads, head_dim);
  if (n_rows > (1 << 28)) return fail(CTHIP_E_UNSUPPORTED, "cthip_kv_append_paged_q4: %d rows in one call (at most 2^28)", n_rows);
  if (n_rows == 0 || n_pages == 0) return 0;
  CTHIP_ARG(k_pages && v_pages && k_rows && v_rows && slots);
  CTHIP_ARG(aligned16(k_pages) && aligned16(v_pages) && k_stride >= (int64_t)kv_heads * head_dim && v_stride >= (int64_t)kv_heads * head_dim);
  return launch_kv4_rows<true>({(unsigned char *)k_pages, (unsigned char *)v_pages, k_rows, v_rows, nullptr, nullptr, k_stride, v_stride, slots, n_rows, n_pages, kv_heads}, head_dim);
}

int cthip_kv_rows_paged_q4(float *k_rows, float *v_rows, const void *k_pages, const void *v_pages, const int *slots, int n_rows, int n_pages, int kv_heads,
                           int head_dim) {
  CTHIP_REQUIRE_INIT();
  CTHIP_ARG(n_rows >= 0 && n_pages >= 0 && n_pages <= INT_MAX / kKvPageRows);
  if (!kv4_shape_ok(kv_heads, head_dim)) return fail(CTHIP_E_UNSUPPORTED, "cthip_kv_rows_paged_q4: %d heads of %d (head sizes 32, 64, 128)", kv_heads, head_dim);
  if (n_rows > (1 << 28)) return fail(CTHIP_E_UNSUPPORTED, "cthip_kv_rows_paged_q4: %d rows in one call (at most 2^28)", n_rows);
  if (n_rows == 0 || n_pages == 0 || (!k_rows && !v_rows)) return 0;
  CTHIP_ARG(slots && (!k_rows || k_pages) && (!v_rows || v_pages) && aligned16(k_pages) && aligned16(v_pages));
  return launch_kv4_rows<false>({(unsigned char *)k_pages, (unsigned char *)v_pages, nullptr, nullptr, k_rows, v_rows, 0, 0, slots, n_rows, n_pages, kv_heads}, head_dim);
}

int cthip_beam_reorder_paged_q4(int *tables_out, int *history_out, void *k_pages, void *v_pages, int n_layers, int n_pages, const int *tables, int table_stride,
                                const int *lens, const int *parents, int n_batch, int n_beams, int kv_heads, int head_dim, const int *history, int cols,
                                const int *tokens, const int *step) {
  CTHIP_REQUIRE_INIT();
  CTHIP_ARG(n_batch >= 0 && n_beams >= 1 && n_layers >= 0 && n_pages >= 0 && n_pages <= INT_MAX / kKvPageRows && table_stride > 0 && cols >= 0);
  if (n_beams > kMaxBeams) return fail(CTHIP_E_UNSUPPORTED, "cthip_beam_reorder_paged_q4: %d beams (at most %d)", n_beams, kMaxBeams);
  if (!kv4_shape_ok(kv_heads, head_dim)) return fail(CTHIP_E_UNSUPPORTED, "cthip_beam_reorder_paged_q4: %d heads of %d (head sizes 32, 64, 128)", kv_heads, head_dim);
  if (n_layers > (1 << 20) || (int64_t)n_batch * n_beams > 65535)
    return fail(CTHIP_E_UNSUPPORTED, "cthip_beam_reorder_paged_q4: %d layers, %d x %d beams (at most 1048576 layers, 65535 beams)", n_layers, n_batch, n_beams);
  if (n_batch == 0) return 0;
  CTHIP_ARG(tables_out && tables && tables_out != tables && lens && parents);
  CTHIP_ARG(n_layers == 0 || n_pages == 0 || (k_pages && v_pages && aligned16(k_pages) && aligned16(v_pages)));
  CTHIP_ARG(!history_out || (history && history_out != history && tokens && step));
  const ReorderArgs a = {tables_out, cols ? history_out : nullptr, (unsigned char *)k_pages, (unsigned char *)v_pages, tables, lens, parents, history, tokens, step,
                         table_stride, n_layers, n_pages, n_beams, cols, kv_heads * kv4_head_bytes(head_dim)};
  const unsigned copies = n_pages ? (unsigned)n_layers : 0u;
  hipLaunchKernelGGL(k_beam_reorder, dim3(1 + copies, (unsigned)(n_batch * n_beams)), dim3(256), 0, state().stream, a);
  CTHIP_LAUNCH_CHECK();
  return 0;
}

}  // extern "C"
