// Attention of a ragged batch of query rows over the 4-bit paged cache (layout: kv4.h).  The reference attends one sequence over
// a dense fp32 cache (external/llm/layers.lisp:3-5,19-33).
//
// out = sum_t p_t v_t / sum_t p_t, p_t = exp(q . k_t / sqrt(Dh) - maximum), over one pass of the pages with a running maximum and
// sum.  One launch: as many workgroups as the card holds, each with an equal part of all (tile of rows, head, page) there are, whatever
// the lengths; a tile that several workgroups have parts of is joined by the last of them, in their order.
//
// What bounds it is the vector unit, not memory: taking the nibbles apart (9 instructions for 8 numbers of a key, 20 for 16 of
// values), the scales (one a number of the 16 x 64 scores, two terms of p d), exponentials.  Per page and 16 rows 450 instructions at
// Dh = 64 and some 650 at 128, of 4 cycles each, against 512 and 1024 cycles of matrix instructions and, at Dh = 128, 9 KB.
//   700-row prompts of 5 sequences, 32 heads over 4 of 64 (25 GFLOP): 109 - 111 us, the vector units busy 67 % of it, the matrix units 17 %.
//   32 sequences of 150 .. 20000, 64 heads over 8 of 128 (159 MB): 45.3 us = 3.5 TB/s; vector units 48 %, matrix units 14 %; some 12 us are what a
//   workgroup does before its first page and after its last.
//   8 sequences of 1500 .. 5000, 32 heads of 128 (93 MB): 28.6 us = 3.25 TB/s, 15 of a tile's 16 rows empty.
//   One sequence of 701, 12 heads of 64: 8.4 us, a chain of round trips: lengths, table, page, record, ticket, records.
#include <algorithm>
#include <type_traits>

#include "kv4.h"
#include "planes.h"

namespace cthip {

struct Kv4Attn {
  float *out;
  const float *q;
  const unsigned char *k_pages, *v_pages;
  const int *tables, *lens, *starts;
  int64_t q_stride;
  int n_pages, table_stride, n_seqs, n_rows, H, Hkv;
  int group;       // query heads of a key / value head
  int piece_log2;  // pages are shared out in pieces of this many
  int *tickets;    // workspace: a counter per job that is shared, zero between calls
  float *parts;    // and the shares' records: 16 rows of unnormalised outputs, their maxima, their sums
};

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f2_any __attribute__((ext_vector_type(2), aligned(4)));  // an 8-byte access at 4-byte alignment
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kTileRows = 16;       // rows (query row, query head of the group) of a tile
constexpr int kSplitSlots = 2048;   // records of shares in the workspace, two a workgroup
constexpr int kJobPieces = 1;       // what a job costs besides its pages, in pieces of them (2: 52 us instead of 50, 34 instead of 31, for the batches above)

// floor(x / d) where that is below 2^21, x below 2^30: the quotient by a reciprocal is off by one at most, which what it leaves shows.  (A division
// of integers is forty instructions that nothing runs beside.)
__device__ __forceinline__ int fast_div(int x, int d) {
  const int q = (int)((float)x * __builtin_amdgcn_rcpf((float)d)), left = x - q * d;
  return q + (left >= d ? 1 : 0) - (left < 0 ? 1 : 0);
}
__device__ __forceinline__ int uniform_fast_div(int x, int d) { return __builtin_amdgcn_readfirstlane(fast_div(x, d)); }

// of three, NaN ignored (fmaxf would first have each operand made a quiet number: an instruction more for each)
__device__ __forceinline__ float max3(float x, float y, float z) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
  return r;
}

// The lane's number, asked for anew each time: held over the loop over pages it would be kept in memory, and come back as a wait for all
// loads on their way.
__device__ __forceinline__ int lane_now() {
  int l;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(l));
  return l;
}

// sum, and maximum, over the lanes up to this one
__device__ __forceinline__ int wave_scan_int(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ int wave_scan_max(int v) {
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x111, 0xF, 0xF, false));  // (a lane that gets nothing: its own)
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x112, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x114, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x118, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x142, 0xA, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x143, 0xC, 0xF, false));
  return v;
}

// the larger of this lane's and the one's 16, or 32, lanes away
__device__ __forceinline__ float max16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Which part of the batch a workgroup takes.  A job is a tile of rows of one key / value head of one sequence.  Its cost is
// its pages in pieces of `piece` (four, one a wavefront, or more where numbers would not fit 32 bits) and kJobPieces for what a job costs
// besides; the jobs' costs laid end to end are cut into as many equal parts as workgroups run at once, so that a long sequence is
// shared by many workgroups and many short ones go to one.  The lengths are on the device only: every wavefront works
// the division out for itself, 64 sequences at a time (0.4 us each: 33 us for 4096 sequences of which one has a row; 57 where each
// 64 waited for their lengths and were gone through again for a job).
struct Batch {
  int first = 0, before = 0;  // of the 64 sequences in the lanes: the first, and the cost in front of it
  int reach = 0;              // the largest start up to the last of them
  int len, row0, rows, tiles, cost, upto;  // this lane's; cost: of one job; upto: of all up to the end of this sequence
  // A wavefront keeps them in LDS while it works on a job: they are needed again for the next one only.
  __device__ __forceinline__ void put(int (*to)[64]) const {
    const int l = lane_now();
    to[0][l] = len, to[1][l] = row0, to[2][l] = rows, to[3][l] = tiles, to[4][l] = cost, to[5][l] = upto;
  }
  __device__ __forceinline__ void get(const int (*from)[64]) {
    const int l = lane_now();
    len = from[0][l], row0 = from[1][l], rows = from[2][l], tiles = from[3][l], cost = from[4][l], upto = from[5][l];
  }
};
struct Read {  // of a sequence
  int len = 0, row0 = 0, end = 0;
  __device__ __forceinline__ Read(const Kv4Attn &a, int first) {
    const int i = first + lane_now();
    if (i < a.n_seqs) len = a.lens[i], row0 = a.starts[i], end = a.starts[i + 1];
  }
};
__device__ __forceinline__ void look(const Kv4Attn &a, const Read &read, Batch &s) {
  s.len = max(read.len, 0), s.row0 = read.row0;
  const int end = min(read.end, a.n_rows);
  // (rows in front of an earlier sequence's are nobody's: no row is two sequences', and the costs of all stay within their bound)
  const int reach = max(s.reach, wave_scan_max(s.row0));
  s.reach = __builtin_amdgcn_readlane(reach, 63);
  s.rows = s.row0 == reach && end > s.row0 ? end - s.row0 : 0;
  s.tiles = (s.rows * a.group + kTileRows - 1) / kTileRows;
  const int pages = a.n_pages > 0 && s.len > 0 ? (int)min(((unsigned)s.len + kKvPageRows - 1) / kKvPageRows, (unsigned)a.table_stride) : 0;
  s.cost = max(1, (pages + (1 << a.piece_log2) - 1) >> a.piece_log2) + kJobPieces;  // (without keys there is still a row to write)
  s.upto = s.before + wave_scan_int(s.tiles * a.Hkv * s.cost);
}
struct Job {
  int seq, head, tile;
  int len, rows, row0;  // of the sequence: keys, rows of this step and the first of them
  int at, cost;         // its place on the line of all costs
};
// the job at a place on the line, which lies in front of its end; fronts: what 64 sequences at a time have in front of them, cost and largest start
__device__ __forceinline__ bool find_job(const Kv4Attn &a, Batch &s, int (*kept)[64], const int (*fronts)[64], int place, Job &j) {
  if (place < s.before || place >= __builtin_amdgcn_readlane(s.upto, 63)) {
    const int lane = lane_now();
    const int block = __popcll(__ballot(lane * 64 < a.n_seqs && fronts[0][lane] <= place)) - 1;
    s.first = 64 * block, s.before = __builtin_amdgcn_readfirstlane(fronts[0][block]), s.reach = __builtin_amdgcn_readfirstlane(fronts[1][block]);
    look(a, Read(a, s.first), s);
    s.put(kept);
  }
  const unsigned long long past = __ballot(s.upto > place);
  if (!past) return false;
  const int l = (int)__builtin_ctzll(past);
  const int tiles = __builtin_amdgcn_readlane(s.tiles, l), all = tiles * a.Hkv;
  j.cost = __builtin_amdgcn_readlane(s.cost, l);
  const int start = __builtin_amdgcn_readlane(s.upto, l) - all * j.cost, job = uniform_fast_div(place - start, j.cost);
  j.at = start + job * j.cost;
  j.seq = s.first + l;
  j.head = tiles == 1 ? job : uniform_fast_div(job, tiles);
  // tiles from both ends in turn: in a prompt's own pages late rows see more than early ones, and a workgroup gets some of each
  const int t = job - j.head * tiles;
  j.tile = t & 1 ? tiles - 1 - (t >> 1) : t >> 1;
  j.len = __builtin_amdgcn_readlane(s.len, l);
  j.rows = __builtin_amdgcn_readlane(s.rows, l);
  j.row0 = __builtin_amdgcn_readlane(s.row0, l);
  return true;
}

// The pages come straight into LDS, into a wavefront's own place: the keys and the values of a head as they lie in memory.  A page's
// key quants are taken to registers when their turn comes, and the next page's are asked for at once; the rest follows when the scores, or the
// outputs, are there.
template <int DH>
struct Kv4Lds {
  static constexpr int HEAD = 36 * DH, WAVE = 2 * HEAD, STATS = 4 * WAVE, SEQS = STATS + 14 * kTileRows * 4, FRONTS = SEQS + 4 * 6 * 64 * 4, Q = FRONTS + 2 * 64 * 4,
                       BYTES = Q + DH / 32 * 2048;
  static constexpr int REQUESTS = DH / 32 + (DH / 32 + 1) / 2;  // of a head's part of a page: 16 bytes a lane, then 4
  static constexpr int SHARES = DH == 32 ? 128 : 256;  // of one tile, at most: their records are added up by one workgroup
  static_assert(WAVE >= kTileRows * (DH + 4) * 4 && 4 * WAVE >= 4 * SHARES * kTileRows, "results, and weights of shares, in the pages' place");
};

// One page for one wavefront and 16 rows.  S^T = K Q^T and O^T = V^T P^T: the row is the lane's number modulo 16 throughout (scores,
// maxima, sums and outputs), lane group g = lane / 16 holds keys 16 s + 4 g + i of the page and channels 4 g + i of a result tile.
//   scores  Numbers as fp16 integers, q as two fp16 terms (22 bits of the row's largest); a block's scale is applied to its 32-wide
//           partial sum.  (The nibbles as they stand are fp16 subnormals n 2^-24 and would need no conversion, but the matrix
//           instruction adds products of subnormals with five bits less: 2.8e-6 of a score instead of 6e-8.)
//   output  2^14 p as two fp16 terms, times the scale d as two again (the rounded product, what that leaves, the second term's): 22
//           bits of each 2^14 p d, or a grid of 2^-24 where it, or 2^14 p, is below 2^-2.  Values as exact fp16 integers, fp32 accumulators.
//           Products stay below 2^15 (fp16 ends at 65504) by a power of two f: 2^f d, f > 0, while all scales seen are below 2^-9, which is exact;
//           2^f p, f >= -4, from a scale of 2 on (on d it would put the page's other scales on fp16's subnormal grid: off by 5 % beside a
//           value of 4e5 that has no weight).  Pages with a scale of 32 or more take the fp32 matrix instructions, p d as one fp32 number, at an
//           eighth of the rate (where all pages have one the batches above take 85 and 57 us, the prompts 239).
template <int DH>
__global__ __launch_bounds__(256, DH == 128 ? 3 : 4) void k_kv4_attn(Kv4Attn a) {
  using L = Kv4Lds<DH>;
  constexpr int NB = DH / 32;
  extern __shared__ __align__(16) unsigned char smem[];
  float (*s_m)[kTileRows] = (float (*)[kTileRows])(smem + L::STATS), (*s_l)[kTileRows] = s_m + 4, (*s_w)[kTileRows] = s_m + 8, *s_sum = s_m[12];
  int *s_ticket = (int *)s_m[13];
  int (*s_seqs)[6][64] = (int (*)[6][64])(smem + L::SEQS);
  int (*s_fronts)[64] = (int (*)[64])(smem + L::FRONTS);  // (every wavefront writes all of it, the same)
  // a wavefront's results lie where its own pages did
  auto s_o = [&](int wave, int row) { return (float *)(smem + wave * L::WAVE) + row * (DH + 4); };
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = a.group;
  int total = 0, longest = 0;
  Batch s;
  for (Read read(a, 0);;) {
    const bool more = s.first + 64 < a.n_seqs;
    if (lane_now() == 0) s_fronts[0][s.first >> 6] = s.before, s_fronts[1][s.first >> 6] = s.reach;
    const Read next(a, more ? s.first + 64 : a.n_seqs);  // (on its way while these are looked at)
    look(a, read, s);
    longest = max(longest, s.tiles ? s.cost : 0);
    total = __builtin_amdgcn_readlane(s.upto, 63);
    if (!more) break;
    s.before = total;
    s.first += 64;
    read = next;
  }
  longest = __builtin_amdgcn_readlane(wave_scan_max(longest), 63);
  s.put(s_seqs[wv]);
  // A part's length: of the whole, or what keeps a tile's shares below their number, or, since its last workgroup reads all of a tile's
  // records, as many pieces as come out about even with that (sqrt(longest / 20): 32768 keys of one head of 128 27.3 -> 22.5 us, 131072 38.0 -> 34.1).
  const int even = __builtin_amdgcn_readfirstlane((int)__builtin_sqrtf(0.05f * (float)longest));
  const int per = max(max(uniform_fast_div(total + (int)gridDim.x - 1, (int)gridDim.x), (longest + L::SHARES - 2) / (L::SHARES - 1)), even);
  // Workgroups are dealt to the eight XCDs in turn.  Neighbours on the line, which may read the same pages and join their shares, on one of
  // them, and all XCDs alike where there are fewer parts than workgroups (one sequence of 2048, 8 heads of 128, 72 parts: 15.3 us on one XCD,
  // 10.8 on eight).
  const int parts = uniform_fast_div(total + per - 1, per), of_xcd = (parts + 7) >> 3, nth = blockIdx.x >> 3;
  const int me = nth < of_xcd ? (int)(blockIdx.x & 7) * of_xcd + nth : parts;
  const int x0 = (int)min((int64_t)me * per, (int64_t)total), x1 = min(total - x0, per) + x0;
  for (int x = x0; x < x1;) {
  Job w;
  if (x != x0) s.get(s_seqs[wv]);
  if (!find_job(a, s, s_seqs[wv], s_fronts, x, w)) break;
  x = w.at + w.cost;
  const int lane = lane_now();
  const int n = lane & 15, g = lane >> 4;
  // this lane's row
  const int rho = w.tile * kTileRows + n, j = fast_div(rho, G);
  const bool active = j < w.rows;
  const int head = w.head * G + rho - j * G;
  const int64_t all = (int64_t)a.table_stride * kKvPageRows;
  const int limit = active ? (int)min((int64_t)w.len - w.rows + j, all - 1) : -1;  // the last key it sees
  // pages that any row / every row of the tile sees (rows rise with n)
  const int j1 = min(w.rows - 1, uniform_fast_div(w.tile * kTileRows + kTileRows - 1, G)), j0 = uniform_fast_div(w.tile * kTileRows, G);
  const int last = (int)min((int64_t)w.len - w.rows + j1, all - 1), least = (int)min((int64_t)w.len - w.rows + j0, all - 1);
  const int pages = a.n_pages > 0 && last >= 0 ? last / kKvPageRows + 1 : 0;
  // its pieces lie on the line behind those that stand for the rest (a job without pages is one piece of none)
  const int pieces = max(1, (pages + (1 << a.piece_log2) - 1) >> a.piece_log2), line = w.at + kJobPieces;
  const int owner = uniform_fast_div(line, per), shares = uniform_fast_div(line + pieces - 1, per) - owner + 1, share = me - owner;
  const int from_piece = max(x0 - line, 0), to_piece = min(x1 - line, pieces);
  if (from_piece >= to_piece) continue;
  const int p0 = from_piece << a.piece_log2, p1 = (int)min((int64_t)pages, (int64_t)to_piece << a.piece_log2);

  // page ids of the next 64 pages of this wavefront, one a lane
  const int *table = a.tables + (int64_t)w.seq * a.table_stride;
  int ids, ids_from;
  auto page_id = [&](int k) {  // k: this wavefront's k-th page (the same in every lane)
    if (k >= ids_from + 64) {
      ids_from = k;
      const int p = p0 + wv + 4 * (k + lane);
      ids = p < p1 ? table[p] : -1;
      asm volatile("" : "+v"(ids));  // (waited for here: behind the branch it would be waited for with all pages on their way, page after page)
    }
    return __builtin_amdgcn_readlane(ids, k - ids_from);
  };
  const int mine = p0 + wv < p1 ? (p1 - p0 - wv + 3) / 4 : 0;  // pages of this wavefront
  {
    const int p = p0 + wv + 4 * lane;
    ids_from = 0;
    ids = p < p1 ? table[p] : -1;
  }
  auto valid = [&](int id) { return id >= 0 && id < a.n_pages; };
  const unsigned char *ring = smem + wv * L::WAVE;
  const unsigned ring_at = (unsigned)(size_t)(__attribute__((address_space(3))) const unsigned char *)ring;
  // a head's part of a page (an absent page's is page 0's: its rows are masked)
  auto ask_quants = [&](const unsigned char *pool, int id, unsigned to) {
    const unsigned char *p = uniform(pool + ((int64_t)(valid(id) ? id : 0) * a.Hkv + w.head) * L::HEAD);
#pragma unroll
    for (int i = 0; i < NB; i++) dma16(p + 1024 * i, 16 * lane, to + 1024 * i);
  };
  auto ask_scales = [&](const unsigned char *pool, int id, unsigned to) {
    const unsigned char *p = uniform(pool + ((int64_t)(valid(id) ? id : 0) * a.Hkv + w.head) * L::HEAD) + 1024 * NB;
    if (NB > 1) {
#pragma unroll
      for (int i = 0; i < NB / 2; i++) dma4(p + 256 * i, 4 * lane, to + 1024 * NB + 256 * i);
    } else if (lane < 32) {
      dma4(p, 4 * lane, to + 1024);
    }
  };
  const unsigned char *const kp = ring, *const vp = ring + L::HEAD;
  const unsigned k_at = ring_at, v_at = ring_at + L::HEAD;
  int id = -1, next = -1;  // of the page that is worked on, and of the one behind it
  if (mine > 0) {
    id = page_id(0);
    ask_quants(a.k_pages, id, k_at), ask_scales(a.k_pages, id, k_at);
    ask_quants(a.v_pages, id, v_at), ask_scales(a.v_pages, id, v_at);
  }

  // The row's query as two fp16 terms, in LDS as the matrix instructions take them: [block][term][lane][8].  (Held in registers they are a
  // quarter of what a wavefront has.)  Every wavefront looks at the whole row, block b is wavefront b's to convert.
  float weight;
  {
    float x[NB][8], mine8[8];
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
#pragma unroll
      for (int e = 0; e < 8; e++) mine8[e] = b == 0 || wv == b ? x[b][e] : mine8[e];
    }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    int bad = odd;
    bad |= __shfl_xor(bad, 16, 64);
    bad |= __shfl_xor(bad, 32, 64);
    // 2^(9 - e), e the exponent of the row's largest, brings that into [2^9, 2^10): fp16's own 11 bits, and 11 below them
    const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 127);
    const float up = __uint_as_float((unsigned)(127 + 9 - e) << 23), down = __uint_as_float((unsigned)(127 - 9 + e) << 23);
    if (wv < NB) {
      half8 hi, lo;
#pragma unroll
      for (int k = 0; k < 8; k++) {
        // the order in which a dword's nibbles come apart: channels 0 2 4 6 1 3 5 7
        const int ch = k < 4 ? (k & 1) * 2 + (k >> 1) * 4 : 1 + (k & 1) * 2 + ((k - 4) >> 1) * 4;
        const float y = bad ? NAN : mine8[ch] * up;  // (every score of the row a NaN, and those that are masked minus infinity: without a key it is zero)
        hi[k] = (_Float16)y;
        lo[k] = (_Float16)(y - (float)hi[k]);
      }
      *(half8 *)(smem + L::Q + wv * 2048 + lane * 16) = hi;
      *(half8 *)(smem + L::Q + wv * 2048 + 1024 + lane * 16) = lo;
    }
    // scores as powers of two: log2(e) / sqrt(DH), and the power of two taken off again
    weight = (DH == 32 ? 0.25503487f : DH == 64 ? 0.18033688f : 0.12751743f) * down;
  }

  f32x4 o[NB][2];
#pragma unroll
  for (int b = 0; b < NB; b++) o[b][0] = o[b][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, l = 0.0f;
  int f = 100;  // outputs are held times 2^f, f in -4 .. 15 (100: no scale seen)

  // What a row's weights are taken against: 2^(m weight - base) = 2^14.  The base is used as it is rounded wherever weights of different maxima
  // meet, so its rounding cancels.
  auto base_of = [&](float top) { return top > -INFINITY ? fmaf(top, weight, -14.0f) : -14.0f; };

  // a number that the compiler does not see through: half * minus + a is then one mixed instruction, where a difference is a conversion more
  float minus = -1.0f;
  asm volatile("" : "+s"(minus));
  // Numbers -8 .. 7 of nibbles: the lower one of a byte set behind 0x6400 reads 1024 + n, the upper one behind 0x5400 reads 64 + n (n the
  // nibble with its upper bit flipped).  Mask and exponent in registers of both kinds: one instruction for the and and the xor.
  uint32_t lower = 0x000F000Fu, upper = 0x00F000F0u, e_lower = 0x64086408u, e_upper = 0x54805480u;
  asm volatile("" : "+s"(lower), "+s"(upper), "+v"(e_lower), "+v"(e_upper));
  auto lower_of = [&](uint32_t u) { return __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, (u & lower) ^ e_lower) - (_Float16)1032.0f); };
  auto upper_of = [&](uint32_t u) { return __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, (u & upper) ^ e_upper) - (_Float16)72.0f); };
  __syncthreads();
  for (int k = 0; k < mine; k++) {
    {
      // Of the wavefronts on a SIMD the oldest goes first, and what it gains the others lose: the last workgroup of a compute unit ended at
      // twice the first one's time, the SIMDs to itself.  So who has more left goes first, by quarters of a part (prompts 122 -> 112 us, the
      // batches 52 -> 48 and 34 -> 30).
      const int left = 4 * (x1 - line - from_piece - (k << 2 >> a.piece_log2));
      if (left > 3 * per) __builtin_amdgcn_s_setprio(3);
      else if (left > 2 * per) __builtin_amdgcn_s_setprio(2);
      else if (left > per) __builtin_amdgcn_s_setprio(1);
      else __builtin_amdgcn_s_setprio(0);
    }
    const int page = p0 + wv + 4 * k;
    const int from = valid(id) ? page * kKvPageRows : INT_MAX - (kKvPageRows - 1);  // (absent: behind every limit)
    const bool whole = from + kKvPageRows - 1 <= least;                            // every row of the tile sees every row of the page (uniform)
    // the scales of block b, rows 16 t + 4 g ..
    auto scales = [&](const unsigned char *p, int t, int b) { return *(const half4 *)(p + 32 * DH + ((4 * t + g) * NB + b) * 8); };
    typedef uint32_t kdw __attribute__((ext_vector_type(NB)));
    typedef unsigned short sdw __attribute__((ext_vector_type(NB)));
    wait_loads<L::REQUESTS>();  // (younger than this page's keys: its values)
    const bool more = k + 1 < mine;
    if (more) next = page_id(k + 1);
    f32x4 s[4];
    kdw kq[4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
      s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      kq[t] = *(const kdw *)(kp + kv4_key_offset(16 * t + n, g, 0, DH));
    }
    wait_lds();
    if (more) ask_quants(a.k_pages, next, k_at);
#pragma unroll
    for (int b = 0; b < NB; b++) {
      const half8 q_hi = *(const half8 *)(smem + L::Q + b * 2048 + lane * 16), q_lo = *(const half8 *)(smem + L::Q + b * 2048 + 1024 + lane * 16);
#pragma unroll
      for (int t = 0; t < 4; t++) {
        const uint32_t u = kq[t][b], v = u >> 8;
        const half8 kk = __builtin_bit_cast(half8, (u32x4){lower_of(u), upper_of(u), lower_of(v), upper_of(v)});  // channels 0 2, 4 6, 1 3, 5 7
        f32x4 x = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, q_lo, f32x4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
        x = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, q_hi, x, 0, 0, 0);
        const half4 d = scales(kp, t, b);
#pragma unroll
        for (int i = 0; i < 4; i++) s[t][i] = fmaf(x[i], (float)d[i], s[t][i]);
      }
    }
    wait_lds();
    if (more) ask_scales(a.k_pages, next, k_at);
    if (!whole) {
      int sees = limit - from - 4 * g;  // of the keys 16 t + i: up to this one
      asm volatile("" : "+v"(sees));
#pragma unroll
      for (int t = 0; t < 4; t++)
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (16 * t + i > sees) s[t][i] = -INFINITY;
    }
    float tops[5];
#pragma unroll
    for (int e = 0; e < 5; e++) tops[e] = max3(s[3 * e / 4][3 * e % 4], s[(3 * e + 1) / 4][(3 * e + 1) % 4], s[(3 * e + 2) / 4][(3 * e + 2) % 4]);
    // (no assembly in front of the exchange of lanes: the waits it needs are the compiler's)
    const float top = max32(max16(fmaxf(max3(tops[0], tops[1], tops[2]), max3(tops[3], tops[4], s[3][3]))));
    if (__ballot(top > m)) {  // a new maximum in some row
      const float m_new = fmaxf(m, top), corr = m > -INFINITY ? __builtin_amdgcn_exp2f(base_of(m) - base_of(m_new)) : 0.0f;
      m = m_new;
      l *= corr;
#pragma unroll
      for (int b = 0; b < NB; b++) o[b][0] *= corr, o[b][1] *= corr;
    }
    const float base = base_of(m);
    if (__ballot(!(fabsf(base) < 4194304.0f))) {  // (seldom: where the base's rounding is a power of two that matters)
      const float from_m = m > -INFINITY ? m : 0.0f;
#pragma unroll
      for (int t = 0; t < 4; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) s[t][i] = __builtin_amdgcn_exp2f(fmaf(s[t][i] - from_m, weight, 14.0f));
    } else {
#pragma unroll
      for (int t = 0; t < 4; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) s[t][i] = __builtin_amdgcn_exp2f(fmaf(s[t][i], weight, -base));
    }
#pragma unroll
    for (int t = 0; t < 4; t++) l += (s[t][0] + s[t][1]) + (s[t][2] + s[t][3]);
    if (more) wait_loads<L::REQUESTS>();  // (younger than this page's values: the next one's keys)
    else wait_loads<0>();
    const sdw vs_now = *(const sdw *)(vp + 32 * DH + lane * NB * 2);
    unsigned large = 0;  // scales of 2 and more have this bit of their exponent
#pragma unroll
    for (int x = 0; x < NB; x++) large |= vs_now[x] & 0x4000u;
    bool plain = whole && f == 0 && !__ballot(large), wide = false;
    if (!plain) {
      float d = 0.0f;  // the largest scale of the page's rows that are there (each lane has a piece of the page's scales)
#pragma unroll
      for (int x = 0; x < NB; x++) {
        const int flat = lane * NB + x, row = flat / (4 * NB) * 4 + flat % 4;
        const float dx = fabsf(half_bits_to_float(vs_now[x]));
        d = fmaxf(d, whole || from + row <= last ? dx : 0.0f);
      }
      d = fminf(wave_max(d), 65504.0f);
      const int e = __builtin_amdgcn_readfirstlane((int)(__float_as_uint(d) >> 23)) - 127;  // (uniform)
      const int fits = e > 0 ? max(-e, -4) : e >= -9 ? 0 : min(-e, 15);  // the power of two that this page asks for
      if (d > 0.0f && f == 100) {
        f = fits;
      } else if (d > 0.0f && e + f > 0 && f > -4) {
        const float by = ldexpf(1.0f, max(-e, -4) - f);
        f = max(-e, -4);
#pragma unroll
        for (int b = 0; b < NB; b++) o[b][0] *= by, o[b][1] *= by;
      }
      wide = e > 4;
      plain = whole && f == 0;
    }
    const float p_by = ldexpf(1.0f, min(f, 0));
    auto outputs = [&](auto plain) {
    constexpr bool PLAIN = decltype(plain)::value;
    const _Float16 by = (_Float16)ldexpf(1.0f, f == 100 ? 0 : max(f, 0));
    // p as two fp16 terms, once for all blocks
    half2v ph[8], pl[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float x0 = s[i >> 1][2 * (i & 1)] * (PLAIN ? 1.0f : p_by), x1 = s[i >> 1][2 * (i & 1) + 1] * (PLAIN ? 1.0f : p_by);
      ph[i] = __builtin_convertvector((f32x2){x0, x1}, half2v);
      pl[i] = __builtin_convertvector((f32x2){fmaf((float)ph[i][0], minus, x0), fmaf((float)ph[i][1], minus, x1)}, half2v);
    }
#pragma unroll
    for (int b = 0; b < NB; b++) {
      const u32x4 vq = *(const u32x4 *)(vp + (b * 16 + n) * kKvPageRows + 16 * g);
#pragma unroll
      for (int part = 0; part < 2; part++) {
        half2v xh[4], xl[4];  // p d: the rounded product of the first term, what that leaves, and the second term's
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const half4 d4 = scales(vp, 2 * part + (i >> 1), b);
          half2v d = i & 1 ? half2v{d4[2], d4[3]} : half2v{d4[0], d4[1]};
          if (!PLAIN) {
            d = d * (half2v){by, by};
            const int at = from + 16 * (2 * part + (i >> 1)) + 4 * g + 2 * (i & 1);
            if (at > limit) d[0] = (_Float16)0.0f;  // (the scale of a row that is not seen may be anything)
            if (at + 1 > limit) d[1] = (_Float16)0.0f;
          }
          xh[i] = ph[4 * part + i] * d;
          xl[i] = __builtin_elementwise_fma(pl[4 * part + i], d, __builtin_elementwise_fma(ph[4 * part + i], d, -xh[i]));
        }
        const half8 hi = __builtin_bit_cast(half8, (u32x4){__builtin_bit_cast(uint32_t, xh[0]), __builtin_bit_cast(uint32_t, xh[1]), __builtin_bit_cast(uint32_t, xh[2]),
                                                           __builtin_bit_cast(uint32_t, xh[3])});
        const half8 lo = __builtin_bit_cast(half8, (u32x4){__builtin_bit_cast(uint32_t, xl[0]), __builtin_bit_cast(uint32_t, xl[1]), __builtin_bit_cast(uint32_t, xl[2]),
                                                           __builtin_bit_cast(uint32_t, xl[3])});
        // bytes 0 1 and 2 3 of a dword as halves
        const uint32_t u0 = __builtin_amdgcn_perm(0, vq[2 * part], 0x0C010C00u), u1 = __builtin_amdgcn_perm(0, vq[2 * part], 0x0C030C02u);
        const uint32_t u2 = __builtin_amdgcn_perm(0, vq[2 * part + 1], 0x0C010C00u), u3 = __builtin_amdgcn_perm(0, vq[2 * part + 1], 0x0C030C02u);
        const half8 v0 = __builtin_bit_cast(half8, (u32x4){lower_of(u0), lower_of(u1), lower_of(u2), lower_of(u3)});
        const half8 v1 = __builtin_bit_cast(half8, (u32x4){upper_of(u0), upper_of(u1), upper_of(u2), upper_of(u3)});
        o[b][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, lo, o[b][0], 0, 0, 0);
        o[b][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, lo, o[b][1], 0, 0, 0);
        o[b][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, hi, o[b][0], 0, 0, 0);
        o[b][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, hi, o[b][1], 0, 0, 0);
      }
    }
    };
    // large scales: four keys 16 t + 4 g + i, one of each lane group, an instruction
    auto outputs_wide = [&]() {
#pragma unroll 1
      for (int t = 0; t < 4; t++) {  // (the first of the scores each time, in turn: little code)
#pragma unroll
        for (int b = 0; b < NB; b++) {
          const uint32_t u = *(const uint32_t *)(vp + (b * 16 + n) * kKvPageRows + 16 * g + 4 * t);
          const half4 d = scales(vp, t, b);
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const float x = from + 16 * t + 4 * g + i > limit ? 0.0f : s[0][i] * ((float)d[i] * p_by);
            o[b][0] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)((int)(u << (28 - 8 * i)) >> 28), x, o[b][0], 0, 0, 0);
            o[b][1] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)((int)(u << (24 - 8 * i)) >> 28), x, o[b][1], 0, 0, 0);
          }
        }
        s[0] = s[1], s[1] = s[2], s[2] = s[3];
      }
    };
    if (wide) outputs_wide();
    else if (plain) outputs(std::true_type());
    else outputs(std::false_type());
    wait_lds();
    if (more) ask_quants(a.v_pages, next, v_at), ask_scales(a.v_pages, next, v_at);
    id = next;
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);

  // the four wavefronts' results meet
  const int tid = wv * 64 + lane_now(), n_out = tid & 15, g_out = (tid >> 4) & 3;
  const int nr = min(kTileRows, w.rows * G - w.tile * kTileRows);  // rows of the tile that there are
  if (g_out == 0) s_m[wv][n_out] = m > -INFINITY ? base_of(m) : -INFINITY, s_l[wv][n_out] = l;
  const float back = ldexpf(1.0f, f == 100 ? 0 : -f);
  if (n_out < nr) {
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int half = 0; half < 2; half++) *(f32x4 *)(s_o(wv, n_out) + b * 32 + half * 16 + 4 * g_out) = o[b][half] * back;
  }
  __syncthreads();
  // a share that goes on from the workgroup before, and one that goes on in the next: a workgroup has one of each at most
  auto record_of = [&](int k) { return a.parts + (int64_t)(2 * (owner + k) + (k == 0)) * kTileRows * (DH + 2); };
  auto weight_of = [](float mk, float lk, float M) { return mk > -INFINITY ? __builtin_amdgcn_exp2f(mk - M) : lk == lk ? 0.0f : 1.0f; };  // (a NaN stays one)
  if (tid < nr) {
    float M = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int x = 0; x < 4; x++) M = fmaxf(M, s_m[x][tid]);
#pragma unroll
    for (int x = 0; x < 4; x++) {
      const float e = weight_of(s_m[x][tid], s_l[x][tid], M);
      s_w[x][tid] = e;
      sum = fmaf(e, s_l[x][tid], sum);
    }
    s_sum[tid] = sum;
    if (shares > 1) {
      float *to = record_of(share) + kTileRows * DH + 2 * tid;
      __hip_atomic_store((unsigned long long *)to, __builtin_bit_cast(unsigned long long, (f32x2){M, sum}), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  __syncthreads();
  // where a pair of channels of a tile's row goes
  auto out_at = [&](int r, int c) {
    const int rr = w.tile * kTileRows + r, jj = fast_div(rr, G);
    return a.out + ((int64_t)(w.row0 + jj) * a.H + w.head * G + rr - jj * G) * DH + c;
  };
  for (int e = tid; e < nr * DH / 2; e += 256) {
    const int r = e / (DH / 2), c = e % (DH / 2) * 2;
    f32x2 x = {0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const f32x2 y = *(const f32x2 *)(s_o(k, r) + c);
      x[0] = fmaf(s_w[k][r], y[0], x[0]), x[1] = fmaf(s_w[k][r], y[1], x[1]);
    }
    if (shares > 1) {
      __hip_atomic_store((unsigned long long *)(record_of(share) + 2 * e), __builtin_bit_cast(unsigned long long, x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    } else {
      const float sum = s_sum[r];
      *(f2_any *)out_at(r, c) = sum != 0.0f ? f2_any{x[0] / sum, x[1] / sum} : f2_any{0.0f, 0.0f};
    }
  }
  if (shares > 1) {
    int *tickets = a.tickets + 2 * owner;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this thread's device-scope stores have reached memory
    __syncthreads();
    if (tid == 0) *s_ticket = __hip_atomic_fetch_add(tickets, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (*s_ticket == shares - 1) {  // (uniform) the last of the job's workgroups adds the shares up, in their order
      if (tid == 0) __hip_atomic_store(tickets, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // the next call counts again
      // Maxima and sums of all shares, asked for at once, then the outputs, eight or sixteen shares at a time: a load after the other would be a
      // round trip to memory for each share.  Up to 16 shares every thread works the weights out for itself (9.3 us for one sequence of 701, 12
      // heads of 64, against 10.4; with all parts on one XCD), else once for all (8192: 14.4 against 15.9).
      if (shares <= 16) {
        f32x2 (*ml)[kTileRows] = (f32x2 (*)[kTileRows])smem;
        if ((tid >> 4) < shares && (tid & 15) < nr)
          ml[tid >> 4][tid & 15] =
              __builtin_bit_cast(f32x2, __hip_atomic_load((const unsigned long long *)(record_of(tid >> 4) + kTileRows * DH + 2 * (tid & 15)), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
        __syncthreads();
        for (int e = tid; e < nr * DH / 2; e += 256) {
          const int r = e / (DH / 2), c = e % (DH / 2) * 2;
          float M = -INFINITY, sum = 0.0f;
          for (int k = 0; k < shares; k++) M = fmaxf(M, ml[k][r][0]);
          f32x2 x = {0.0f, 0.0f};
          for (int k0 = 0; k0 < shares; k0 += 8) {
            unsigned long long y[8];
#pragma unroll
            for (int k = 0; k < 8; k++) y[k] = __hip_atomic_load((const unsigned long long *)(record_of(min(k0 + k, shares - 1)) + 2 * e), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
            for (int k = 0; k < 8; k++) {
              if (k0 + k < shares) {
                const f32x2 z = __builtin_bit_cast(f32x2, y[k]), s = ml[k0 + k][r];
                const float f = weight_of(s[0], s[1], M);
                sum = fmaf(f, s[1], sum);
                x[0] = fmaf(f, z[0], x[0]), x[1] = fmaf(f, z[1], x[1]);
              }
            }
          }
          *(f2_any *)out_at(r, c) = sum != 0.0f ? f2_any{x[0] / sum, x[1] / sum} : f2_any{0.0f, 0.0f};
        }
      } else {
        float (*weights)[kTileRows] = (float (*)[kTileRows])smem;
        {
          const int r = tid & 15;
          f32x2 z[L::SHARES / 16];
          float M = -INFINITY, sum = 0.0f;
#pragma unroll
          for (int i = 0; i < L::SHARES / 16; i++) {
            const int k = (tid >> 4) + 16 * i;
            z[i] = f32x2{-INFINITY, 0.0f};
            if (k < shares && r < nr)
              z[i] = __builtin_bit_cast(f32x2, __hip_atomic_load((const unsigned long long *)(record_of(k) + kTileRows * DH + 2 * r), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
          }
#pragma unroll
          for (int i = 0; i < L::SHARES / 16; i++) M = fmaxf(M, z[i][0]);
          M = max32(max16(M));
          s_m[wv][r] = M;  // (four lanes, the same)
          __syncthreads();
          M = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
#pragma unroll
          for (int i = 0; i < L::SHARES / 16; i++) {
            const int k = (tid >> 4) + 16 * i;
            const float f = weight_of(z[i][0], z[i][1], M);
            if (k < shares) weights[k][r] = f;
            sum = fmaf(f, z[i][1], sum);
          }
          sum += __shfl_xor(sum, 16, 64);
          sum += __shfl_xor(sum, 32, 64);
          s_l[wv][r] = sum;
          __syncthreads();
        }
        for (int e = tid; e < nr * DH / 2; e += 256) {
          const int r = e / (DH / 2), c = e % (DH / 2) * 2;
          const float sum = (s_l[0][r] + s_l[1][r]) + (s_l[2][r] + s_l[3][r]);
          f32x2 x = {0.0f, 0.0f};
          for (int k0 = 0; k0 < shares; k0 += 16) {
            unsigned long long y[16];
#pragma unroll
            for (int k = 0; k < 16; k++) y[k] = __hip_atomic_load((const unsigned long long *)(record_of(min(k0 + k, shares - 1)) + 2 * e), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
            for (int k = 0; k < 16; k++) {
              if (k0 + k < shares) {
                const f32x2 z = __builtin_bit_cast(f32x2, y[k]);
                const float f = weights[k0 + k][r];
                x[0] = fmaf(f, z[0], x[0]), x[1] = fmaf(f, z[1], x[1]);
              }
            }
          }
          *(f2_any *)out_at(r, c) = sum != 0.0f ? f2_any{x[0] / sum, x[1] / sum} : f2_any{0.0f, 0.0f};
        }
      }
    }
  }
  __syncthreads();  // the next job's results go through the same LDS
  }
}

}  // namespace cthip

using namespace cthip;

extern "C" {

int64_t cthip_sdpa_paged_q4_workspace(int head_dim) {
  if (!kv4_shape_ok(1, head_dim)) return fail(CTHIP_E_BAD_ARG, "cthip_sdpa_paged_q4_workspace: head size %d (32, 64, 128)", head_dim);
  return 4ll * kSplitSlots * (1 + kTileRows * (head_dim + 2));  // a ticket and a record each
}

int cthip_sdpa_paged_q4(float *out, const float *q, int64_t q_stride, const void *k_pages, const void *v_pages, int n_pages, const int *tables, int table_stride,
                        const int *lens, const int *starts, int n_seqs, int n_rows, int H, int Hkv, int Dh, void *workspace) {
  CTHIP_REQUIRE_INIT();
  CTHIP_ARG(n_seqs >= 0 && n_rows >= 0 && n_pages >= 0 && n_pages <= INT_MAX / kKvPageRows && table_stride > 0 && table_stride <= INT_MAX / kKvPageRows);
  CTHIP_ARG(H > 0 && Hkv > 0 && H % Hkv == 0);
  if (!kv4_shape_ok(Hkv, Dh) || H > 65535) return fail(CTHIP_E_UNSUPPORTED, "cthip_sdpa_paged_q4: %d heads over %d of %d (at most 65535 heads, head sizes 32, 64, 128)", H, Hkv, Dh);
  if (n_seqs > kKv4MaxSeqs) return fail(CTHIP_E_UNSUPPORTED, "cthip_sdpa_paged_q4: %d sequences in one call (at most %d)", n_seqs, kKv4MaxSeqs);
  if (n_seqs == 0 || n_rows == 0) return 0;
  CTHIP_ARG(out && q && out != q && tables && lens && starts && workspace && q_stride >= (int64_t)H * Dh);
  CTHIP_ARG(n_pages == 0 || (k_pages && v_pages));
  CTHIP_ARG((((uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)workspace) & 15) == 0);
  // rows of a tile share a key / value head: at most this many tiles of all sequences, and as many jobs a head
  const int64_t tiles = (int64_t)n_rows * (H / Hkv) / kTileRows + (n_seqs < n_rows ? n_seqs : n_rows), jobs = tiles * Hkv;
  if (jobs > (1 << 21) || n_rows > (1 << 20))
    return fail(CTHIP_E_UNSUPPORTED, "cthip_sdpa_paged_q4: %d rows of %d heads in one call (at most 2^20 rows, and 2^21 tiles of 16 heads of them)", n_rows, H);
  // as many workgroups as run at once (three or four a compute unit for their registers and pages; with two or three prompts took 119 us
  // where these took 112, the batches 50 and 32 where these took 48 and 30), a multiple of the XCDs
  const int at_once = std::min(kSplitSlots / 2, state().compute_units * (Dh == 128 ? 3 : 4) / 8 * 8);
  int piece = 2;  // (the line is shorter than 2^30, and a workgroup's part of it below what fast_div holds for)
  while (jobs * ((table_stride >> piece) + 1 + kJobPieces) > std::min((int64_t)INT_MAX / 2, (int64_t)at_once << 20)) piece++;
  const Kv4Attn a = {out,     q,     (const unsigned char *)k_pages, (const unsigned char *)v_pages, tables, lens, starts, q_stride, n_pages, table_stride, n_seqs, n_rows, H, Hkv,
                     H / Hkv, piece, (int *)workspace, (float *)workspace + kSplitSlots};
  const dim3 grid((unsigned)at_once), block(256);
#define ATT(DH_) hipLaunchKernelGGL(k_kv4_attn<DH_>, grid, block, Kv4Lds<DH_>::BYTES, state().stream, a)
  switch (Dh) {
    case 32: ATT(32); break;
    case 64: ATT(64); break;
    default: ATT(128); break;
  }
#undef ATT
  CTHIP_LAUNCH_CHECK();
  return 0;
}

}  // extern "C"
