// Beam search's selection: the n_beams best of (beam, token) by score[beam] + log softmax(logits[beam])[token].  The reference
// decodes greedily (apps/gpt2/gpt2.lisp:97-113); this is its !argmax (api/high-level-ops.lisp:314-343) for several hypotheses.
//
// The logits are read once: a row is cut into slices, a workgroup holds a slice in registers, 16 or 32 values a thread, and leaves its
// maximum, its sum of exponentials and its n_beams best in order.  A second launch joins the rows' sums and merges the sorted lists,
// a workgroup a request.  (As one launch, the last of a request's workgroups merging, stores had to reach memory and a ticket be
// drawn before a workgroup could end, and the merge's registers were everybody's: 62 us instead of 25 for 48 x 8 beams of 32000.)
// Where there is much to read, half the time is the logits' way and half what a workgroup does with its slice once it is there -- a
// bound from below on the n_beams best, found lane by lane, and the candidates' way through LDS: 384 rows of 32000 (49 MB) 17.4 us + 8.4
// for the merge.  Smaller chunks with the next one on its way while one is worked on (29 - 37 us) do that more often; a looser
// bound by fewer steps (28.4) has more candidates.
// Exponentials, and the sums of a thread's 16 or 32, are in 32 bits (off by 2^-21 of a row's sum at most: that much of a score, alike for all of a
// beam's candidates); sums over threads and slices, logarithms and what candidates are compared by in 64: within a beam no rounding turns two
// round, between beams scores that are closer than 2^-21 may be.
#include <algorithm>

#include "common.h"

namespace cthip {

constexpr int kMaxSelectBeams = 32;
constexpr int kSelectThreads = 256, kMaxSlices = 32, kSelectList = 2048;
constexpr int kMergeList = 6144;  // list entries that the merge keeps in LDS, at most

struct BeamArgs {
  int *tokens, *parents;
  float *scores_out;
  int *finished_out;
  const float *logits;
  int64_t stride;
  const float *scores;
  const int *finished;
  int batch, beams, vocab, eos;
  int slices, slice;       // of a row, and the values of one
  unsigned char *records;  // one a slice: sum, maximum, then the best (logit, token) pairs
  int list_bytes;          // of the merge's LDS: for all of a request's lists, or 0 where they are too many
};

// NaN counts as minus infinity
__device__ __forceinline__ float beam_logit(float x) { return fmaxf(x, -INFINITY); }
// (value, index) pairs in order: the higher value, then the lower index
__device__ __forceinline__ bool beam_before(float a, int i, float b, int j) { return a > b || (a == b && i < j); }
struct BeamPair {
  float x;
  int token;
};
template <int CTRL>
__device__ __forceinline__ double dpp_d(double v) {
  const int2 w = __builtin_bit_cast(int2, v);
  return __builtin_bit_cast(double, make_int2(__builtin_amdgcn_update_dpp(0, w.x, CTRL, 0xF, 0xF, true), __builtin_amdgcn_update_dpp(0, w.y, CTRL, 0xF, 0xF, true)));
}
__device__ __forceinline__ double lane_bcast_d(double v, int lane) {
  const int2 w = __builtin_bit_cast(int2, v);
  return __builtin_bit_cast(double, make_int2(__builtin_amdgcn_readlane(w.x, lane), __builtin_amdgcn_readlane(w.y, lane)));
}
__device__ __forceinline__ double wave_sum_d(double v) {
  v += dpp_d<0xB1>(v);
  v += dpp_d<0x4E>(v);
  v += dpp_d<0x141>(v);
  v += dpp_d<0x140>(v);
  return (lane_bcast_d(v, 0) + lane_bcast_d(v, 16)) + (lane_bcast_d(v, 32) + lane_bcast_d(v, 48));
}
template <int VPT>
__global__ __launch_bounds__(kSelectThreads) void k_beam_slice(BeamArgs a) {
  constexpr int CHUNK = VPT * kSelectThreads;
  __shared__ BeamPair list[kSelectList];
  __shared__ BeamPair best[kMaxSelectBeams];  // of the chunks so far, in order
  __shared__ float s_f[4];
  __shared__ BeamPair s_p[4];
  __shared__ double s_d[4];
  __shared__ int s_count;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, K = a.beams;
  const int row = blockIdx.x / a.slices, part = blockIdx.x - row * a.slices;
  // a beam that is finished, or has no score, has no use for its logits
  const float score = beam_logit(a.scores[row]);
  if (score == -INFINITY || (a.finished && a.finished[row])) return;
  {
    const float *x = a.logits + (int64_t)row * a.stride;
    const int v0 = part * a.slice, v1 = min(a.vocab, v0 + a.slice);
    float top = -INFINITY;
    double sum = 0.0;
    int kept = 0;
    for (int c0 = v0; c0 < v1; c0 += CHUNK) {
      float v[VPT];
#pragma unroll
      for (int j = 0; j < VPT / 4; j++) {
        const int at = c0 + 4 * (tid + kSelectThreads * j);
        if (at + 4 <= v1) {
          const f4_any y = *(const f4_any *)(x + at);
#pragma unroll
          for (int e = 0; e < 4; e++) v[4 * j + e] = y[e];
        } else {
#pragma unroll
          for (int e = 0; e < 4; e++) v[4 * j + e] = at + e < v1 ? x[at + e] : -INFINITY;
        }
      }
      if (tid == 0) s_count = 0;
      float mine = -INFINITY;
#pragma unroll
      for (int j = 0; j < VPT / 4; j++) {
#pragma unroll
        for (int e = 0; e < 4; e++) v[4 * j + e] = beam_logit(v[4 * j + e]);
        mine = fmaxf(mine, fmaxf(fmaxf(v[4 * j], v[4 * j + 1]), fmaxf(v[4 * j + 2], v[4 * j + 3])));
      }
      // The K-th largest of a wavefront's 64 maxima: at least K values are that large, so it bounds the K-th best from below; of the four
      // wavefronts' the largest does.
      float left = mine, bound = -INFINITY;
      for (int k = 0; k < K; k++) {
        bound = wave_max(left);
        const unsigned long long those = __ballot(left == bound);
        if (lane == (int)__builtin_ctzll(those)) left = -INFINITY;  // (below any maximum; among minus infinities nothing changes)
      }
      const float wave_top = wave_max(mine);
      if (lane == 0) s_f[wv] = bound, s_p[wv].x = wave_top;
      __syncthreads();
      bound = fmaxf(fmaxf(s_f[0], s_f[1]), fmaxf(s_f[2], s_f[3]));
      const float chunk_top = fmaxf(fmaxf(s_p[0].x, s_p[1].x), fmaxf(s_p[2].x, s_p[3].x));
      if (kept == K) bound = fmaxf(bound, best[K - 1].x);
      // sums: a thread's in 32 bits, then in 64
      const float new_top = fmaxf(top, chunk_top);
      float part_sum = 0.0f;
      if (fabsf(new_top) < INFINITY) {  // (uniform)
#pragma unroll
        for (int e = 0; e < VPT; e++) part_sum += __builtin_amdgcn_exp2f((v[e] - new_top) * 1.44269504f);
      } else if (new_top > 0.0f) {  // infinities have all the weight
#pragma unroll
        for (int e = 0; e < VPT; e++) part_sum += v[e] == new_top ? 1.0f : 0.0f;
      }
      if (top > -INFINITY && top < new_top) sum *= exp((double)top - (double)new_top);
      sum += (double)part_sum;
      top = new_top;
      // candidates, in any order
      int more = 0;
      if (mine >= bound) {  // (seldom)
#pragma unroll
        for (int e = 0; e < VPT; e++) {
          const int at = c0 + 4 * (tid + kSelectThreads * (e >> 2)) + (e & 3);
          if (v[e] >= bound && at < v1) {
            const int to = atomicAdd(&s_count, 1);
            if (to < kSelectList) list[to] = {v[e], at};
            else more = 1;
          }
        }
      }
      if (tid < kept) {
        const int to = atomicAdd(&s_count, 1);
        if (to < kSelectList) list[to] = best[tid];
        else more = 1;
      }
      const bool over = __syncthreads_or(more);
      const int count = min(s_count, kSelectList), keep = min(K, kept + min(v1 - c0, CHUNK));
      if (!over) {
        // each candidate's place is the number of those before it
        for (int at = tid; at < count; at += kSelectThreads) {
          const BeamPair me = list[at];
          int rank = 0;
#pragma unroll 4
          for (int k = 0; k < count; k++) {
            const BeamPair p = list[k];
            rank += (p.x > me.x) | ((p.x == me.x) & (p.token < me.token));
          }
          if (rank < keep) best[rank] = me;
        }
      } else {
        // (more equal ones than the list holds) one after the other, the best behind the last
        const BeamPair old = tid < kept ? best[tid] : BeamPair{-INFINITY, INT_MAX};
        BeamPair last = {INFINITY, -1};
        for (int k = 0; k < keep; k++) {
          BeamPair p = {-INFINITY, INT_MAX};
          auto look = [&](float y, int at) {
            if (beam_before(last.x, last.token, y, at) && beam_before(y, at, p.x, p.token)) p = {y, at};
          };
#pragma unroll
          for (int e = 0; e < VPT; e++) {
            const int at = c0 + 4 * (tid + kSelectThreads * (e >> 2)) + (e & 3);
            if (at < v1) look(v[e], at);
          }
          look(old.x, old.token);
          for (int o = 32; o > 0; o >>= 1) {
            const float y = __shfl_xor(p.x, o, 64);
            const int at = __shfl_xor(p.token, o, 64);
            if (beam_before(y, at, p.x, p.token)) p = {y, at};
          }
          if (lane == 0) s_p[wv] = p;
          __syncthreads();
          last = s_p[0];
          for (int w = 1; w < 4; w++)
            if (beam_before(s_p[w].x, s_p[w].token, last.x, last.token)) last = s_p[w];
          __syncthreads();
          if (tid == 0) best[k] = last;
        }
      }
      kept = keep;
      __syncthreads();
    }
    sum = wave_sum_d(sum);
    if (lane == 0) s_d[wv] = sum;
    __syncthreads();
    unsigned char *rec = a.records + (int64_t)blockIdx.x * (24 + 8 * K);
    if (tid < K) ((BeamPair *)(rec + 24))[tid] = tid < kept ? best[tid] : BeamPair{-INFINITY, INT_MAX};
    if (tid == 0) {
      *(double *)rec = (s_d[0] + s_d[1]) + (s_d[2] + s_d[3]);
      *(float *)(rec + 8) = top;
    }
  }
}

// one workgroup a request
__global__ __launch_bounds__(kSelectThreads) void k_beam_merge(BeamArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  BeamPair *const list = (BeamPair *)smem;
  __shared__ double s_base[kMaxSelectBeams];  // of each beam: what a logit less the row's maximum is added to
  __shared__ float s_top[kMaxSelectBeams];
  __shared__ int s_state[kMaxSelectBeams];
  __shared__ double s_y[kSelectThreads];  // candidates
  __shared__ BeamPair s_p[kSelectThreads];
  __shared__ int s_b[kSelectThreads], s_count;
  __shared__ float s_bound;
  // sums and maxima of the request's slices, and how much of each slice's list is used up
  double *const s_sums = (double *)(smem + a.list_bytes);
  float *const s_tops = (float *)(s_sums + a.beams * a.slices);
  int *const s_taken = (int *)(s_tops + a.beams * a.slices);
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, K = a.beams, request = blockIdx.x, slices_in_all = K * a.slices, record_bytes = 24 + 8 * K;
  const int b0 = request * K;
  const unsigned char *recs = a.records + (int64_t)b0 * a.slices * record_bytes;
  const int entries = slices_in_all * K;
  const bool held = entries * (int)sizeof(BeamPair) <= a.list_bytes;
  auto entry = [&](int i) { return ((const BeamPair *)(recs + (int64_t)(i / K) * record_bytes + 24))[i % K]; };
  // what there is to read is asked for at once; where a thread has more than one of a kind, the others behind it
  const bool has_entry = held && tid < entries, has_slice = tid < slices_in_all;
  BeamPair first_entry = {};
  float first_top = 0.0f, score = 0.0f;
  double first_sum = 0.0;
  int done = 0;
  if (has_entry) first_entry = entry(tid);
  if (has_slice) first_top = *(const float *)(recs + (int64_t)tid * record_bytes + 8), first_sum = *(const double *)(recs + (int64_t)tid * record_bytes);
  if (tid < K) score = a.scores[b0 + tid];
  if (tid < K && a.finished) done = a.finished[b0 + tid];
  // (lists of beams that had no use for theirs hold anything, and are not looked at)
  if (has_entry) list[tid] = first_entry;
  if (has_slice) s_tops[tid] = first_top, s_sums[tid] = first_sum, s_taken[tid] = 0;
  if (held)
    for (int i = tid + kSelectThreads; i < entries; i += kSelectThreads) list[i] = entry(i);
  for (int i = tid + kSelectThreads; i < slices_in_all; i += kSelectThreads) {
    s_tops[i] = *(const float *)(recs + (int64_t)i * record_bytes + 8);
    s_sums[i] = *(const double *)(recs + (int64_t)i * record_bytes);
    s_taken[i] = 0;
  }
  if (tid < K) {
    const float s = beam_logit(score);
    s_state[tid] = s == -INFINITY ? 0 : done ? 1 : 2;  // no candidates, one, a row of them
    s_base[tid] = (double)s;
    s_top[tid] = 0.0f;
  }
  __syncthreads();
  if (tid < K && s_state[tid] == 2) {
    float top = -INFINITY;
    for (int i = 0; i < a.slices; i++) top = fmaxf(top, s_tops[tid * a.slices + i]);
    s_top[tid] = top;
    if (top == -INFINITY) s_state[tid] = 0;
  }
  __syncthreads();
  for (int i = tid; i < slices_in_all; i += kSelectThreads) {
    const int k = i / a.slices;
    if (s_state[k] == 2) {
      const float t = s_tops[i], top = s_top[k];
      s_sums[i] = t == top ? s_sums[i] : t > -INFINITY ? s_sums[i] * exp((double)t - (double)top) : 0.0;
    }
  }
  __syncthreads();
  if (tid < K && s_state[tid] == 2) {
    double sum = 0.0;
    for (int i = 0; i < a.slices; i++) sum += s_sums[tid * a.slices + i];
    s_base[tid] -= log(sum);
  }
  __syncthreads();
  // List i = beam * slices + slice is lane i % 64's.  Candidates of minus infinity come behind all others: in the order (beam, logit, token),
  // which the lists of a beam's slices have among themselves.
  auto head = [&](int i, int at) { return held ? list[i * K + at] : ((const BeamPair *)(recs + (int64_t)i * record_bytes + 24))[at]; };
  auto value = [&](int beam, BeamPair p) {
    const double z = s_base[beam] + (p.x == s_top[beam] ? 0.0 : (double)p.x - (double)s_top[beam]);
    return p.x > -INFINITY && z == z ? z : -INFINITY;  // (a score of infinity less a logit of infinity is no number)
  };
  auto before = [](double y1, int b1, BeamPair p1, double y2, int b2, BeamPair p2) {
    return y1 > y2 || (y1 == y2 && (b1 < b2 || (b1 == b2 && beam_before(p1.x, p1.token, p2.x, p2.token))));
  };
  // this lane's best: of the heads of its lists
  double y;
  int beam, which;
  BeamPair p;
  const float per = 1.0f / (float)a.slices;
  auto look = [&]() {
    y = -INFINITY, beam = INT_MAX, which = -1, p = {-INFINITY, INT_MAX};
    for (int l = lane; l < slices_in_all; l += 64) {
      const int b = (int)(((float)l + 0.5f) * per), state = s_state[b], n = s_taken[l];  // (exact: l < 1024)
      // a beam without candidates has its tokens at minus infinity, a finished one its eos and the others at minus infinity: in its first list
      if (n >= K || (state != 2 && l != b * a.slices)) continue;
      BeamPair h;
      double z;
      if (state == 2) h = head(l, n), z = h.token == INT_MAX ? -INFINITY : value(b, h);
      else if (state == 0) h = {-INFINITY, n}, z = -INFINITY;
      else h = {n == 0 ? 0.0f : -INFINITY, n == 0 ? a.eos : n - 1 + (n - 1 >= a.eos)}, z = n == 0 ? s_base[b] : -INFINITY;
      if (h.token != INT_MAX && before(z, b, h, y, beam, p)) y = z, beam = b, p = h, which = l;
    }
  };
  auto put = [&](int k, double z, int b, BeamPair h) {
    a.tokens[b0 + k] = h.token;
    a.parents[b0 + k] = b;
    a.scores_out[b0 + k] = (float)z;
    if (a.finished_out) a.finished_out[b0 + k] = h.token == a.eos || (a.finished && a.finished[b0 + b]);
  };
  if (wv == 0) {
    // the K-th largest of the lanes' best, in 32 bits (rounding keeps the order): the K best are among those that reach it
    look();
    float left = which >= 0 ? (float)y : -INFINITY, bound = -INFINITY;
    for (int k = 0; k < K; k++) {
      bound = wave_max(left);
      const unsigned long long those = __ballot(left == bound);
      if (lane == (int)__builtin_ctzll(those)) left = -INFINITY;
    }
    if (lane == 0) s_bound = bound, s_count = 0;
  }
  __syncthreads();
  const float bound = s_bound;
  if (bound > -INFINITY) {
    for (int i = tid; i < entries; i += kSelectThreads) {
      const int l = i / K, n = i - l * K, b = l / a.slices, state = s_state[b];
      BeamPair h = {-INFINITY, 0};
      double z = -INFINITY;
      if (state == 2) h = head(l, n), z = value(b, h);
      else if (state == 1 && n == 0 && l == b * a.slices) h = {0.0f, a.eos}, z = s_base[b];
      if ((float)z >= bound) {
        const int to = atomicAdd(&s_count, 1);
        if (to < kSelectThreads) s_y[to] = z, s_p[to] = h, s_b[to] = b;
      }
    }
  }
  __syncthreads();
  const int count = s_count;
  if (bound > -INFINITY && count <= kSelectThreads) {  // each one's place is the number of those before it
    if (tid < count) {
      int rank = 0;
      const double my = s_y[tid];
      const BeamPair mp = s_p[tid];
      const int mb = s_b[tid];
#pragma unroll 4
      for (int k = 0; k < count; k++) {  // (no short cuts: a branch would wait for each part of a candidate in turn)
        const double cy = s_y[k];
        const BeamPair cp = s_p[k];
        const int cb = s_b[k];
        const int earlier = (cp.x > mp.x) | ((cp.x == mp.x) & (cp.token < mp.token));
        rank += (cy > my) | ((cy == my) & ((cb < mb) | ((cb == mb) & earlier)));
      }
      if (rank < K) put(rank, my, mb, mp);
    }
    return;
  }
  if (wv != 0) return;
  // fewer than K candidates, or very many equal ones: one after the other
  for (int k = 0; k < K; k++) {
    // rounded to 32 bits the largest stays among the largest; where several lanes have that, they are compared in turn
    const float near = which >= 0 ? (float)y : -INFINITY;
    const float top = wave_max(near);
    unsigned long long those = __ballot(which >= 0 && near == top);
    int winner = (int)__builtin_ctzll(those);
    if (those & (those - 1)) {
      double wy = lane_bcast_d(y, winner);
      int wb = __builtin_amdgcn_readlane(beam, winner);
      BeamPair wp = {lane_bcast(p.x, winner), __builtin_amdgcn_readlane(p.token, winner)};
      for (those &= those - 1; those; those &= those - 1) {
        const int c = (int)__builtin_ctzll(those), cb = __builtin_amdgcn_readlane(beam, c);
        const double cy = lane_bcast_d(y, c);
        const BeamPair cp = {lane_bcast(p.x, c), __builtin_amdgcn_readlane(p.token, c)};
        if (before(cy, cb, cp, wy, wb, wp)) winner = c, wy = cy, wb = cb, wp = cp;
      }
    }
    if (lane == winner) {
      put(k, y, beam, p);
      s_taken[which]++;
      look();
    }
  }
}

}  // namespace cthip

using namespace cthip;

extern "C" {

int64_t cthip_beam_select_workspace(int n_batch, int n_beams) {
  if (n_batch < 0 || n_beams < 1 || n_beams > kMaxSelectBeams) return fail(CTHIP_E_BAD_ARG, "cthip_beam_select_workspace: %d x %d beams (at most %d)", n_batch, n_beams, kMaxSelectBeams);
  // (the records take what n_batch * n_beams gives; what is asked for besides is not used, and kept since callers work the size out themselves)
  return 256 + 4ll * n_batch + (int64_t)n_batch * n_beams * kMaxSlices * (24 + 8 * n_beams);
}

int cthip_beam_select(int *tokens, int *parents, float *scores_out, int *finished_out, const float *logits, int64_t logits_stride, const float *scores,
                      const int *finished, int n_batch, int n_beams, int vocab, int eos, void *workspace) {
  CTHIP_REQUIRE_INIT();
  CTHIP_ARG(n_batch >= 0 && n_beams >= 1 && vocab >= 1 && vocab >= n_beams && vocab <= (1 << 30) && logits_stride >= vocab && eos >= -1 && eos < vocab);
  if (n_beams > kMaxSelectBeams || (int64_t)n_batch * n_beams > (1 << 18))
    return fail(CTHIP_E_UNSUPPORTED, "cthip_beam_select: %d x %d beams (at most %d, and 2^18 in all)", n_batch, n_beams, kMaxSelectBeams);
  CTHIP_ARG(eos >= 0 || !finished);
  if (n_batch == 0) return 0;
  CTHIP_ARG(tokens && parents && scores_out && logits && scores && workspace && ((uintptr_t)workspace & 15) == 0);
  CTHIP_ARG(scores_out != scores && (!finished_out || finished_out != finished));
  // A slice is what a workgroup holds in registers (rows that need more than kMaxSlices have longer ones): 16 values a thread while that is at most
  // four workgroups a compute unit, 32 otherwise.  4 beams of 50257: 10.0 us with 16 values, 10.8 with 32; 64 of 50257: 11.9 and 11.8; 384 of
  // 32000: 26.5 and 25.2; 128 of 128256: 34.9 and 30.6.
  const int64_t rows = (int64_t)n_batch * n_beams;
  const int small = (vocab + 16 * kSelectThreads - 1) / (16 * kSelectThreads);
  const bool few = small <= kMaxSlices && rows * small <= 4 * state().compute_units;
  const int slices = few ? small : std::min(kMaxSlices, (vocab + 32 * kSelectThreads - 1) / (32 * kSelectThreads));
  const int slice = ((vocab + slices - 1) / slices + 3) / 4 * 4;
  const int in_use = (vocab + slice - 1) / slice, entries = n_beams * in_use * n_beams;
  const int list_bytes = entries <= kMergeList ? (int)sizeof(BeamPair) * entries : 0;
  const BeamArgs a = {tokens, parents, scores_out, finished_out, logits, logits_stride, scores, finished, n_batch, n_beams, vocab, eos, in_use, slice,
                      (unsigned char *)workspace, list_bytes};
  if (few) hipLaunchKernelGGL(k_beam_slice<16>, dim3((unsigned)(rows * in_use)), dim3(kSelectThreads), 0, state().stream, a);
  else hipLaunchKernelGGL(k_beam_slice<32>, dim3((unsigned)(rows * in_use)), dim3(kSelectThreads), 0, state().stream, a);
  CTHIP_LAUNCH_CHECK();
  hipLaunchKernelGGL(k_beam_merge, dim3((unsigned)n_batch), dim3(kSelectThreads), (unsigned)(list_bytes + 16 * n_beams * in_use), state().stream, a);
  CTHIP_LAUNCH_CHECK();
  return 0;
}

}  // extern "C"
