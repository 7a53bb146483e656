// Verification of drafted tokens against the target's probabilities, from random numbers that are given.  The reference takes the most
// probable token (apps/gpt2/gpt2.lisp:97-113: cthip_argmax); with no drafts this is sampling by the target's probabilities.
//
// Draft x of a row, drawn from q, stays where u q(x) < p(x); the first that does not is replaced by a token drawn from max(p - q, 0), and behind
// the last that stays one more is drawn from p: what comes out is distributed as the target's own samples are.  Drawn is the lowest token at which the running sum of
// the weights is above u times their sum.  u q is exact in 64 bits, differences and sums are taken in 64: near a border between two
// tokens 32 bits would settle for a neighbour once in some thousand draws from a large vocabulary.
//
// Two launches.  A row is cut into slices; a workgroup finds its sequence's first rejected draft for itself (one load of two
// numbers a draft) and leaves its slice's sums, the replacement's and, in case that one is nothing, the target's own.  Then a wavefront
// finds the slice and a workgroup the token in it, eight side by side a thread.  Bound by the two rows of the vocabulary that a sequence needs, and
// by two launches of four to six round trips each where those are short.  (One launch of a workgroup a sequence would read 64 rows with 64 of 256 compute units; one in which the last of a sequence's workgroups, by ticket, finds the token has not
// been built.)
//   64 sequences of 1 .. 5 rows, 128256 tokens (65.7 MB needed): 13.3 + 7 us; the sums at 5 TB/s.
//   48 sequences of up to 8 rows, 32000 tokens: 5.7 + 6.1 us.  One sequence of 5 rows, 50257 tokens: 3.9 + 5.0 us.
#include <algorithm>

#include "common.h"

namespace cthip {

constexpr int kDraftThreads = 256, kDraftSlices = 64;
constexpr int kDraftWorkspace = 2048;  // bytes a sequence
constexpr int kDraftEach = 8;          // tokens that a thread looks at side by side, at most
static_assert(16 * kDraftSlices + 4 <= kDraftWorkspace, "the sums of a sequence's slices");

// A probability of the draft's: below nothing, nothing; NaN stays NaN (it rejects its draft, and what it is taken off weighs nothing)
__device__ __forceinline__ float draft_part(float q) { return q < 0.0f ? 0.0f : q; }

struct DraftArgs {
  int *tokens_out, *accepted, *lens_out;
  const float *target, *draft;
  int64_t target_stride, draft_stride;
  const int *tokens;
  const float *uniforms;
  const int *starts, *positions, *lens;
  int n_rows, vocab, slices, slice;
  int each;  // slices that a workgroup sums up, one after the other
  unsigned char *workspace;
  // of a sequence: of each slice the weights' sum, of each slice the target's; and its drafts that stay, -1 where it sits out
  __device__ __forceinline__ double *sums(int seq) const { return (double *)(workspace + (int64_t)seq * kDraftWorkspace); }
  __device__ __forceinline__ int *stays(int seq) const { return (int *)(sums(seq) + 2 * kDraftSlices); }
};

__device__ __forceinline__ double draft_wave_sum(double v) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// The rows of a sequence, those of drafts that stay, and the token row that the last one is drawn from
struct Verified {
  int row0, rows, stay;
  bool there;
  __device__ __forceinline__ Verified(const DraftArgs &a, int seq) {
    const int lane = threadIdx.x & 63;
    row0 = a.starts[seq];
    const int end = a.starts[seq + 1];
    there = row0 >= 0 && end > row0 && end <= a.n_rows;
    rows = there ? end - row0 : 0;
    stay = 0;
    if (!there) return;
    there = !a.positions || a.positions[row0] >= 0;
    if (!there) return;
    for (int j0 = 0; j0 < rows - 1; j0 += 64) {  // (every wavefront for itself)
      const int j = j0 + lane;
      bool good = true;
      if (j < rows - 1) {
        const int x = a.tokens[row0 + j + 1];
        good = x >= 0 && x < a.vocab;
        if (good) {
          const float p = a.target[(int64_t)(row0 + j) * a.target_stride + x], q = a.draft ? draft_part(a.draft[(int64_t)(row0 + j) * a.draft_stride + x]) : 1.0f;
          good = (double)a.uniforms[row0 + j] * (double)q < (double)p;
        }
      }
      const unsigned long long bad = __ballot(!good);
      if (bad) {
        stay = j0 + (int)__builtin_ctzll(bad);
        return;
      }
    }
    stay = rows - 1;
  }
};

// What a token weighs: a difference that is NaN or below nothing, as nothing
struct DraftRow {
  const float *p, *q;
  int taken;  // the rejected draft, where there are no probabilities of the draft's: the whole of them was its
  __device__ __forceinline__ DraftRow(const DraftArgs &a, int row0, int rows, int stay) {
    p = a.target + (int64_t)(row0 + stay) * a.target_stride;
    const bool rejected = stay < rows - 1;
    q = rejected && a.draft ? a.draft + (int64_t)(row0 + stay) * a.draft_stride : nullptr;
    taken = rejected && !a.draft ? a.tokens[row0 + stay + 1] : -1;
  }
  __device__ __forceinline__ void at(int t, double &w, double &own) const {
    const float x = p[t];
    own = x > 0.0f ? (double)x : 0.0;
    const double left = (double)x - (q ? (double)draft_part(q[t]) : 0.0);
    w = t == taken ? 0.0 : left > 0.0 ? left : 0.0;
  }
};

__global__ __launch_bounds__(kDraftThreads) void k_draft_slice(DraftArgs a) {
  __shared__ double part[kDraftSlices][2][kDraftThreads / 64];  // of its slices
  const int seq = blockIdx.y, tid = threadIdx.x;
  const Verified v(a, seq);
  if (blockIdx.x == 0 && tid == 0) a.stays(seq)[0] = v.there ? v.stay : -1;
  if (!v.there) return;
  const DraftRow row(a, v.row0, v.rows, v.stay);
  const int s0 = blockIdx.x * a.each, n = min(a.slices - s0, a.each);
  for (int s = 0; s < n; s++) {
    double w = 0.0, own = 0.0;
    const int t1 = min(a.vocab, (s0 + s + 1) * a.slice);
    for (int t = (s0 + s) * a.slice + tid; t < t1; t += kDraftThreads) {
      double x, y;
      row.at(t, x, y);
      w += x, own += y;
    }
    w = draft_wave_sum(w), own = draft_wave_sum(own);
    if ((tid & 63) == 0) part[s][0][tid >> 6] = w, part[s][1][tid >> 6] = own;
  }
  __syncthreads();
  if (tid < 2 * n) {
    const double *sums = part[tid >> 1][tid & 1];
    a.sums(seq)[kDraftSlices * (tid & 1) + s0 + (tid >> 1)] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  }
}

// inclusive, over a wavefront
__device__ __forceinline__ double draft_wave_scan(double v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(v, o, 64);
    if (lane >= o) v += y;
  }
  return v;
}

__global__ __launch_bounds__(kDraftThreads) void k_draft_token(DraftArgs a) {
  __shared__ double part[2][kDraftThreads / 64];
  __shared__ int s_found[2], s_last;
  const int seq = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  // (all of these at once)
  const int row0 = a.starts[seq], end = a.starts[seq + 1], stay = a.stays(seq)[0];
  const int rows = row0 >= 0 && end > row0 && end <= a.n_rows ? end - row0 : 0;
  const double *sums = a.sums(seq);
  const double left = lane < a.slices ? sums[lane] : 0.0, all = lane < a.slices ? sums[kDraftSlices + lane] : 0.0;
  if (tid == 0) {
    a.accepted[seq] = max(stay, 0);
    if (a.lens_out) a.lens_out[seq] = a.lens[seq] - (stay >= 0 ? rows - 1 - stay : 0);
  }
  if (stay < 0) {
    for (int j = tid; j < rows; j += kDraftThreads) a.tokens_out[row0 + j] = -1;
    return;
  }
  const float u = a.uniforms[row0 + rows - 1];
  const DraftRow row(a, row0, rows, stay);
  int token = -1;
  double mine = left, upto = draft_wave_scan(left), total = __shfl(upto, 63, 64);
  const bool own = !(total > 0.0);  // nothing is left of the target behind the draft's: by roundings alone, then its own
  if (own) mine = all, upto = draft_wave_scan(all), total = __shfl(upto, 63, 64);
  if (total > 0.0) {
    const double goal = (double)u * total;
    // the first slice that reaches past the goal, or the last that weighs anything
    const unsigned long long past = __ballot(upto > goal && mine > 0.0), any = __ballot(mine > 0.0);
    const int s = past ? (int)__builtin_ctzll(past) : 63 - (int)__builtin_clzll(any);
    double before = s > 0 ? __shfl(upto, s - 1, 64) : 0.0;
    const int t1 = min(a.vocab, (s + 1) * a.slice);
    if (tid == 0) s_last = -1;
    int last = -1;
    // a thread's tokens lie side by side: their sums, over the workgroup, and then the one among them
    for (int t0 = s * a.slice, round = 0; t0 < t1; t0 += kDraftEach * kDraftThreads, round ^= 1) {
      const int each = min(kDraftEach, (t1 - t0 + kDraftThreads - 1) / kDraftThreads), t = t0 + tid * each, end = min(t + each, t1);
      double w[kDraftEach], sum = 0.0;
#pragma unroll
      for (int e = 0; e < kDraftEach; e++) {
        double o = 0.0;
        w[e] = 0.0;
        if (t + e < end) row.at(t + e, w[e], o);
        if (own) w[e] = o;
      }
#pragma unroll
      for (int e = 0; e < kDraftEach; e++) sum += w[e];
      const double scan = draft_wave_scan(sum);
      if (lane == 63) part[round][wv] = scan;
      if (tid == 0) s_found[round] = INT_MAX;
      __syncthreads();
      double front = before + scan - sum;
#pragma unroll
      for (int k = 0; k < kDraftThreads / 64; k++) {
        if (k < wv) front += part[round][k];
        before += part[round][k];
      }
      if (sum > 0.0) {
        int found = INT_MAX;
#pragma unroll
        for (int e = 0; e < kDraftEach; e++) {
          front += w[e];
          if (w[e] > 0.0) {
            last = t + e;
            if (found == INT_MAX && front > goal) found = t + e;
          }
        }
        if (found != INT_MAX) atomicMin(&s_found[round], found);
      }
      __syncthreads();
      if (s_found[round] != INT_MAX) {
        token = s_found[round];
        break;
      }
    }
    if (token < 0) {  // (sums of other orders, or a number that is not below one)
      if (last >= 0) atomicMax(&s_last, last);
      __syncthreads();
      token = s_last;
    }
  }
  for (int j = tid; j < rows; j += kDraftThreads) a.tokens_out[row0 + j] = j < stay ? a.tokens[row0 + j + 1] : j == stay ? token : -1;
}

}  // namespace cthip

using namespace cthip;

extern "C" {

int64_t cthip_draft_verify_workspace(int n_seqs) {
  if (n_seqs < 0) return fail(CTHIP_E_BAD_ARG, "cthip_draft_verify_workspace: %d sequences", n_seqs);
  return (int64_t)n_seqs * kDraftWorkspace;
}

int cthip_draft_verify(int *tokens_out, int *accepted, int *lens_out, const float *target, int64_t target_stride, const float *draft, int64_t draft_stride, const int *tokens,
                       const float *uniforms, const int *starts, const int *positions, const int *lens, int n_seqs, int n_rows, int vocab, void *workspace) {
  CTHIP_REQUIRE_INIT();
  CTHIP_ARG(n_seqs >= 0 && n_rows >= 0 && vocab >= 1 && vocab <= (1 << 30) && target_stride >= vocab && (!draft || draft_stride >= vocab));
  if (n_seqs > 65535) return fail(CTHIP_E_UNSUPPORTED, "cthip_draft_verify: %d sequences in one call (at most 65535)", n_seqs);
  if (n_seqs == 0) return 0;
  CTHIP_ARG(accepted && starts && workspace && ((uintptr_t)workspace & 15) == 0 && (!lens_out || lens));
  CTHIP_ARG(n_rows == 0 || (tokens_out && target && tokens && uniforms && tokens_out != tokens));
  const int slices = std::min(kDraftSlices, (vocab + 1023) / 1024), slice = (vocab + slices - 1) / slices;
  // As many workgroups as run at once, eight a compute unit: each has to find the row first (64 rows of 128256: a workgroup a slice 15.0 us, so 13.3; half as many
  // slices 12.3, and the second launch 10.2 instead of 7).
  const int at_once = 8 * state().compute_units, each = (int)std::min((int64_t)slices, ((int64_t)n_seqs * slices + at_once - 1) / at_once);
  const DraftArgs a = {tokens_out, accepted, lens_out, target, draft, target_stride, draft_stride, tokens, uniforms, starts, positions, lens, n_rows, vocab, (vocab + slice - 1) / slice, slice, each,
                       (unsigned char *)workspace};
  hipLaunchKernelGGL(k_draft_slice, dim3((unsigned)((a.slices + each - 1) / each), (unsigned)n_seqs), dim3(kDraftThreads), 0, state().stream, a);
  CTHIP_LAUNCH_CHECK();
  hipLaunchKernelGGL(k_draft_token, dim3((unsigned)n_seqs), dim3(kDraftThreads), 0, state().stream, a);
  CTHIP_LAUNCH_CHECK();
  return 0;
}

}  // extern "C"
