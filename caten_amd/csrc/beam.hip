// Beam search's selection: the n_beams best of (beam, token) by score[beam] + log softmax(logits[beam])[token].  The reference
// decodes greedily (apps/gpt2/gpt2.lisp:97-113); this is its !argmax (api/high-level-ops.lisp:314-343) for several hypotheses.
#include "common.h"

namespace cthip {

constexpr int kMaxSelectBeams = 32;
constexpr int kSelectThreads = 1024;

struct BeamArgs {
  int *tokens, *parents;
  float *scores_out;
  int *finished_out;
  const float *logits;
  int64_t stride;
  const float *scores;
  const int *finished;
  int batch, beams, vocab, eos;
  unsigned char *ws;
};
// a row's record in the workspace: its maximum, its sum of exponentials, its best tokens with their logits in order
struct BeamRow {
  double sum;
  float top;
  float x[kMaxSelectBeams];
  int token[kMaxSelectBeams];
};

// NaN counts as minus infinity
__device__ __forceinline__ float beam_logit(float x) { return x == x ? x : -INFINITY; }
// (value, index) pairs in order: the higher value, then the lower index
__device__ __forceinline__ bool beam_before(float a, int i, float b, int j) { return a > b || (a == b && i < j); }

__global__ __launch_bounds__(kSelectThreads) void k_beam_row(BeamArgs a) {
  __shared__ float sv[kSelectThreads / 64];
  __shared__ int si[kSelectThreads / 64];
  __shared__ double ss[kSelectThreads / 64];
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const float *x = a.logits + (int64_t)row * a.stride;
  BeamRow *out = (BeamRow *)a.ws + row;
  float last = INFINITY;
  int last_i = -1;
  float top = 0.0f;
  for (int k = 0; k < a.beams; k++) {
    float best = -INFINITY;
    int at = INT_MAX;
    for (int v = tid; v < a.vocab; v += kSelectThreads) {
      const float y = beam_logit(x[v]);
      if (beam_before(last, last_i, y, v) && beam_before(y, v, best, at)) best = y, at = v;
    }
    for (int o = 32; o > 0; o >>= 1) {
      const float y = __shfl_xor(best, o, 64);
      const int v = __shfl_xor(at, o, 64);
      if (beam_before(y, v, best, at)) best = y, at = v;
    }
    if (lane == 0) sv[wv] = best, si[wv] = at;
    __syncthreads();
    best = sv[0], at = si[0];
    for (int w = 1; w < kSelectThreads / 64; w++)
      if (beam_before(sv[w], si[w], best, at)) best = sv[w], at = si[w];
    __syncthreads();
    if (k == 0) top = best;
    if (tid == 0) out->x[k] = best, out->token[k] = at;
    last = best, last_i = at;
  }
  double sum = 0.0;
  for (int v = tid; v < a.vocab; v += kSelectThreads) {
    const float y = beam_logit(x[v]);
    sum += y == top ? 1.0 : (double)expf(y - top);
  }
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if (lane == 0) ss[wv] = sum;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kSelectThreads / 64; w++) sum += ss[w];
    out->sum = sum, out->top = top;
  }
}

__global__ __launch_bounds__(64) void k_beam_merge(BeamArgs a) {
  const int b0 = blockIdx.x * a.beams;
  if (threadIdx.x != 0) return;
  int at[kMaxSelectBeams] = {};
  for (int j = 0; j < a.beams; j++) {
    double best = -INFINITY;
    int who = -1, token = 0;
    for (int k = 0; k < a.beams; k++) {
      const BeamRow *r = (const BeamRow *)a.ws + b0 + k;
      const float s = beam_logit(a.scores[b0 + k]);
      const bool done = a.finished && a.finished[b0 + k];
      double y;
      int t;
      if (s == -INFINITY || (!done && r->top == -INFINITY)) {
        y = -INFINITY;
        t = at[k];
      } else if (done) {
        y = at[k] == 0 ? (double)s : -INFINITY;
        t = at[k] == 0 ? a.eos : at[k] - 1 + (at[k] - 1 >= a.eos);
      } else {
        const float v = r->x[at[k]];
        y = v == -INFINITY ? -INFINITY : (double)s + ((v == r->top ? 0.0 : (double)v - (double)r->top) - log(r->sum));
        t = r->token[at[k]];
      }
      if (who < 0 || y > best) best = y, who = k, token = t;
    }
    at[who]++;
    a.tokens[b0 + j] = token;
    a.parents[b0 + j] = who;
    a.scores_out[b0 + j] = (float)best;
    if (a.finished_out) a.finished_out[b0 + j] = (a.finished && a.finished[b0 + who]) || token == a.eos;
  }
}

}  // namespace cthip

using namespace cthip;

extern "C" {

int64_t cthip_beam_select_workspace(int n_batch, int n_beams) {
  if (n_batch < 0 || n_beams < 1 || n_beams > kMaxSelectBeams) return fail(CTHIP_E_BAD_ARG, "cthip_beam_select_workspace: %d x %d beams (at most %d)", n_batch, n_beams, kMaxSelectBeams);
  return 256 + 4ll * n_batch + (int64_t)n_batch * n_beams * 32 * (24 + 8 * n_beams);
}

int cthip_beam_select(int *tokens, int *parents, float *scores_out, int *finished_out, const float *logits, int64_t logits_stride, const float *scores,
                      const int *finished, int n_batch, int n_beams, int vocab, int eos, void *workspace) {
  CTHIP_REQUIRE_INIT();
  CTHIP_ARG(n_batch >= 0 && n_beams >= 1 && vocab >= 1 && vocab >= n_beams && logits_stride >= vocab && eos >= -1 && eos < vocab);
  if (n_beams > kMaxSelectBeams || (int64_t)n_batch * n_beams > (1 << 24))
    return fail(CTHIP_E_UNSUPPORTED, "cthip_beam_select: %d x %d beams (at most %d, and 2^24 in all)", n_batch, n_beams, kMaxSelectBeams);
  CTHIP_ARG(eos >= 0 || !finished);
  if (n_batch == 0) return 0;
  CTHIP_ARG(tokens && parents && scores_out && logits && scores && workspace && ((uintptr_t)workspace & 15) == 0);
  CTHIP_ARG(scores_out != scores && (!finished_out || finished_out != finished));
  const BeamArgs a = {tokens, parents, scores_out, finished_out, logits, logits_stride, scores, finished, n_batch, n_beams, vocab, eos, (unsigned char *)workspace};
  hipLaunchKernelGGL(k_beam_row, dim3((unsigned)(n_batch * n_beams)), dim3(kSelectThreads), 0, state().stream, a);
  CTHIP_LAUNCH_CHECK();
  hipLaunchKernelGGL(k_beam_merge, dim3((unsigned)n_batch), dim3(64), 0, state().stream, a);
  CTHIP_LAUNCH_CHECK();
  return 0;
}

}  // extern "C"
