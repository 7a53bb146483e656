// Attention of a ragged batch of query rows over the 4-bit paged cache (layout: kv4.h).  The reference attends one sequence over
// a dense fp32 cache (external/llm/layers.lisp:3-5,19-33).
#include "kv4.h"

namespace cthip {

struct Kv4Attn {
  float *out;
  const float *q;
  const unsigned char *k_pages, *v_pages;
  const int *tables, *lens, *starts;
  int64_t q_stride;
  int n_pages, table_stride, n_seqs, n_rows, H, Hkv;
};

// one workgroup per (row, query head): the keys of a page by four lanes each, then a channel per thread over the page's rows
template <int DH>
__global__ __launch_bounds__(256) void k_kv4_attn(Kv4Attn a) {
  constexpr int NB = DH / 32, PARTS = 256 / DH;
  __shared__ float p_s[64], red[4], o_s[256];
  __shared__ int seq_s;
  const int r = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, hk = h / (a.H / a.Hkv);
  if (tid == 0) seq_s = -1;
  __syncthreads();
  for (int i = tid; i < a.n_seqs; i += 256)
    if (a.starts[i] <= r && r < a.starts[i + 1]) seq_s = i;
  __syncthreads();
  const int i = seq_s;
  if (i < 0) return;
  const int pos = a.lens[i] - (a.starts[i + 1] - a.starts[i]) + r - a.starts[i];
  const int T = (int)min((int64_t)pos + 1, (int64_t)a.table_stride * kKvPageRows);
  const int key = tid >> 2, g = tid & 3, c = tid % DH, part = tid / DH;
  float q[NB][8];
  for (int b = 0; b < NB; b++)
    for (int j = 0; j < 8; j++) q[b][j] = a.q[r * a.q_stride + h * DH + b * 32 + g * 8 + j];
  const float scale = 1.0f / sqrtf((float)DH);
  float m = -INFINITY, l = 0.0f, o = 0.0f;
  for (int t0 = 0; t0 < T; t0 += 64) {
    const int page = a.tables[(int64_t)i * a.table_stride + t0 / 64];
    if (page < 0 || page >= a.n_pages) continue;  // (uniform)
    const unsigned char *kh = a.k_pages + ((int64_t)page * a.Hkv + hk) * kv4_head_bytes(DH), *vh = a.v_pages + ((int64_t)page * a.Hkv + hk) * kv4_head_bytes(DH);
    float s = 0.0f;
    for (int b = 0; b < NB; b++) {
      const uint32_t w = *(const uint32_t *)(kh + kv4_key_offset(key, g, b, DH));
      float d = 0.0f;
      for (int j = 0; j < 4; j++) {
        d = fmaf(q[b][j], (float)((int)(w << (28 - 8 * j)) >> 28), d);
        d = fmaf(q[b][4 + j], (float)((int)(w << (24 - 8 * j)) >> 28), d);
      }
      s = fmaf(d, half_bits_to_float(*(const unsigned short *)(kh + kv4_scale_offset(key, b, DH))), s);
    }
    s += dpp_f<0xB1>(s);
    s += dpp_f<0x4E>(s);
    s = t0 + key < T ? s * scale : -INFINITY;
    float top = s;
    for (int x = 4; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
    if ((tid & 63) == 0) red[tid >> 6] = top;
    __syncthreads();
    const float m_new = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    const float p = t0 + key < T ? expf(s - m_new) : 0.0f;
    if (g == 0) p_s[key] = p;
    const float corr = expf(m - m_new);
    m = m_new;
    __syncthreads();
    l *= corr;
    o *= corr;
    for (int k = part; k < 64 && t0 + k < T; k += PARTS) {
      const int v = vh[kv4_value_offset(k, c >> 5, c & 15)];
      o = fmaf(p_s[k] * half_bits_to_float(*(const unsigned short *)(vh + kv4_scale_offset(k, c >> 5, DH))), (float)((int)((uint32_t)v << (c & 16 ? 24 : 28)) >> 28), o);
      l += p_s[k];
    }
    __syncthreads();
  }
  o_s[tid] = o;
  __shared__ float l_s[256];
  l_s[tid] = l;
  __syncthreads();
  if (tid < DH) {
    float O = 0.0f, L = 0.0f;
    for (int x = 0; x < PARTS; x++) O += o_s[tid + x * DH], L += l_s[tid + x * DH];
    a.out[((int64_t)r * a.H + h) * DH + tid] = L != 0.0f ? O / L : 0.0f;  // (a NaN stays one)
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
  const Kv4Attn a = {out, q, (const unsigned char *)k_pages, (const unsigned char *)v_pages, tables, lens, starts, q_stride, n_pages, table_stride, n_seqs, n_rows, H, Hkv};
  const dim3 grid((unsigned)n_rows, (unsigned)H), block(256);
  switch (Dh) {
    case 32: hipLaunchKernelGGL(k_kv4_attn<32>, grid, block, 0, state().stream, a); break;
    case 64: hipLaunchKernelGGL(k_kv4_attn<64>, grid, block, 0, state().stream, a); break;
    default: hipLaunchKernelGGL(k_kv4_attn<128>, grid, block, 0, state().stream, a); break;
  }
  CTHIP_LAUNCH_CHECK();
  return 0;
}

}  // extern "C"
