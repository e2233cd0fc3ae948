// The rows that a step of many sequences adds: q and k normed and rotated by
// positions of several axes, k and v written to the paged cache
// (gm_rope_append; qwen/forward.py:81-97, 179-199 for one sequence).
//
// A pair (x_i, x_{i + rd/2}) turns by a = pos inv_freq_i:
//   x_i' = x_i cos a - x_{i + rd/2} sin a,  x_{i + rd/2}' = x_{i + rd/2} cos a + x_i sin a.
// a reaches 1e6 and more, where fp32 keeps 0.06 of it, so turns = pos inv_freq /
// 2 pi is formed in 64 bits and only its fraction goes on in 32.  One block per
// token: its sines and cosines are formed once, in LDS, and serve all heads.  A
// row of Dh elements is Dh / 8 lanes of 16-byte loads (two for fp32), the norm a
// sum over those lanes; the partner of an element comes through LDS.
// Bound: HBM for prompts (bytes in and out once), the chain of latencies
// (position, sine, row, LDS, store) for a step's few tokens, whose heads then go
// to blocks of their own.
#include "kernels.h"
#include "serving.h"

namespace {

constexpr double kInv2Pi = 0.15915494309189533577;

template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

template <int Dh, int QT>
__global__ void __launch_bounds__(256) k_rope_append(gm_rope_append_args A, bool vec) {
  constexpr int LPR = Dh / 8, RPP = 256 / LPR;                 // lanes per row, rows per pass
  __shared__ float cs[Dh / 2], sn[Dh / 2];
  __shared__ __attribute__((aligned(16))) float rows[RPP][Dh];
  const int t = blockIdx.x, half = A.rope_dim >> 1;
  const int sub = threadIdx.x / LPR, i0 = (threadIdx.x % LPR) * 8;
  const int nrow = A.n_head + 2 * A.n_head_kv;
  for (int i = threadIdx.x; i < half; i += 256) {
    int ax = A.axis ? A.axis[i] : 0;
    if (ax < 0 || ax >= A.n_axes) ax = 0;
    const double r = (double)A.positions[(int64_t)ax * A.T + t] * (A.inv_freq[i] * kInv2Pi);
    float s, c;
    sincospif((float)(2.0 * (r - rint(r))), &s, &c);
    cs[i] = c;
    sn[i] = s;
  }
  const int slot = A.slots[t];
  const bool keep = slot >= 0 && slot < A.n_rows;
  __syncthreads();
  for (int r0 = blockIdx.y * RPP; r0 < nrow; r0 += gridDim.y * RPP) {      // the same count for every lane
    const int r = r0 + sub;
    const bool live = r < nrow;
    const bool isq = r < A.n_head, isk = !isq && r < A.n_head + A.n_head_kv;
    const int h = isq ? r : isk ? r - A.n_head : r - A.n_head - A.n_head_kv;
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.f;
    if (live) {
      const void* src = isq ? A.q : isk ? A.k : A.v;
      const int64_t st = isq ? A.q_stride_t : isk ? A.k_stride_t : A.v_stride_t;
      const int64_t sh = isq ? A.q_stride_h : isk ? A.k_stride_h : A.v_stride_h;
      gm_load<8>(src, t * st + h * sh + i0, QT, vec, x);
    }
    const float* nw = isq ? A.q_norm : isk ? A.k_norm : nullptr;
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
    ss = row_sum<LPR>(ss);
    if (nw) {
      const float f = 1.0f / sqrtf(ss / (float)Dh + A.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (x[e] * f) * nw[i0 + e];
    }
    __syncthreads();                                            // the last pass has read its rows
#pragma unroll
    for (int e = 0; e < 8; ++e) rows[sub][i0 + e] = x[e];
    __syncthreads();
    if (live && (isq || isk)) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = i0 + e;
        if (i < half) x[e] = x[e] * cs[i] - rows[sub][i + half] * sn[i];
        else if (i < 2 * half) x[e] = x[e] * cs[i - half] + rows[sub][i - half] * sn[i - half];
      }
    }
    if (live && isq) {
      gm_store<8>(A.q_out, ((int64_t)t * A.n_head + h) * Dh + i0, A.out_type, x);
    } else if (live && keep) {
      gm_store<8>(isk ? A.k_pages : A.v_pages, ((int64_t)slot * A.n_head_kv + h) * Dh + i0, A.cache_type, x);
    }
  }
}

template <int Dh>
int launch(const gm_rope_append_args* a, hipStream_t s) {
  const bool vec = gm_rows_aligned(a->q, a->in_type, a->q_stride_t, a->q_stride_h) &&
                   gm_rows_aligned(a->k, a->in_type, a->k_stride_t, a->k_stride_h) &&
                   gm_rows_aligned(a->v, a->in_type, a->v_stride_t, a->v_stride_h);
  constexpr int RPP = 256 / (Dh / 8);
  const int passes = (a->n_head + 2 * a->n_head_kv + RPP - 1) / RPP;
  const dim3 grid(a->T, a->T < 512 ? passes : 1);
  switch (a->in_type) {
    case GM_QTYPE_F32: k_rope_append<Dh, GM_QTYPE_F32><<<grid, 256, 0, s>>>(*a, vec); break;
    case GM_QTYPE_F16: k_rope_append<Dh, GM_QTYPE_F16><<<grid, 256, 0, s>>>(*a, vec); break;
    default: k_rope_append<Dh, GM_QTYPE_BF16><<<grid, 256, 0, s>>>(*a, vec); break;
  }
  GM_TRY(hipGetLastError());
  return GM_OK;
}

}  // namespace

int gm_rope_append_run(const gm_rope_append_args* a, hipStream_t s) {
  switch (a->head_dim) {
    case 64: return launch<64>(a, s);
    case 128: return launch<128>(a, s);
    default: return launch<256>(a, s);
  }
}
