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
// sum over those lanes; the partner of an element comes through LDS.  Two passes
// of rows are on their way before the sines, and before the rows they follow.
// Bound: HBM for prompts (bytes in and out once): 16,384 tokens of 48 heads of 128,
// 16 bits, 99 us, 4.1 TB/s (106 with the compiler's 82 registers and five blocks a CU,
// 118 without the loads ahead); 2,021 of 20 heads of 256 from fp32 17 us, 3.6 TB/s.  The
// chain of latencies (position, sine, row, LDS, store) for a step's few tokens, whose
// heads then go to blocks of their own: 8 tokens 4.3 us.
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

// 8 elements as they lie in memory.
template <int QT>
struct Raw {
  static constexpr int N = QT == GM_QTYPE_F32 ? 2 : 1;
  gm_u32x4 w[N];
  __device__ __forceinline__ void load(const void* p, int64_t i, bool vec) {
    if constexpr (QT == GM_QTYPE_F32) {
      const uint32_t* q = static_cast<const uint32_t*>(p) + i;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (vec) w[h] = *reinterpret_cast<const gm_u32x4*>(q + 4 * h);
        else w[h] = gm_u32x4{q[4 * h], q[4 * h + 1], q[4 * h + 2], q[4 * h + 3]};
      }
    } else {
      const uint16_t* q = static_cast<const uint16_t*>(p) + i;
      if (vec) {
        w[0] = *reinterpret_cast<const gm_u32x4*>(q);
      } else {
#pragma unroll
        for (int d = 0; d < 4; ++d) w[0][d] = (uint32_t)q[2 * d] | (uint32_t)q[2 * d + 1] << 16;
      }
    }
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    if constexpr (QT == GM_QTYPE_F32) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(w[e / 4][e % 4]);
    } else {
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        x[2 * d] = GmT16<QT>::lo(w[0][d]);
        x[2 * d + 1] = GmT16<QT>::hi(w[0][d]);
      }
    }
  }
};

__device__ __forceinline__ void lds8(const float* p, float (&v)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const gm_f32x4 q = *reinterpret_cast<const gm_f32x4*>(p + 4 * h);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[4 * h + e] = q[e];
  }
}

template <int Dh, int QT>
__global__ void __launch_bounds__(256, 6) k_rope_append(gm_rope_append_args A, bool vec) {
  constexpr int LPR = Dh / 8, RPP = 256 / LPR;                 // lanes per row, rows per pass
  __shared__ __attribute__((aligned(16))) float cs[Dh / 2], sn[Dh / 2];
  __shared__ __attribute__((aligned(16))) float rows[RPP][Dh]; // a row's lanes are of one wave: no barrier
  const int t = blockIdx.x, half = A.rope_dim >> 1;
  const int sub = threadIdx.x / LPR, i0 = (threadIdx.x % LPR) * 8;
  const int nrow = A.n_head + 2 * A.n_head_kv, step = gridDim.y * RPP;
  auto load = [&](int r, Raw<QT>& raw) {
    const bool isq = r < A.n_head, isk = !isq && r < A.n_head + A.n_head_kv;
    const int h = isq ? r : isk ? r - A.n_head : r - A.n_head - A.n_head_kv;
    const void* src = isq ? A.q : isk ? A.k : A.v;
    const int64_t st = isq ? A.q_stride_t : isk ? A.k_stride_t : A.v_stride_t;
    const int64_t sh = isq ? A.q_stride_h : isk ? A.k_stride_h : A.v_stride_h;
    if (r < nrow) raw.load(src, t * st + h * sh + i0, vec);
  };
  // two passes ahead: their loads pass the sines, and the rows before them
  int r0 = blockIdx.y * RPP;
  Raw<QT> raw[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
#pragma unroll
    for (int h = 0; h < Raw<QT>::N; ++h) raw[u].w[h] = gm_u32x4{0u, 0u, 0u, 0u};
    load(r0 + u * step + sub, raw[u]);
  }
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
  auto pass = [&](int r, const Raw<QT>& raw) {
    const bool live = r < nrow;
    const bool isq = r < A.n_head, isk = !isq && r < A.n_head + A.n_head_kv;
    const int h = isq ? r : isk ? r - A.n_head : r - A.n_head - A.n_head_kv;
    float x[8];
    raw.get(x);
    if (A.q_norm || A.k_norm) {
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
    }
    __builtin_amdgcn_wave_barrier();                            // LDS keeps a wave's order; so must the compiler
    *reinterpret_cast<gm_f32x4*>(&rows[sub][i0]) = gm_f32x4{x[0], x[1], x[2], x[3]};
    *reinterpret_cast<gm_f32x4*>(&rows[sub][i0 + 4]) = gm_f32x4{x[4], x[5], x[6], x[7]};
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (isq || isk) {
      if ((half & 7) == 0) {                                    // the lane's 8 turn as one
        if (i0 < 2 * half) {
          const bool low = i0 < half;
          const int at = low ? i0 : i0 - half;
          float c[8], s[8], y[8];
          lds8(cs + at, c);
          lds8(sn + at, s);
          lds8(&rows[sub][low ? i0 + half : at], y);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = low ? x[e] * c[e] - y[e] * s[e] : x[e] * c[e] + y[e] * s[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int i = i0 + e;
          if (i < half) x[e] = x[e] * cs[i] - rows[sub][i + half] * sn[i];
          else if (i < 2 * half) x[e] = x[e] * cs[i - half] + rows[sub][i - half] * sn[i - half];
        }
      }
    }
    if (live && isq) {
      gm_store<8>(A.q_out, ((int64_t)t * A.n_head + h) * Dh + i0, A.out_type, x);
    } else if (live && keep) {
      gm_store<8>(isk ? A.k_pages : A.v_pages, ((int64_t)slot * A.n_head_kv + h) * Dh + i0, A.cache_type, x);
    }
  };
  for (; r0 < nrow; r0 += 2 * step) {                           // the same count for every lane
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = r0 + u * step;
      if (r >= nrow) break;
      const Raw<QT> now = raw[u];
      load(r + 2 * step + sub, raw[u]);
      pass(r + sub, now);
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
