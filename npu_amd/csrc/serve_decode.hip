// Attention of one new token per sequence over a cache in pages
// (gm_paged_attention): out = softmax(scale q K^T) V per query head.
//
// Work: rounds of 32 keys.  The sequences' rounds lie one behind the other, and
// block i of nblk (at most R) takes the rounds i R / nblk .. (i + 1) R / nblk of one kv head,
// whatever sequences they belong to: blocks differ by one round at most, however
// the lengths differ, and the host needs no length.  A block's four waves take its
// rounds in turn, each with a running maximum, sum and output of its own, and are
// joined in LDS where a sequence (or the block) ends.  A sequence that lies in one
// block is written at once; others leave {m, l, o} per block, and k_paged_join adds
// them up in the blocks' order.
//
// A round in a wave, heads of the kv head's group as the 16 columns of
// v_mfma_f32_16x16x32 (lane = (g, n) = (lane / 16, lane % 16)):
//   S^T = K Q^T      A = key n, dims 32 c + 8 g ..: 16 bytes straight from the
//                    cache; the lane gets keys 4 g + r and 16 + 4 g + r of head n
//   O^T += V^T P^T   the contraction's order is free, so k slot 8 g + j stands for
//                    key 4 g + j (j < 4) or 16 + 4 g + j - 4: the scores are the B
//                    operand as they lie.  A needs 8 keys of one dim: the lane loads
//                    8 dims of each of those 8 keys (16 bytes, 16 lanes a row's 256)
//                    and turns the 8 x 8 block with one v_perm per register; MFMA i
//                    then has row n = dim 8 n + i
// so K and V pass from memory to the MFMAs without LDS, every byte once.
// Bound: HBM; 32 keys of 256 dims (32 KB) cost a wave about 900 cycles of MFMA,
// perm and softmax, a fifth of what the card's rate leaves it.  Measured, with the join:
// 4 x 131,071 positions of 8 x 128 (2.1 GB) 356 us, 6.0 TB/s; 64 ragged ones up to 8,192 of
// 2 x 256 84 us; one of 4,001 with fp32 queries 16 us, the latencies of two launches.
//
// fp32 queries (NP > 1): q and p go as NP planes of the cache's type (three of
// bf16: exact; two of f16, q scaled to 2^9 .. 2^10 and p to 2^15: 22 bits).  The
// MFMAs round their sums towards -infinity, so every other chunk of dims takes -q,
// every other round -p, and a round's part of the output is formed by itself.
#include "kernels.h"
#include "serving.h"

namespace {

constexpr int kRound = 32;          // keys of a round
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_inff();

size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

struct Dec {
  gm_paged_attn_args a;
  float* part;      // [2 nblk][Hkv row groups][RG][Dh]
  float* ml;        // [2 nblk][Hkv row groups][RG][2]
  int nblk;         // blocks along the rounds
  int G, RG, NG;    // heads of a kv head, of them in a row group, row groups
  int cap;          // positions that a table holds
  bool qvec, gvec;
};

__device__ __forceinline__ int seq_len(const Dec& P, int b) { return min(max(P.a.lengths[b], 0), P.cap); }

// Round r's block: the i with i R / nblk <= r < (i + 1) R / nblk.
__device__ __forceinline__ int block_of(int r, int R, int nblk) {
  return (int)((((int64_t)r + 1) * nblk - 1) / R);
}

// pre[b] = rounds before sequence b, b = 0 .. n_seq; one block of 256 threads.
__device__ __forceinline__ void scan_rounds(const Dec& P, int* pre, int* wsum) {
  const int n = P.a.n_seq, per = (n + 255) / 256, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b0 = min(tid * per, n), b1 = min(b0 + per, n);
  int own = 0;
  for (int b = b0; b < b1; ++b) own += (seq_len(P, b) + kRound - 1) / kRound;
  int inc = own;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl_up(inc, o, 64);
    if (lane >= o) inc += v;
  }
  if (lane == 63) wsum[wave] = inc;
  __syncthreads();
  int at = inc - own;
  for (int w = 0; w < wave; ++w) at += wsum[w];
  for (int b = b0; b < b1; ++b) {
    pre[b] = at;
    at += (seq_len(P, b) + kRound - 1) / kRound;
  }
  if (tid == 255) pre[n] = at;
  __syncthreads();
}

__device__ __forceinline__ void load_gate(const Dec& P, int b, int h, int d, float (&g)[4]) {
  const gm_paged_attn_args& A = P.a;
  g[0] = g[1] = g[2] = g[3] = 0.f;
  if (A.gate) gm_load<4>(A.gate, b * A.gate_stride_t + h * A.gate_stride_h + d, A.gate_type, P.gvec, g);
}

// Four outputs of one head: o / l (0 where there was no key), times sigmoid(gate g).
__device__ __forceinline__ void write_out(const Dec& P, int b, int h, int d, gm_f32x4 o, float l, const float (&g)[4]) {
  const gm_paged_attn_args& A = P.a;
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = o[e] / l;
    if (A.gate) v[e] *= 1.0f / (1.0f + expf(-g[e]));
    if (l == 0.f) v[e] = 0.f;
  }
  gm_store<4>(A.out, ((int64_t)b * A.n_head + h) * A.head_dim + d, A.q_type, v);
}

// v = the NP planes of 8 values, largest first.
template <int QT, int NP>
__device__ __forceinline__ void planes(const float (&v)[8], gm_u32x4 (&pl)[NP]) {
  using T = GmT16<QT>;
  float r[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = v[e];
#pragma unroll
  for (int p = 0; p < NP; ++p) {
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      pl[p][d] = T::pack(r[2 * d], r[2 * d + 1]);
      if (p + 1 < NP) {
        r[2 * d] -= T::lo(pl[p][d]);
        r[2 * d + 1] -= T::hi(pl[p][d]);
      }
    }
  }
}

// Blocks that a CU holds, one of a block's waves on each SIMD.  One more or less than this:
// fp32 queries at 64 x 4,000 positions of 2 x 256 113 us (one: 128), 16 bits at 4 x 131,071
// of 8 x 128 375 (two: 421), fp32 there with 4 heads 197 (two: 205), 32 x 8,000 of 8 x 64
// 104 (three: 108).
constexpr int per_cu(int Dh) { return Dh == 256 ? 2 : Dh == 128 ? 3 : 4; }

template <int Dh, int QT, int NP>
__global__ void __launch_bounds__(256, per_cu(Dh)) k_paged_attn(Dec P) {
  using T = GmT16<QT>;
  constexpr bool QLDS = NP > 1 || Dh == 256;        // queries in LDS: registers would spill
  constexpr int NC = Dh / 32;                       // MFMAs of a 16-key tile
  constexpr int VD = Dh < 128 ? 4 : 8;              // dims of a V row in a lane
  constexpr int DG = Dh / (16 * VD);                // V loads a row
  constexpr int LDO = Dh + 4;                       // floats between two heads' outputs in LDS
  constexpr float kShift = QT == GM_QTYPE_F16 ? 15.f : 0.f;        // p in f16: no subnormals to speak of
  constexpr int QB = QLDS ? NP * NC * 1024 : 0, OB = 4 * 16 * LDO * 4;
  __shared__ __attribute__((aligned(16))) char buf[QB > OB ? QB : OB];
  __shared__ float mls[4][16][2];
  __shared__ float qsc[16];
  __shared__ int wsum[4];
  extern __shared__ int pre[];                      // [n_seq + 1]
  const gm_paged_attn_args& A = P.a;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15;
  const int hk = blockIdx.y / P.NG, gb = blockIdx.y % P.NG;
  const int h0 = hk * P.G + gb * P.RG, nh = min(P.RG, P.G - gb * P.RG);    // the block's query heads
  scan_rounds(P, pre, wsum);
  const int R = pre[A.n_seq], i = blockIdx.x;
  if (i == 0) {                                     // sequences without a key
    for (int b = threadIdx.x / 64; b < A.n_seq; b += 4)
      if (pre[b] == pre[b + 1])
        for (int u = lane; u < nh * (Dh / 4); u += 64)
          write_out(P, b, h0 + u / (Dh / 4), 4 * (u % (Dh / 4)), gm_f32x4{0.f, 0.f, 0.f, 0.f}, 0.f, {});
  }
  const int nb = min(P.nblk, R);                    // blocks that have a round, all of them
  if (i >= nb) return;
  const int r0 = (int)((int64_t)i * R / nb), r1 = (int)((int64_t)(i + 1) * R / nb);
  int b;                                            // the sequence of round r0: the last with pre[b] <= r0
  {
    int lo = 0, hi = A.n_seq - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (pre[mid] <= r0) lo = mid;
      else hi = mid - 1;
    }
    b = lo;
  }
  const int64_t ldr = (int64_t)A.n_head_kv * Dh;    // elements of a cache row
  const uint16_t* kp = static_cast<const uint16_t*>(A.k_pages) + (int64_t)hk * Dh + 8 * g;
  const uint16_t* vp = static_cast<const uint16_t*>(A.v_pages) + (int64_t)hk * Dh + VD * n;
  for (int s0 = r0; s0 < r1; ++b) {
    const int s1 = min(r1, pre[b + 1]), len = seq_len(P, b);
    if (s0 >= s1) continue;                         // a sequence without a key
    // ---- the queries: head n of the lane (those past nh repeat the last)
    const int64_t qrow = b * A.q_stride_t + (int64_t)(h0 + min(n, nh - 1)) * A.q_stride_h;
    gm_u32x4 qf[NP > 1 ? 1 : NC];                   // with QLDS on its way there
    float qs = A.scale;
    if constexpr (NP == 1) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const uint16_t* q = static_cast<const uint16_t*>(A.q) + qrow + 32 * c + 8 * g;
        if (P.qvec) {
          qf[c] = *reinterpret_cast<const gm_u32x4*>(q);
        } else {
#pragma unroll
          for (int d = 0; d < 4; ++d) qf[c][d] = (uint32_t)q[2 * d] | (uint32_t)q[2 * d + 1] << 16;
        }
        if constexpr (QLDS)
          if (c % 4 == wave) *reinterpret_cast<gm_u32x4*>(buf + (c * 64 + lane) * 16) = qf[c];
      }
      if constexpr (QLDS) __syncthreads();
    } else {
      // wave w stages heads 4 w .. 4 w + 3, 16 lanes a head
      const int hr = 4 * wave + g;
      const int64_t row = b * A.q_stride_t + (int64_t)(h0 + min(hr, nh - 1)) * A.q_stride_h;
      float x[(Dh + 127) / 128][8], big = 0.f;
#pragma unroll
      for (int u = 0; u < (Dh + 127) / 128; ++u) {
        const int d = 128 * u + 8 * n;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[u][e] = 0.f;
        if (d < Dh) gm_load<8>(A.q, row + d, GM_QTYPE_F32, P.qvec, x[u]);
#pragma unroll
        for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(x[u][e]));
      }
      float f = 1.f, back = 1.f;
      if constexpr (QT == GM_QTYPE_F16) {
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) big = fmaxf(big, __shfl_xor(big, o, 64));
        // 2^(9 - exponent): what is lost below it is 2^-34 of the row's largest value
        const int ex = (int)(__float_as_uint(big) >> 23);
        if (ex > 9 && ex < 240) {
          f = __uint_as_float((uint32_t)(263 - ex) << 23);
          back = __uint_as_float((uint32_t)(ex - 9) << 23);
        }
      }
#pragma unroll
      for (int u = 0; u < (Dh + 127) / 128; ++u) {
        const int d = 128 * u + 8 * n;
        if (d >= Dh) continue;
        const int c = d / 32;
        gm_u32x4 pl[NP];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[u][e] *= c & 1 ? -f : f;
        planes<QT, NP>(x[u], pl);
#pragma unroll
        for (int p = 0; p < NP; ++p)
          *reinterpret_cast<gm_u32x4*>(buf + ((p * NC + c) * 64 + (d % 32) / 8 * 16 + hr) * 16) = pl[p];
      }
      if (n == 0) qsc[hr] = back;
      __syncthreads();
      qs *= qsc[n];
    }
    gm_f32x4 acc[DG][VD];
#pragma unroll
    for (int d = 0; d < DG; ++d)
#pragma unroll
      for (int e = 0; e < VD; ++e) acc[d][e] = gm_f32x4{0.f, 0.f, 0.f, 0.f};
    float m = kNegInf, l = 0.f;
    const int32_t* table = A.block_table + b * A.table_stride;
    // the cache row of key (lane % 32) of round r, -1 if there is none
    auto row_of = [&](int r) {
      const int key = (r - pre[b]) * kRound + (lane & 31);
      int id = -1;
      if (key < len) id = table[key / A.page_size];
      return id >= 0 && id < A.n_pages ? id * A.page_size + key % A.page_size : -1;
    };
    int next = s0 + wave < s1 ? row_of(s0 + wave) : -1;
    for (int r = s0 + wave; r < s1; r += 4) {
      const int row = next;
      const uint32_t ok = (uint32_t)__ballot(row >= 0);
      const int safe = max(row, 0);
      gm_u32x4 kf[2][NC];
      uint32_t vf[8][DG][VD / 2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint16_t* src = kp + __shfl(safe, 16 * t + n, 64) * ldr;
#pragma unroll
        for (int c = 0; c < NC; ++c)
          kf[t][c] = gm_ld<true>(reinterpret_cast<const gm_u32x4*>(src + 32 * c));
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint16_t* src = vp + __shfl(safe, (j < 4 ? 4 * g + j : 12 + 4 * g + j), 64) * ldr;
#pragma unroll
        for (int d = 0; d < DG; ++d) {
          if constexpr (VD == 8) {
            const gm_u32x4 w = gm_ld<true>(reinterpret_cast<const gm_u32x4*>(src + 128 * d));
#pragma unroll
            for (int e = 0; e < 4; ++e) vf[j][d][e] = w[e];
          } else {
            const gm_u32x2 w = gm_ld<true>(reinterpret_cast<const gm_u32x2*>(src));
            vf[j][d][0] = w[0];
            vf[j][d][1] = w[1];
          }
        }
      }
      if (r + 4 < s1) next = row_of(r + 4);
      // ---- scores
      gm_f32x4 s[2];
      int q0 = lane * 16;                            // of the queries in LDS, unknown to the compiler, which
      asm("" : "+v"(q0));                            // would else keep them all in registers over the rounds
      if constexpr (NP == 1) {
        s[0] = s[1] = gm_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          gm_u32x4 q;
          if constexpr (QLDS) q = *reinterpret_cast<const gm_u32x4*>(buf + c * 1024 + q0);
          else q = qf[c];
#pragma unroll
          for (int t = 0; t < 2; ++t) s[t] = T::mfma16(kf[t][c], q, s[t]);
        }
      } else {
        gm_f32x4 odd[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) s[t] = odd[t] = gm_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int p = NP - 1; p >= 0; --p)
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            const gm_u32x4 q = *reinterpret_cast<const gm_u32x4*>(buf + (p * NC + c) * 1024 + q0);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              if (c & 1) odd[t] = T::mfma16(kf[t][c], q, odd[t]);
              else s[t] = T::mfma16(kf[t][c], q, s[t]);
            }
          }
#pragma unroll
        for (int t = 0; t < 2; ++t) s[t] -= odd[t];
      }
      float p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = s[j >> 2][j & 3] * qs;
      if (ok != 0xffffffffu) {                       // the last round, or a page that is none
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool live = ok >> (j < 4 ? 4 * g + j : 12 + 4 * g + j) & 1;
          p[j] = live ? p[j] : kNegInf;
#pragma unroll
          for (int d = 0; d < DG; ++d)               // 0 times what lies there may be NaN
#pragma unroll
            for (int e = 0; e < VD / 2; ++e) vf[j][d][e] = live ? vf[j][d][e] : 0u;
        }
      }
      float mn = fmaxf(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])), fmaxf(fmaxf(p[4], p[5]), fmaxf(p[6], p[7])));
      mn = fmaxf(mn, __shfl_xor(mn, 16, 64));
      mn = fmaxf(fmaxf(mn, __shfl_xor(mn, 32, 64)), m);
      const float mr = mn == kNegInf ? 0.f : mn;     // every key so far masked
      const float al = exp2f((m - mr) * kLog2e);
      m = mn;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = exp2f(fmaf(p[j] - mr, kLog2e, kShift));
      gm_u32x4 pp[NP];
      planes<QT, NP>(p, pp);
      if constexpr (NP == 1) {                       // as rounded: few keys then divide the rounding out
#pragma unroll
        for (int w = 0; w < 4; ++w) sum = T::add(pp[0][w], sum);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += p[j];
      }
      l = fmaf(l, al, sum);
      const uint32_t flip = NP > 1 && (r & 4) ? 0x80008000u : 0u;
      const float sgn = NP > 1 && (r & 4) ? -1.f : 1.f;
      if constexpr (NP > 1) {
#pragma unroll
        for (int q = 0; q < NP; ++q)
#pragma unroll
          for (int d = 0; d < 4; ++d) pp[q][d] ^= flip;
      }
      // ---- outputs
#pragma unroll
      for (int d = 0; d < DG; ++d)
#pragma unroll
        for (int e = 0; e < VD; ++e) {
          gm_u32x4 v;
#pragma unroll
          for (int w = 0; w < 4; ++w)
            v[w] = __builtin_amdgcn_perm(vf[2 * w + 1][d][e / 2], vf[2 * w][d][e / 2],
                                         e & 1 ? 0x07060302u : 0x05040100u);
          if constexpr (NP == 1) {
            acc[d][e] = T::mfma16(v, pp[0], acc[d][e] * al);
          } else {
            gm_f32x4 w = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int q = NP - 1; q >= 0; --q) w = T::mfma16(v, pp[q], w);
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[d][e][c] = fmaf(acc[d][e][c], al, sgn * w[c]);
          }
        }
    }
    // ---- the waves joined
    const int nact = min(4, s1 - s0);
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (g == 0) {
      mls[wave][n][0] = m;
      mls[wave][n][1] = l;
    }
    __syncthreads();                                 // also: the queries' planes have been read
    float M = mls[0][n][0];
    for (int w = 1; w < nact; ++w) M = fmaxf(M, mls[w][n][0]);
    const float f = m == kNegInf ? 0.f : exp2f((m - M) * kLog2e);
    float* os = reinterpret_cast<float*>(buf);
    if (wave < nact && n < nh) {
#pragma unroll
      for (int d = 0; d < DG; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int e = 0; e < VD; e += 4)
            *reinterpret_cast<gm_f32x4*>(os + (wave * 16 + n) * LDO + 16 * VD * d + VD * (4 * g + q) + e) =
                gm_f32x4{acc[d][e][q] * f, acc[d][e + 1][q] * f, acc[d][e + 2][q] * f, acc[d][e + 3][q] * f};
    }
    __syncthreads();
    const bool whole = s0 == pre[b] && s1 == pre[b + 1];
    const int64_t slot = ((int64_t)(2 * i + (s0 == pre[b] ? 1 : 0)) * gridDim.y + blockIdx.y) * P.RG;
    for (int u = threadIdx.x; u < nh * (Dh / 4); u += 256) {
      const int h = u / (Dh / 4), d = 4 * (u % (Dh / 4));
      float Mh = mls[0][h][0], lh = 0.f;
      for (int w = 1; w < nact; ++w) Mh = fmaxf(Mh, mls[w][h][0]);
      gm_f32x4 o = {0.f, 0.f, 0.f, 0.f};
      for (int w = 0; w < nact; ++w) {
        o += *reinterpret_cast<const gm_f32x4*>(os + (w * 16 + h) * LDO + d);
        const float mw = mls[w][h][0];
        lh = fmaf(mls[w][h][1], mw == kNegInf ? 0.f : exp2f((mw - Mh) * kLog2e), lh);
      }
      if (whole) {
        float gt[4];
        load_gate(P, b, h0 + h, d, gt);
        write_out(P, b, h0 + h, d, o, lh, gt);
      } else {
        *reinterpret_cast<gm_f32x4*>(P.part + (slot + h) * Dh + d) = o;
        if (d == 0) {
          P.ml[2 * (slot + h)] = Mh;
          P.ml[2 * (slot + h) + 1] = lh;
        }
      }
    }
    __syncthreads();                                 // before the next sequence writes LDS
    s0 = s1;
  }
}

// The parts of sequence b, head h (block b n_head + h), where it lies in more than
// one block of k_paged_attn: out = sum_p o_p e^(m_p - M) / sum_p l_p e^(m_p - M).  Bound by
// latency (lengths, maxima, parts): 7 us for 126 parts of 16 heads, 8 us for 1,024 blocks
// of a few parts.  512 threads where there are fewer blocks than CUs (one sequence of 4,001:
// 17.5 us in all, 18.5 with 256), else 256 (256 sequences of 32 heads: 204 and 219).
template <int Dh, int NT>
__global__ void __launch_bounds__(NT) k_paged_join(Dec P) {
  constexpr int TP = Dh / 4, NGR = NT / TP;
  __shared__ int64_t red[NT / 64][2];
  __shared__ float fred[NT / 64];
  __shared__ __attribute__((aligned(16))) float os[NGR][Dh];
  extern __shared__ float wt[];                      // [nblk]
  const gm_paged_attn_args& A = P.a;
  const int b = blockIdx.x / A.n_head, h = blockIdx.x % A.n_head, tid = threadIdx.x;
  const int wave = tid >> 6, lane = tid & 63;
  int64_t before = 0, all = 0;
  for (int j = tid; j < A.n_seq; j += NT) {
    const int c = (seq_len(P, j) + kRound - 1) / kRound;
    all += c;
    before += j < b ? c : 0;
  }
  before = gm_wave_sum(before);
  all = gm_wave_sum(all);
  if (lane == 0) {
    red[wave][0] = before;
    red[wave][1] = all;
  }
  __syncthreads();
  before = all = 0;
  for (int w = 0; w < NT / 64; ++w) {
    before += red[w][0];
    all += red[w][1];
  }
  const int mine = (seq_len(P, b) + kRound - 1) / kRound, R = (int)all;
  if (mine == 0) return;
  const int nb = min(P.nblk, R);
  const int i0 = block_of((int)before, R, nb), i1 = block_of((int)before + mine - 1, R, nb);
  if (i0 == i1) return;
  const int np = i1 - i0 + 1, hk = h / P.G, hg = h - hk * P.G, gy = hk * P.NG + hg / P.RG, hr = hg % P.RG;
  // part p: the first block's second slot, the others' first
  auto slot = [&](int p) {
    return ((int64_t)(2 * (i0 + p) + (p == 0 ? 1 : 0)) * (A.n_head_kv * P.NG) + gy) * P.RG + hr;
  };
  const int grp = tid / TP, d = 4 * (tid % TP);
  float gt[4];                                       // loaded before the waits
  load_gate(P, b, h, d, gt);
  float M = kNegInf;
  for (int p = tid; p < np; p += NT) {
    const float v = P.ml[2 * slot(p)];
    wt[p] = v;
    M = fmaxf(M, v);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
  if (lane == 0) fred[wave] = M;
  __syncthreads();
  for (int w = 0; w < NT / 64; ++w) M = fmaxf(M, fred[w]);
  __syncthreads();
  for (int p = tid; p < np; p += NT) {
    const float v = wt[p];
    wt[p] = v == kNegInf ? 0.f : exp2f((v - M) * kLog2e);
  }
  __syncthreads();
  gm_f32x4 o = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
#pragma unroll 4
  for (int p = grp; p < np; p += NGR) {
    const int64_t sl = slot(p);
    const float f = wt[p];
    const gm_f32x4 v = *reinterpret_cast<const gm_f32x4*>(P.part + sl * Dh + d);
    l = fmaf(P.ml[2 * sl + 1], f, l);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(v[e], f, o[e]);
  }
  __shared__ float ls[NGR];
  *reinterpret_cast<gm_f32x4*>(&os[grp][d]) = o;
  if (d == 0) ls[grp] = l;
  __syncthreads();
  if (grp > 0) return;
  for (int q = 1; q < NGR; ++q) {
    o += *reinterpret_cast<const gm_f32x4*>(&os[q][d]);
    l += ls[q];
  }
  write_out(P, b, h, d, o, l, gt);
}

// As many blocks as the CUs hold at once; more would only leave more parts to join.
Dec plan(const gm_paged_attn_args* a) {
  Dec P{};
  P.a = *a;
  P.G = a->n_head / a->n_head_kv;
  P.RG = P.G < 16 ? P.G : 16;
  P.NG = (P.G + 15) / 16;
  const int64_t cap = (int64_t)a->table_width * a->page_size;
  P.cap = (int)(cap < 0x7fffff00 ? cap : 0x7fffff00);
  const int64_t rounds = (int64_t)a->n_seq * ((P.cap + kRound - 1) / kRound);
  const int ny = a->n_head_kv * P.NG;
  const int held = 256 * per_cu(a->head_dim);
  const int64_t most = ny < held ? held / ny : 1;
  P.nblk = (int)(rounds < 1 ? 1 : rounds < most ? rounds : most);
  return P;
}

size_t part_bytes(const Dec& P) {
  return align256((size_t)2 * P.nblk * P.a.n_head_kv * P.NG * P.RG * P.a.head_dim * 4);
}

template <int Dh, int QT, int NP>
int launch(const Dec& P, hipStream_t s) {
  const size_t lds = (size_t)(P.a.n_seq + 1) * 4;
  k_paged_attn<Dh, QT, NP><<<dim3(P.nblk, P.a.n_head_kv * P.NG), 256, lds, s>>>(P);
  GM_TRY(hipGetLastError());
  if (P.nblk == 1) return GM_OK;
  const int heads = P.a.n_seq * P.a.n_head;
  if (heads < 256) k_paged_join<Dh, 512><<<heads, 512, (size_t)P.nblk * 4, s>>>(P);
  else k_paged_join<Dh, 256><<<heads, 256, (size_t)P.nblk * 4, s>>>(P);
  GM_TRY(hipGetLastError());
  return GM_OK;
}

template <int Dh>
int launch_types(const Dec& P, hipStream_t s) {
  const bool f32 = P.a.q_type == GM_QTYPE_F32;
  if (P.a.cache_type == GM_QTYPE_BF16)
    return f32 ? launch<Dh, GM_QTYPE_BF16, 3>(P, s) : launch<Dh, GM_QTYPE_BF16, 1>(P, s);
  return f32 ? launch<Dh, GM_QTYPE_F16, 2>(P, s) : launch<Dh, GM_QTYPE_F16, 1>(P, s);
}

}  // namespace

size_t gm_paged_attn_ws(const gm_paged_attn_args* a) {
  const Dec P = plan(a);
  return part_bytes(P) + align256((size_t)2 * P.nblk * a->n_head_kv * P.NG * P.RG * 8);
}

int gm_paged_attn_run(const gm_paged_attn_args* a, uint8_t* ws, hipStream_t s) {
  Dec P = plan(a);
  P.part = reinterpret_cast<float*>(ws);
  P.ml = reinterpret_cast<float*>(ws + part_bytes(P));
  P.qvec = gm_rows_aligned(a->q, a->q_type, a->q_stride_t, a->q_stride_h);
  P.gvec = a->gate && gm_rows_aligned(a->gate, a->gate_type, a->gate_stride_t, a->gate_stride_h);
  switch (a->head_dim) {
    case 64: return launch_types<64>(P, s);
    case 128: return launch_types<128>(P, s);
    default: return launch_types<256>(P, s);
  }
}
