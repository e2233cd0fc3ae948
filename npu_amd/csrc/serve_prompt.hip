// Causal attention over packed prompts (gm_prompt_attention), keys packed or in
// the cache's pages: out = softmax(scale q K^T + mask) V in one pass over the keys
// with a running maximum m and sum l per row.
//
// Rows: a kv head's rows of one sequence are its tokens x G = n_head / n_head_kv
// heads, head fastest, so that a block's rows share nearly all their keys.  A block
// is 4 waves of 32 rows; K and V tiles of kKT keys go from memory straight to LDS,
// the next while the present one is used.
//
// v_mfma_f32_32x32x16, lane (hf, n) = (lane / 32, lane % 32):
//   S^T = K Q^T     A = key n, dims 16 c + 8 hf ..: 16 bytes of LDS; the lane gets
//                   keys 8 (r / 4) + 4 hf + r % 4 of row n, r < 16: a row's scores
//                   are in two lanes, and its maximum and sum need one swap
//   O^T += V^T P^T  the contraction's order is free: k slot 8 hf + j of MFMA u stands
//                   for key 16 u + 8 (j / 4) + 4 hf + j % 4, so the scores rounded to
//                   16 bits are the B operand as they lie; A = 4 keys x 16 dims per
//                   16 lanes by the transposing LDS read, two of them an MFMA
// LDS rows keep their 16-byte granules g at g ^ f(key) so that neither read meets a
// bank twice.  The rescaling of l and o by a new maximum waits until it has grown by
// 2^kLazy; p is then at most 2^(kLazy + kShift).
//
// A masked key has p = 0, and 0 times a V value that is not finite would be NaN: a
// tile with a masked key looks at its V first, and where it must multiplies the
// finite values alone and counts the others by the rows that see them.
#include "kernels.h"
#include "serving.h"

namespace {

constexpr int kWaves = 4, kRows = 32 * kWaves;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_inff();

struct Pmt {
  gm_prompt_attn_args a;
  int G;
  bool qvec, gvec;
};

typedef short gm_i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) gm_i16x4 gm_lds_i16x4;

// Rows lane 4 k .. 4 k + 3 of a 16-lane group point at (row k, 4 values each); lane
// i gets value i of the four rows.
__device__ __forceinline__ gm_u32x2 read_tr(const char* p) {
  const gm_i16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((gm_lds_i16x4*)p);
  return __builtin_bit_cast(gm_u32x2, v);
}

// 16 bytes per lane from memory to LDS, lane l's at dst + 16 l.
__device__ __forceinline__ void to_lds(const void* src, char* dst) {
  __builtin_amdgcn_global_load_lds(src, dst, 16, 0, 0);
}

// {own, other half's} of a value, in the same order in both lanes of a row.
__device__ __forceinline__ void both_halves(float v, float& a, float& b) {
  const uint32_t u = __float_as_uint(v);
  const auto w = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  a = __uint_as_float(w[0]);
  b = __uint_as_float(w[1]);
}

template <int QT>
__device__ __forceinline__ bool odd16(uint32_t w) {       // either 16-bit value infinite or NaN
  constexpr uint32_t E = QT == GM_QTYPE_BF16 ? 0x7f80u : 0x7c00u;
  return (w & E) == E || (w & E << 16) == E << 16;
}

// A 16-bit value that is not finite as a number that a tile's worth of them can be
// counted by: 1 for inf, 128 for -inf, 16384 for NaN; 0 for a finite one.
template <int QT>
__device__ __forceinline__ uint32_t odd_kind(uint32_t w) {
  constexpr bool B = QT == GM_QTYPE_BF16;
  constexpr uint32_t E = B ? 0x7f80u : 0x7c00u;
  if ((w & E) != E) return 0u;
  if (w & (0x7fffu ^ E)) return B ? 0x4680u : 0x7400u;
  return w & 0x8000u ? (B ? 0x4300u : 0x5800u) : (B ? 0x3f80u : 0x3c00u);
}
// The sum of at most 64 values that the count stands for.
__device__ __forceinline__ float odd_value(float count) {
  const int c = (int)count, pos = c & 127, neg = c >> 7 & 127;
  if (c >= 16384 || (pos && neg)) return __builtin_nanf("");
  return pos ? __builtin_inff() : neg ? kNegInf : 0.f;
}

// O^T += V^T P^T of a tile whose V is not all finite: the finite values' products,
// then what the rows that see the others get of them.  vb: the lane's place in V;
// left: the tile's last key that its row sees, and ok: the keys that have a page,
// both less the lane's 4 hf.
template <int Dh, int QT>
__device__ __attribute__((noinline)) void pv_odd(const char* vb, int left, unsigned long long ok, const uint32_t* p,
                                                 gm_f32x16* o) {
  using T = GmT16<QT>;
  constexpr int NS = Dh == 256 ? 1 : 2, ND = Dh / 32, RB = 2 * Dh;
  const uint32_t one = QT == GM_QTYPE_BF16 ? 0x3f80u : 0x3c00u;
#pragma unroll 1
  for (int d = 0; d < ND; ++d) {
    gm_f32x16 x, od = o[d];
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = 0.f;
#pragma unroll 1
    for (int u = 0; u < 2 * NS; ++u) {
      // granule bits are an XOR in the address's low bits, whose base is a tile's
      const uintptr_t place = reinterpret_cast<uintptr_t>(vb) ^ (uintptr_t)(64 * d & 255 & (RB - 1));
      const char* at = reinterpret_cast<const char*>(place) + 16 * u * RB + 256 * (d / 4);
      const gm_u32x2 lo = read_tr(at), hi = read_tr(at + 8 * RB);
      gm_u32x4 v = {lo[0], lo[1], hi[0], hi[1]}, kind, seen;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        kind[w] = odd_kind<QT>(v[w] & 0xffffu) | odd_kind<QT>(v[w] >> 16) << 16;
        v[w] &= (kind[w] & 0xffffu ? 0u : 0xffffu) | (kind[w] >> 16 ? 0u : 0xffff0000u);
        const int key = 16 * u + 8 * (w >> 1) + 2 * (w & 1);
        const uint32_t okw = (uint32_t)(ok >> key);
        seen[w] = (key <= left && (okw & 1) ? one : 0u) | (key + 1 <= left && (okw & 2) ? one << 16 : 0u);
      }
      od = T::mfma32(v, gm_u32x4{p[4 * u], p[4 * u + 1], p[4 * u + 2], p[4 * u + 3]}, od);
      x = T::mfma32(kind, seen, x);
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) od[e] += odd_value(x[e]);
    o[d] = od;
  }
}

template <int Dh, int QT, bool PAGED>
__global__ void __launch_bounds__(64 * kWaves, 2) k_prompt_attn(Pmt P) {
  using T = GmT16<QT>;
  constexpr int KT = Dh == 256 ? 32 : 64;              // keys of a tile
  constexpr int NS = KT / 32, NC = Dh / 16, ND = Dh / 32, NGR = Dh / 8, RB = 2 * Dh;
  constexpr int TILE = KT * RB, NI = TILE / (1024 * kWaves);
  constexpr float kShift = QT == GM_QTYPE_F16 ? 11.f : 0.f, kLazy = QT == GM_QTYPE_F16 ? 4.f : 8.f;
  extern __shared__ __attribute__((aligned(1024))) char lds[];      // [2][K, V][TILE]
  __shared__ int votes[kWaves];
  const gm_prompt_attn_args& A = P.a;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, hf = lane >> 5, n = lane & 31;
  const int hk = blockIdx.x % A.n_head_kv, bi = blockIdx.x / A.n_head_kv;
  // sequence b's blocks start at cu_q[b] G / kRows + b: never fewer than it needs
  auto cuq = [&](int b) { return min(max(A.cu_q[b], 0), A.n_q); };
  int below = 0;
  for (int b0 = 0; b0 < A.n_seq; b0 += 64 * kWaves) {
    const int b = b0 + (int)threadIdx.x;
    below += __popcll(__ballot(b < A.n_seq && (int)((int64_t)cuq(min(b, A.n_seq - 1)) * P.G / kRows) + b <= bi));
  }
  if (lane == 0) votes[wave] = below;
  __syncthreads();
  const int b = votes[0] + votes[1] + votes[2] + votes[3] - 1;
  if (b < 0) return;
  const int q0 = cuq(b), nq = max(cuq(b + 1) - q0, 0);
  const int nblk = (int)(((int64_t)nq * P.G + kRows - 1) / kRows);
  const int local = bi - (int)((int64_t)q0 * P.G / kRows) - b;
  if (local >= nblk) return;
  const int blk = nblk - 1 - local;                        // the longest first
  int k0 = 0, nk;
  if constexpr (PAGED) {
    const int64_t cap = (int64_t)A.table_width * A.page_size;
    nk = max(A.lengths[b], 0);
    if (nk > cap) nk = (int)cap;
  } else {
    k0 = min(max(A.cu_k[b], 0), A.n_k);
    nk = max(min(max(A.cu_k[b + 1], 0), A.n_k) - k0, 0);
  }
  const int rows = nq * P.G, r = blk * kRows + wave * 32 + n;
  const int rc = min(r, rows - 1), t = rc / P.G, h = hk * P.G + (rc - t * P.G);
  const int ahead = nk - nq;                               // keys before the first row's own
  const int last = ahead + t;                              // the row's last key
  const int wlast0 = ahead + min(blk * kRows + wave * 32, rows - 1) / P.G;         // the wave's first row's
  const int wlast1 = ahead + min(blk * kRows + wave * 32 + 31, rows - 1) / P.G;    // its last row's
  const int nkeys = max(ahead + min(blk * kRows + kRows - 1, rows - 1) / P.G + 1, 0);   // of the block
  const int ntile = (nkeys + KT - 1) / KT;

  gm_u32x4 qf[NC];
  {
    const uint16_t* q = static_cast<const uint16_t*>(A.q) + (int64_t)(q0 + t) * A.q_stride_t +
                        (int64_t)h * A.q_stride_h + 8 * hf;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (P.qvec) {
        qf[c] = *reinterpret_cast<const gm_u32x4*>(q + 16 * c);
      } else {
#pragma unroll
        for (int d = 0; d < 4; ++d)
          qf[c][d] = (uint32_t)q[16 * c + 2 * d] | (uint32_t)q[16 * c + 2 * d + 1] << 16;
      }
    }
  }
  // the cache row of key (lane % KT) of a tile; keys past the last repeat it, -1: no page
  const int32_t* table = PAGED ? A.block_table + b * A.table_stride : nullptr;
  auto row_of = [&](int tile) {
    const int key = min(tile * KT + (lane & (KT - 1)), nkeys - 1);
    if constexpr (!PAGED) return k0 + key;
    const int id = table[key / A.page_size];
    return id >= 0 && id < A.n_pages ? id * A.page_size + key % A.page_size : -1;
  };
  const int64_t kst = PAGED ? (int64_t)A.n_head_kv * Dh : A.k_stride_t;
  const int64_t vst = PAGED ? (int64_t)A.n_head_kv * Dh : A.v_stride_t;
  const uint16_t* kp = static_cast<const uint16_t*>(A.k) + hk * (PAGED ? Dh : A.k_stride_h);
  const uint16_t* vp = static_cast<const uint16_t*>(A.v) + hk * (PAGED ? Dh : A.v_stride_h);
  auto fk = [](int key) { return NGR == 8 ? key & 7 : key & 15; };
  auto fv = [](int key) { return NGR == 8 ? (key >> 1 & 1) * 4 : (key & 3) * 4; };
  auto load = [&](int row, int buf) {                      // row: of key (lane % KT)
    char* kd = lds + 2 * buf * TILE;
    const int safe = max(row, 0);
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int gi = (wave * NI + j) * 64 + lane, key = gi / NGR, gr = gi % NGR;
      const int64_t at = __shfl(safe, key, 64);
      to_lds(kp + at * kst + 8 * (gr ^ fk(key)), kd + (wave * NI + j) * 1024);
      to_lds(vp + at * vst + 8 * (gr ^ fv(key)), kd + TILE + (wave * NI + j) * 1024);
    }
  };
  // a lane's places in a tile: its key's row of K, its key of four of V
  const int i16 = lane & 15;
  const int kbase = n * RB + ((hf ^ fk(n)) << 4);
  const int vkey = 4 * hf + (i16 >> 2), vgr = 2 * (lane >> 4 & 1) + ((i16 & 3) >> 1);
  const int vbase = vkey * RB + ((vgr ^ fv(vkey)) << 4) + 8 * (i16 & 1);

  gm_f32x16 o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
  const float c1 = A.scale * kLog2e;
  float m = kNegInf, mref = 0.f, l = 0.f;

  int row = 0, next = 0;
  if (ntile > 0) {
    row = row_of(0);
    load(row, 0);
    if (ntile > 1) next = row_of(1);
  }
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  for (int it = 0; it < ntile; ++it) {
    const int buf = it & 1;
    const unsigned long long full = KT == 64 ? ~0ull : 0xffffffffull;
    const unsigned long long ok = PAGED ? __ballot(row >= 0) & full : full;
    if (it + 1 < ntile) load(next, buf ^ 1);
    row = next;
    if (it + 2 < ntile) next = row_of(it + 2);
    if (it * KT <= wlast1) {
      const char* K = lds + 2 * buf * TILE;
      const char* V = K + TILE;
      gm_f32x16 s[NS];
#pragma unroll
      for (int u = 0; u < NS; ++u) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[u][e] = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const gm_u32x4 k = *reinterpret_cast<const gm_u32x4*>(
              K + 32 * u * RB + (kbase ^ (32 * c & (16 * (NGR < 16 ? 8 : 16) - 1))) + 256 * (c / 8) * (NGR > 16));
          s[u] = T::mfma32(k, qf[c], s[u]);
        }
      }
      const bool masked = it * KT + KT - 1 > wlast0 || ok != full;
      if (masked) {
        const int left = last - it * KT - 4 * hf;
        uint32_t okh[NS];
#pragma unroll
        for (int u = 0; u < NS; ++u) okh[u] = (uint32_t)(ok >> (32 * u)) >> (4 * hf);
#pragma unroll
        for (int u = 0; u < NS; ++u)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            constexpr int W = 32;
            const int key = W * u + 8 * (e >> 2) + (e & 3);      // and 4 hf
            s[u][e] = key <= left && (!PAGED || (okh[u] >> (key - W * u) & 1)) ? s[u][e] : kNegInf;
          }
      }
      float mt = kNegInf;
#pragma unroll
      for (int u = 0; u < NS; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e) mt = fmaxf(mt, s[u][e]);
      float ma, mb;
      both_halves(mt, ma, mb);
      mt = fmaxf(ma, mb) * c1;
      if (__any(mt > m + kLazy)) {
        const float mn = fmaxf(m, mt), mr = mn == kNegInf ? 0.f : mn;
        const float al = __builtin_amdgcn_exp2f(m - mr);
        m = mn;
        mref = mr;
        l *= al;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[d][e] *= al;
      }
      uint32_t p[NS][8];
      float sum = 0.f;
      const float sub = mref - kShift;
#pragma unroll
      for (int u = 0; u < NS; ++u)
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const float a = __builtin_amdgcn_exp2f(fmaf(s[u][e], c1, -sub));
          const float b2 = __builtin_amdgcn_exp2f(fmaf(s[u][e + 1], c1, -sub));
          sum += a + b2;
          p[u][e / 2] = T::pack(a, b2);
        }
      l += sum;
      bool odd = false;
      if (masked) {
        for (int j = lane; j < TILE / 16; j += 64) {
          const gm_u32x4 v = *reinterpret_cast<const gm_u32x4*>(V + 16 * j);
#pragma unroll
          for (int e = 0; e < 4; ++e) odd |= odd16<QT>(v[e]);
        }
        odd = __any(odd);
      }
      if (__builtin_expect(!odd, 1)) {
#pragma unroll
        for (int u = 0; u < 2 * NS; ++u) {                 // 16 keys
          const gm_u32x4 pb = {p[u >> 1][4 * (u & 1)], p[u >> 1][4 * (u & 1) + 1], p[u >> 1][4 * (u & 1) + 2],
                               p[u >> 1][4 * (u & 1) + 3]};
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            const char* at = V + 16 * u * RB + (vbase ^ (64 * d & 255 & (RB - 1))) + 256 * (d / 4);
            const gm_u32x2 lo = read_tr(at), hi = read_tr(at + 8 * RB);
            o[d] = T::mfma32(gm_u32x4{lo[0], lo[1], hi[0], hi[1]}, pb, o[d]);
          }
        }
      } else {
        // rare, and the wave has no registers left for it: o and p go through memory
        gm_f32x16 om[ND];
        uint32_t pm[NS * 8];
#pragma unroll
        for (int d = 0; d < ND; ++d) om[d] = o[d];
#pragma unroll
        for (int e = 0; e < NS * 8; ++e) pm[e] = p[e / 8][e % 8];
        pv_odd<Dh, QT>(V + vbase, last - it * KT - 4 * hf, ok >> (4 * hf), pm, om);
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] = om[d];
      }
    }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
  }
  float la, lb;
  both_halves(l, la, lb);
  l = la + lb;
  if (r >= rows) return;
  const int64_t orow = ((int64_t)(q0 + t) * A.n_head + h) * Dh;
  const int64_t grow = (int64_t)(q0 + t) * A.gate_stride_t + (int64_t)h * A.gate_stride_h;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int dim = 32 * d + 2 * e + 4 * hf;
      float v[4], g[4];
      if (A.gate) gm_load<4>(A.gate, grow + dim, A.gate_type, P.gvec, g);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        v[c] = o[d][e + c] * inv;
        if (A.gate) v[c] *= 1.0f / (1.0f + __builtin_amdgcn_exp2f(-g[c] * kLog2e));
        if (l == 0.f) v[c] = 0.f;
      }
      gm_store<4>(A.out, orow + dim, QT, v);
    }
}

template <int Dh, int QT, bool PAGED>
int launch(const Pmt& P, hipStream_t s) {
  constexpr int KT = Dh == 256 ? 32 : 64;
  constexpr size_t lds = (size_t)4 * KT * 2 * Dh;
  const int64_t nblk = (int64_t)P.a.n_q * P.G / kRows + P.a.n_seq, grid = nblk * P.a.n_head_kv;
  if (grid > 0x7fffffff) return gm_fail_arg("gm_prompt_attention: too many rows");
  if (int rc = gm_set_smem(k_prompt_attn<Dh, QT, PAGED>, lds)) return rc;
  k_prompt_attn<Dh, QT, PAGED><<<(unsigned)grid, 64 * kWaves, lds, s>>>(P);
  GM_TRY(hipGetLastError());
  return GM_OK;
}

template <int Dh>
int launch_types(const Pmt& P, hipStream_t s) {
  const bool paged = P.a.block_table != nullptr;
  if (P.a.type == GM_QTYPE_BF16)
    return paged ? launch<Dh, GM_QTYPE_BF16, true>(P, s) : launch<Dh, GM_QTYPE_BF16, false>(P, s);
  return paged ? launch<Dh, GM_QTYPE_F16, true>(P, s) : launch<Dh, GM_QTYPE_F16, false>(P, s);
}

}  // namespace

int gm_prompt_attn_run(const gm_prompt_attn_args* a, hipStream_t s) {
  Pmt P{};
  P.a = *a;
  P.G = a->n_head / a->n_head_kv;
  P.qvec = gm_rows_aligned(a->q, a->type, a->q_stride_t, a->q_stride_h);
  P.gvec = a->gate && gm_rows_aligned(a->gate, a->gate_type, a->gate_stride_t, a->gate_stride_h);
  switch (a->head_dim) {
    case 64: return launch_types<64>(P, s);
    case 128: return launch_types<128>(P, s);
    default: return launch_types<256>(P, s);
  }
}
