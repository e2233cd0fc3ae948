// Causal attention over packed prompts (gm_prompt_attention), keys packed or in
// the cache's pages: out = softmax(scale q K^T + mask) V in one pass over the keys,
// with a row's exponentials taken relative to a fixed reference.
//
// Rows: a kv head's rows of one sequence are its tokens x G = n_head / n_head_kv
// heads, head fastest, so that a block's rows share nearly all their keys.  A wave has
// 32 rows; K and V tiles of KT keys go from memory straight to LDS, one tile ahead.
// The longest blocks of all sequences start first.
//
// v_mfma_f32_32x32x16, lane (hf, n) = (lane / 32, lane % 32):
//   S^T = K Q^T     A = key n, dims 16 c + 8 hf ..: 16 bytes of LDS; the lane gets
//                   keys 8 (r / 4) + 4 hf + r % 4 of row n, r < 16: a row's scores
//                   are in two lanes
//   O^T += V^T P^T  the contraction's order is free: k slot 8 hf + j of MFMA u stands
//                   for key 16 u + 8 (j / 4) + 4 hf + j % 4, so the scores rounded to
//                   16 bits are the B operand as they lie; A = 4 keys x 16 dims per
//                   16 lanes by the transposing LDS read, two of them an MFMA
// LDS rows keep their 16-byte granules g at g ^ f(key) so that neither read meets a
// bank twice (SQ_LDS_BANK_CONFLICT 0).  The scores of a tile are formed while the
// probabilities of the one before it are.
//
// The reference that a row's scores are taken relative to is the maximum of its first
// tile, and stays: bf16 has fp32's range, and an fp16 probability may grow to 2^15
// times that tile's largest.  So the loop neither finds maxima nor rescales o (which
// would take a second set of its registers).  A row that outgrows it sends its block
// through twice more: the true maxima, then with those.  References are whole, so that
// another one scales p by a power of two and rounds it alike.
//
// A masked key has p = 0, and 0 times a V value that is not finite would be NaN: such
// values are cleared in the tiles with a mask, and added at the end to the rows that
// see them.
//
// Bound: MFMA, with the exponentials beside them; for short prompts the latency of a
// block's first loads and its epilogue.  Measured: 16,000 tokens of 16 heads of 256 on 2,
// bf16, 2.29 ms (915 TFLOP/s of the 1,110 of a large product); 8,192 tokens in 11 prompts,
// 32 heads of 128 on 8, fp16, 136 us (675); 301 tokens in 5, 16 of 256, 30 us.  With a
// running maximum and the rescaling the first took 15.6 ms, its registers spilled.
#include "kernels.h"
#include "serving.h"

namespace {

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

// Sum over the wave's lanes.
__device__ __forceinline__ int wave_sum64(int v) {
  v += GM_DPP_I(v, GM_ROW_ROR8);
  v += GM_DPP_I(v, GM_ROW_ROR4);
  v += GM_DPP_I(v, GM_QPERM_2301);
  v += GM_DPP_I(v, GM_QPERM_1032);
  return (__builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16)) +
         (__builtin_amdgcn_readlane(v, 32) + __builtin_amdgcn_readlane(v, 48));
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

// Clears the values of a tile that are not finite; whether there were any (the same
// for the whole block).
template <int QT, int TILE, int NW>
__device__ __forceinline__ bool clear_odd(char* tile) {
  constexpr int N = TILE / (16 * 64 * NW);
  gm_u32x4 v[N];
  bool odd = false;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    v[j] = *reinterpret_cast<const gm_u32x4*>(tile + 16 * (64 * NW * j + (int)threadIdx.x));
#pragma unroll
    for (int e = 0; e < 4; ++e) odd |= odd16<QT>(v[j][e]);
  }
  if (!__syncthreads_or(odd)) return false;
#pragma unroll
  for (int j = 0; j < N; ++j) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      v[j][e] &= (odd_kind<QT>(v[j][e] & 0xffffu) ? 0u : 0xffffu) | (odd_kind<QT>(v[j][e] >> 16) ? 0u : 0xffff0000u);
    *reinterpret_cast<gm_u32x4*>(tile + 16 * (64 * NW * j + (int)threadIdx.x)) = v[j];
  }
  __syncthreads();
  return true;
}

// NW waves of 32 rows each, KT keys a tile; the last QL of the Dh / 16 pieces of the
// queries in LDS instead of registers; LK, LV: LDS reads ahead of their MFMAs.
template <int Dh, int QT, bool PAGED, int NW, int KT, int QL, int LK, int LV, int WPS>
__global__ void __launch_bounds__(64 * NW, WPS) k_prompt_attn(Pmt P) {
  using T = GmT16<QT>;
  constexpr int NS = KT / 32, NC = Dh / 16, ND = Dh / 32, NGR = Dh / 8, RB = 2 * Dh;
  constexpr int TILE = KT * RB, NI = TILE / (1024 * NW), ROWS = 32 * NW, QR = NC - QL;
  // p = 2^(score - reference + kStart) of the first tile's maximum (pass 0), kExact of the
  // row's (pass 2); a tile's p of a row sum to at most kMost
  constexpr bool F16 = QT == GM_QTYPE_F16;
  constexpr float kStart = 0.f, kExact = F16 ? 14.f : 0.f, kMost = F16 ? 32768.f : 0x1p80f;
  extern __shared__ __attribute__((aligned(1024))) char lds[];      // K [2][TILE], V [2][TILE], queries [NW][QL][1024]
  __shared__ int votes[NW];
  const gm_prompt_attn_args& A = P.a;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, hf = lane >> 5, n = lane & 31;
  const int hk = blockIdx.x % A.n_head_kv, bi = blockIdx.x / A.n_head_kv;
  auto cuq = [&](int b) { return min(max(A.cu_q[b], 0), A.n_q); };
  auto blocks = [&](int b) { return (int)(((int64_t)max(cuq(b + 1) - cuq(b), 0) * P.G + ROWS - 1) / ROWS); };
  int b, blk;
  if (A.n_seq <= 64) {
    // block bi of all blocks from the last of every sequence down to the first: the
    // longest start first.  Lane l has sequence l; level L holds the sequences with
    // more than L blocks
    const int nb = lane < A.n_seq ? blocks(lane) : 0;
    auto down_to = [&](int level) { return wave_sum64(max(nb - level, 0)); };     // blocks on this level and above
    if (bi >= down_to(0)) return;
    int lo = 0, hi = 1;                                    // bi is on level lo or above, below hi
    while (bi < down_to(hi)) lo = hi, hi *= 2;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (bi < down_to(mid)) lo = mid;
      else hi = mid;
    }
    blk = lo;
    const unsigned long long on = __ballot(nb > lo);
    int skip = bi - down_to(lo + 1);
    unsigned long long rest = on;
    while (skip-- > 0) rest &= rest - 1;
    b = __ffsll(rest) - 1;
  } else {
    // sequence b's blocks start at cu_q[b] G / ROWS + b: never fewer than it needs
    int below = 0;
    for (int b0 = 0; b0 < A.n_seq; b0 += 64 * NW) {
      const int c = b0 + (int)threadIdx.x;
      below += __popcll(__ballot(c < A.n_seq && (int)((int64_t)cuq(min(c, A.n_seq - 1)) * P.G / ROWS) + c <= bi));
    }
    if (lane == 0) votes[wave] = below;
    __syncthreads();
    b = -1;
#pragma unroll
    for (int w = 0; w < NW; ++w) b += votes[w];
    if (b < 0) return;
    const int nblk = blocks(b), local = bi - (int)((int64_t)cuq(b) * P.G / ROWS) - b;
    if (local >= nblk) return;
    blk = nblk - 1 - local;                                // the longest first
  }
  b = __builtin_amdgcn_readfirstlane(b);
  blk = __builtin_amdgcn_readfirstlane(blk);
  const int q0 = cuq(b), nq = max(cuq(b + 1) - q0, 0);
  int k0 = 0, nk;
  if constexpr (PAGED) {
    const int64_t cap = min((int64_t)A.table_width * A.page_size, (int64_t)0x7fffff00);   // room to round up
    nk = max(A.lengths[b], 0);
    if (nk > cap) nk = (int)cap;
  } else {
    k0 = min(max(A.cu_k[b], 0), A.n_k);
    nk = max(min(max(A.cu_k[b + 1], 0), A.n_k) - k0, 0);
  }
  const int rows = nq * P.G, r0 = blk * ROWS + wave * 32;
  const int ahead = nk - nq;                               // keys before the first row's own
  const int nkeys = max(ahead + min(blk * ROWS + ROWS - 1, rows - 1) / P.G + 1, 0);   // of the block
  const int ntile = (nkeys + KT - 1) / KT;
  // token and head of the lane's row, worked out where they are needed: kept, they would
  // take registers from the loop
  auto row_at = [&](int& t, int& h) {
    int rc = min(r0 + n, rows - 1);
    asm volatile("" : "+v"(rc));
    t = rc / P.G;
    h = hk * P.G + (rc - t * P.G);
  };
  gm_u32x4 qf[QR];
  char* const ql = lds + 4 * TILE + (wave * QL * 64 + lane) * 16;
  {
    int t, h;
    row_at(t, h);
    const uint16_t* q = static_cast<const uint16_t*>(A.q) + (int64_t)(q0 + t) * A.q_stride_t +
                        (int64_t)h * A.q_stride_h + 8 * hf;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      gm_u32x4 w;
      if (P.qvec) {
        w = *reinterpret_cast<const gm_u32x4*>(q + 16 * c);
      } else {
#pragma unroll
        for (int d = 0; d < 4; ++d) w[d] = (uint32_t)q[16 * c + 2 * d] | (uint32_t)q[16 * c + 2 * d + 1] << 16;
      }
      if (c < QR) qf[c] = w;
      else *reinterpret_cast<gm_u32x4*>(ql + (c - QR) * 1024) = w;
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
  // a tile of K or V to LDS; row: of key (lane % KT)
  auto load = [&](const uint16_t* src, int64_t st, bool isk, int row, int at0) {
    const int safe = max(row, 0);
    int ln = lane;                                         // what follows from it is formed anew, not kept
    asm volatile("" : "+v"(ln));
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int gi = (wave * NI + j) * 64 + ln, key = gi / NGR, gr = gi % NGR;
      const int64_t at = __shfl(safe, key, 64);
      to_lds(src + at * st + 8 * (gr ^ (isk ? fk(key) : fv(key))), lds + at0 + (wave * NI + j) * 1024);
    }
  };
  // a lane's places in a tile: its key's row of K, its key of four of V
  const int i16 = lane & 15;
  const int kbase = n * RB + ((hf ^ fk(n)) << 4);
  const int vkey = 4 * hf + (i16 >> 2), vgr = 2 * (lane >> 4 & 1) + ((i16 & 3) >> 1);
  const int vbase = vkey * RB + ((vgr ^ fv(vkey)) << 4) + 8 * (i16 & 1);
  constexpr int KX = NGR < 16 ? 127 : 255;                 // address bits that the XORs reach

  gm_f32x16 o[ND], s[NS];
  const float c1 = A.scale * kLog2e;
  float sub = 0.f, l = 0.f, top = kNegInf;                 // what is subtracted from a score, sum, largest score
  constexpr unsigned long long full = KT == 64 ? ~0ull : 0xffffffffull;

  // MFMA j of a tile's scores, j = NC u + c: its K, and its queries where they are in LDS
  auto read_k = [&](int ka, int j) {
    const int u = j / NC, c = j % NC;
    return *reinterpret_cast<const gm_u32x4*>(lds + (ka ^ (32 * c & KX)) + 32 * u * RB + 256 * (c / 8) * (NGR > 16));
  };
  auto read_q = [&](int j) { return *reinterpret_cast<const gm_u32x4*>(ql + (j % NC - QR) * 1024); };
  // MFMA j of a tile's outputs, j = ND u + d: 16 keys, 32 dims
  auto read_v = [&](int va, int j) {
    const int u = j / ND, d = j % ND;
    const char* at = lds + (va ^ (64 * d & 255 & (RB - 1))) + 16 * u * RB + 256 * (d / 4);
    const gm_u32x2 lo = read_tr(at), hi = read_tr(at + 8 * RB);
    return gm_u32x4{lo[0], lo[1], hi[0], hi[1]};
  };
  // The scores x of a tile; beside(j) after MFMA j.  Every step is held in its place:
  // left to itself the compiler waits for each read right after it.
  auto scores = [&](int tile, gm_f32x16 (&x)[NS], auto beside) {
    int ka = kbase + (tile & 1) * TILE;                    // formed anew for every tile: the XORs, kept, take registers
    asm volatile("" : "+v"(ka));
    gm_u32x4 kr[LK], qr[LK];
#pragma unroll
    for (int j = 0; j < LK; ++j) {
      kr[j] = read_k(ka, j);
      if (j % NC >= QR) qr[j] = read_q(j);
    }
#pragma unroll
    for (int u = 0; u < NS; ++u)
#pragma unroll
      for (int e = 0; e < 16; ++e) x[u][e] = 0.f;
#pragma unroll
    for (int j = 0; j < NS * NC; ++j) {
      __builtin_amdgcn_sched_barrier(0);
      const int c = j % NC;
      x[j / NC] = T::mfma32(kr[j % LK], c < QR ? qf[c < QR ? c : 0] : qr[j % LK], x[j / NC]);
      if (j + LK < NS * NC) {
        kr[j % LK] = read_k(ka, j + LK);
        if ((j + LK) % NC >= QR) qr[j % LK] = read_q(j + LK);
      }
      beside(j);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto row_max = [&](gm_f32x16 (&x)[NS]) {
    float v = x[0][0];
#pragma unroll
    for (int u = 0; u < NS; ++u)
#pragma unroll
      for (int e = 0; e < 16; ++e) v = fmaxf(v, x[u][e]);
    float va, vb;
    both_halves(v, va, vb);
    top = fmaxf(top, fmaxf(va, vb));
  };
  auto mask = [&](int tile, unsigned long long ok, gm_f32x16 (&x)[NS]) {
    int t, h;
    row_at(t, h);
#pragma unroll
    for (int u = 0; u < NS; ++u) {
      const uint32_t okh = (uint32_t)(ok >> (32 * u)) >> (4 * hf);
      const int left = ahead + t - tile * KT - 32 * u - 4 * hf;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int key = 8 * (e >> 2) + (e & 3);            // and 4 hf
        x[u][e] = key <= left && (!PAGED || (okh >> key & 1)) ? x[u][e] : kNegInf;
      }
    }
  };
  auto okay = [&](int row) { return PAGED ? __ballot(row >= 0) & full : full; };
  // rows of tile it, of the next one (to be loaded), of the one after that
  int rw = 0, rw1 = 0, rw2 = 0;
  const int first = ahead + blk * ROWS / P.G;              // the last key of the block's first row
  int it0 = ntile;                                         // the first tile with a mask
  bool odd = false;                                        // some tile with a mask held a V that is not finite
  // pass 0 takes a row's first tile as its reference; where that was not enough (the
  // same for the whole block), pass 1 finds the maximum and pass 2 takes that
  for (int pass = 0; pass < 3; ++pass) {
    bool far = false;                                      // a score too far from its row's reference
    l = 0.f;
    if (pass == 2) sub = (top == kNegInf ? 0.f : rintf(top * c1)) - kExact;
    else top = kNegInf;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
    // K of tile j lies in buffer j % 2, V in 2 + j % 2; in round it K of it + 2 and V of
    // it + 1 are on their way, and the scores of it + 1 are formed beside the rest of it
    if (ntile > 0) {
      rw = row_of(0);
      load(kp, kst, true, rw, 0);
      load(vp, vst, false, rw, 2 * TILE);
      if (ntile > 1) {
        rw1 = row_of(1);
        load(kp, kst, true, rw1, TILE);
      }
      if (ntile > 2) rw2 = row_of(2);
    }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    bool masked = false;
    auto finish = [&](int tile, int row, gm_f32x16 (&x)[NS]) {           // the scores of a tile are there
      const unsigned long long ok = okay(row);
      masked = tile * KT + KT - 1 > first || ok != full;   // for some row of the block
      if (masked) mask(tile, ok, x);
      if (pass == 1 || (pass == 0 && tile == 0)) {
        row_max(x);
        sub = (top == kNegInf ? 0.f : rintf(top * c1)) - kStart;
        far |= top == kNegInf;
      }
    };
    if (ntile > 0) {
      scores(0, s, [](int) {});
      finish(0, rw, s);
    }
    __syncthreads();                                       // tile 0 of K is read
    for (int it = 0; it < ntile; ++it) {
      if (it + 2 < ntile) load(kp, kst, true, rw2, (it & 1) * TILE);
      if (it + 1 < ntile) load(vp, vst, false, rw1, (2 + ((it + 1) & 1)) * TILE);
      const int rw3 = it + 3 < ntile ? row_of(it + 3) : 0;
      if (masked) {
        it0 = min(it0, it);
        odd |= clear_odd<QT, TILE, NW>(lds + (2 + (it & 1)) * TILE);
      }
      // the next tile's scores (past the last: what lies there, never used), and beside
      // them this one's probabilities and the first reads of its V
      gm_f32x16 sn[NS];
      uint32_t p[NS * 8];
      float sum = 0.f;
      gm_u32x4 vr[LV];
      int va = vbase + (2 + (it & 1)) * TILE;
      asm volatile("" : "+v"(va));
      constexpr int NQK = NS * NC, PER = (NS * 8 + NQK - 1) / NQK;
      scores(it + 1, sn, [&](int j) {
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          const int w = PER * j + e;
          if (w < NS * 8) {
            const float a = __builtin_amdgcn_exp2f(fmaf(s[w / 8][2 * w % 16], c1, -sub));
            const float b2 = __builtin_amdgcn_exp2f(fmaf(s[w / 8][2 * w % 16 + 1], c1, -sub));
            p[w] = T::pack(a, b2);
            sum = T::add(p[w], sum);                        // as rounded: a row of few keys then divides the rounding out
          }
        }
        if (j >= NQK - LV) vr[j - (NQK - LV)] = read_v(va, j - (NQK - LV));
      });
      l += sum;
      far |= sum > kMost;                                   // NaN is no reason: it stays NaN
      if (pass != 1) {
#pragma unroll
        for (int j = 0; j < 2 * NS * ND; ++j) {
          const int u = j / ND;
          o[j % ND] = T::mfma32(vr[j % LV], gm_u32x4{p[4 * u], p[4 * u + 1], p[4 * u + 2], p[4 * u + 3]}, o[j % ND]);
          if (j + LV < 2 * NS * ND) vr[j % LV] = read_v(va, j + LV);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
#pragma unroll
      for (int u = 0; u < NS; ++u) s[u] = sn[u];
      if (it + 1 < ntile) finish(it + 1, rw1, s);
      rw1 = rw2;
      rw2 = rw3;
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
    }
    if (pass == 0 && !__syncthreads_or(far)) break;
  }
  // ---- out: 64 dims at a time through LDS, so that a row's are stored together
  constexpr int LDO = 68, OUTS = NW * 32 * LDO * 4;        // floats of a row in LDS; bytes of all, a V tile behind them
  static_assert(OUTS % 1024 == 0);
  const uint32_t one = F16 ? 0x3c00u : 0x3f80u;
  float la, lb;
  both_halves(l, la, lb);
  const float lt = la + lb, inv = lt == 0.f ? 0.f : 1.0f / lt;
  float* const os = reinterpret_cast<float*>(lds) + wave * 32 * LDO;
  os[n * LDO + 64] = lt;                                   // beside the 64 dims
  // in step i the lane has 8 dims of the wave's row 8 i + lane / 8
  const int od = 8 * (lane & 7);
  int64_t orow[4], grow[4];
  bool live[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + 8 * i + (lane >> 3), rc = min(r, rows - 1), t = rc / P.G, h = hk * P.G + (rc - t * P.G);
    live[i] = r < rows;
    orow[i] = ((int64_t)(q0 + t) * A.n_head + h) * Dh + od;
    grow[i] = (int64_t)(q0 + t) * A.gate_stride_t + (int64_t)h * A.gate_stride_h + od;
  }
#pragma unroll
  for (int d0 = 0; d0 < ND; d0 += 2) {
    float g[4][8];
    if (A.gate) {
#pragma unroll
      for (int i = 0; i < 4; ++i) gm_load<8>(A.gate, grow[i] + 32 * d0, A.gate_type, P.gvec, g[i]);
    }
#pragma unroll
    for (int d = d0; d < d0 + 2; ++d) {
      gm_f32x16 x = o[d];
      if (odd) {
        // what the row gets of the values that were cleared: the MFMAs count those it sees
        gm_f32x16 c;
#pragma unroll
        for (int e = 0; e < 16; ++e) c[e] = 0.f;
        int t, h;
        row_at(t, h);
#pragma unroll 1
        for (int it = it0; it < ntile; ++it) {
          __syncthreads();                                 // the tile before is read
          rw = row_of(it);
          load(vp, vst, false, rw, OUTS);
          __builtin_amdgcn_s_waitcnt(0);
          __syncthreads();
          const unsigned long long ok = okay(rw) >> (4 * hf);
          const int left = ahead + t - it * KT - 4 * hf;
#pragma unroll 1
          for (int u = 0; u < 2 * NS; ++u) {
            const char* at = lds + ((vbase + OUTS) ^ (64 * d & 255 & (RB - 1))) + 16 * u * RB + 256 * (d / 4);
            const gm_u32x2 lo = read_tr(at), hi = read_tr(at + 8 * RB);
            const gm_u32x4 v = {lo[0], lo[1], hi[0], hi[1]};
            gm_u32x4 kind, seen;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              kind[w] = odd_kind<QT>(v[w] & 0xffffu) | odd_kind<QT>(v[w] >> 16) << 16;
              const int key = 16 * u + 8 * (w >> 1) + 2 * (w & 1);         // and 4 hf
              const uint32_t okw = (uint32_t)(ok >> key);
              seen[w] = (key <= left && (okw & 1) ? one : 0u) | (key + 1 <= left && (okw & 2) ? one << 16 : 0u);
            }
            c = T::mfma32(kind, seen, c);
          }
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] += odd_value(c[e]);
      }
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<gm_f32x4*>(os + n * LDO + 32 * (d - d0) + 2 * e + 4 * hf) =
            gm_f32x4{x[e] * inv, x[e + 1] * inv, x[e + 2] * inv, x[e + 3] * inv};
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();                       // the wave's own rows: no other wave reads them
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float* src = os + (8 * i + (lane >> 3)) * LDO + od;
      const gm_f32x4 x0 = *reinterpret_cast<const gm_f32x4*>(src), x1 = *reinterpret_cast<const gm_f32x4*>(src + 4);
      float v[8] = {x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
      if (A.gate) {
        const bool any = os[(8 * i + (lane >> 3)) * LDO + 64] != 0.f;    // the row has a key
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float f = 1.0f / (1.0f + __builtin_amdgcn_exp2f(-g[i][e] * kLog2e));
          v[e] = any ? v[e] * f : 0.f;
        }
      }
      if (live[i]) gm_store<8>(A.out, orow[i] + 32 * d0, QT, v);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
}

template <int Dh, int QT, bool PAGED, int NW, int KT, int QL, int LK, int LV, int WPS>
int launch(const Pmt& P, hipStream_t s) {
  constexpr size_t tiles = (size_t)4 * KT * 2 * Dh + NW * QL * 1024, outs = (size_t)NW * 32 * 68 * 4 + KT * 2 * Dh;
  constexpr size_t lds = tiles > outs ? tiles : outs;
  constexpr int ROWS = 32 * NW;
  const int64_t nblk = (int64_t)P.a.n_q * P.G / ROWS + P.a.n_seq, grid = nblk * P.a.n_head_kv;
  if (grid > 0x7fffffff) return gm_fail_arg("gm_prompt_attention: too many rows");
  auto kern = k_prompt_attn<Dh, QT, PAGED, NW, KT, QL, LK, LV, WPS>;
  if (int rc = gm_set_smem(kern, lds)) return rc;
  kern<<<(unsigned)grid, 64 * NW, lds, s>>>(P);
  GM_TRY(hipGetLastError());
  return GM_OK;
}

template <int Dh, int QT, bool PAGED>
int launch_size(const Pmt& P, hipStream_t s) {
  if constexpr (Dh == 256) {
    // heads of 256 take 128 registers for o and 64 for q: two waves a SIMD hold that only
    // with 10 of the 16 pieces of q in LDS, which one block of 8 waves a CU has room for
    // (16,000 tokens: 2.3 ms; all in registers and spilled 2.95, one wave a SIMD 3.3).
    // Where such blocks would leave CUs idle, 4 waves with everything in registers
    // (301 tokens: 29.7 us against 33.5)
    if ((int64_t)P.a.n_q * P.a.n_head / 256 < 256) return launch<Dh, QT, PAGED, 4, 32, 0, 4, 4, 1>(P, s);
    return launch<Dh, QT, PAGED, 8, 32, 10, 2, 2, 2>(P, s);
  } else {
    return launch<Dh, QT, PAGED, 4, 32, 0, 4, 3, 2>(P, s);
  }
}

template <int Dh>
int launch_types(const Pmt& P, hipStream_t s) {
  const bool paged = P.a.block_table != nullptr;
  if (P.a.type == GM_QTYPE_BF16)
    return paged ? launch_size<Dh, GM_QTYPE_BF16, true>(P, s) : launch_size<Dh, GM_QTYPE_BF16, false>(P, s);
  return paged ? launch_size<Dh, GM_QTYPE_F16, true>(P, s) : launch_size<Dh, GM_QTYPE_F16, false>(P, s);
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
