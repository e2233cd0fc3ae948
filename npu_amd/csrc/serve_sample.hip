// One token per row of logits (gm_sample): temperature, top-k, top-p, min-p and
// the inverse of the kept weights' running sum at u.
//
// The pick is that of the definition in 64 bits: weights w = e^((x - max) / t) and
// all their sums are fp64, so that u times the total falls between the same two
// running sums.  fp64 FMAs run at the fp32 rate here; the exponential is a table of
// 64 powers in LDS and five terms.
//
// k_sample_groups   every group of 512 logits: its maximum, the maximum of every lane's
//                   8 and, for rows without a top-k, the group's sum of weights.  The
//                   one pass over all logits.
// k_sample_pick     one block per row.  A histogram of the lanes' maxima over their
//                   distance from the row's finds a distance that the filters cannot
//                   pass: where k maxima are nearer, or maxima that weigh top_p of the
//                   total, or by min-p itself.  Only lanes with a maximum that near are
//                   read again, and up to kCand candidates are ranked against each
//                   other in LDS.  More than that (a flat nucleus, a large k): the same
//                   histogram over all values finds the bin where the filter ends, and
//                   only that bin's are ranked (or cut bit by bit, if they too are many).
// Kept tokens run in the vocabulary's order, so nothing is ever sorted as a whole.
// No result depends on the order of atomics: they count, or add fixed-point values.
// Bound: HBM and, without top-k, the fp64 exponentials of the first kernel; for few
// rows the second kernel's chain of block-wide steps.
#include "kernels.h"
#include "serving.h"

namespace {

constexpr int kGroup = 512;         // logits of a group: 8 per lane of a wave
constexpr int kCand = 1024;         // candidates ranked in LDS, one per thread
constexpr int kBins = 2048;         // bins of the distance from the maximum ...
constexpr float kBinsPerE = 32.f;   // ... 1/32 wide, in units of the temperature
constexpr int kList = 4096;         // lanes of 8 logits that are read again
constexpr float kNegInf = -__builtin_inff();
constexpr float kPosInf = __builtin_inff();

size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

struct Smp {
  gm_sample_args a;
  float* gmax;       // [n_row][ng]
  double* gsum;      // [n_row][ng]
  void* lmax;        // [n_row][ng][64] in the logits' type
  int ng;
  bool vec;          // rows start at multiples of 16 bytes
};

struct RowParam {
  float t, top_p, min_p;
  int top_k;         // 0: none
  bool greedy;
};

__device__ __forceinline__ RowParam row_param(const gm_sample_args& A, int row) {
  RowParam r;
  r.t = A.temperature ? A.temperature[row] : A.temperature_all;
  r.top_k = A.top_k ? A.top_k[row] : A.top_k_all;
  r.top_p = A.top_p ? A.top_p[row] : A.top_p_all;
  r.min_p = A.min_p ? A.min_p[row] : A.min_p_all;
  r.greedy = !(r.t > 0.f);
  if (r.top_k <= 0 || r.top_k >= A.vocab) r.top_k = 0;
  if (!(r.top_p < 1.f)) r.top_p = 1.f;                 // NaN too: no filter
  if (r.top_p <= 0.f) {                                // the largest alone
    r.top_p = 1.f;
    r.top_k = 1;
  }
  if (!(r.min_p > 0.f)) r.min_p = 0.f;
  if (r.min_p > 1.f) r.min_p = 1.f;
  return r;
}

// 2^(j / 64), j < 64.
__device__ __forceinline__ void exp_table(double* tab) {
  if (threadIdx.x < 64) tab[threadIdx.x] = exp2((double)threadIdx.x * (1.0 / 64));
}

constexpr double kUnits = 92.332482616893656877;       // 64 / ln 2
constexpr double kFar = -700.0 * kUnits;               // weights below e^-700 count as 0

// 2^(y / 64), kFar <= y <= 0, within 3e-16 of it and 2e-16 |y / 64| more: y = k + f with
// |f| <= 1/2, 2^(k % 64 / 64) from the table, 2^(k / 64) straight into the exponent.  k
// is in the low bits of a sum with 1.5 x 2^52.
__device__ __forceinline__ double fexp(double y, const double* tab) {
  constexpr double magic = 6755399441055744.0, c = 0.010830424696249145;      // ln 2 / 64
  const double t = y + magic;
  const int ki = (int)(uint32_t)__double_as_longlong(t);
  const double f = y - (t - magic);
  double p = fma(f, c * c * c * c * c / 120, c * c * c * c / 24);
  p = fma(f, p, c * c * c / 6);
  p = fma(f, p, c * c / 2);
  p = fma(f, p, c);
  const double s = tab[ki & 63];
  return __longlong_as_double(__double_as_longlong(fma(s, f * p, s)) + ((long long)(ki >> 6) << 52));
}

// The weight of x beside the maximum m; units = 64 / (ln 2 t).
__device__ __forceinline__ double weight(float x, float m, double units, const double* tab) {
  if (!(x > kNegInf)) return 0.0;                      // NaN, -inf
  if (x == m) return 1.0;
  if (m == kPosInf) return 0.0;
  const double y = ((double)x - (double)m) * units;
  return y < kFar ? 0.0 : fexp(y, tab);
}

// The 8 logits of a lane in group gr; index of the j-th: at(j).  Past the end -inf.
struct Lane8 {
  float x[8];
  int i0, step;
  __device__ __forceinline__ int at(int j) const { return i0 + (j & 3) + (j >> 2) * step; }
};
__device__ __forceinline__ Lane8 load8(const Smp& P, int row, int gr, int lane) {
  const gm_sample_args& A = P.a;
  const int V = A.vocab;
  Lane8 r;
  // fp32: two loads of four, 256 apart; 16 bits: one of eight
  const bool f32 = A.type == GM_QTYPE_F32;
  r.step = f32 ? 256 : 4;
  r.i0 = gr * kGroup + lane * (f32 ? 4 : 8);
  const int64_t base = (int64_t)row * A.row_stride;
  if (P.vec && (gr + 1) * kGroup <= V) {
    if (f32) {
      float lo[4], hi[4];
      gm_load<4>(A.logits, base + r.i0, GM_QTYPE_F32, true, lo);
      gm_load<4>(A.logits, base + r.i0 + 256, GM_QTYPE_F32, true, hi);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        r.x[j] = lo[j];
        r.x[4 + j] = hi[j];
      }
    } else {
      gm_load<8>(A.logits, base + r.i0, A.type, true, r.x);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = r.at(j);
      r.x[j] = i < V ? gm_elem(A.logits, base + i, A.type) : kNegInf;
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) r.x[j] = r.x[j] > kNegInf ? r.x[j] + 0.f : kNegInf;   // NaN -> -inf, -0 -> 0
  return r;
}

__device__ __forceinline__ Lane8 load8(const Smp& P, int row, int gr) { return load8(P, row, gr, threadIdx.x & 63); }

// Maximum over the wave's lanes.
__device__ __forceinline__ float wave_max64(float v) {
  v = fmaxf(v, GM_DPP_F(v, GM_ROW_ROR8));
  v = fmaxf(v, GM_DPP_F(v, GM_ROW_ROR4));
  v = fmaxf(v, GM_DPP_F(v, GM_QPERM_2301));
  v = fmaxf(v, GM_DPP_F(v, GM_QPERM_1032));
  const int b = __builtin_bit_cast(int, v);
  const float r0 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 0));
  const float r1 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 16));
  const float r2 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 32));
  const float r3 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 48));
  return fmaxf(fmaxf(r0, r1), fmaxf(r2, r3));
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// U groups of a wave, loaded together: 4, or 1 where there are few rows (one row of
// 248,320: 4.5 us with 4).
template <int U>
__global__ void __launch_bounds__(256) k_sample_groups(Smp P) {
  __shared__ double tab[64];
  exp_table(tab);
  __syncthreads();
  const int row = blockIdx.y, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const RowParam rp = row_param(P.a, row);
  const bool sums = !rp.greedy && rp.top_k == 0;
  const bool lanes = !rp.greedy && (rp.top_k > 1 || rp.top_p < 1.f || rp.min_p > 0.f);
  const double units = kUnits / (double)rp.t;
  const int g0 = (blockIdx.x * 4 + wave) * U;
  Lane8 v[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (g0 + u < P.ng) v[u] = load8(P, row, g0 + u);
  double s[U];
  float gm[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    s[u] = 0.0;
    gm[u] = kNegInf;
    if (g0 + u >= P.ng) continue;
    float m = v[u].x[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) m = fmaxf(m, v[u].x[j]);
    if (lanes) {
      const int64_t at = ((int64_t)row * P.ng + g0 + u) * 64 + lane;
      if (P.a.type == GM_QTYPE_F32) static_cast<float*>(P.lmax)[at] = m;
      else if (P.a.type == GM_QTYPE_BF16) static_cast<uint16_t*>(P.lmax)[at] = (uint16_t)GmT16<GM_QTYPE_BF16>::pack(m, m);
      else static_cast<uint16_t*>(P.lmax)[at] = (uint16_t)GmT16<GM_QTYPE_F16>::pack(m, m);
    }
    gm[u] = m = wave_max64(m);
    if (sums && m > kNegInf) {
      float low = v[u].x[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) low = fminf(low, v[u].x[j]);
      if (m < kPosInf && !__any(!(((double)low - (double)m) * units >= kFar))) {
        // the usual group: all finite and near enough (77 us with the tests per value at
        // 256 rows of 248,320)
#pragma unroll
        for (int j = 0; j < 8; ++j) s[u] += fexp(((double)v[u].x[j] - (double)m) * units, tab);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) s[u] += weight(v[u].x[j], m, units, tab);
      }
    }
  }
  if (sums) {
    if constexpr (U == 4) {
      // four sums over the lanes in 7 exchanges: pairs of lanes first take two groups
      // each, then one; lane l ends with group l % 4
      const bool o1 = lane & 1, o2 = lane & 2;
      const double a = (o1 ? s[1] : s[0]) + __shfl_xor(o1 ? s[0] : s[1], 1, 64);
      const double b = (o1 ? s[3] : s[2]) + __shfl_xor(o1 ? s[2] : s[3], 1, 64);
      double c = (o2 ? b : a) + __shfl_xor(o2 ? a : b, 2, 64);
#pragma unroll
      for (int o = 4; o < 64; o <<= 1) c += __shfl_xor(c, o, 64);
      if (lane < 4 && g0 + lane < P.ng) P.gsum[(int64_t)row * P.ng + g0 + lane] = c;
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const double c = wave_sum(s[u]);
        if (lane == 0 && g0 + u < P.ng) P.gsum[(int64_t)row * P.ng + g0 + u] = c;
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (lane == u && g0 + u < P.ng) P.gmax[(int64_t)row * P.ng + g0 + u] = gm[u];
}

// ---- block-wide steps of k_sample_pick (1024 threads)
constexpr int kThreads = 1024, kWaves = 16;

__device__ __forceinline__ float block_max(float v, float* red) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float m = red[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) m = fmaxf(m, red[w]);
  return m;
}

__device__ __forceinline__ int block_min(int v, int* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  int m = red[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) m = min(m, red[w]);
  return m;
}

__device__ __forceinline__ int block_max_u(uint32_t v, int* red) {
  return (int)~(uint32_t)(block_min((int)(~v ^ 0x80000000u), red) ^ 0x80000000u);
}

// Running sum over the threads, the own value with it; all: the sum.
template <typename T>
__device__ __forceinline__ T block_scan(T v, T* red, T* all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const T u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 63) red[wave] = v;
  __syncthreads();
  T before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) before += red[w];
    total += red[w];
  }
  *all = total;
  return v + before;
}

// Floats as integers of the same order.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct Shared {
  double tab[64];
  double dred[kWaves];
  unsigned long long ured[kWaves];
  float fred[kWaves];
  int ired[kWaves];
  int count;
  int bin;
  unsigned long long above;
  int above_n;
  unsigned long long cand[kCand];       // descending value, then index: (~key << 32) | index
  double w[kCand];
  int id[kCand];
  unsigned long long mass[kBins];       // fixed point
  unsigned int cnt[kBins];
};

static_assert(sizeof(Shared::mass) >= kList * sizeof(int));

// Where the filters end: kept are the values above `key`, and of that value the
// indices up to `id`.
struct Cut {
  uint32_t key;
  int id;
};
__device__ __forceinline__ bool kept(float x, int i, const Cut& c) {
  const uint32_t k = key_of(x);
  return k > c.key || (k == c.key && i <= c.id);
}

struct Row {
  int row;
  float xmax;
  float per_bin;     // bins per unit of x
  double units;
  double fix;        // fixed point of the histogram's masses: the sum of all fits 63 bits
};

// The thread's candidate (tid < n) among S.cand, ranked: its weight goes to S.w and
// its entry's index to S.id at its rank.  Returns its rank.
__device__ __forceinline__ int rank_candidates(Shared& S, int n, unsigned long long mine, double w) {
  int rank = 0;
  if ((int)threadIdx.x < n) {
    for (int j = 0; j < n; ++j) rank += S.cand[j] < mine ? 1 : 0;
    S.w[rank] = w;
    S.id[rank] = (int)(uint32_t)mine;
  }
  __syncthreads();
  return rank;
}

__device__ __forceinline__ float value_of(unsigned long long c) {
  const uint32_t k = ~(uint32_t)(c >> 32);
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// Adds a wave's lanes to S.cnt[bin] and S.mass[bin] (bin < 0: none).  Lanes that
// all have one bin add once.
__device__ __forceinline__ void hist_add(Shared& S, int bin, unsigned long long m) {
  const unsigned long long on = __ballot(bin >= 0);
  if (on == 0) return;
  const int first = __shfl(bin, __ffsll(on) - 1, 64);
  if (__ballot(bin >= 0 && bin != first) == 0) {
    unsigned long long s = bin >= 0 ? m : 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) {
      atomicAdd(&S.cnt[first], (unsigned)__popcll(on));
      atomicAdd(&S.mass[first], s);
    }
  } else if (bin >= 0) {
    atomicAdd(&S.cnt[bin], 1u);
    atomicAdd(&S.mass[bin], m);
  }
}

__device__ __forceinline__ void hist_clear(Shared& S) {
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += kThreads) {
    S.cnt[i] = 0;
    S.mass[i] = 0;
  }
  __syncthreads();
}

// The bin (bin 0 holds the largest values) where the running count reaches `k`
// (by_count) or the running mass `m`: S.bin, with what lies before it in S.above,
// S.above_n.  The last bin that holds anything where it is never reached.
__device__ __forceinline__ void hist_find(Shared& S, bool by_count, unsigned long long k, double m, double fix) {
  constexpr int PER = kBins / kThreads;
  __syncthreads();
  unsigned long long c[PER], s[PER], cs = 0, ss = 0, all;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    c[j] = S.cnt[threadIdx.x * PER + j];
    s[j] = S.mass[threadIdx.x * PER + j];
    cs += c[j];
    ss += s[j];
  }
  unsigned long long nb = block_scan<unsigned long long>(cs, S.ured, &all) - cs;
  unsigned long long sb = block_scan<unsigned long long>(ss, S.ured, &all) - ss;
  int hit = kBins, last = -1;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const unsigned long long nn = nb + c[j], sn = sb + s[j];
    const bool reach = by_count ? nn >= k : (double)sn >= m * fix;
    if (c[j]) {
      if (reach && hit == kBins) hit = threadIdx.x * PER + j;
      last = threadIdx.x * PER + j;
    }
    nb = nn;
    sb = sn;
  }
  int bin = block_min(hit, S.ired);
  if (bin == kBins) bin = -block_min(-last, S.ired);
  if (bin / PER == (int)threadIdx.x) {
    // back to what lies before the bin
#pragma unroll
    for (int j = PER - 1; j >= 0; --j)
      if ((int)threadIdx.x * PER + j >= bin) {
        nb -= c[j];
        sb -= s[j];
      }
    S.bin = bin;
    S.above = sb;
    S.above_n = (int)nb;
  }
  __syncthreads();
}

// The bin of a value by its distance from the maximum; it never falls as x does.
__device__ __forceinline__ int dist_bin(float x, const Row& R) {
  if (!(x > kNegInf)) return -1;
  if (x == R.xmax) return 0;
  const float d = (R.xmax - x) * R.per_bin;
  return d < (float)(kBins - 1) ? (int)d : kBins - 1;
}

// For the groups of this wave that may hold something of bin `limit` or nearer, four
// at a time: f(group, its values).
template <typename F>
__device__ __forceinline__ void each_group(const Smp& P, const float* gmax, const Row& R, int limit, F f) {
  constexpr int U = 4;
  for (int g0 = (threadIdx.x >> 6) * U; g0 < P.ng; g0 += kWaves * U) {
    Lane8 v[U];
    bool on[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = g0 + u < P.ng ? dist_bin(gmax[g0 + u], R) : -1;
      on[u] = b >= 0 && b <= limit;
      if (on[u]) v[u] = load8(P, R.row, g0 + u);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (on[u]) f(g0 + u, v[u]);
  }
}

// The cut at the k-th value (by_count) or where the running weight, from the
// largest on, reaches m; *total: the weight of what is kept.  gs[g]: group g's kept
// weight of at least minw; *whole: whether that is all of it, or what the bin of the
// cut keeps is not in it yet.
__device__ Cut find_cut(const Smp& P, Shared& S, const float* gmax, double* gs, int* ec, const Row& R, int limit,
                        bool by_count, int k, double m, double minw, double* total, bool* whole) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  hist_clear(S);
  each_group(P, gmax, R, limit, [&](int, const Lane8& v) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      int bin = dist_bin(v.x[j], R);
      if (bin > limit) bin = -1;
      unsigned long long w = 0;
      if (bin >= 0 && !by_count) w = (unsigned long long)(weight(v.x[j], R.xmax, R.units, S.tab) * R.fix);
      hist_add(S, bin, w);
    }
  });
  hist_find(S, by_count, (unsigned long long)k, m, R.fix);
  const int bin = S.bin, members = (int)S.cnt[bin], above_n = S.above_n;
  // the groups' weight above the bin in 64 bits, and the bin's members: how many a group
  // has, their least and largest key, and themselves if they are few
  if (threadIdx.x == 0) S.count = 0;
  for (int g = threadIdx.x; g < P.ng; g += kThreads) {
    gs[g] = 0.0;
    ec[g] = 0;
  }
  __syncthreads();
  double sum = 0.0;
  uint32_t least = 0xffffffffu, most = 0u;
  each_group(P, gmax, R, bin, [&](int g, const Lane8& v) {
    double own = 0.0;
    int e = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int b = dist_bin(v.x[j], R);
      if (b >= 0 && b < bin) {
        const double w = weight(v.x[j], R.xmax, R.units, S.tab);
        sum += w;
        own += w >= minw ? w : 0.0;
      }
      if (b == bin) {
        const uint32_t key = key_of(v.x[j]);
        least = min(least, key);
        most = max(most, key);
        ++e;
        if (members <= kCand) S.cand[atomicAdd(&S.count, 1)] = (unsigned long long)~key << 32 | (uint32_t)v.at(j);
      }
    }
    own = wave_sum(own);
    e = gm_wave_sum(e);
    if (lane == 0) {
      gs[g] = own;
      ec[g] = e;
    }
  });
  double above;
  block_scan<double>(sum, S.dred, &above);
  least = ~(uint32_t)block_max_u(~least, S.ired);
  most = (uint32_t)block_max_u(most, S.ired);
  Cut c;
  *whole = false;
  if (least != most && members <= kCand) {
    __syncthreads();
    const unsigned long long mine = (int)threadIdx.x < members ? S.cand[threadIdx.x] : 0;
    const double w = (int)threadIdx.x < members ? weight(value_of(mine), R.xmax, R.units, S.tab) : 0.0;
    const int rank = rank_candidates(S, members, mine, w);
    double all;
    const double ws = (int)threadIdx.x < members ? S.w[threadIdx.x] : 0.0;
    const double run = block_scan<double>(ws, S.dred, &all);                 // thread r: rank r
    const bool in = (int)threadIdx.x < members &&
                    (by_count ? above_n + (int)threadIdx.x < k : threadIdx.x == 0 || above + (run - ws) < m);
    int n;
    block_scan<int>(in ? 1 : 0, S.ired, &n);
    if (n < 1) n = 1;
    if ((int)threadIdx.x == n - 1) S.w[0] = above + run;
    if ((int)threadIdx.x < members && rank == n - 1) S.cand[0] = mine;
    __syncthreads();
    c.key = ~(uint32_t)(S.cand[0] >> 32);
    c.id = (int)(uint32_t)S.cand[0];
    *total = S.w[0];
    __syncthreads();
    return c;
  }
  // many members, or equals: the keys' distance from the largest in digits of 11 bits
  // (none if all are one value; 16-bit logits leave the low bits of a key alone)
  const int low = P.a.type == GM_QTYPE_F32 ? 0 : P.a.type == GM_QTYPE_BF16 ? 16 : 13;
  const uint32_t span = (most - least) >> low;
  double over = above;                                  // weight above what is left
  int over_n = above_n, equal = members;
  uint32_t gap = 0, known = 0;                          // settled digits of the gap, and their mask
  for (int top = 32 - __clz(span | 1) - (span == 0); top > 0;) {
    const int bits = top < 11 ? top : 11, shift = top - bits;
    hist_clear(S);
    each_group(P, gmax, R, bin, [&](int, const Lane8& v) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t d = (most - key_of(v.x[j])) >> low;
        const bool on = dist_bin(v.x[j], R) == bin && (d & known) == gap;
        unsigned long long w = 0;
        if (on && !by_count) w = (unsigned long long)(weight(v.x[j], R.xmax, R.units, S.tab) * R.fix);
        hist_add(S, on ? (int)(d >> shift & ((1u << bits) - 1)) : -1, w);
      }
    });
    hist_find(S, by_count, by_count ? (unsigned long long)(k - over_n) : 0, m - over, R.fix);
    over_n += S.above_n;
    equal = (int)S.cnt[S.bin];
    gap |= (uint32_t)S.bin << shift;
    known |= ((1u << bits) - 1) << shift;
    top = shift;
    // the weight above in 64 bits: values of the settled digits nearer than this one
    double part = 0.0;
    const uint32_t g1 = gap, kn = known, sh = (uint32_t)shift;
    if (by_count) {
      // only wanted at the end, where it is formed from the cut itself
    } else {
      each_group(P, gmax, R, bin, [&](int, const Lane8& v) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t d = (most - key_of(v.x[j])) >> low;
          const uint32_t before = kn & ~(((1u << bits) - 1) << sh);
          if (dist_bin(v.x[j], R) == bin && (d & before) == (g1 & before) && (d & kn) < g1)
            part += weight(v.x[j], R.xmax, R.units, S.tab);
        }
      });
    }
    double more;
    block_scan<double>(part, S.dred, &more);
    over += more;
    __syncthreads();
  }
  c.key = most - (gap << low);
  if (by_count && span) {
    // the weight of the bin's values above the cut's
    double part = 0.0, more;
    each_group(P, gmax, R, bin, [&](int, const Lane8& v) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (dist_bin(v.x[j], R) == bin && key_of(v.x[j]) > c.key) part += weight(v.x[j], R.xmax, R.units, S.tab);
    });
    block_scan<double>(part, S.dred, &more);
    over += more;
  }
  const float x = value_of((unsigned long long)~c.key << 32);
  const double w1 = weight(x, R.xmax, R.units, S.tab);
  double need = by_count ? (double)(k - over_n) : w1 > 0.0 ? ceil((m - over) / w1) : (double)equal;
  need = fmin(fmax(need, 1.0), (double)equal);
  const int nth = (int)need;
  *total = over + need * w1;
  if (span) {
    // how many of exactly this value every group has
    __syncthreads();
    each_group(P, gmax, R, bin, [&](int g, const Lane8& v) {
      int e = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) e += v.x[j] > kNegInf && key_of(v.x[j]) == c.key ? 1 : 0;
      e = gm_wave_sum(e);
      if (lane == 0) ec[g] = e;
    });
    __syncthreads();
  }
  // the nth index that holds x: the groups in order, every thread some
  const int per = (P.ng + kThreads - 1) / kThreads, g0 = min((int)threadIdx.x * per, P.ng), g1 = min(g0 + per, P.ng);
  int own = 0, all;
  for (int g = g0; g < g1; ++g) own += ec[g];
  int run = block_scan<int>(own, S.ired, &all) - own;
  for (int g = g0; g < g1; ++g) {
    const int e = ec[g], in = min(max(nth - run, 0), e);
    if (e > 0 && in > 0 && run + e >= nth) {             // the group of the nth
      S.bin = g;
      S.above_n = nth - run;
    }
    if (w1 >= minw) gs[g] += (double)in * w1;
    run += e;
  }
  __syncthreads();
  *whole = span == 0;
  if (wave == 0) {
    const Lane8 v = load8(P, R.row, S.bin);
    // the group's equals in index order, one after the other
    int left = S.above_n, at = -1;
    uint32_t mine = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) mine |= (v.x[j] > kNegInf && key_of(v.x[j]) == c.key ? 1u : 0u) << j;
    while (left > 0) {
      int best = 0x7fffffff;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (mine >> j & 1) best = min(best, v.at(j));
      int first = best;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) first = min(first, __shfl_xor(first, o, 64));
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (v.at(j) == first) mine &= ~(1u << j);
      at = first;
      --left;
    }
    if (threadIdx.x == 0) S.count = at;
  }
  __syncthreads();
  c.id = S.count;
  __syncthreads();
  return c;
}

__global__ void __launch_bounds__(kThreads) k_sample_pick(Smp P) {
  extern __shared__ __attribute__((aligned(16))) char dyn[];
  Shared& S = *reinterpret_cast<Shared*>(dyn);
  double* gs = reinterpret_cast<double*>(dyn + sizeof(Shared));          // [ng]
  float* gmax = reinterpret_cast<float*>(gs + P.ng);                     // [ng]
  int* ec = reinterpret_cast<int*>(gmax + P.ng);                         // [ng]
  const gm_sample_args& A = P.a;
  const int row = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  exp_table(S.tab);
  const RowParam rp = row_param(A, row);
  float mx = kNegInf;
  for (int g = tid; g < P.ng; g += kThreads) {
    gmax[g] = P.gmax[(int64_t)row * P.ng + g];
    mx = fmaxf(mx, gmax[g]);
  }
  if (tid == 0) S.count = 0;
  Row R;
  R.row = row;
  R.xmax = block_max(mx, S.fred);
  const double inv = 1.0 / (double)rp.t;
  R.units = kUnits / (double)rp.t;
  R.per_bin = (float)(inv * (double)kBinsPerE);
  R.fix = ldexp(1.0, 62 - (32 - __clz(A.vocab)));
  if (R.xmax == kNegInf) {
    if (tid == 0) A.ids[row] = -1;
    return;
  }
  if (rp.greedy || rp.top_k == 1) {                     // the lowest index of the maximum
    int g = 0x7fffffff;
    for (int i = tid; i < P.ng; i += kThreads)
      if (gmax[i] == R.xmax) g = min(g, i);
    g = block_min(g, S.ired);
    if (wave == 0) {
      const Lane8 v = load8(P, row, g);
      int at = 0x7fffffff;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (v.x[j] == R.xmax) at = min(at, v.at(j));
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) at = min(at, __shfl_xor(at, o, 64));
      if (lane == 0) A.ids[row] = at;
    }
    return;
  }
  const bool by_p = rp.top_p < 1.f, by_k = rp.top_k > 0, by_min = rp.min_p > 0.f;
  const double minw = (double)rp.min_p;
  double all = 0.0;                                     // the weight of everything
  if (!by_k) {
    double s = 0.0;
    for (int g = tid; g < P.ng; g += kThreads) {
      const double v = gmax[g] == kNegInf ? 0.0 : P.gsum[(int64_t)row * P.ng + g] * weight(gmax[g], R.xmax, R.units, S.tab);
      gs[g] = v;
      s += v;
    }
    block_scan<double>(s, S.dred, &all);
  }
  const double u = (double)A.u[row];
  // ---- the farthest bin that may hold something kept, or counted by a filter before
  int limit = kBins - 1;
  const int nl = P.ng * 64;
  const int64_t l0 = (int64_t)row * nl;
  if (by_k || by_p) {
    hist_clear(S);
    constexpr int U = 4;
    for (int i0 = tid; i0 < nl; i0 += kThreads * U) {
      float x[U];
#pragma unroll
      for (int e = 0; e < U; ++e) {
        const int i = i0 + e * kThreads;
        x[e] = i < nl ? gm_elem(P.lmax, l0 + i, A.type) : kNegInf;
      }
#pragma unroll
      for (int e = 0; e < U; ++e) {
        const int bin = dist_bin(x[e], R);
        if (bin < 0) continue;
        if (by_k) {
          atomicAdd(&S.cnt[bin], 1u);
        } else {
          // a little less than it weighs
          const float w = x[e] == R.xmax ? 1.f : __builtin_amdgcn_exp2f((x[e] - R.xmax) * (float)inv * 1.44269504f) * 0.9999f;
          atomicAdd(&S.cnt[bin], 1u);
          atomicAdd(&S.mass[bin], (unsigned long long)(w * 0x1p40f));
        }
      }
    }
    const double want = (double)rp.top_p * all;
    hist_find(S, by_k, (unsigned long long)rp.top_k, want, 0x1p40);
    const bool reached = by_k ? S.above_n + (int)S.cnt[S.bin] >= rp.top_k
                              : (double)(S.above + S.mass[S.bin]) >= want * 0x1p40;
    if (reached) limit = S.bin;
    __syncthreads();
  }
  if (by_min && !(by_k && by_p)) {
    // one bin more than the threshold's: the test itself is the weight's
    const double d = -log((double)rp.min_p) * (double)kBinsPerE + 1.0;
    if (d < (double)limit) limit = (int)d;
  }
  // ---- few candidates: ranked in LDS
  if (limit < kBins - 1) {
    int* const list = reinterpret_cast<int*>(S.mass);                    // kList of them
    if (tid == 0) S.bin = 0;
    __syncthreads();
    constexpr int U = 4;
    for (int i0 = tid; i0 < nl; i0 += kThreads * U) {
      float x[U];
#pragma unroll
      for (int e = 0; e < U; ++e) {
        const int i = i0 + e * kThreads;
        x[e] = i < nl ? gm_elem(P.lmax, l0 + i, A.type) : kNegInf;
      }
#pragma unroll
      for (int e = 0; e < U; ++e) {
        const int bin = dist_bin(x[e], R);
        if (bin < 0 || bin > limit) continue;
        const int at = atomicAdd(&S.bin, 1);
        if (at < kList) list[at] = i0 + e * kThreads;
      }
    }
    __syncthreads();
    const int nlist = S.bin;
    if (nlist <= kList) {
      for (int i = tid; i < nlist; i += kThreads) {
        const Lane8 v = load8(P, row, list[i] >> 6, list[i] & 63);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int bin = dist_bin(v.x[j], R);
          if (bin < 0 || bin > limit) continue;
          const int at = atomicAdd(&S.count, 1);
          if (at < kCand) S.cand[at] = (unsigned long long)~key_of(v.x[j]) << 32 | (uint32_t)v.at(j);
        }
      }
    }
    __syncthreads();
    const int n = nlist <= kList ? S.count : kCand + 1;
    if (n <= kCand) {
      const unsigned long long mine = tid < n ? S.cand[tid] : 0;
      const double w = tid < n ? weight(value_of(mine), R.xmax, R.units, S.tab) : 0.0;
      rank_candidates(S, n, mine, w);
      // from here on thread r has the candidate of rank r
      const bool in_k = tid < n && (!by_k || tid < rp.top_k);
      const double ws = in_k ? S.w[tid] : 0.0;
      const int id = tid < n ? S.id[tid] : 0x7fffffff;
      double tk;
      const double run = block_scan<double>(ws, S.dred, &tk);
      if (!by_k) tk = all;
      bool in = in_k && ws > 0.0;
      if (by_p) in = in && (tid == 0 || run - ws < (double)rp.top_p * tk);
      if (by_min) in = in && (tid == 0 || ws >= minw);
      // the kept ones in the vocabulary's order
      int nk;
      block_scan<int>(in ? 1 : 0, S.ired, &nk);
      __syncthreads();
      if (tid < n) S.id[tid] = in ? id : 0x7fffffff;
      __syncthreads();
      if (in) {
        int place = 0;
        for (int j = 0; j < n; ++j) place += S.id[j] < id ? 1 : 0;
        S.w[place] = ws;
        S.cand[place] = (unsigned long long)id;
      }
      __syncthreads();
      double total;
      const double cum = block_scan<double>(tid < nk ? S.w[tid] : 0.0, S.dred, &total);
      int pick = tid < nk && cum > u * total ? tid : 0x7fffffff;
      pick = block_min(pick, S.ired);
      if (tid == 0) A.ids[row] = (int64_t)S.cand[pick < nk ? pick : nk - 1];
      return;
    }
  }
  // ---- many: the cut, then the kept weight of every group
  Cut c{0u, 0x7fffffff};
  bool whole = false;
  double tk;
  if (by_k) c = find_cut(P, S, gmax, gs, ec, R, limit, true, rp.top_k, 0.0, minw, &tk, &whole);
  if (by_p)
    c = find_cut(P, S, gmax, gs, ec, R, limit, false, 0, (double)rp.top_p * (by_k ? tk : all), minw, &tk, &whole);
  const bool cut = by_k || by_p;
  auto kept_w = [&](float x, int i) {
    if (!(x > kNegInf) || (cut && !kept(x, i, c))) return 0.0;
    const double w = weight(x, R.xmax, R.units, S.tab);
    return w >= minw ? w : 0.0;
  };
  if ((cut && !whole) || (!cut && by_min)) {
    for (int g = tid; g < P.ng; g += kThreads) gs[g] = 0.0;
    __syncthreads();
    each_group(P, gmax, R, limit, [&](int g, const Lane8& v) {
      if (cut && key_of(gmax[g]) < c.key) return;
      double s = 0.0;
#pragma unroll
      for (int j = 0; j < 8; ++j) s += kept_w(v.x[j], v.at(j));
      s = wave_sum(s);
      if (lane == 0) gs[g] = s;
    });
    __syncthreads();
  }
  // the group where the running weight passes u times the total
  const int per = (P.ng + kThreads - 1) / kThreads, gb = min(tid * per, P.ng), ge = min(gb + per, P.ng);
  double own = 0.0, total;
  for (int g = gb; g < ge; ++g) own += gs[g];
  const double run = block_scan<double>(own, S.dred, &total);
  const double want = u * total;
  int hit = 0x7fffffff, last = -1;
  double before = run - own, start = 0.0;
  for (int g = gb; g < ge; ++g) {
    const double next = before + gs[g];
    if (gs[g] > 0.0) {
      last = g;
      if (next > want && hit == 0x7fffffff) {
        hit = g;
        start = before;
      }
    }
    before = next;
  }
  const int first = block_min(hit, S.ired);
  const int g = first != 0x7fffffff ? first : -block_min(-last, S.ired);
  if (hit == first && first != 0x7fffffff) S.w[0] = start;
  __syncthreads();
  if (wave > 0) return;
  // within the group: the lanes' values in index order
  const Lane8 v = load8(P, row, g);
  double sum = first != 0x7fffffff ? S.w[0] : 0.0;
  int pick = 0x7fffffff, tail = -1;
  const int halves = A.type == GM_QTYPE_F32 ? 2 : 1, w8 = 8 / halves;
#pragma unroll
  for (int hf = 0; hf < 2; ++hf) {
    double mine = 0.0;                                   // hf past the type's halves adds nothing
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j / w8 == hf) mine += kept_w(v.x[j], v.at(j));
    double inc = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double up = __shfl_up(inc, o, 64);
      if (lane >= o) inc += up;
    }
    double at = sum + (inc - mine);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j / w8 == hf) {
        const double x = kept_w(v.x[j], v.at(j));
        at += x;
        if (x > 0.0) {
          tail = max(tail, v.at(j));
          if (at > want) pick = min(pick, v.at(j));
        }
      }
    sum += __shfl(inc, 63, 64);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    pick = min(pick, __shfl_xor(pick, o, 64));
    tail = max(tail, __shfl_xor(tail, o, 64));
  }
  // no running sum passed it (the order of rounding, or u = 1): the last kept one
  if (lane == 0) A.ids[row] = first != 0x7fffffff && pick != 0x7fffffff ? pick : tail;
}

int groups(const gm_sample_args* a) { return (a->vocab + kGroup - 1) / kGroup; }

}  // namespace

size_t gm_sample_ws(const gm_sample_args* a) {
  const size_t n = (size_t)a->n_row * groups(a);
  return align256(n * 8) + align256(n * 4) + align256(n * 64 * gm_elem_bytes(a->type));
}

int gm_sample_run(const gm_sample_args* a, uint8_t* ws, hipStream_t s) {
  Smp P{};
  P.a = *a;
  P.ng = groups(a);
  const size_t n = (size_t)a->n_row * P.ng;
  P.gsum = reinterpret_cast<double*>(ws);
  P.gmax = reinterpret_cast<float*>(ws + align256(n * 8));
  P.lmax = ws + align256(n * 8) + align256(n * 4);
  P.vec = gm_rows_aligned(a->logits, a->type, a->row_stride, 0);
  if (a->n_row >= 8) k_sample_groups<4><<<dim3((P.ng + 15) / 16, a->n_row), 256, 0, s>>>(P);
  else k_sample_groups<1><<<dim3((P.ng + 3) / 4, a->n_row), 256, 0, s>>>(P);
  GM_TRY(hipGetLastError());
  const size_t lds = sizeof(Shared) + (size_t)P.ng * 16;
  if (int rc = gm_set_smem(k_sample_pick, lds)) return rc;
  k_sample_pick<<<a->n_row, kThreads, lds, s>>>(P);
  GM_TRY(hipGetLastError());
  return GM_OK;
}
