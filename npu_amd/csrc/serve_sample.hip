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
//                   histogram over all values.  Its weights are fp32 in fixed point, with
//                   a bound on their error, so that it leaves an interval of bins (nearly
//                   always one) that holds the end of the filter; one pass in 64 bits sums
//                   what lies above, and only the interval's values are ranked (or cut
//                   digit by digit of their bits, if they too are many).
// Kept tokens run in the vocabulary's order, so nothing is ever sorted as a whole.
// No result depends on the order of atomics: they count, or add fixed-point values.
// Bound: HBM and, without top-k, the fp64 exponentials of the first kernel; for few
// rows the second kernel's chain of block-wide steps, for many flat rows its two passes.
//
// Measured, first and second kernel: one row of 248,320 fp32 with all filters 3 + 22 us;
// 64 rows of 248,320 fp32 with mixed filters 20 (3.2 TB/s) + 31 us; 256 rows of 248,320 bf16
// and their nuclei 67 us (1.9 TB/s, beside its 64 M exponentials) + 200.  The 200 are those of
// the few flat rows, each on one CU: 50 for the histogram, 80 for the pass in 64 bits, 50
// instructions a value in both; rows of up to kCand candidates are done after 20 to 60.
#include "kernels.h"
#include "serving.h"

namespace {

constexpr int kGroup = 512;         // logits of a group: 8 per lane of a wave
constexpr int kCand = 1024;         // candidates ranked in LDS, one per thread
constexpr int kBins = 4096;         // bins of the distance from the maximum ...
constexpr int kFine = 2048;         // ... these 1/128 wide in units of the temperature, the
constexpr float kBinsPerE = 128.f;  // others 1/8: the ranges end 16 and 272 away
constexpr int kList = 8192;         // lanes of 8 logits that are read again
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

// The least of unsigned values.
__device__ __forceinline__ uint32_t block_min_u(uint32_t v, int* red) {
  return (uint32_t)block_min((int)(v ^ 0x80000000u), red) ^ 0x80000000u;
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

// Floats as integers of the same order, without the bits that the logits' type does
// not have (low: 0 for fp32, 16 for bf16, 13 for fp16).
__device__ __forceinline__ uint32_t key_of(float x, int low) {
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u ? ~b : b | 0x80000000u) >> low;
}
__device__ __forceinline__ float value_of(uint32_t key, int low) {
  const uint32_t k = key << low;
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~(k | ((1u << low) - 1)));
}

struct Shared {
  double tab[64];
  double dred[kWaves];
  unsigned long long ured[kWaves];
  float fred[kWaves];
  int ired[kWaves];
  int count;
  int lo, hi;                           // of hist_find
  int group, nth, id_of;                // of the equals at a cut
  unsigned long long above;
  unsigned long long cand[kCand];       // descending value, then index: (~key << 32) | index
  double w[kCand];
  int id[kCand];
  unsigned long long mass[kBins];       // fixed point, or counts
};

static_assert(sizeof(Shared::mass) >= kList * sizeof(int));

// Where the filters end: kept are the values above `key`, and of that value the
// indices up to `id`.
struct Cut {
  uint32_t key;
  int id;
};
__device__ __forceinline__ bool kept(float x, int i, const Cut& c, int low) {
  const uint32_t k = key_of(x, low);
  return k > c.key || (k == c.key && i <= c.id);
}

struct Row {
  int row, low;
  float xmax;
  float per_bin;     // bins per unit of x
  float octaves;     // powers of two per unit of x
  double units;
};

// The candidate `mine` of thread tid < n among S.cand[0 .. n), ranked: its weight goes to
// S.w and its index to S.id at its rank.  Returns its rank.
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

// The last bin has no end, and a row may have most of its values there: it is not counted,
// but marked as one that reaches whatever is looked for.
constexpr unsigned long long kMark = 1ull << 62;

__device__ __forceinline__ void hist_clear(Shared& S) {
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kBins / kThreads; ++i) S.mass[threadIdx.x + i * kThreads] = 0;
  __syncthreads();
}

// S.lo, S.hi: the bins (bin 0 holds the largest values) where the running mass reaches
// tlo and thi, 0 < tlo <= thi; S.above: the mass before S.lo.  Where tlo is never reached
// S.lo is the last bin that holds anything, and where thi is not S.hi is kBins.
__device__ __forceinline__ void hist_find(Shared& S, unsigned long long tlo, unsigned long long thi) {
  constexpr int PER = kBins / kThreads;
  __syncthreads();
  unsigned long long c[PER], own = 0, all;
  int last = -1;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    c[j] = S.mass[threadIdx.x * PER + j];
    own += c[j];
    if (c[j]) last = threadIdx.x * PER + j;
  }
  if (threadIdx.x == 0) {
    S.lo = 0;
    S.hi = kBins;
    S.above = 0;
  }
  unsigned long long before = block_scan<unsigned long long>(own, S.ured, &all) - own;
  const int end = -block_min(-last, S.ired);            // two barriers behind the clear above
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int bin = threadIdx.x * PER + j;
    const unsigned long long after = before + c[j];
    if ((before < tlo && after >= tlo) || (all < tlo && bin == end)) {
      S.lo = bin;
      S.above = before;
    }
    if (before < thi && after >= thi) S.hi = bin;
    before = after;
  }
  __syncthreads();
}

// The bin of a value by its distance from the maximum; it never falls as x does.  Top-k
// with a low temperature ends far out: with all bins 1/128 wide, 64 rows with a 300th
// value 33 temperatures away took 750 us instead of 50.
__device__ __forceinline__ int dist_bin(float x, const Row& R) {
  const float d = (R.xmax - x) * R.per_bin;
  // the two slopes' lesser; NaN (an infinite maximum or reach) goes to the last bin
  const float b = fminf(fminf(d, fmaf(d, 1.f / 16, (float)kFine * (15.f / 16))), (float)(kBins - 1));
  const int bin = x == R.xmax ? 0 : (int)b;
  return x > kNegInf ? bin : -1;
}

// The least x whose bin is below `bin`, NaN for bin 0: two comparisons sort a value among
// the bins' ends instead of its bin.
__device__ __forceinline__ float bin_end(int bin, const Row& R) {
  uint32_t no = key_of(kNegInf, 0), yes = key_of(R.xmax, 0);
  while (yes - no > 1) {                                // 32 times at most
    const uint32_t mid = no + (yes - no) / 2;
    if (dist_bin(value_of(mid, 0), R) < bin) yes = mid;
    else no = mid;
  }
  return bin > 0 ? value_of(yes, 0) : __builtin_nanf("");
}

// The weight of x where dist_bin is not the last: no further than 272 temperatures.
__device__ __forceinline__ double near_weight(float x, const Row& R, const double* tab) {
  return fexp(x == R.xmax ? 0.0 : ((double)x - (double)R.xmax) * R.units, tab);
}

// A weight in fp32 as a multiple of 2^-32, rounded down.  The exponent's rounding is the
// largest of its errors: 2^-24 of up to 32 (smaller weights are 0), thrice, is 6e-6 of the
// weight.  kHigh and kLow below leave 3e-5 for it, and one unit per value for the rounding
// down.
__device__ __forceinline__ unsigned long long mass_of(float x, const Row& R) {
  const float w = x == R.xmax ? 1.f : __builtin_amdgcn_exp2f((x - R.xmax) * R.octaves);
  return (unsigned long long)__float2uint_rz(fmaxf(w, 0.f) * 4294967040.f);
}
constexpr double kHigh = 1.0 + 0x1p-15, kLow = 1.0 - 0x1p-15;

// f(index, maximum) for the lanes' maxima, 16 of a thread loaded together.
template <typename F>
__device__ __forceinline__ void each_max(const Smp& P, int row, F f) {
  constexpr int U = 4;
  const int n = P.ng * 16;                              // fours of them
  const int64_t l0 = (int64_t)row * P.ng * 64;
  for (int i0 = threadIdx.x; i0 < n; i0 += kThreads * U) {
    float x[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * kThreads;
      if (i < n) {
        gm_load<4>(P.lmax, l0 + (int64_t)i * 4, P.a.type, true, x[u]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[u][e] = kNegInf;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) f((i0 + u * kThreads) * 4 + e, x[u][e]);
  }
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

// The cut at the k-th value (by_count) or where the running weight, from the largest on,
// reaches m, among the values of bin `limit` or nearer; all of those where neither
// happens.  *total: the weight of what is kept.  gs[g]: group g's kept weight, of tokens
// of at least minw; ec[g] is scratch.  All threads of the block call it.
__device__ __forceinline__ Cut find_cut(const Smp& P, Shared& S, const float* gmax, double* gs, unsigned long long* ec,
                                        const Row& R, int limit, bool by_count, int k, double m, double minw,
                                        double* total) {
  const int tid = threadIdx.x, lane = tid & 63;
  hist_clear(S);
  bool far = false;
  each_group(P, gmax, R, limit, [&](int, const Lane8& v) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int bin = dist_bin(v.x[j], R);
      if (bin == kBins - 1) far = true;
      else if (bin >= 0 && bin <= limit) atomicAdd(&S.mass[bin], by_count ? 1ull : mass_of(v.x[j], R));
    }
  });
  if (far && limit == kBins - 1) S.mass[kBins - 1] = kMark;
  if (by_count) {
    hist_find(S, (unsigned long long)k, (unsigned long long)k);
  } else {
    const double lo = m * (0x1p32 / kHigh) - (double)P.a.vocab - 1.0, hi = m * (0x1p32 / kLow) + 1.0;
    hist_find(S, (unsigned long long)fmax(lo, 1.0), (unsigned long long)fmax(hi, 1.0));
  }
  const int lo = S.lo, hi = min(max(S.hi, lo), limit);
  const int above_n = by_count ? (int)S.above : 0;
  const float xa = bin_end(lo, R), xm = bin_end(hi + 1, R);      // above the interval x >= xa, with it x >= xm
  const bool by_min = minw > 0.0;
  // the weight above the interval in 64 bits, and its members: how many, their least and
  // largest key, and themselves if they are few
  if (tid == 0) S.count = 0;
  for (int g = tid; g < P.ng; g += kThreads) {
    gs[g] = 0.0;
    ec[g] = 0;
  }
  __syncthreads();
  double sum = 0.0;
  uint32_t least = 0xffffffffu, most = 0u;
  each_group(P, gmax, R, hi, [&](int g, const Lane8& v) {
    double own = 0.0;
    bool in = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      // no branch: the eight exponentials overlap
      const bool up = v.x[j] >= xa;
      const double e = near_weight(up ? v.x[j] : R.xmax, R, S.tab), w = up ? e : 0.0;
      if (by_min) sum += w;
      own += by_min && w < minw ? 0.0 : w;
      in |= v.x[j] >= xm && !up;
    }
    if (in) {
      const bool room = *static_cast<volatile int*>(&S.count) <= kCand;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (!(v.x[j] >= xm) || v.x[j] >= xa) continue;
        const uint32_t key = key_of(v.x[j], R.low);
        least = min(least, key);
        most = max(most, key);
        const int at = room ? atomicAdd(&S.count, 1) : kCand;      // past kCand their number has no use
        if (at < kCand) S.cand[at] = (unsigned long long)~key << 32 | (uint32_t)v.at(j);
      }
    }
    if (!by_min) sum += own;
    own = wave_sum(own);
    if (lane == 0) gs[g] = own;
  });
  double above;
  block_scan<double>(sum, S.dred, &above);
  least = block_min_u(least, S.ired);
  most = ~block_min_u(~most, S.ired);
  const int members = S.count;
  Cut c;
  if (members <= kCand) {
    const unsigned long long mine = tid < members ? S.cand[tid] : 0;
    const double w = tid < members ? weight(value_of(~(uint32_t)(mine >> 32), R.low), R.xmax, R.units, S.tab) : 0.0;
    const int rank = rank_candidates(S, members, mine, w);
    // from here on thread r has the candidate of rank r
    double all;
    const double ws = tid < members ? S.w[tid] : 0.0;
    const double run = block_scan<double>(ws, S.dred, &all);
    const bool in = tid < members && (by_count ? above_n + tid < k : tid == 0 || above + (run - ws) < m);
    int n;
    block_scan<int>(in ? 1 : 0, S.ired, &n);
    if (n < 1) n = 1;
    // a group's kept members in multiples of 2^-54 of the largest weight: 512 of them fit
    if (tid < n && tid < members && ws >= minw)
      atomicAdd(&ec[S.id[tid] / kGroup], (unsigned long long)__double2ull_rz(ws * 0x1p54));
    __syncthreads();
    if (tid == n - 1) S.w[0] = above + run;
    if (tid < members && rank == n - 1) S.cand[0] = mine;
    for (int g = tid; g < P.ng; g += kThreads) gs[g] += (double)ec[g] * 0x1p-54;
    __syncthreads();
    c.key = ~(uint32_t)(S.cand[0] >> 32);
    c.id = (int)(uint32_t)S.cand[0];
    *total = S.w[0];
    __syncthreads();
    return c;
  }
  // many members: their keys' distance from the largest in digits of 12 bits, 3 of them
  // at most (none if all are one value)
  const uint32_t span = most - least;
  const double top_w = weight(value_of(most, R.low), R.xmax, R.units, S.tab);
  // fixed point for the members' weights: top_w below 2^(62 - the vocabulary's bits)
  const int up = 62 - (32 - __clz(P.a.vocab)) - (top_w > 0.0 ? ilogb(top_w) + 1 : 0);
  const double fix = ldexp(1.0, up);
  unsigned long long left = by_count ? (unsigned long long)max(k - above_n, 1)
                                     : (unsigned long long)fmin(fmax((m - above) * fix, 1.0), 0x1p62);
  uint32_t gap = 0, known = 0;                          // settled digits of the distance, and their mask
  int top = span ? 32 - __clz(span) : 0;
  for (int digit = 0; digit < 3; ++digit) {
    if (top == 0) break;
    const int bits = min(top, 12), shift = top - bits;
    const uint32_t mask = (1u << bits) - 1;
    hist_clear(S);
    each_group(P, gmax, R, hi, [&](int, const Lane8& v) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (!(v.x[j] >= xm) || v.x[j] >= xa) continue;
        const uint32_t d = most - key_of(v.x[j], R.low);
        if ((d & known) != gap) continue;
        const unsigned long long one =
            by_count ? 1ull : __double2ull_rz(weight(v.x[j], R.xmax, R.units, S.tab) * fix);
        atomicAdd(&S.mass[d >> shift & mask], one);
      }
    });
    hist_find(S, left, left);
    left = left > S.above ? left - S.above : 1;
    gap |= (uint32_t)S.lo << shift;
    known |= mask << shift;
    top = shift;
    __syncthreads();
  }
  c.key = most - gap;
  // the members above the cut's value in 64 bits, and how many every group has of it
  double part = 0.0, more;
  int near = 0, near_all;
  each_group(P, gmax, R, hi, [&](int g, const Lane8& v) {
    double own = 0.0;
    int e = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (!(v.x[j] >= xm) || v.x[j] >= xa) continue;
      const uint32_t key = key_of(v.x[j], R.low);
      if (key > c.key) {
        const double w = weight(v.x[j], R.xmax, R.units, S.tab);
        part += w;
        own += w >= minw ? w : 0.0;
        ++near;
      }
      e += key == c.key ? 1 : 0;
    }
    own = wave_sum(own);
    e = gm_wave_sum(e);
    if (lane == 0) {
      gs[g] += own;
      ec[g] = (unsigned long long)e;
    }
  });
  block_scan<double>(part, S.dred, &more);
  block_scan<int>(near, S.ired, &near_all);
  // the nth index that holds the cut's value: the groups in order, every thread some
  const int per = (P.ng + kThreads - 1) / kThreads, g0 = min(tid * per, P.ng), g1 = min(g0 + per, P.ng);
  int own = 0, equal;
  for (int g = g0; g < g1; ++g) own += (int)ec[g];
  int run = block_scan<int>(own, S.ired, &equal) - own;
  const double w1 = weight(value_of(c.key, R.low), R.xmax, R.units, S.tab);
  const double over = above + more;
  const double need = by_count ? (double)(k - above_n - near_all) : w1 > 0.0 ? ceil((m - over) / w1) : (double)equal;
  const int nth = max((int)fmin(need, (double)equal), 1);
  *total = over + (double)nth * w1;
  if (tid == 0) {
    S.group = 0;
    S.nth = 0;
    S.id_of = 0x7fffffff;
  }
  __syncthreads();
  for (int g = g0; g < g1; ++g) {
    const int e = (int)ec[g], in = min(max(nth - run, 0), e);
    if (in > 0 && run + e >= nth) {                      // the group of the nth
      S.group = g;
      S.nth = in;
    }
    if (w1 >= minw) gs[g] += (double)in * w1;
    run += e;
  }
  __syncthreads();
  if (tid < 64) {
    const Lane8 v = load8(P, R.row, S.group);
    const int want = S.nth, w8 = P.a.type == GM_QTYPE_F32 ? 4 : 8;
    int before = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {                        // index order: lanes, then their fours of fp32's second half
      int mine = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) mine += j / w8 == h && v.x[j] > kNegInf && key_of(v.x[j], R.low) == c.key ? 1 : 0;
      int inc = mine;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int other = __shfl_up(inc, o, 64);
        if (lane >= o) inc += other;
      }
      int at = before + inc - mine;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j / w8 == h && v.x[j] > kNegInf && key_of(v.x[j], R.low) == c.key && ++at == want) S.id_of = v.at(j);
      before += __shfl(inc, 63, 64);
    }
  }
  __syncthreads();
  c.id = S.id_of;
  __syncthreads();
  return c;
}

__global__ void __launch_bounds__(kThreads) k_sample_pick(Smp P) {
  extern __shared__ __attribute__((aligned(16))) char dyn[];
  Shared& S = *reinterpret_cast<Shared*>(dyn);
  double* gs = reinterpret_cast<double*>(dyn + sizeof(Shared));                 // [ng]
  unsigned long long* ec = reinterpret_cast<unsigned long long*>(gs + P.ng);    // [ng]
  float* gmax = reinterpret_cast<float*>(ec + P.ng);                            // [ng]
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
  R.low = A.type == GM_QTYPE_F32 ? 0 : A.type == GM_QTYPE_BF16 ? 16 : 13;
  R.xmax = block_max(mx, S.fred);
  const double inv = 1.0 / (double)rp.t;
  R.units = kUnits / (double)rp.t;
  R.per_bin = (float)(inv * (double)kBinsPerE);
  R.octaves = (float)(inv * 1.4426950408889634);
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
  if (by_k || by_p) {
    hist_clear(S);
    each_max(P, row, [&](int, float x) {
      const int bin = dist_bin(x, R);
      if (bin >= 0 && bin < kBins - 1) atomicAdd(&S.mass[bin], by_k ? 1ull : mass_of(x, R));
    });
    const unsigned long long want =
        by_k ? (unsigned long long)rp.top_k : (unsigned long long)((double)rp.top_p * all * (0x1p32 / kLow)) + 1;
    hist_find(S, want, want);
    limit = min(limit, S.hi);
    __syncthreads();
  }
  if (by_min && !(by_k && by_p)) {
    // one bin more than the threshold's: the test itself is the weight's
    const double d = -log((double)rp.min_p) * (double)kBinsPerE;
    const double b = (d < kFine ? d : kFine + (d - kFine) * (1.0 / 16)) + 1.0;
    if (b < (double)limit) limit = (int)b;
  }
  // ---- few candidates: ranked in LDS
  if (limit < kBins - 1) {
    int* const list = reinterpret_cast<int*>(S.mass);                    // kList of them
    if (tid == 0) S.lo = 0;
    __syncthreads();
    each_max(P, row, [&](int i, float x) {
      const int bin = dist_bin(x, R);
      if (bin < 0 || bin > limit) return;
      const int at = atomicAdd(&S.lo, 1);
      if (at < kList) list[at] = i;
    });
    __syncthreads();
    const int nlist = S.lo;
    if (nlist <= kList) {
      for (int i = tid; i < nlist; i += kThreads) {
        const Lane8 v = load8(P, row, list[i] >> 6, list[i] & 63);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int bin = dist_bin(v.x[j], R);
          if (bin < 0 || bin > limit) continue;
          const int at = atomicAdd(&S.count, 1);
          if (at < kCand) S.cand[at] = (unsigned long long)~key_of(v.x[j], R.low) << 32 | (uint32_t)v.at(j);
        }
      }
    }
    __syncthreads();
    const int n = nlist <= kList ? S.count : kCand + 1;
    if (n <= kCand) {
      const unsigned long long mine = tid < n ? S.cand[tid] : 0;
      const double w = tid < n ? weight(value_of(~(uint32_t)(mine >> 32), R.low), R.xmax, R.units, S.tab) : 0.0;
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
  const bool cut = by_k || by_p;
  double tk = all;
#pragma nounroll
  for (int f = by_k ? 0 : 1; f < (by_p ? 2 : 1); ++f)      // the k largest, then their nucleus
    c = find_cut(P, S, gmax, gs, ec, R, limit, f == 0, rp.top_k, (double)rp.top_p * tk, minw, &tk);
  auto kept_w = [&](float x, int i) {
    if (!(x > kNegInf) || (cut && !kept(x, i, c, R.low))) return 0.0;
    const double w = weight(x, R.xmax, R.units, S.tab);
    return w >= minw ? w : 0.0;
  };
  if (!cut && by_min) {
    for (int g = tid; g < P.ng; g += kThreads) gs[g] = 0.0;
    __syncthreads();
    each_group(P, gmax, R, limit, [&](int g, const Lane8& v) {
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
  // a kept weight is somewhere: the maximum's is 1
  const int g = first != 0x7fffffff ? first : max(-block_min(-last, S.ired), 0);
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
  const size_t lds = sizeof(Shared) + (size_t)P.ng * 20;
  // one limit for every vocabulary: two threads' calls must not lower it for each other
  constexpr size_t most = sizeof(Shared) + ((1 << 21) / kGroup) * 20;
  static_assert(most <= 160 * 1024);
  if (lds > 65536)
    if (int rc = gm_set_smem(k_sample_pick, most)) return rc;
  k_sample_pick<<<a->n_row, kThreads, lds, s>>>(P);
  GM_TRY(hipGetLastError());
  return GM_OK;
}
