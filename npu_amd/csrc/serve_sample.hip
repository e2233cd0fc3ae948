// One token per row of logits (gm_sample): temperature, top-k, top-p, min-p and
// the inverse of the kept weights' running sum at u.
//
// The pick is that of the definition in 64 bits: weights w = e^((x - max) / t) and
// all their sums are fp64, so that u times the total falls between the same two
// running sums.  fp64 FMAs run at the fp32 rate here; the exponential is a table of
// 64 powers in LDS and five terms (14 instructions instead of the library's 40).
//
// k_sample_groups   every group of 512 logits: its maximum and, for rows without a
//                   top-k, its sum of weights.  The one pass over all logits.
// k_sample_pick     one block per row.  Whatever passes the filters is at least the
//                   k-th largest group maximum (k groups hold such a value each) or
//                   what min-p leaves, so few groups are read again; up to kCand
//                   candidates are ranked against each other in LDS.  More than that
//                   (a nucleus without top-k, a large k): a histogram of the distance
//                   from the maximum finds the bin where the filter ends, and only
//                   that bin's values are ranked (or cut bit by bit, if they too are
//                   many).
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
constexpr float kNegInf = -__builtin_inff();
constexpr float kPosInf = __builtin_inff();

size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

struct Smp {
  gm_sample_args a;
  float* gmax;       // [n_row][ng]
  double* gsum;      // [n_row][ng]
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

// e^y for y <= 0 within 2e-16: y = k ln2 / 64 + z, |z| < 0.0055, the powers of
// 2^(1/64) from the table.
__device__ __forceinline__ double fexp(double y, const double* tab) {
  y = fmax(y, -800.0);                                 // 0 below -745
  const double k = rint(y * 92.332482616893656877);    // 64 / ln 2
  double z = fma(k, -0x1.62e42fefa39efp-7, y);         // ln 2 / 64, its leading bits and the rest
  z = fma(k, -0x1.abc9e3b39803fp-62, z);
  double p = fma(z, 1.0 / 120, 1.0 / 24);
  p = fma(z, p, 1.0 / 6);
  p = fma(z, p, 0.5);
  p = fma(z, p, 1.0);
  const int ki = (int)k;
  const double s = tab[ki & 63];
  return ldexp(fma(s, z * p, s), ki >> 6);
}

// The weight of x beside the maximum m (inv = 1 / t).
__device__ __forceinline__ double weight(float x, float m, double inv, const double* tab) {
  if (!(x > kNegInf)) return 0.0;                      // NaN, -inf
  if (x == m) return 1.0;
  if (m == kPosInf) return 0.0;
  return fexp(((double)x - (double)m) * inv, tab);
}

// The 8 logits of a lane in group gr; index of the j-th: at(j).  Past the end -inf.
struct Lane8 {
  float x[8];
  int i0, step;
  __device__ __forceinline__ int at(int j) const { return i0 + (j & 3) + (j >> 2) * step; }
};
__device__ __forceinline__ Lane8 load8(const Smp& P, int row, int gr) {
  const gm_sample_args& A = P.a;
  const int lane = threadIdx.x & 63, V = A.vocab;
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

__global__ void __launch_bounds__(256) k_sample_groups(Smp P) {
  __shared__ double tab[64];
  exp_table(tab);
  __syncthreads();
  const int row = blockIdx.y, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const RowParam rp = row_param(P.a, row);
  const bool sums = !rp.greedy && rp.top_k == 0;
  const double inv = 1.0 / (double)rp.t;
  constexpr int U = 4;                                 // groups of a wave, loaded together
  const int g0 = (blockIdx.x * 4 + wave) * U;
  Lane8 v[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (g0 + u < P.ng) v[u] = load8(P, row, g0 + u);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (g0 + u >= P.ng) break;
    float m = v[u].x[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) m = fmaxf(m, v[u].x[j]);
    m = wave_max(m);
    double s = 0.0;
    if (sums && m > kNegInf) {
#pragma unroll
      for (int j = 0; j < 8; ++j) s += weight(v[u].x[j], m, inv, tab);
      s = wave_sum(s);
    }
    if (lane == 0) {
      P.gmax[(int64_t)row * P.ng + g0 + u] = m;
      P.gsum[(int64_t)row * P.ng + g0 + u] = s;
    }
  }
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
  double inv;
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

__device__ __forceinline__ int dist_bin(float x, const Row& R) {
  if (!(x > kNegInf)) return -1;
  if (x == R.xmax) return 0;
  if (R.xmax == kPosInf) return kBins - 1;
  const double d = ((double)R.xmax - (double)x) * R.inv * (double)kBinsPerE;
  return d < (double)(kBins - 1) ? (int)d : kBins - 1;
}

// The cut at the k-th value (by_count) or where the running weight, from the
// largest on, reaches m; *total: the weight of what is kept.
__device__ Cut find_cut(const Smp& P, Shared& S, const float* gmax, const Row& R, bool by_count, int k, double m,
                        double* total) {
  const int wave = threadIdx.x >> 6;
  hist_clear(S);
  for (int gr = wave; gr < P.ng; gr += kWaves) {
    const Lane8 v = load8(P, R.row, gr);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int bin = dist_bin(v.x[j], R);
      hist_add(S, bin, bin < 0 ? 0 : (unsigned long long)(weight(v.x[j], R.xmax, R.inv, S.tab) * R.fix));
    }
  }
  hist_find(S, by_count, (unsigned long long)k, m, R.fix);
  const int bin = S.bin, members = (int)S.cnt[bin];
  int above_n = S.above_n;
  // the weight above the bin in 64 bits, and the bin's members if they are few
  if (threadIdx.x == 0) S.count = 0;
  __syncthreads();
  double sum = 0.0;
  for (int gr = wave; gr < P.ng; gr += kWaves) {
    const Lane8 v = load8(P, R.row, gr);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int b = dist_bin(v.x[j], R);
      if (b >= 0 && b < bin) sum += weight(v.x[j], R.xmax, R.inv, S.tab);
      if (b == bin && members <= kCand)
        S.cand[atomicAdd(&S.count, 1)] = (unsigned long long)~key_of(v.x[j]) << 32 | (uint32_t)v.at(j);
    }
  }
  double above;
  block_scan<double>(sum, S.dred, &above);
  Cut c;
  if (members <= kCand) {
    __syncthreads();
    const unsigned long long mine = (int)threadIdx.x < members ? S.cand[threadIdx.x] : 0;
    const double w = (int)threadIdx.x < members ? weight(value_of(mine), R.xmax, R.inv, S.tab) : 0.0;
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
  // many members: 11, 11 and 10 bits of the key, then the index among equals
  uint32_t prefix = 0;
  int shift = 21, bits = 11;
  uint32_t known = 0;                                   // mask of the bits that are settled
  double over = above;                                  // weight above what is left
  int over_n = above_n;
  for (int pass = 0; pass < 3; ++pass) {
    hist_clear(S);
    for (int gr = wave; gr < P.ng; gr += kWaves) {
      const Lane8 v = load8(P, R.row, gr);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t key = key_of(v.x[j]);
        const bool on = dist_bin(v.x[j], R) == bin && (key & known) == prefix;
        const int digit = (int)(~key >> shift & ((1u << bits) - 1));     // 0: the largest
        hist_add(S, on ? digit : -1,
                 on ? (unsigned long long)(weight(v.x[j], R.xmax, R.inv, S.tab) * R.fix) : 0);
      }
    }
    hist_find(S, by_count, by_count ? (unsigned long long)(k - over_n) : 0, m - over, R.fix);
    const uint32_t digit = (uint32_t)S.bin;
    over += (double)S.above / R.fix;
    over_n += S.above_n;
    prefix |= (~digit & ((1u << bits) - 1)) << shift;
    known |= ((1u << bits) - 1) << shift;
    if (pass < 2) {
      bits = pass == 0 ? 11 : 10;
      shift -= bits;
    }
    __syncthreads();
  }
  const int equal = (int)S.cnt[S.bin];
  const float x = __uint_as_float(prefix & 0x80000000u ? prefix & 0x7fffffffu : ~prefix);
  const double w1 = weight(x, R.xmax, R.inv, S.tab);
  double need = by_count ? (double)(k - over_n) : w1 > 0.0 ? ceil((m - over) / w1) : (double)equal;
  need = fmin(fmax(need, 1.0), (double)equal);
  const int nth = (int)need;
  *total = over + need * w1;
  // the nth index that holds x: groups in order, 1024 at a time
  c.key = prefix;
  c.id = -1;
  int seen = 0;
  for (int g0 = 0; g0 < P.ng && c.id < 0; g0 += kThreads) {
    __syncthreads();
    for (int gr = g0 + wave; gr < min(g0 + kThreads, P.ng); gr += kWaves) {
      const Lane8 v = load8(P, R.row, gr);
      int e = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) e += v.x[j] > kNegInf && key_of(v.x[j]) == prefix ? 1 : 0;
      e = gm_wave_sum(e);
      if ((threadIdx.x & 63) == 0) S.id[gr - g0] = e;
    }
    __syncthreads();
    const int own = g0 + (int)threadIdx.x < P.ng ? S.id[threadIdx.x] : 0;
    int all;
    const int run = block_scan<int>(own, S.ired, &all) + seen;
    if (run >= nth && run - own < nth) {
      S.bin = g0 + (int)threadIdx.x;
      S.above_n = nth - (run - own);
    }
    __syncthreads();
    if (seen + all >= nth) {
      if (wave == 0) {
        const Lane8 v = load8(P, R.row, S.bin);
        // the group's equals in index order: as many passes as the value has places
        int left = S.above_n, at = -1;
        uint32_t mine = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) mine |= (v.x[j] > kNegInf && key_of(v.x[j]) == prefix ? 1u : 0u) << j;
        while (left > 0) {
          int best = 0x7fffffff;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (mine >> j & 1) best = min(best, v.at(j));
          int low = best;
#pragma unroll
          for (int o = 32; o > 0; o >>= 1) low = min(low, __shfl_xor(low, o, 64));
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (v.at(j) == low) mine &= ~(1u << j);
          at = low;
          --left;
        }
        if (threadIdx.x == 0) S.count = at;
      }
      __syncthreads();
      c.id = S.count;
    }
    seen += all;
  }
  __syncthreads();
  return c;
}

__global__ void __launch_bounds__(kThreads) k_sample_pick(Smp P) {
  extern __shared__ __attribute__((aligned(16))) char dyn[];
  Shared& S = *reinterpret_cast<Shared*>(dyn);
  double* gs = reinterpret_cast<double*>(dyn + sizeof(Shared));          // [ng]
  float* gmax = reinterpret_cast<float*>(gs + P.ng);                     // [ng]
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
  R.inv = 1.0 / (double)rp.t;
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
  // ---- the least value that may be kept or counted
  float bound = kNegInf;
  if (by_k && rp.top_k <= P.ng) {
    int hit = -1;
    for (int i = tid; i < P.ng; i += kThreads) {        // the k-th largest group maximum
      int above = 0;
      const float own = gmax[i];
      for (int j = 0; j < P.ng; ++j) above += gmax[j] > own || (gmax[j] == own && j < i) ? 1 : 0;
      if (above == rp.top_k - 1) hit = i;
    }
    hit = -block_min(-hit, S.ired);
    bound = gmax[hit];
  }
  if (by_min && !(by_k && by_p)) {
    // what is a little below stays in: the test itself is the weight's
    const double low = (double)R.xmax + (double)rp.t * (log((double)rp.min_p) * 1.000001 - 1e-6);
    const float lf = (float)low;
    bound = fmaxf(bound, lf - fabsf(lf) * 1e-6f);
  }
  const double minw = (double)rp.min_p;
  double all = 0.0;                                     // the weight of everything
  if (!by_k) {
    double s = 0.0;
    for (int g = tid; g < P.ng; g += kThreads) {
      const double v = gmax[g] == kNegInf ? 0.0 : P.gsum[(int64_t)row * P.ng + g] * weight(gmax[g], R.xmax, R.inv, S.tab);
      gs[g] = v;
      s += v;
    }
    block_scan<double>(s, S.dred, &all);
  }
  const double u = (double)A.u[row];
  // ---- few candidates: ranked in LDS
  if (bound > kNegInf) {
    for (int g = wave; g < P.ng; g += kWaves) {
      if (!(gmax[g] >= bound)) continue;
      const Lane8 v = load8(P, row, g);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (v.x[j] >= bound && v.x[j] > kNegInf) {
          const int at = atomicAdd(&S.count, 1);
          if (at < kCand) S.cand[at] = (unsigned long long)~key_of(v.x[j]) << 32 | (uint32_t)v.at(j);
        }
    }
    __syncthreads();
    const int n = S.count;
    if (n <= kCand) {
      const unsigned long long mine = tid < n ? S.cand[tid] : 0;
      const double w = tid < n ? weight(value_of(mine), R.xmax, R.inv, S.tab) : 0.0;
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
  if (by_k) {
    double tk;
    c = find_cut(P, S, gmax, R, true, rp.top_k, 0.0, &tk);
    if (by_p) {
      double none;
      c = find_cut(P, S, gmax, R, false, 0, (double)rp.top_p * tk, &none);
    }
  } else if (by_p) {
    double none;
    c = find_cut(P, S, gmax, R, false, 0, (double)rp.top_p * all, &none);
  }
  const bool cut = by_k || by_p;
  auto kept_w = [&](float x, int i) {
    if (!(x > kNegInf) || (cut && !kept(x, i, c))) return 0.0;
    const double w = weight(x, R.xmax, R.inv, S.tab);
    return w >= minw ? w : 0.0;
  };
  if (cut || by_min) {
    for (int g = wave; g < P.ng; g += kWaves) {
      double s = 0.0;
      if (gmax[g] > kNegInf && (!cut || key_of(gmax[g]) >= c.key)) {
        const Lane8 v = load8(P, row, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) s += kept_w(v.x[j], v.at(j));
        s = wave_sum(s);
      }
      if (lane == 0) gs[g] = s;
    }
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
  return align256(n * 8) + align256(n * 4);
}

int gm_sample_run(const gm_sample_args* a, uint8_t* ws, hipStream_t s) {
  Smp P{};
  P.a = *a;
  P.ng = groups(a);
  P.gsum = reinterpret_cast<double*>(ws);
  P.gmax = reinterpret_cast<float*>(ws + align256((size_t)a->n_row * P.ng * 8));
  P.vec = gm_rows_aligned(a->logits, a->type, a->row_stride, 0);
  k_sample_groups<<<dim3((P.ng + 15) / 16, a->n_row), 256, 0, s>>>(P);
  GM_TRY(hipGetLastError());
  const size_t lds = sizeof(Shared) + (size_t)P.ng * 12;
  if (int rc = gm_set_smem(k_sample_pick, lds)) return rc;
  k_sample_pick<<<a->n_row, kThreads, lds, s>>>(P);
  GM_TRY(hipGetLastError());
  return GM_OK;
}
