// sample.cu - the next token of each request from its logits and one given random number.
//
//   w_i = exp((x_i - max x) / T);  order: larger x first, of equal ones the lower index first
//   top-k: the first k of the order;  top-p: of those the shortest prefix with >= p of their sum;
//   min-p: of those the ones with w_i >= min_p;  token = first index i with
//   sum_{kept j <= i} w_j > u * sum_{kept j} w_j.   T <= 0: the first of the order.
//
// No sort: the kept set is a prefix of the order, so it is given by one value and, among the
// logits that equal it, an index. A cluster of CTAs has a row, each a contiguous slice; slices
// are joined through distributed shared memory, every CTA computing the same decisions, and a
// pass over the row ends with one cluster barrier.
//
// * Common path: with top-k or top-p, a histogram of the row over the distance (max - x) / T
//   gives the bins that the prefix ends in: by count exactly, by mass nearly (count and mean
//   place in the bin are kept, the mass follows). Logits in front of them only add their
//   weights to a warp's sum; the members go to a list per warp in index order. A second
//   histogram, of the lists alone with exact masses, leaves a few that are ranked against each
//   other directly. The sums say which warp holds the token; all warps of that CTA sum a
//   part of its share, and the one that holds it looks for the index. Four passes over the
//   slice, the first from HBM, the others from L1 or L2.
//
// * General path, for rows that do not fit that (too many near logits or equal ones, cuts deep in
//   the tail, larger vocabularies): histograms of the whole row, first linear in the distance,
//   then in the bits of the values of the bin the prefix ends in, until one value is left; the
//   draw walks 512-byte segments in index order. Each pass reads the slice again (L1 / L2).
//
// What bounds it. Many rows: dependent instructions (~120 a logit, all passes together; half of the
// issue slots taken by 24 warps on an SM) and the barriers between passes. 256 rows of 128,000 fp32,
// top-p: 265 us, 131 MB from HBM once, 0.49 TB/s, where a read alone takes 20 us. Few rows: a chain of
// ~30 barriers and the latency of each pass (one row of 128,000: 24 us). The general path: 190 us for
// one row of 300,001 with top-p, 199 for 8 of 262,208 with top-k and top-p. Measured and not kept: the
// slice in registers over all passes (unrolled, it misses the instruction cache: slower by half),
// 8-wide fp32 groups (8 % slower), a larger share of shared memory (no change).
//
// Rounding. The answer is an index, and a cut that falls on another side of a sum changes it,
// so weights and sums are wider than 32-bit floats: common path, 30-bit weights (Exp2Table) as
// 64-bit integers, whose order of addition does not matter, cut off to units of 2^-45 of the largest (2^-43
// for 2^18 logits) and dropped below 2^-46 of it: a sum is right to 2^-28 of itself and a unit for
// each logit. General path, weights by 64-bit exp() (2^-46 of each: its argument is rounded too),
// summed in doubles in a fixed order, or for a cut as integers of 2^-61 of the row's sum and less.
#include <climits>
#include <cmath>
#include <cooperative_groups.h>

#include "common.cuh"
#include "dbk_internal.h"

namespace cg = cooperative_groups;

namespace dbk {
namespace {

// Threads of a CTA. Many rows (256 x 128,000 fp32: 265 us): small CTAs, three on an SM, whose phases
// hide each other's barriers (80 registers a thread, 16 to 104 bytes of them spilled; four have 64
// and spill 88 to 428: 273 us; five: 293). At most one CTA per SM: larger ones, for a slice's passes are
// chains of dependent instructions (one row of 128,000: 24 us with 512 threads; two to an SM, with
// 64 registers: 27).
constexpr int kManyThreads = 256, kManyCtas = 3, kFewThreads = 512, kMaxWarps = 32;
constexpr int kBins = 256;
constexpr float kFine = 14.f;       // log2 distances of the general path's first histogram
constexpr float kFar = 46.f;        // and of its second; past it weights are nothing to the common path
constexpr int kMaxCluster = 8;
constexpr int kMaxVocab = 1 << 20;
constexpr int kMaxSlice = 32768;    // logits of a CTA, at most (with 256 threads 32 rounds of a warp)
constexpr unsigned long long kNone = ~0ull;

struct SampleArgs {
  const void* logits;
  const float* u;
  const float* temperature;   // [batch] or nullptr (temp for all)
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int64_t* out;
  float temp, p, mp;
  int k;
  int batch, vocab, cluster, iters;
  double unit;                // fixed-point units of a weight of 1: 2^(45 - lower_bits)
  int lower_bits;
};

struct Hist {
  unsigned long long mass[kBins];
  unsigned int count[kBins];
};

struct SampleShared {
  Hist hist[2];                       // alternate between passes: one cluster barrier each
  double sum[2];
  unsigned long long far[2], idx[2];
  float top[2];
  double warp_d[kMaxWarps];
  unsigned long long warp_m[kMaxWarps];
  unsigned int warp_c[kMaxWarps];
  unsigned long long cum_mass[kBins];
  unsigned int cum_count[kBins];
  int found;
  double found_base;
};

__device__ __forceinline__ unsigned int order_key(float x) {   // ascending with x; +0 = -0
  const unsigned int b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int n = 4;
  static constexpr uint32_t kNegInf = 0xff800000u;
  // 32-bit word w of the `left` logits at e, -inf behind them
  __device__ __forceinline__ static uint32_t word(const float* e, int w, int left) {
    return w < left ? __float_as_uint(e[w]) : kNegInf;
  }
  __device__ __forceinline__ static void unpack(const uint4& v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y);
    f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  }
};
template <> struct Vec<__half> {
  static constexpr int n = 8;
  static constexpr uint32_t kNegInf = 0xfc00fc00u;
  __device__ __forceinline__ static uint32_t word(const __half* e, int w, int left) {
    const uint16_t* b = reinterpret_cast<const uint16_t*>(e) + 2 * w;
    return (2 * w < left ? b[0] : kNegInf & 0xffffu) | (uint32_t)(2 * w + 1 < left ? b[1] : kNegInf & 0xffffu) << 16;
  }
  __device__ __forceinline__ static void unpack(const uint4& v, float (&f)[8]) { unpack8<__half>(v, f); }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int n = 8;
  static constexpr uint32_t kNegInf = 0xff80ff80u;
  __device__ __forceinline__ static uint32_t word(const __nv_bfloat16* e, int w, int left) {
    const uint16_t* b = reinterpret_cast<const uint16_t*>(e) + 2 * w;
    return (2 * w < left ? b[0] : kNegInf & 0xffffu) | (uint32_t)(2 * w + 1 < left ? b[1] : kNegInf & 0xffffu) << 16;
  }
  __device__ __forceinline__ static void unpack(const uint4& v, float (&f)[8]) { unpack8<__nv_bfloat16>(v, f); }
};

__device__ __forceinline__ float fast_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A row's parameters and extent.
struct Row {
  float temp, p, mp, u;
  int k, row, rank, head, nvec, v0, v1;     // vectors of the row and of this CTA
  int whole;                                // vectors that lie in the tensor in full
  const uint4* base;                        // vector 0
};

template <typename T>
__device__ __forceinline__ Row load_row(const SampleArgs& a) {
  constexpr int VN = Vec<T>::n;
  Row r;
  r.row = blockIdx.x / a.cluster;
  r.rank = blockIdx.x - r.row * a.cluster;
  r.temp = a.temperature ? __ldcg(a.temperature + r.row) : a.temp;
  r.k = a.top_k ? __ldcg(a.top_k + r.row) : a.k;
  r.p = a.top_p ? __ldcg(a.top_p + r.row) : a.p;
  r.mp = a.min_p ? __ldcg(a.min_p + r.row) : a.mp;
  r.mp = r.mp > 0.f ? fminf(r.mp, 1.f) : 0.f;             // (NaN: off)
  r.u = fminf(fmaxf(__ldcg(a.u + r.row), 0.f), 0x1.fffffep-1f);
  // The row in whole 16-byte vectors: vector 0 starts `head` logits before it.
  const long long start = (long long)r.row * a.vocab;
  r.head = (int)(start % VN);
  r.base = reinterpret_cast<const uint4*>(static_cast<const T*>(a.logits) + (start - r.head));
  r.nvec = (r.head + a.vocab + VN - 1) / VN;
  r.whole = (int)min((long long)r.nvec, ((long long)a.batch * a.vocab - (start - r.head)) / VN);
  const int per = (r.nvec + a.cluster - 1) / a.cluster;
  r.v0 = min(r.rank * per, r.nvec);
  r.v1 = min(r.v0 + per, r.nvec);
  return r;
}

// Vector v as it lies in memory; -inf where it is not of this CTA's slice or past the tensor.
template <typename T>
__device__ __forceinline__ uint4 fetch_vec(const SampleArgs& a, const Row& r, int v) {
  constexpr int VN = Vec<T>::n;
  // The load comes without a branch, so that several of them are in flight.
  const uint32_t ninf = Vec<T>::kNegInf;
  const uint4 none = make_uint4(ninf, ninf, ninf, ninf);
  uint4 raw = r.whole > 0 ? r.base[min(v, r.whole - 1)] : none;
  if (v >= r.v1) raw = none;
  else if (v >= r.whole) {                   // the tensor's last logits: element by element
    const int n = (int)((long long)a.batch * a.vocab - (long long)r.row * a.vocab + r.head - (long long)v * VN);
    const T* e = reinterpret_cast<const T*>(r.base + v);
    raw.x = Vec<T>::word(e, 0, n);
    raw.y = Vec<T>::word(e, 1, n);
    raw.z = Vec<T>::word(e, 2, n);
    raw.w = Vec<T>::word(e, 3, n);
  }
  return raw;
}
// Its logits as floats; NaN and what is not of the row as -inf.
template <typename T>
__device__ __forceinline__ void decode_vec(const SampleArgs& a, const Row& r, int v, const uint4& raw,
                                           float (&f)[Vec<T>::n]) {
  constexpr int VN = Vec<T>::n;
  Vec<T>::unpack(raw, f);
#pragma unroll
  for (int e = 0; e < VN; ++e) f[e] = fmaxf(f[e], -INFINITY);            // NaN
  if (v == 0 || v == r.nvec - 1) {
#pragma unroll
    for (int e = 0; e < VN; ++e) {
      const int i = v * VN + e - r.head;
      if (i < 0 || i >= a.vocab) f[e] = -INFINITY;
    }
  }
}
template <typename T>
__device__ __forceinline__ void load_vec(const SampleArgs& a, const Row& r, int v, float (&f)[Vec<T>::n]) {
  decode_vec<T>(a, r, v, fetch_vec<T>(a, r, v), f);
}

__device__ __forceinline__ float log2_per_logit(float temp) {
  return fmaxf(fminf(1.4426950408889634f / fmaxf(temp, 1e-38f), 1e30f), 1e-30f);
}

// The general path of one row whose maximum is M; every CTA of the cluster calls it.
template <typename T, int NT>
__device__ __noinline__ void general_row(const SampleArgs& a, const Row& R, float M, SampleShared& sh,
                                         double* seg) {
  constexpr int VN = Vec<T>::n;
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int C = a.cluster, row = R.row, rank = R.rank, head = R.head, v0 = R.v0, v1 = R.v1;
  const float temp = R.temp, p = R.p, mp = R.mp;
  const int k = R.k;
  const bool greedy = !(temp > 0.f);
  auto load = [&](int v, float (&f)[VN]) { load_vec<T>(a, R, v, f); };
  int phase = 0;
  const float cl = log2_per_logit(temp);
  const double dM = (double)M, dT = (double)temp;
  auto dist = [&](float x) { return (x == M ? 0.f : M - x) * cl; };          // log2 of max w / w, for bins
  auto fine = [&](float x) -> double {                                       // w
    if (x == M) return 1.0;
    if (x == -INFINITY) return 0.0;
    const double w = exp(((double)x - dM) / dT);
    return w > 0.0 ? w : 0.0;                       // (0 / 0 of infinite logits and temperatures)
  };

  // Find the first index, in index order, at which the running sum of value(x, i) over the whole
  // row passes `target` (target(total) of the row's sum). Every CTA gets the index.
  auto locate = [&](auto&& segment_value, auto&& element_value, auto&& target_of) -> int {
    const int segs = a.iters * (NT / 32);
    for (int it = 0; it < a.iters; ++it) {
      float f[VN];
      const int v = v0 + it * NT + tid;
      load(v, f);
      double s = segment_value(f, v * VN - head);
      if (__any_sync(0xffffffffu, s != 0.0)) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      }
      if (lane == 0) seg[it * (NT / 32) + warp] = s;
    }
    __syncthreads();
    const int chunk = (segs + NT - 1) / NT;
    const int s0 = min(tid * chunk, segs), s1 = min(s0 + chunk, segs);
    double mine = 0.0;
    for (int s = s0; s < s1; ++s) mine += seg[s];
    double inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double t = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += t;
    }
    if (lane == 31) sh.warp_d[warp] = inc;
    __syncthreads();
    double before = 0.0, all = 0.0;
#pragma unroll
    for (int w = 0; w < (NT / 32); ++w) {
      if (w == warp) before = all;
      all += sh.warp_d[w];
    }
    const int ph = phase++ & 1;
    if (tid == 0) sh.sum[ph] = all;
    cluster.sync();
    double total = 0.0, cta = 0.0;
    for (int r = 0; r < C; ++r) {
      if (r == rank) cta = total;
      total += *cluster.map_shared_rank(&sh.sum[ph], r);
    }
    const double target = target_of(total);
    unsigned long long hit = kNone;
    // The parts of the line that CTAs and threads hold meet exactly (every border is one and the
    // same rounded sum on both sides), so one thread holds the target; it walks its segments.
    const bool here = cta <= target && target < cta + all;
    double excl = __shfl_up_sync(0xffffffffu, inc, 1);
    if (lane == 0) excl = 0.0;
    double at = cta + (before + excl);
    if (here && at <= target && target < cta + (before + inc)) {
      int s = s0;
      double next = at;                               // the sum in front of the next segment
      for (int t = s0; t < s1 && next <= target; ++t) {
        if (seg[t] == 0.0) continue;
        s = t;
        at = next;
        next += seg[t];
      }
      sh.found = s;
      sh.found_base = at;
    }
    __syncthreads();
    if (here && warp == 0) {
      const int s = sh.found;
      const double at = sh.found_base;
      float f[VN];
      const int v = v0 + (s / (NT / 32)) * NT + (s % (NT / 32)) * 32 + lane;
      load(v, f);
      double w[VN], own = 0.0;
#pragma unroll
      for (int e = 0; e < VN; ++e) { w[e] = element_value(f[e], v * VN - head + e); own += w[e]; }
      double run = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double t = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += t;
      }
      run = at + run - own;
      int first = INT_MAX, last = -1;
#pragma unroll
      for (int e = 0; e < VN; ++e) {
        run += w[e];
        if (w[e] > 0.0) {
          last = v * VN - head + e;
          if (run > target && first == INT_MAX) first = last;
        }
      }
      first = __reduce_min_sync(0xffffffffu, first);
      last = __reduce_max_sync(0xffffffffu, last);
      hit = (unsigned long long)(first != INT_MAX ? first : last);
    }
    if (tid == 0) sh.idx[ph] = hit;
    cluster.sync();
    for (int r = 0; r < C; ++r) {
      const unsigned long long i = *cluster.map_shared_rank(&sh.idx[ph], r);
      if (i != kNone) return (int)i;
    }
    return -1;
  };
  auto sum_of = [&](auto&& element_value) {
    return [&, element_value](const float (&f)[VN], int i) {
      double s = 0.0;
#pragma unroll
      for (int e = 0; e < VN; ++e) s += element_value(f[e], i + e);
      return s;
    };
  };

  if (greedy) {                                     // the first logit that equals the maximum
    auto same = [&](float x, int) { return x == M ? 1.0 : 0.0; };
    const int i = locate(sum_of(same), same, [](double) { return 0.0; });
    if (rank == 0 && tid == 0) a.out[row] = i;
    cluster.sync();
    return;
  }

  // ---------------------------------------------------------------- the prefix's last value
  unsigned int kx = 0;                              // kept: keys above kx, and of the equal ones
  int cut = -1;                                     // those with an index up to cut
  const bool by_k = k > 0 && k < a.vocab, by_p = p < 1.f;
  if (by_k || by_p) {
    // One pass: `place` gives a logit's bin (or -1), the histograms of all CTAs are joined, and
    // cum_count / cum_mass hold their running sums.
    // Units of a weight: the row's sum takes 61 to 62 bits of 63, whatever its logits are, so that a
    // rounding of each of 2^20 weights is 2^-42 of it.
    double unit = 1.0;
    auto fixed = [&](float x) { return by_p ? (unsigned long long)__double2ll_rn(fine(x) * unit) : 0ull; };
    if (by_p) {
      double z = 0.0;
      for (int v = v0 + tid; v < v1; v += NT) {
        float f[VN];
        load(v, f);
        float some = 0.f;
#pragma unroll
        for (int e = 0; e < VN; ++e) some += fast_ex2(-dist(f[e]));
        z += (double)some;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
      if (lane == 0) sh.warp_d[warp] = z;
      __syncthreads();
      const int ph = phase++ & 1;
      if (tid == 0) {
        double t = 0.0;
        for (int w = 0; w < (NT / 32); ++w) t += sh.warp_d[w];
        sh.sum[ph] = t;
      }
      cluster.sync();
      z = 0.0;
      for (int r = 0; r < C; ++r) z += *cluster.map_shared_rank(&sh.sum[ph], r);
      unit = ldexp(1.0, 61 - ilogb(fmax(z, 1.0)));  // (z is right to 2^-10)
    }
    unsigned long long rest = 0;                    // mass of the logits `place` sends past the end
    auto histogram = [&](auto&& place, bool first) {
      const int ph = phase++ & 1;
      Hist& h = sh.hist[ph];
      for (int i = tid; i < kBins; i += NT) { h.mass[i] = 0; h.count[i] = 0; }
      __syncthreads();
      unsigned long long tail = 0;
      for (int v = v0 + tid; v < v1; v += NT) {
        float f[VN];
        load(v, f);
#pragma unroll
        for (int e = 0; e < VN; ++e) {
          const int b = place(f[e], dist(f[e]));
          if (b >= 0) {
            atomicAdd(&h.count[b], 1u);
            if (by_p) atomicAdd(&h.mass[b], fixed(f[e]));
          } else if (first) {
            tail += fixed(f[e]);
          }
        }
      }
      if (first) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) tail += __shfl_xor_sync(0xffffffffu, tail, o);
        if (lane == 0) sh.warp_m[warp] = tail;
        __syncthreads();
        if (tid == 0) {
          unsigned long long t = 0;
          for (int w = 0; w < (NT / 32); ++w) t += sh.warp_m[w];
          sh.far[ph] = t;
        }
      }
      cluster.sync();
      unsigned long long m = 0;
      unsigned int c = 0;
      if (tid < kBins) {
        for (int r = 0; r < C; ++r) {
          const Hist* o = cluster.map_shared_rank(&h, r);
          m += o->mass[tid];
          c += o->count[tid];
        }
      }
      if (first) {
        rest = 0;
        for (int r = 0; r < C; ++r) rest += *cluster.map_shared_rank(&sh.far[ph], r);
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long tm = __shfl_up_sync(0xffffffffu, m, o);
        const unsigned int tc = __shfl_up_sync(0xffffffffu, c, o);
        if (lane >= o) { m += tm; c += tc; }
      }
      if (lane == 31) { sh.warp_m[warp] = m; sh.warp_c[warp] = c; }
      __syncthreads();
      if (tid < kBins) {
        for (int w = 0; w < warp; ++w) { m += sh.warp_m[w]; c += sh.warp_c[w]; }
        sh.cum_mass[tid] = m;
        sh.cum_count[tid] = c;
      }
      if (tid == 0) sh.found = kBins;
      __syncthreads();
    };
    // First bin at which the running count (or mass) reaches `need`; kBins if none does.
    auto crossing = [&](bool count, unsigned long long need) -> int {
      if (tid < kBins) {
        const unsigned long long now = count ? sh.cum_count[tid] : sh.cum_mass[tid];
        const unsigned long long prev = tid == 0 ? 0 : (count ? sh.cum_count[tid - 1] : sh.cum_mass[tid - 1]);
        if (now >= need && prev < need) sh.found = tid;
      }
      __syncthreads();
      const int b = sh.found;
      __syncthreads();
      if (tid == 0) sh.found = kBins;
      __syncthreads();
      return b;
    };
    constexpr float kNear = kBins / kFine, kWide = kBins / (kFar - kFine);
    auto near_bin = [&](float, float d) { return d < kFine ? min((int)(d * kNear), kBins - 1) : -1; };
    auto wide_bin = [&](float, float d) {
      return d >= kFine && d < kFar ? min((int)((d - kFine) * kWide), kBins - 1) : -1;
    };
    auto past_bin = [&](float x, float d) { return d >= kFar && x > -INFINITY ? 0 : -1; };

    // The prefix that reaches `need` (a count, or a mass): sets kx and cut; returns its mass.
    // The first histogram has been made already.
    auto search = [&](bool count, unsigned long long need) -> unsigned long long {
      unsigned long long above = 0;                 // mass above the current range
      int b = crossing(count, need), stage = 0;
      auto take = [&](int n) {                      // the first n bins lie in front
        if (n == 0) return;
        need -= count ? (unsigned long long)sh.cum_count[n - 1] : sh.cum_mass[n - 1];
        above += sh.cum_mass[n - 1];
        __syncthreads();
      };
      while (b == kBins) {                          // past this histogram: the next
        take(kBins);
        if (++stage == 3) { kx = 0; cut = -1; return above; }      // all that weigh anything
        if (stage == 1) histogram(wide_bin, false);
        else histogram(past_bin, false);
        b = crossing(count, need);
      }
      take(b);
      // Keys the bin can hold: its edges, four values more on each side (the distance has three
      // roundings), members by the bin itself.
      const float lo = stage == 2 ? kFar : stage == 1 ? kFine + b / kWide : b / kNear;
      const float hi = stage == 2 ? INFINITY : stage == 1 ? kFine + (b + 1) / kWide : (b + 1) / kNear;
      unsigned int khi = order_key(M - lo / cl * (1.f - 2e-6f)), klo = order_key(M - hi / cl * (1.f + 2e-6f));
      khi = khi > 0xffffffffu - 4 ? 0xffffffffu : khi + 4;
      klo = stage == 2 || klo < 5 ? 1 : klo - 4;
      // from here up a key is surely not of a later bin
      const unsigned int sure = stage == 2 ? 0 : order_key(M - hi / cl * (1.f - 2e-6f)) + 4;
      const int bin = b;
      for (;;) {
        int shift = 0;
        while (((khi - klo) >> shift) >= kBins) ++shift;
        histogram([&](float x, float d) {
          if ((stage == 2 ? past_bin(x, d) : stage == 1 ? wide_bin(x, d) : near_bin(x, d)) != bin) return -1;
          const unsigned int key = order_key(x);
          return key > khi || key < klo ? -1 : (int)((khi - key) >> shift);
        }, false);
        b = crossing(count, need);
        if (b == kBins) b = kBins - 1;              // cannot be: the bin's members are in the range
        take(b);
        const unsigned int n = sh.cum_count[b] - (b > 0 ? sh.cum_count[b - 1] : 0);
        const unsigned long long m = sh.cum_mass[b] - (b > 0 ? sh.cum_mass[b - 1] : 0);
        __syncthreads();
        khi -= (unsigned int)b << shift;
        const unsigned int width = 1u << shift;
        if (khi - klo >= width) klo = khi - width + 1;
        if ((n <= 1 && klo >= sure) || klo == khi) {
          // One logit, or n equal ones of which the first `kept` by index stay.
          unsigned long long kept = n;
          if (n > 1) kept = count ? need : (m / n == 0 ? n : (need + m / n - 1) / (m / n));
          if (kept >= n) {
            kx = klo - 1;
            cut = -1;
            return above + m;
          }
          kx = klo;
          auto tie = [&](float x, int) { return order_key(x) == kx ? 1.0 : 0.0; };
          const double last = (double)kept - 1.0;
          // (with the histogram still wanted by the caller this is only reached last)
          cut = locate(sum_of(tie), tie, [&](double) { return last; });
          return above + m / n * kept;
        }
      }
    };

    histogram(near_bin, true);
    const unsigned long long near_mass = sh.cum_mass[kBins - 1];
    unsigned long long Z = near_mass + rest;
    bool fresh = true;                              // the first histogram is in cum_*
    if (by_k) {
      Z = search(true, (unsigned long long)k);
      fresh = false;
    }
    if (by_p) {
      if (!fresh) histogram(near_bin, true);
      const double need = ceil((double)fmaxf(p, 0.f) * (double)Z);
      search(false, need < 1.0 ? 1ull : (unsigned long long)need);
    }
  }

  // ---------------------------------------------------------------- the draw
  const bool cuts = by_k || by_p;
  const bool low = mp > 0.f;
  auto kept = [&](float x, int i) {
    if (cuts) {
      const unsigned int key = order_key(x);
      if (!(key > kx || (key == kx && i <= cut))) return false;
    }
    if (low) {                                      // by the 32-bit weight but next to the border
      const float d = dist(x), w = fast_ex2(-d);
      if (w > mp * 1.001f) return true;
      if (w < mp * 0.999f && (mp > 1e-30f || d < 100.f)) return false;
      return fine(x) >= (double)mp;
    }
    return true;
  };
  auto weight = [&](float x, int i) { return kept(x, i) ? fine(x) : 0.0; };
  const int i = locate(sum_of(weight), weight, [&](double total) { return (double)R.u * total; });
  if (rank == 0 && tid == 0) a.out[row] = i;
  cluster.sync();
}

// f(r, value of p in the r-th CTA) for all CTAs of the cluster, the loads issued together.
template <typename V, typename F>
__device__ __forceinline__ void for_cluster(int C, const V* p, F&& f) {
  cg::cluster_group cluster = cg::this_cluster();
  V v[kMaxCluster];
#pragma unroll
  for (int r = 0; r < kMaxCluster; ++r)
    if (r < C) v[r] = *cluster.map_shared_rank(const_cast<V*>(p), r);
#pragma unroll
  for (int r = 0; r < kMaxCluster; ++r)
    if (r < C) f(r, v[r]);
}

// Row maximum over the cluster (after its barrier `top` may be reused by the next row only).
template <int NT>
__device__ __forceinline__ float cluster_max(float M, float* warp_top, float* top, int C) {
  cg::cluster_group cluster = cg::this_cluster();
  M = warp_max(M);
  if ((threadIdx.x & 31) == 0) warp_top[threadIdx.x >> 5] = M;
  __syncthreads();
  if (threadIdx.x < 32) {
    M = warp_max(threadIdx.x < NT / 32 ? warp_top[threadIdx.x] : -INFINITY);
    if (threadIdx.x == 0) *top = M;
  }
  cluster.sync();
  M = -INFINITY;
  for_cluster(C, top, [&](int, float v) { M = fmaxf(M, v); });
  return M;
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT) sample_general_kernel(const __grid_constant__ SampleArgs a) {
  constexpr int VN = Vec<T>::n;
  __shared__ SampleShared sh;
  extern __shared__ double seg[];                 // [iters * warps] sums of 32 * VN logits
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const Row R = load_row<T>(a);
  float M = -INFINITY;
  for (int v = R.v0 + threadIdx.x; v < R.v1; v += 4 * NT) {
    float f[4][VN];
#pragma unroll
    for (int q = 0; q < 4; ++q) load_vec<T>(a, R, v + q * NT, f[q]);
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int e = 0; e < VN; ++e) M = fmaxf(M, f[q][e]);
  }
  M = cluster_max<NT>(M, reinterpret_cast<float*>(sh.warp_d), &sh.top[0], a.cluster);
  if (M == -INFINITY) {                            // nothing to choose from
    if (R.rank == 0 && threadIdx.x == 0) a.out[R.row] = -1;
    cg::this_cluster().sync();
    return;
  }
  general_row<T, NT>(a, R, M, sh, seg);
}

// ------------------------------------------------------------------ common path
constexpr int kCand = 256;                // members of the sub-bin the prefix ends in
constexpr int kCoarse = 512;              // bins of the first histogram (every CTA reads all CTAs')
constexpr int kHead = (int)(4.f * kCoarse / kFar);   // bins of the weights above 1/16
constexpr int kParts = 2;                 // of a CTA's warps, with a histogram each: 15 bits of count
static_assert(kMaxSlice / kParts < 1 << 15, "a part's count");
constexpr int kSub = 64;                  // and of the second
constexpr float kBinsPerLog2 = kCoarse / kFar;
constexpr float kPlaces = 8.f * kCoarse - 0.5f;   // places (eighths of a bin) that count

// floor(2^(30 + j / 256))
__device__ const unsigned int kExp2[256] = {
    0x40000000u, 0x402c6be9u, 0x4058f6a7u, 0x4085a050u, 0x40b268f9u, 0x40df50b8u, 0x410c57a1u, 0x41397dcbu,
    0x4166c34cu, 0x41942838u, 0x41c1aca7u, 0x41ef50adu, 0x421d1461u, 0x424af7d9u, 0x4278fb2bu, 0x42a71e6cu,
    0x42d561b3u, 0x4303c517u, 0x433248adu, 0x4360ec8cu, 0x438fb0cbu, 0x43be957fu, 0x43ed9abfu, 0x441cc0a3u,
    0x444c0740u, 0x447b6eadu, 0x44aaf701u, 0x44daa053u, 0x450a6abau, 0x453a564du, 0x456a6322u, 0x459a9151u,
    0x45cae0f1u, 0x45fb521au, 0x462be4e2u, 0x465c9960u, 0x468d6fadu, 0x46be67e0u, 0x46ef8210u, 0x4720be54u,
    0x47521cc5u, 0x47839d7au, 0x47b5408bu, 0x47e70610u, 0x4818ee21u, 0x484af8d5u, 0x487d2645u, 0x48af7689u,
    0x48e1e9b9u, 0x49147feeu, 0x4947393eu, 0x497a15c4u, 0x49ad1597u, 0x49e038d0u, 0x4a137f87u, 0x4a46e9d6u,
    0x4a7a77d4u, 0x4aae299bu, 0x4ae1ff43u, 0x4b15f8e5u, 0x4b4a169bu, 0x4b7e587du, 0x4bb2bea4u, 0x4be7492au,
    0x4c1bf828u, 0x4c50cbb7u, 0x4c85c3f1u, 0x4cbae0eeu, 0x4cf022c9u, 0x4d25899bu, 0x4d5b157eu, 0x4d90c68bu,
    0x4dc69cdcu, 0x4dfc988cu, 0x4e32b9b4u, 0x4e69006du, 0x4e9f6cd3u, 0x4ed5feffu, 0x4f0cb70cu, 0x4f439513u,
    0x4f7a9930u, 0x4fb1c37cu, 0x4fe91412u, 0x50208b0du, 0x50582887u, 0x508fec9cu, 0x50c7d765u, 0x50ffe8feu,
    0x51382181u, 0x5170810au, 0x51a907b4u, 0x51e1b59au, 0x521a8ad7u, 0x52538786u, 0x528cabc3u, 0x52c5f7a9u,
    0x52ff6b54u, 0x533906e0u, 0x5372ca67u, 0x53acb607u, 0x53e6c9dau, 0x542105fdu, 0x545b6a8bu, 0x5495f7a0u,
    0x54d0ad5au, 0x550b8bd3u, 0x55469329u, 0x5581c377u, 0x55bd1cdau, 0x55f89f6fu, 0x56344b52u, 0x5670209fu,
    0x56ac1f75u, 0x56e847eeu, 0x57249a29u, 0x57611642u, 0x579dbc56u, 0x57da8c83u, 0x581786e5u, 0x5854ab9bu,
    0x5891fac0u, 0x58cf7474u, 0x590d18d3u, 0x594ae7fau, 0x5988e209u, 0x59c7071cu, 0x5a055751u, 0x5a43d2c6u,
    0x5a827999u, 0x5ac14be9u, 0x5b0049d4u, 0x5b3f7377u, 0x5b7ec8f1u, 0x5bbe4a61u, 0x5bfdf7e5u, 0x5c3dd19bu,
    0x5c7dd7a3u, 0x5cbe0a1bu, 0x5cfe6922u, 0x5d3ef4d7u, 0x5d7fad59u, 0x5dc092c6u, 0x5e01a53fu, 0x5e42e4e2u,
    0x5e8451cfu, 0x5ec5ec25u, 0x5f07b404u, 0x5f49a98bu, 0x5f8bccdbu, 0x5fce1e12u, 0x60109d50u, 0x60534ab7u,
    0x60962665u, 0x60d9307au, 0x611c6918u, 0x615fd05eu, 0x61a3666du, 0x61e72b64u, 0x622b1f66u, 0x626f4291u,
    0x62b39508u, 0x62f816ebu, 0x633cc85au, 0x6381a978u, 0x63c6ba64u, 0x640bfb40u, 0x64516c2eu, 0x64970d4eu,
    0x64dcdec3u, 0x6522e0adu, 0x6569132fu, 0x65af7669u, 0x65f60a7fu, 0x663ccf91u, 0x6683c5c3u, 0x66caed35u,
    0x6712460au, 0x6759d065u, 0x67a18c67u, 0x67e97a34u, 0x683199edu, 0x6879ebb6u, 0x68c26fb1u, 0x690b2601u,
    0x69540ec8u, 0x699d2a2bu, 0x69e6784cu, 0x6a2ff94fu, 0x6a79ad55u, 0x6ac39484u, 0x6b0daeffu, 0x6b57fce8u,
    0x6ba27e65u, 0x6bed3398u, 0x6c381ca6u, 0x6c8339b2u, 0x6cce8ae1u, 0x6d1a1056u, 0x6d65ca37u, 0x6db1b8a7u,
    0x6dfddbcbu, 0x6e4a33c8u, 0x6e96c0c2u, 0x6ee382deu, 0x6f307a41u, 0x6f7da70fu, 0x6fcb096fu, 0x7018a185u,
    0x70666f76u, 0x70b47367u, 0x7102ad7fu, 0x71511de3u, 0x719fc4b9u, 0x71eea226u, 0x723db650u, 0x728d015du,
    0x72dc8373u, 0x732c3cb9u, 0x737c2d55u, 0x73cc556du, 0x741cb528u, 0x746d4cacu, 0x74be1c20u, 0x750f23abu,
    0x75606373u, 0x75b1dba1u, 0x76038c5bu, 0x765575c7u, 0x76a7980fu, 0x76f9f358u, 0x774c87ccu, 0x779f5590u,
    0x77f25ccdu, 0x78459dacu, 0x78991853u, 0x78ecccecu, 0x7940bb9eu, 0x7994e491u, 0x79e947efu, 0x7a3de5dfu,
    0x7a92be8au, 0x7ae7d219u, 0x7b3d20b6u, 0x7b92aa88u, 0x7be86fb9u, 0x7c3e7072u, 0x7c94acddu, 0x7ceb2523u,
    0x7d41d96du, 0x7d98c9e6u, 0x7deff6b6u, 0x7e476008u, 0x7e9f0606u, 0x7ef6e8dau, 0x7f4f08aeu, 0x7fa765acu,
};

// 2^t for t <= 0 with 30 bits, as a multiple of 2^-unit_bits: t in 64 bits, formed with 40 bits
// behind the point by adding 1.5 * 2^12; its 8 leading fraction bits index 2^(j / 256), the
// other 32 (r < 2^-8) give 2^r - 1 = z + z^2 / 2 + z^3 / 6, z = r ln 2, in 32-bit floats: 2^-23 of
// at most 2^-8.5. The table is in shared memory, 4 copies against bank conflicts.
struct Exp2Table {
  unsigned int v[256][4];
  __device__ __forceinline__ void fill() {
    if (threadIdx.x < 256) {
      const unsigned int t = kExp2[threadIdx.x];
      *reinterpret_cast<uint4*>(v[threadIdx.x]) = make_uint4(t, t, t, t);
    }
  }
  // max(0, 2^(diff * per) * 2^unit_bits), diff <= 0, diff * per > -kFar - 1; lower_bits = 45 - unit_bits
  __device__ __forceinline__ unsigned long long operator()(double diff, double per, int lower_bits) const {
    const double u = fma(diff, per, 6144.0);
    const unsigned int hi = (unsigned int)__double2hiint(u), lo = (unsigned int)__double2loint(u);
    const unsigned int t = v[hi & 255][threadIdx.x & 3];
    const int n = (int)((hi >> 8) & 0xfff) - 2048;              // floor(t)
    const float z = (__uint_as_float((lo >> 9) | 0x3f800000u) - 1.f) * (0.6931471805599453f / 256.f);
    const float q = fmaf(z * z, fmaf(z, 1.f / 6.f, 0.5f), z);
    const unsigned int qi = __float_as_uint(q + 0.00390625f) & 0x7fffffu;   // units of 2^-31
    const unsigned int w = t + __umulhi(t, qi << 1);
    return ((unsigned long long)w << 15) >> (lower_bits - n);
  }
};

struct Cand {
  unsigned int key;
  int idx;
  unsigned long long mass;
};

template <int NT>
struct FastShared {
  static constexpr int kWarps = NT / 32, kList = (NT == kManyThreads ? 2048 : 4096) / kWarps;   // listed logits of a warp
  static constexpr int kRounds = kMaxSlice / (4 * NT);                // rounds of vectors of a warp, at most
  static_assert(kRounds <= 32, "a lane per round");
  Exp2Table table;
  union {
    unsigned int coarse[kParts][kCoarse]; // count << 17 | sum of places in the bin (eighths)
    Cand all[kCand];                      // later: the members of every CTA
  };
  float x[kWarps][kList];
  int idx[kWarps][kList];
  unsigned long long mass[kWarps][kList]; // 0: not kept
  unsigned long long round_sum[kRounds];
  unsigned long long sub_mass[kSub];
  unsigned int sub_count[kSub];
  Cand mine[2][kCand];                    // this CTA's members, one buffer per search
  int n_mine[2];
  unsigned long long cum_mass[kSub];
  unsigned int cum_count[kSub];
  unsigned long long head[1], above[1], sum[1], total[1];   // read by the other CTAs
  int crowded[1], first[1];
  float top[1], warp_top[kWarps];
  unsigned long long warp_m[kWarps], warp_n[kWarps];
  unsigned int warp_c[kWarps];
  float warp_f[kWarps], warp_near[kWarps];
  int bin, any_crowded, k_bin, lo_bin, hi_bin;
  unsigned int k_count, hi_count, lo_before;
  unsigned long long sum_above, sum_all, cut_mass;
  unsigned int cut_key;
  int cut_idx;
};

// Sum over the warp of values below 2^57, as two sums of halves.
__device__ __forceinline__ unsigned long long warp_sum_u64(unsigned long long v) {
  const unsigned int lo = __reduce_add_sync(0xffffffffu, (unsigned int)v & 0x3ffffffu);
  const unsigned int mid = __reduce_add_sync(0xffffffffu, (unsigned int)(v >> 26) & 0x3ffffffu);
  const unsigned int hi = __reduce_add_sync(0xffffffffu, (unsigned int)(v >> 52));
  return lo + ((unsigned long long)mid << 26) + ((unsigned long long)hi << 52);
}
__device__ __forceinline__ unsigned long long warp_scan_u64(unsigned long long v) {   // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long t = __shfl_up_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) >= o) v += t;
  }
  return v;
}

// w >= min_p in 64 bits, for weights next to the border.
__device__ __noinline__ bool reaches(float v, float M, float temp, float mp) {
  return (v == M ? 1.0 : exp(((double)v - (double)M) / (double)temp)) >= (double)mp;
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT, NT == kManyThreads ? kManyCtas : 1) sample_kernel(const __grid_constant__ SampleArgs a) {
  constexpr int VN = Vec<T>::n;
  extern __shared__ double dyn[];
  using Shared = FastShared<NT>;
  constexpr int kList = Shared::kList;
  Shared& sh = *reinterpret_cast<Shared*>(dyn);
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, C = a.cluster;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const Row R = load_row<T>(a);
  const bool greedy = !(R.temp > 0.f);

  // Warp w has the w-th contiguous part of the slice, in 512-byte rounds of its lanes, so
  // warp, round, lane, element is index order.
  // (Loops over the rounds are not unrolled: straight-line code for a slice is several times the
  // instruction cache, and took 5 to 10 times as long.)
  const int rounds = (R.v1 - R.v0 + NT - 1) / NT;
  const int first_v = R.v0 + warp * rounds * 32 + lane;
  sh.table.fill();
  for (int i = tid; i < kParts * kCoarse / 4; i += NT)
    reinterpret_cast<uint4*>(sh.coarse)[i] = make_uint4(0, 0, 0, 0);
  if (tid < kSub) { sh.sub_mass[tid] = 0; sh.sub_count[tid] = 0; }
  if (tid < 2) sh.n_mine[tid] = 0;
  if (tid == 0) {
    sh.crowded[0] = 0;
    sh.first[0] = INT_MAX;
    sh.k_bin = sh.lo_bin = sh.hi_bin = kCoarse;
    sh.head[0] = 0;
  }
  constexpr int kAhead = 32 / VN;                  // loads in flight: 32 registers of them
  // body(i, logits) for the warp's rounds, the next vectors in flight (two by name: a move from one
  // register to the next would wait for its load).
  auto each_round = [&](auto&& body) {
    uint4 p0 = fetch_vec<T>(a, R, first_v), p1 = fetch_vec<T>(a, R, rounds > 1 ? first_v + 32 : INT_MAX);
#pragma unroll 1
    for (int i = 0; i < rounds; i += 2) {
      float x[VN];
      decode_vec<T>(a, R, first_v + i * 32, p0, x);
      p0 = fetch_vec<T>(a, R, i + 2 < rounds ? first_v + (i + 2) * 32 : INT_MAX);
      body(i, x);
      if (i + 1 < rounds) {
        decode_vec<T>(a, R, first_v + (i + 1) * 32, p1, x);
        p1 = fetch_vec<T>(a, R, i + 3 < rounds ? first_v + (i + 3) * 32 : INT_MAX);
        body(i + 1, x);
      }
    }
  };
  float M = -INFINITY;
#pragma unroll 1
  for (int i = 0; i < rounds; i += kAhead) {
    float f[kAhead][VN];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) load_vec<T>(a, R, i + q < rounds ? first_v + (i + q) * 32 : INT_MAX, f[q]);
#pragma unroll
    for (int q = 0; q < kAhead; ++q)
#pragma unroll
      for (int e = 0; e < VN; ++e) M = fmaxf(M, f[q][e]);
  }
  M = cluster_max<NT>(M, sh.warp_top, &sh.top[0], C);
  if (M == -INFINITY) {                            // nothing to choose from
    if (R.rank == 0 && tid == 0) a.out[R.row] = -1;
    cluster.sync();
    return;
  }
  // To the general path: infinite logits, which share the draw; draws that may end among the weights
  // this path drops (2^18 of less than 2^-46: 2^-28 of the largest).
  if ((M == INFINITY || R.u < 0x1p-24f) && !greedy) {
    cluster.sync();
    general_row<T, NT>(a, R, M, *reinterpret_cast<SampleShared*>(dyn), dyn + sizeof(SampleShared) / sizeof(double));
    return;
  }
  if (greedy) {                                    // the first logit that equals the maximum
    int at = INT_MAX;
#pragma unroll 1
    for (int i = 0; i < rounds; ++i) {
      float x[VN];
      load_vec<T>(a, R, first_v + i * 32, x);
#pragma unroll
      for (int e = 0; e < VN; ++e)
        if (x[e] == M) at = min(at, (first_v + i * 32) * VN + e - R.head);
    }
    at = __reduce_min_sync(0xffffffffu, at);
    if (lane == 0 && at != INT_MAX) atomicMin(&sh.first[0], at);
    cluster.sync();
    if (R.rank == 0 && tid == 0) {
      for_cluster(C, &sh.first[0], [&](int, int v) { at = min(at, v); });
      a.out[R.row] = at;
    }
    cluster.sync();
    return;
  }

  const float cl = log2_per_logit(R.temp);
  const double dM = (double)M;
  const double per = fmax(fmin(1.4426950408889634 / fmax((double)R.temp, 1e-38), 1e30), 1e-30);
  const float places = cl * (8.f * kBinsPerLog2);
  // Distance in eighths of a bin. Every pass forms it anew and must get the same value: rounded here,
  // so that no pass's product goes unrounded into a sum of its own.
  auto place = [&](float v) { return __fmul_rn(__fsub_rn(M, v), places); };
  auto units = [&](float v) { return sh.table((double)v - dM, per, a.lower_bits); };   // place < kPlaces
  // w >= min_p: by the units but for those next to the border.
  const double mp_units = (double)R.mp * a.unit;
  const unsigned long long mp_no = R.mp > 0.f ? (unsigned long long)fmax(mp_units * 0.999999 - 2.0, 0.0) : 0;
  const unsigned long long mp_yes = R.mp > 0.f ? (unsigned long long)(mp_units * 1.000001) + 3 : 0;
  auto passes = [&](float v, unsigned long long m) {
    if (m >= mp_yes) return true;
    if (m < mp_no) return false;
    return reaches(v, M, R.temp, R.mp);
  };
  const bool by_p = R.p < 1.f;
  bool by_k = R.k > 0 && R.k < a.vocab;

  // ---------------------------------------------------------------- bins the prefix ends in
  // Logits in bins below lo are in it, those in lo..hi are listed, those behind are not in it.
  int lo = kCoarse, hi = kCoarse;
  unsigned int before_lo = 0;
  if (by_k || by_p) {
    unsigned long long heavy = 0;
    unsigned int* const hist = sh.coarse[warp * kParts / (NT / 32)];
    each_round([&](int, const float (&x)[VN]) {
      bool some = false;
#pragma unroll
      for (int e = 0; e < VN; ++e) {
        const float y = place(x[e]);
        some |= y < 8 * kHead - 0.5f;
        if (y < kPlaces) {                         // nearest place, by adding 1.5 * 2^23
          const unsigned int at = __float_as_uint(y + 12582912.f) & (8 * kCoarse - 1);
          atomicAdd(&hist[at >> 3], (1u << 17) | (at & 7));
        }
      }
      if (by_p && __any_sync(0xffffffffu, some)) {
#pragma unroll
        for (int e = 0; e < VN; ++e) heavy += place(x[e]) < 8 * kHead - 0.5f ? units(x[e]) : 0;
      }
    });
    if (by_p && heavy) atomicAdd(&sh.head[0], heavy);
    cluster.sync();
    constexpr int PT = 2;                          // bins of a thread, of the first kCoarse / 2
    static_assert(kCoarse / PT <= NT, "bins per thread");
    unsigned int c[PT] = {0, 0}, off[PT] = {0, 0};
    if (tid < kCoarse / PT)
#pragma unroll
      for (int part = 0; part < kParts; ++part)
        for_cluster(C, reinterpret_cast<const uint2*>(sh.coarse[part]) + tid, [&](int, const uint2& v) {
          c[0] += v.x >> 17;
          c[1] += v.y >> 17;
          off[0] += v.x & 0x1ffff;
          off[1] += v.y & 0x1ffff;
        });
    float f[PT], square = 0.f, near = 0.f;         // near: what the bins say of the head
    unsigned long long head_units = 0;
    if (by_p) for_cluster(C, &sh.head[0], [&](int, unsigned long long v) { head_units += v; });
    unsigned int c_sum = 0;
    float f_sum = 0.f;
#pragma unroll
    for (int q = 0; q < PT; ++q) {
      const float mean = c[q] ? __fdividef((float)off[q], (float)c[q]) * 0.125f : 0.f;
      const float w = fast_ex2(-((float)(tid * PT + q) + mean) * (1.f / kBinsPerLog2));
      f[q] = (float)c[q] * w;
      if (tid * PT + q < kHead) near += f[q];
      else square += f[q] * w;
      c_sum += c[q];
      f_sum += f[q];
    }
    unsigned int c_inc = c_sum;
    float f_inc = f_sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned int tc = __shfl_up_sync(0xffffffffu, c_inc, o);
      const float tf = __shfl_up_sync(0xffffffffu, f_inc, o);
      if (lane >= o) { c_inc += tc; f_inc += tf; }
    }
    square = warp_sum(square);
    near = warp_sum(near);
    constexpr int BW = kCoarse / PT / 32;          // warps with bins
    if (lane == 31 && warp < BW) {
      sh.warp_c[warp] = c_inc;
      sh.warp_f[warp] = f_inc;
      sh.warp_top[warp] = square;
      sh.warp_near[warp] = near;
    }
    __syncthreads();
    unsigned int c_at = c_inc - c_sum, c_all = 0;
    float f_at = f_inc - f_sum, f_all = 0.f;
    square = near = 0.f;
#pragma unroll
    for (int w = 0; w < BW; ++w) {
      if (w < warp) { c_at += sh.warp_c[w]; f_at += sh.warp_f[w]; }
      c_all += sh.warp_c[w];
      f_all += sh.warp_f[w];
      square += sh.warp_top[w];
      near += sh.warp_near[w];
    }
    by_k = by_k && (unsigned int)R.k <= c_all;     // else all of weight are kept
    // The heaviest (the head, d < 4) have their exact sum; of the others a weight is known to half
    // a place (0.4 %), a sum of many to less: about 0.0025 of the root of the sum of their squares.
    // Three times that, and a part in 5,000 for the bins' curvature.
    const float extra = (float)((double)head_units / a.unit) - near;
    f_all += extra;
    const float slack = 0.0075f * sqrtf(square) + 2e-4f * f_all;
    const float want = fmaxf(R.p, 0.f) * f_all, f_lo = want - slack, f_hi = want + slack;
#pragma unroll
    for (int q = 0; q < PT; ++q) {
      const unsigned int c_to = c_at + c[q];
      const float f_to = f_at + f[q];
      const int b = tid * PT + q;
      const float sure = b < kHead - 1 ? f_to * 1.005f : f_to + extra;      // inside the head: 0.4 %
      const float least = b < kHead - 1 ? f_to * 0.995f : f_to + extra;
      if (by_k && c_at < (unsigned int)R.k && (unsigned int)R.k <= c_to) {
        sh.k_bin = b;
        sh.k_count = c_to;
        sh.lo_before = c_at;
      }
      if (!by_k) {                                 // the first bins that reach f_lo and f_hi
        const unsigned int at_lo = __ballot_sync(0xffffffffu, c[q] && sure >= f_lo);
        const unsigned int at_hi = __ballot_sync(0xffffffffu, c[q] && least >= f_hi);
        if (at_lo && lane == __ffs(at_lo) - 1) atomicMin(&sh.lo_bin, b);
        if (at_hi && lane == __ffs(at_hi) - 1) atomicMin(&sh.hi_bin, b);
      }
      c_at = c_to;
      f_at = f_to;
    }
    __syncthreads();
    if (by_k) {
      hi = sh.k_bin;
      const bool whole = by_p || sh.k_count * 8 <= (unsigned int)(C * (NT / 32) * kList);
      lo = whole ? 0 : hi;
      before_lo = whole ? 0 : sh.lo_before;
    } else if (by_p) {
      hi = min(sh.hi_bin, kCoarse - 1);
      lo = min(sh.lo_bin, hi);
    }
  }
  const bool cuts = by_k || by_p;

  // ---------------------------------------------------------------- weights and lists
  int n = 0;                                       // listed by this warp
  unsigned long long above = 0, above_kept = 0, sum = 0;     // of this thread: in front, in all
  const bool all_weights = by_p && !by_k;          // top-p of the whole row: its sum
  const float y_lo = lo < kCoarse ? 8.f * lo - 0.5f : INFINITY, y_hi = hi < kCoarse - 1 ? 8.f * hi + 7.5f : INFINITY;
  each_round([&](int i, const float (&x)[VN]) {
    int where[VN];                                 // 0 in front, 1 listed, 2 behind
    unsigned long long m[VN];
    bool some = false, any = false;
#pragma unroll
    for (int e = 0; e < VN; ++e) {
      const float y = place(x[e]);
      where[e] = y < y_lo ? 0 : (y < y_hi ? 1 : 2);
      if (!(y < kPlaces)) where[e] = 3;            // weighs nothing
      some |= where[e] == 1;
      any |= where[e] < (all_weights ? 3 : 2);
    }
    if (!__any_sync(0xffffffffu, any)) return;     // no weight wanted in this round
    unsigned long long in_front = 0;
#pragma unroll
    for (int e = 0; e < VN; ++e) {
      m[e] = where[e] < 3 ? units(x[e]) : 0;
      if (where[e] == 0) in_front += m[e];
    }
    above += in_front;
    if (all_weights) {
#pragma unroll
      for (int e = 0; e < VN; ++e) sum += m[e];
    }
    if (R.mp > 0.f) {
#pragma unroll
      for (int e = 0; e < VN; ++e)
        if (where[e] == 0 && passes(x[e], m[e])) above_kept += m[e];
    }
    if (cuts && __any_sync(0xffffffffu, some)) {
      int at = n, all = 0;
#pragma unroll
      for (int e = 0; e < VN; ++e) {
        const unsigned int bal = __ballot_sync(0xffffffffu, where[e] == 1);
        at += __popc(bal & ((1u << lane) - 1));
        all += __popc(bal);
      }
#pragma unroll
      for (int e = 0; e < VN; ++e)
        if (where[e] == 1) {
          if (at < kList) {
            sh.x[warp][at] = x[e];
            sh.idx[warp][at] = (first_v + i * 32) * VN + e - R.head;
            sh.mass[warp][at] = m[e];
          }
          ++at;
        }
      n += all;
    }
  });
  unsigned int cut_key = 0xffffffffu;              // kept of the listed: keys above, or equal with
  int cut_idx = -1;                                // an index up to cut_idx
  unsigned long long own = R.mp > 0.f ? above_kept : above;
  if (cuts) {
    if (lane == 0 && n > kList) sh.crowded[0] = 1;
    n = min(n, kList);
    __syncwarp();
    const float sub = (float)kSub / (8.f * (float)(hi + 1 - lo));
    auto sub_bin = [&](float v) { return max(0, min((int)((place(v) - y_lo) * sub), kSub - 1)); };
    for (int t = lane; t < n; t += 32) {
      const int b = sub_bin(sh.x[warp][t]);
      atomicAdd(&sh.sub_count[b], 1u);
      atomicAdd(&sh.sub_mass[b], sh.mass[warp][t]);
    }
    above = warp_sum_u64(above);
    sum = warp_sum_u64(sum);
    __syncthreads();
    if (lane == 0) { sh.warp_m[warp] = above; sh.warp_n[warp] = sum; }
    __syncthreads();
    if (warp == 0) {
      const unsigned long long f = warp_sum_u64(lane < NT / 32 ? sh.warp_m[lane] : 0);
      const unsigned long long g = warp_sum_u64(lane < NT / 32 ? sh.warp_n[lane] : 0);
      if (lane == 0) { sh.above[0] = f; sh.sum[0] = g; }
    }
    cluster.sync();
    unsigned long long m = 0;
    unsigned int c = 0;
    if (tid < kSub) {
      for_cluster(C, &sh.sub_mass[tid], [&](int, unsigned long long v) { m += v; });
      for_cluster(C, &sh.sub_count[tid], [&](int, unsigned int v) { c += v; });
    } else if (tid == kSub) {
      unsigned long long f = 0, g = 0;
      int crowded = 0;
      for_cluster(C, &sh.above[0], [&](int, unsigned long long v) { f += v; });
      for_cluster(C, &sh.sum[0], [&](int, unsigned long long v) { g += v; });
      for_cluster(C, &sh.crowded[0], [&](int, int v) { crowded |= v; });
      sh.sum_above = f;
      sh.sum_all = g;
      sh.any_crowded = crowded;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long tm = __shfl_up_sync(0xffffffffu, m, o);
      const unsigned int tc = __shfl_up_sync(0xffffffffu, c, o);
      if (lane >= o) { m += tm; c += tc; }
    }
    if (lane == 31) { sh.warp_m[warp] = m; sh.warp_c[warp] = c; }
    __syncthreads();
    if (tid < kSub) {
      for (int w = 0; w < warp; ++w) { m += sh.warp_m[w]; c += sh.warp_c[w]; }
      sh.cum_mass[tid] = m;
      sh.cum_count[tid] = c;
    }
    __syncthreads();
    // The prefix of the listed that reaches `need` (a count, or a mass) in the order: false if
    // they do not hold its end. Leaves its last member and its mass.
    int turn = 0;
    unsigned long long cut_mass = 0;
    auto search = [&](bool count, unsigned long long need) -> bool {
      const unsigned long long have = count ? (unsigned long long)sh.cum_count[kSub - 1] : sh.cum_mass[kSub - 1];
      if (sh.any_crowded || need == 0 || have < need) return false;
      if (tid < kSub) {
        const unsigned long long now = count ? sh.cum_count[tid] : sh.cum_mass[tid];
        const unsigned long long prev = tid == 0 ? 0 : (count ? sh.cum_count[tid - 1] : sh.cum_mass[tid - 1]);
        if (now >= need && prev < need) sh.bin = tid;
      }
      __syncthreads();
      const int b = sh.bin;
      const unsigned int members = sh.cum_count[b] - (b > 0 ? sh.cum_count[b - 1] : 0);
      if (members > kCand) return false;
      if (b > 0) need -= count ? (unsigned long long)sh.cum_count[b - 1] : sh.cum_mass[b - 1];
      const unsigned long long front_bins = b > 0 ? sh.cum_mass[b - 1] : 0;
      for (int t = lane; t < n; t += 32) {
        const float v = sh.x[warp][t];
        if (sub_bin(v) == b) {
          const int at = atomicAdd(&sh.n_mine[turn], 1);
          sh.mine[turn][at] = Cand{order_key(v), sh.idx[warp][t], sh.mass[warp][t]};
        }
      }
      cluster.sync();
      int base = 0;                                // warp r brings the r-th CTA's members
      int count_r = 0;
      for_cluster(C, &sh.n_mine[turn], [&](int r, int v) {
        base += r < warp ? v : 0;
        count_r = r == warp ? v : count_r;
      });
      if (warp < C) {                              // ((NT / 32) >= kMaxCluster)
        const Cand* o = cluster.map_shared_rank(&sh.mine[turn][0], warp);
        for (int t = lane; t < count_r; t += 32) sh.all[base + t] = o[t];
      }
      __syncthreads();
      if (tid < (int)members) {
        const Cand me = sh.all[tid];
        unsigned long long front = 0, rank = 0;
        for (unsigned int t = 0; t < members; ++t) {
          const Cand o = sh.all[t];
          if (o.key > me.key || (o.key == me.key && o.idx < me.idx)) { front += o.mass; ++rank; }
        }
        if (count ? rank + 1 == need : front < need && need <= front + me.mass) {
          sh.cut_key = me.key;
          sh.cut_idx = me.idx;
          sh.cut_mass = front_bins + front + me.mass;
        }
      }
      __syncthreads();
      cut_key = sh.cut_key;
      cut_idx = sh.cut_idx;
      cut_mass = sh.cut_mass;
      ++turn;
      return true;
    };
    bool ok = true;
    unsigned long long Z = sh.sum_all;
    if (by_k) {
      ok = search(true, (unsigned long long)(R.k - before_lo));
      Z = cut_mass;                                // with top-p, lo is 0: nothing in front
    }
    if (ok && by_p) {
      const double need = ceil((double)fmaxf(R.p, 0.f) * (double)Z);
      const unsigned long long units_needed = need < 1.0 ? 1ull : (unsigned long long)need;
      ok = units_needed > sh.sum_above && search(false, units_needed - sh.sum_above);
    }
    if (!ok) {                                     // alike in every CTA of the cluster
      cluster.sync();
      general_row<T, NT>(a, R, M, *reinterpret_cast<SampleShared*>(dyn), dyn + sizeof(SampleShared) / sizeof(double));
      return;
    }
    for (int t = lane; t < n; t += 32) {
      const float v = sh.x[warp][t];
      const unsigned int key = order_key(v);
      const unsigned long long w = sh.mass[warp][t];
      const bool kept = (key > cut_key || (key == cut_key && sh.idx[warp][t] <= cut_idx)) && passes(v, w);
      if (kept) own += w;
      else sh.mass[warp][t] = 0;
    }
  }

  // ---------------------------------------------------------------- the draw
  own = warp_sum_u64(own);
  __syncthreads();
  if (lane == 0) sh.warp_m[warp] = own;
  __syncthreads();
  const unsigned long long of_lane = lane < NT / 32 ? sh.warp_m[lane] : 0;
  const unsigned long long cta = warp_sum_u64(of_lane);
  unsigned long long lead = 0;                     // in front of this CTA
  if (tid == 0) sh.total[0] = cta;
  cluster.sync();
  unsigned long long Z = 0;
  for_cluster(C, &sh.total[0], [&](int r, unsigned long long v) {
    if (r == R.rank) lead += Z;
    Z += v;
  });
  cluster.barrier_arrive();                        // its memory is not read any more
  const unsigned long long target = (unsigned long long)((double)R.u * (double)Z);
  if (lead <= target && target < lead + cta) {     // one CTA of the cluster
    // Its warps agree on the one that holds the target.
    const unsigned long long upto_warp = warp_scan_u64(of_lane);
    const int owner = __ffs(__ballot_sync(0xffffffffu, lead + upto_warp > target)) - 1;
    unsigned long long run = lead + __shfl_sync(0xffffffffu, upto_warp - of_lane, owner);
    int hit = -1;
    if (lo == 0) {                                 // all that is kept is listed, in index order
      if (warp == owner) {
        for (int t0 = 0; t0 < n && hit < 0; t0 += 32) {
          const unsigned long long w = t0 + lane < n ? sh.mass[warp][t0 + lane] : 0;
          const unsigned long long inc = warp_scan_u64(w);
          const unsigned int bal = __ballot_sync(0xffffffffu, w > 0 && run + inc > target);
          if (bal) hit = sh.idx[warp][t0 + __ffs(bal) - 1];
          run += __shfl_sync(0xffffffffu, inc, 31);
        }
      }
    } else {
      // All warps sum its rounds, then it looks into the one that holds the target.
      const int owner_v = first_v + (owner - warp) * rounds * 32;
      unsigned long long w[VN];
      auto kept_of = [&](int i) {                  // kept weights of this lane's vector of round i
        float x[VN];
        load_vec<T>(a, R, owner_v + i * 32, x);
        unsigned long long sum = 0;
#pragma unroll
        for (int e = 0; e < VN; ++e) {
          const float y = place(x[e]);
          const int id = (owner_v + i * 32) * VN + e - R.head;
          const unsigned int key = order_key(x[e]);
          w[e] = 0;
          if (y < kPlaces && (y < y_lo || (y < y_hi && (key > cut_key || (key == cut_key && id <= cut_idx))))) {
            w[e] = units(x[e]);
            if (R.mp > 0.f && !passes(x[e], w[e])) w[e] = 0;
          }
          sum += w[e];
        }
        return sum;
      };
#pragma unroll 1
      for (int i = warp; i < rounds; i += NT / 32) {
        const unsigned long long sum = warp_sum_u64(kept_of(i));
        if (lane == 0) sh.round_sum[i] = sum;
      }
      __syncthreads();
      if (warp == owner) {
        const unsigned long long mine = lane < rounds ? sh.round_sum[lane] : 0;
        const unsigned long long upto = warp_scan_u64(mine);
        const int i = __ffs(__ballot_sync(0xffffffffu, run + upto > target)) - 1;
        run += __shfl_sync(0xffffffffu, upto - mine, i);
        const unsigned long long sum = kept_of(i);
        unsigned long long at = run + warp_scan_u64(sum) - sum;
        int first = INT_MAX;
#pragma unroll
        for (int e = 0; e < VN; ++e) {
          at += w[e];
          if (w[e] > 0 && at > target && first == INT_MAX) first = (owner_v + i * 32) * VN + e - R.head;
        }
        hit = __reduce_min_sync(0xffffffffu, first);
      }
    }
    if (warp == owner && lane == 0) a.out[R.row] = hit;
  }
  cluster.barrier_wait();                          // nobody leaves while its memory is read
}

template <typename T, int NT>
int launch_rows(SampleArgs a, const DeviceInfo& dev, cudaStream_t st, int C, int nvec) {
  a.cluster = C;
  a.iters = ((nvec + C - 1) / C + NT - 1) / NT;
  size_t smem = (size_t)a.iters * (NT / 32) * sizeof(double);
  const void* kern;
  if ((int64_t)nvec * Vec<T>::n <= (int64_t)C * kMaxSlice) {
    kern = reinterpret_cast<const void*>(&sample_kernel<T, NT>);
    smem += sizeof(SampleShared);
    if (smem < sizeof(FastShared<NT>)) smem = sizeof(FastShared<NT>);
  } else {
    kern = reinterpret_cast<const void*>(&sample_general_kernel<T, NT>);
  }
  if (int rc = allow_dynamic_smem(kern, dev, smem)) return rc;
  return launch_pdl_cluster(kern, dim3((unsigned)(a.batch * C)), dim3(NT), C, smem, st, &a);
}

template <typename T>
int launch_sample(const SampleArgs& a, const DeviceInfo& dev, cudaStream_t st) {
  constexpr int VN = Vec<T>::n;
  // vectors of a row: more when rows start inside a vector
  const int nvec = a.vocab / VN + (a.vocab % VN ? 2 : 0);
  // CTAs per row: slices of at most kMaxSlice logits, and more of them while SMs have none (few
  // rows: large CTAs) or fewer than kManyCtas, as long as every thread still has a vector.
  int C = 1;
  while (C < kMaxCluster && (int64_t)nvec * VN > (int64_t)C * kMaxSlice) C *= 2;
  if ((int64_t)a.batch * C > dev.num_sms) {
    while (C < kMaxCluster && (int64_t)a.batch * 2 * C <= kManyCtas * dev.num_sms && nvec / (2 * C) >= kManyThreads) C *= 2;
    return launch_rows<T, kManyThreads>(a, dev, st, C, nvec);
  }
  while (C < kMaxCluster && (int64_t)a.batch * 2 * C <= dev.num_sms && nvec / (2 * C) >= kFewThreads) C *= 2;
  return launch_rows<T, kFewThreads>(a, dev, st, C, nvec);
}

}  // namespace
}  // namespace dbk

using namespace dbk;

extern "C" int dbk_sample(const void* logits, const float* uniforms, const float* temperature,
                          const int32_t* top_k, const float* top_p, const float* min_p,
                          int64_t* tokens, int batch, int vocab, float temperature_all,
                          int top_k_all, float top_p_all, float min_p_all, int dtype,
                          void* stream) {
  if (dtype != DBK_F16 && dtype != DBK_BF16 && dtype != DBK_F32) return DBK_EDTYPE;
  if (batch < 0 || batch > (1 << 24) || vocab < 1 || vocab > kMaxVocab) return DBK_ESHAPE;
  if (!(temperature_all == temperature_all) || !(top_p_all == top_p_all) || !(min_p_all == min_p_all))
    return DBK_ESHAPE;
  if (batch == 0) return DBK_OK;
  if (!logits || !uniforms || !tokens) return DBK_ENULL;
  if (!aligned16(logits)) return DBK_EALIGN;
  const size_t rows = (size_t)batch * 4;
  const Span outs[] = {{tokens, 2 * rows}};
  const Span ins[] = {{logits, (size_t)batch * vocab * (dtype == DBK_F32 ? 4 : 2)}, {uniforms, rows},
                      {temperature, rows}, {top_k, rows}, {top_p, rows}, {min_p, rows}};
  if (outputs_overlap(outs, ins)) return DBK_ESHAPE;
  DeviceInfo dev;
  if (int rc = current_device_info(&dev)) return rc;
  SampleArgs a{};
  a.logits = logits; a.u = uniforms; a.temperature = temperature; a.top_k = top_k;
  a.top_p = top_p; a.min_p = min_p; a.out = tokens; a.batch = batch; a.vocab = vocab;
  a.temp = temperature_all; a.k = top_k_all; a.p = top_p_all; a.mp = min_p_all;
  int bits = 1;
  while ((1 << bits) < vocab + 1) ++bits;
  a.lower_bits = 62 - bits < 45 ? 45 - (62 - bits) : 0;        // a row's sum stays below 2^63
  a.unit = std::ldexp(1.0, 45 - a.lower_bits);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == DBK_F32) return launch_sample<float>(a, dev, st);
  return dtype == DBK_F16 ? launch_sample<__half>(a, dev, st) : launch_sample<__nv_bfloat16>(a, dev, st);
}
