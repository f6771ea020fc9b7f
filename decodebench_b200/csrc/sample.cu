// sample.cu - the next token of each request from its logits and one given random number.
//
//   w_i = exp((x_i - max x) / T);  order: larger x first, of equal ones the lower index first
//   top-k: the first k of the order;  top-p: of those the shortest prefix with >= p of their sum;
//   min-p: of those the ones with w_i >= min_p;  token = first index i with
//   sum_{kept j <= i} w_j > u * sum_{kept j} w_j.   T <= 0: the first of the order.
//
// No sort: the kept set is a prefix of the order, so it is given by one value and, among the
// logits that equal it, an index. The value is found by histograms (count and mass) of 256
// bins: first linear in (max - x) / T, then in the bits of the values of the bin the prefix
// ends in, until one value is left (two or three histograms, only the first of which sees
// more than a few logits). The draw walks 512-byte segments of the row in index order.
//
// A cluster of CTAs has a row, each a contiguous slice that it reads again in every pass: the
// slice comes from HBM once and then from L1/L2. Slices are joined through distributed shared
// memory, one cluster barrier per pass, every CTA computing the same decisions.
//
// Rounding. The answer is an index, and a cut that falls on another side of a sum changes it,
// so sums are 64-bit: weights above 2^-kFine of the largest by 64-bit exp(), smaller ones by
// 32-bit exponentials (2^-21 of at most 2^-kFine), histogram masses as 64-bit integers (whose
// order of addition does not matter), the rest in doubles in a fixed order.
#include <climits>
#include <cmath>
#include <cooperative_groups.h>

#include "common.cuh"
#include "dbk_internal.h"

namespace cg = cooperative_groups;

namespace dbk {
namespace {

constexpr int kSmpThreads = 512;
constexpr int kSmpWarps = kSmpThreads / 32;
constexpr int kBins = 256;
constexpr float kFine = 14.f;       // log2 distance up to which weights are 64-bit
constexpr float kFar = 46.f;        // and past which they are nothing
constexpr int kMaxCluster = 8;
constexpr int kMaxVocab = 1 << 20;
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
  double unit;                // fixed-point units of a weight of 1
};

struct Hist {
  unsigned long long mass[kBins];
  unsigned int count[kBins];
};

struct SampleShared {
  Hist hist[2];                       // alternate between passes: one cluster barrier each
  double sum[2];
  unsigned long long idx[2];
  float top[2];
  double warp_d[kSmpWarps];
  unsigned long long warp_m[kSmpWarps];
  unsigned int warp_c[kSmpWarps];
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
  __device__ __forceinline__ static void unpack(const uint4& v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y);
    f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  }
  __device__ __forceinline__ static float one(const float* p) { return *p; }
};
template <> struct Vec<__half> {
  static constexpr int n = 8;
  __device__ __forceinline__ static void unpack(const uint4& v, float (&f)[8]) { unpack8<__half>(v, f); }
  __device__ __forceinline__ static float one(const __half* p) { return __half2float(*p); }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int n = 8;
  __device__ __forceinline__ static void unpack(const uint4& v, float (&f)[8]) { unpack8<__nv_bfloat16>(v, f); }
  __device__ __forceinline__ static float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
};

__device__ __forceinline__ float fast_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__global__ void __launch_bounds__(kSmpThreads) sample_kernel(const __grid_constant__ SampleArgs a) {
  constexpr int VN = Vec<T>::n;
  __shared__ SampleShared sh;
  extern __shared__ double seg[];                 // [iters * warps] sums of 32 * VN logits
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int C = a.cluster, row = blockIdx.x / C, rank = blockIdx.x - row * C;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");

  const float temp = a.temperature ? __ldg(a.temperature + row) : a.temp;
  const int k = a.top_k ? __ldg(a.top_k + row) : a.k;
  const float p = a.top_p ? __ldg(a.top_p + row) : a.p;
  const float mp = fminf(a.min_p ? __ldg(a.min_p + row) : a.mp, 1.f);
  const bool greedy = !(temp > 0.f);

  // The row in whole 16-byte vectors: vector 0 starts `head` logits before it.
  const long long start = (long long)row * a.vocab;
  const int head = (int)(start % VN);
  const int nvec = (head + a.vocab + VN - 1) / VN;
  const int per = (nvec + C - 1) / C;
  const int v0 = min(rank * per, nvec), v1 = min(v0 + per, nvec);
  const T* base = static_cast<const T*>(a.logits) + (start - head);
  const long long room = (long long)a.batch * a.vocab - (start - head);    // logits from base to the end

  // Logits of one vector as floats; what is not of this row, and NaN, as -inf.
  auto load = [&](int v, float (&f)[VN]) {
    if (v >= v1) {
#pragma unroll
      for (int e = 0; e < VN; ++e) f[e] = -INFINITY;
      return;
    }
    const long long at = (long long)v * VN;
    if (at + VN <= room) {
      Vec<T>::unpack(*reinterpret_cast<const uint4*>(base + at), f);
    } else {
#pragma unroll
      for (int e = 0; e < VN; ++e) f[e] = at + e < room ? Vec<T>::one(base + at + e) : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < VN; ++e) f[e] = fmaxf(f[e], -INFINITY);            // NaN
    if (v == 0 || v == nvec - 1) {
#pragma unroll
      for (int e = 0; e < VN; ++e) {
        const int i = v * VN + e - head;
        if (i < 0 || i >= a.vocab) f[e] = -INFINITY;
      }
    }
  };

  int phase = 0;
  // ---------------------------------------------------------------- maximum
  float M = -INFINITY;
  for (int v = v0 + tid; v < v1; v += 4 * kSmpThreads) {
    float f[4][VN];
#pragma unroll
    for (int q = 0; q < 4; ++q) load(v + q * kSmpThreads, f[q]);
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int e = 0; e < VN; ++e) M = fmaxf(M, f[q][e]);
  }
  M = warp_max(M);
  float* wmax = reinterpret_cast<float*>(sh.warp_d);
  if (lane == 0) wmax[warp] = M;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kSmpWarps; ++w) M = fmaxf(M, wmax[w]);
    sh.top[0] = M;
  }
  cluster.sync();
  M = -INFINITY;
  for (int r = 0; r < C; ++r) M = fmaxf(M, *cluster.map_shared_rank(&sh.top[0], r));
  if (M == -INFINITY) {                            // nothing to choose from
    if (rank == 0 && tid == 0) a.out[row] = -1;
    cluster.sync();
    return;
  }

  const float cl = fmaxf(fminf(1.4426950408889634f / fmaxf(temp, 1e-38f), 1e30f), 1e-30f);
  const double dM = (double)M, dT = (double)temp;
  auto dist = [&](float x) { return (x == M ? 0.f : M - x) * cl; };          // log2 of max w / w
  auto fine = [&](float x) { return x == M ? 1.0 : exp(((double)x - dM) / dT); };
  auto fixed = [&](float x, float d) -> unsigned long long {
    const double w = d < kFine ? fine(x) : (double)fast_ex2(-d);
    return (unsigned long long)__double2ll_rn(w * a.unit);
  };

  // Find the first index, in index order, at which the running sum of value(x, i) over the whole
  // row passes `target` (target(total) of the row's sum). Every CTA gets the index.
  auto locate = [&](auto&& segment_value, auto&& element_value, auto&& target_of) -> int {
    const int segs = a.iters * kSmpWarps;
    for (int it = 0; it < a.iters; ++it) {
      float f[VN];
      const int v = v0 + it * kSmpThreads + tid;
      load(v, f);
      double s = segment_value(f, v * VN - head);
      if (__any_sync(0xffffffffu, s != 0.0)) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      }
      if (lane == 0) seg[it * kSmpWarps + warp] = s;
    }
    __syncthreads();
    const int chunk = (segs + kSmpThreads - 1) / kSmpThreads;
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
    for (int w = 0; w < kSmpWarps; ++w) {
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
      const int v = v0 + (s / kSmpWarps) * kSmpThreads + (s % kSmpWarps) * 32 + lane;
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
    double rest = 0.0;                              // mass of the logits `place` sends past the end
    auto histogram = [&](auto&& place, bool first) {
      const int ph = phase++ & 1;
      Hist& h = sh.hist[ph];
      for (int i = tid; i < kBins; i += kSmpThreads) { h.mass[i] = 0; h.count[i] = 0; }
      __syncthreads();
      double tail = 0.0;
      for (int v = v0 + tid; v < v1; v += kSmpThreads) {
        float f[VN];
        load(v, f);
        float far = 0.f;
#pragma unroll
        for (int e = 0; e < VN; ++e) {
          const float d = dist(f[e]);
          const int b = place(f[e], d);
          if (b >= 0) {
            atomicAdd(&h.count[b], 1u);
            atomicAdd(&h.mass[b], fixed(f[e], d));
          } else if (first) {
            far += fast_ex2(-d);
          }
        }
        tail += (double)far;
      }
      if (first) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) tail += __shfl_xor_sync(0xffffffffu, tail, o);
        if (lane == 0) sh.warp_d[warp] = tail;
        __syncthreads();
        if (tid == 0) {
          double t = 0.0;
          for (int w = 0; w < kSmpWarps; ++w) t += sh.warp_d[w];
          sh.sum[ph] = t;
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
        rest = 0.0;
        for (int r = 0; r < C; ++r) rest += *cluster.map_shared_rank(&sh.sum[ph], r);
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

    // The prefix that reaches `need` (a count, or a mass): sets kx and cut; returns its mass.
    // The first histogram has been made already.
    auto search = [&](bool count, unsigned long long need) -> unsigned long long {
      unsigned long long above = 0;                 // mass above the current range
      int b = crossing(count, need);
      bool wide = false;
      if (b == kBins) {                             // past the first histogram: the far one
        const unsigned long long got = count ? (unsigned long long)sh.cum_count[kBins - 1] : sh.cum_mass[kBins - 1];
        above = sh.cum_mass[kBins - 1];
        need -= got;
        __syncthreads();
        histogram(wide_bin, false);
        b = crossing(count, need);
        wide = true;
        if (b == kBins) { kx = 0; cut = -1; return above + sh.cum_mass[kBins - 1]; }   // everything
      }
      if (b > 0) { need -= count ? (unsigned long long)sh.cum_count[b - 1] : sh.cum_mass[b - 1]; above += sh.cum_mass[b - 1]; }
      __syncthreads();
      // Keys the bin can hold: its edges, four values more on each side (the distance has three
      // roundings), members by the bin itself.
      const float lo = wide ? kFine + b / kWide : b / kNear, hi = wide ? kFine + (b + 1) / kWide : (b + 1) / kNear;
      unsigned int khi = order_key(M - lo / cl * (1.f - 2e-6f)), klo = order_key(M - hi / cl * (1.f + 2e-6f));
      khi = khi > 0xffffffffu - 4 ? 0xffffffffu : khi + 4;
      klo = klo < 5 ? 1 : klo - 4;
      // from here up a key is surely not of a later bin
      const unsigned int sure = order_key(M - hi / cl * (1.f - 2e-6f)) + 4;
      const int bin = b;
      for (;;) {
        int shift = 0;
        while (((khi - klo) >> shift) >= kBins) ++shift;
        histogram([&](float x, float d) {
          if ((wide ? wide_bin(x, d) : near_bin(x, d)) != bin) return -1;
          const unsigned int key = order_key(x);
          return key > khi || key < klo ? -1 : (int)((khi - key) >> shift);
        }, false);
        b = crossing(count, need);
        if (b == kBins) b = kBins - 1;              // cannot be: the bin's members are in the range
        if (b > 0) { need -= count ? (unsigned long long)sh.cum_count[b - 1] : sh.cum_mass[b - 1]; above += sh.cum_mass[b - 1]; }
        const unsigned int n = sh.cum_count[b] - (b > 0 ? sh.cum_count[b - 1] : 0);
        const unsigned long long m = sh.cum_mass[b] - (b > 0 ? sh.cum_mass[b - 1] : 0);
        __syncthreads();
        khi -= (unsigned int)b << shift;
        const unsigned int width = 1u << shift;
        if (khi - klo >= width) klo = khi - width + 1;
        if ((n <= 1 && klo >= sure) || klo == khi) {
          // One logit, or n equal ones of which the first `take` by index are kept.
          unsigned long long take = n;
          if (n > 1) take = count ? need : (m / n == 0 ? n : (need + m / n - 1) / (m / n));
          if (take >= n) {
            kx = klo - 1;
            cut = -1;
            return above + m;
          }
          kx = klo;
          auto tie = [&](float x, int) { return order_key(x) == kx ? 1.0 : 0.0; };
          const double last = (double)take - 1.0;
          // (with the histogram still wanted by the caller this is only reached last)
          cut = locate(sum_of(tie), tie, [&](double) { return last; });
          return above + m / n * take;
        }
      }
    };

    histogram(near_bin, true);
    const unsigned long long near_mass = sh.cum_mass[kBins - 1];
    unsigned long long Z = near_mass + (unsigned long long)__double2ll_rn(rest * a.unit);
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
  auto kept = [&](float x, int i, float d) {
    if (d >= kFar) return false;
    if (cuts) {
      const unsigned int key = order_key(x);
      if (!(key > kx || (key == kx && i <= cut))) return false;
    }
    if (low) {
      const float w = fast_ex2(-d);
      if (w < mp * 0.999f) return false;
      if (w <= mp * 1.001f) return fine(x) >= (double)mp;
    }
    return true;
  };
  auto weight = [&](float x, int i) {
    const float d = dist(x);
    if (!kept(x, i, d)) return 0.0;
    return d < kFine ? fine(x) : (double)fast_ex2(-d);
  };
  const float u = fminf(fmaxf(__ldg(a.u + row), 0.f), 0x1.fffffep-1f);
  const int i = locate(sum_of(weight), weight, [&](double total) { return (double)u * total; });
  if (rank == 0 && tid == 0) a.out[row] = i;
  cluster.sync();
}

template <typename T>
int launch_sample(SampleArgs a, const DeviceInfo& dev, cudaStream_t st) {
  constexpr int VN = Vec<T>::n;
  // CTAs per row: more while the rows alone leave SMs idle and a slice keeps every thread busy.
  int C = 1;
  while (C < kMaxCluster && (int64_t)a.batch * C < 2 * dev.num_sms && a.vocab / (2 * C) >= kSmpThreads * VN) C *= 2;
  a.cluster = C;
  const int nvec = (a.vocab + VN - 1) / VN + 1;
  a.iters = ((nvec + C - 1) / C + kSmpThreads - 1) / kSmpThreads;
  const size_t smem = (size_t)a.iters * kSmpWarps * sizeof(double);
  const void* kern = reinterpret_cast<const void*>(&sample_kernel<T>);
  if (int rc = allow_dynamic_smem(kern, dev, smem)) return rc;
  return launch_pdl_cluster(kern, dim3((unsigned)(a.batch * C)), dim3(kSmpThreads), C, smem, st, &a);
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
  DeviceInfo dev;
  if (int rc = current_device_info(&dev)) return rc;
  SampleArgs a{};
  a.logits = logits; a.u = uniforms; a.temperature = temperature; a.top_k = top_k;
  a.top_p = top_p; a.min_p = min_p; a.out = tokens; a.batch = batch; a.vocab = vocab;
  a.temp = temperature_all; a.k = top_k_all; a.p = top_p_all; a.mp = min_p_all;
  int bits = 1;
  while ((1 << bits) < vocab + 1) ++bits;
  a.unit = std::ldexp(1.0, 62 - bits);             // a row's sum stays below 2^63
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == DBK_F32) return launch_sample<float>(a, dev, st);
  return dtype == DBK_F16 ? launch_sample<__half>(a, dev, st) : launch_sample<__nv_bfloat16>(a, dev, st);
}
