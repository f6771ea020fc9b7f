// paged.cu - what a scheduler step does around the attention of new tokens: page tables, slots
// and positions from the requests' lengths, and RoPE plus cache append of a packed chunk.
//
// Both kernels keep the next kernel in the stream from starting before they are done (no early
// release of dependents, writes fenced): dbk_flashdecode reads lengths, page tables and all but
// the newest cache rows ahead of its own dependency wait.
#include <climits>

#include "common.cuh"
#include "dbk_internal.h"

namespace dbk {
namespace {

// ------------------------------------------------------------------ page plan
//   seq_len[b] = ctx[b] + new[b]                 cu[b] = sum of new before b
//   pages b needs: ceil(seq_len / page_size), it has ceil(ctx / page_size); the ones it lacks
//   are the next entries of the free list, requests in order;
//   token t of request b, at position p: slot = table[b][p / page_size] * page_size + p % page_size.
// Every CTA computes both prefix sums over the requests by itself (a few KB from L2, one
// block scan) and then serves its share of table entries and tokens by binary search: one
// launch and no second pass. Bound by the latency of one launch: 3.5 us for 8 requests of one
// token, 5.6 us for 512 requests with 16,384 tokens.
constexpr int kPlanThreads = 256;
constexpr int kPlanMaxBatch = 16384;        // two int32 prefix arrays in shared memory

struct PlanArgs {
  const int32_t *ctx, *fresh, *free_list;
  int32_t* table;
  int32_t *seq_lens, *cu, *positions, *used;
  int64_t* slots;
  int batch, n_free, page_size, max_pages, tokens;
};

struct PlanSeq { long long ctx, add, have, want; };   // tokens; pages before and missing

__device__ __forceinline__ PlanSeq plan_seq(const PlanArgs& a, int b) {
  PlanSeq s;
  s.ctx = max(__ldcg(a.ctx + b), 0);
  s.add = max(__ldcg(a.fresh + b), 0);
  s.have = ((unsigned)s.ctx + (unsigned)(a.page_size - 1)) / (unsigned)a.page_size;
  const long long need = min((s.ctx + s.add + a.page_size - 1) / a.page_size, (long long)a.max_pages);
  s.want = max(need - s.have, 0ll);
  return s;
}

__device__ __forceinline__ int clip31(long long v) { return (int)min(v, (long long)INT_MAX); }

// Last i in [0, n) with at[i] <= v (at[0] = 0 <= v, ascending; of equal entries the last).
__device__ __forceinline__ int last_at(const int* at, int n, int v) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (at[mid] <= v) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(const __grid_constant__ PlanArgs a) {
  extern __shared__ int s_at[];                 // first token and first free page of each request
  int* tok_at = s_at;
  int* page_at = s_at + a.batch;
  __shared__ long long w_tok[kPlanThreads / 32], w_page[kPlanThreads / 32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int per = (a.batch + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
  long long tok = 0, page = 0;
  for (int b = b0; b < b1; ++b) {
    const PlanSeq s = plan_seq(a, b);
    tok += s.add;
    page += s.want;
  }
  long long it = tok, ip = page;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long vt = __shfl_up_sync(0xffffffffu, it, o), vp = __shfl_up_sync(0xffffffffu, ip, o);
    if (lane >= o) { it += vt; ip += vp; }
  }
  if (lane == 31) { w_tok[warp] = it; w_page[warp] = ip; }
  __syncthreads();
  long long all_tok = 0, all_page = 0, pre_tok = 0, pre_page = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    if (w == warp) { pre_tok = all_tok; pre_page = all_page; }
    all_tok += w_tok[w];
    all_page += w_page[w];
  }
  tok = pre_tok + it - tok;
  page = pre_page + ip - page;
  const bool first = blockIdx.x == 0;
  for (int b = b0; b < b1; ++b) {
    const PlanSeq s = plan_seq(a, b);
    tok_at[b] = clip31(tok);
    page_at[b] = clip31(page);
    if (first) {
      a.cu[b] = clip31(tok);
      a.seq_lens[b] = clip31(s.ctx + s.add);
    }
    tok += s.add;
    page += s.want;
  }
  if (first && tid == 0) {
    a.cu[a.batch] = clip31(all_tok);
    a.used[0] = clip31(all_page);
  }
  __syncthreads();

  const int gsize = gridDim.x * kPlanThreads, g0 = blockIdx.x * kPlanThreads + tid;
  const int n_page = clip31(all_page), n_tok = (int)min(all_tok, (long long)a.tokens);
  for (long long i = g0; i < n_page; i += gsize) {
    const int b = last_at(page_at, a.batch, (int)i);
    const PlanSeq s = plan_seq(a, b);
    a.table[(size_t)b * a.max_pages + s.have + (i - page_at[b])] = i < a.n_free ? __ldcg(a.free_list + i) : -1;
  }
  for (long long i = g0; i < a.tokens; i += gsize) {
    int pos = 0;
    long long slot = -1;
    if (i < n_tok) {
      const int b = last_at(tok_at, a.batch, (int)i);
      const PlanSeq s = plan_seq(a, b);
      pos = clip31(s.ctx + (i - tok_at[b]));
      const int lp = pos / a.page_size;
      int pg = -1;
      if (lp < s.have) {
        if (lp < a.max_pages) pg = __ldcg(a.table + (size_t)b * a.max_pages + lp);
      } else if (lp - s.have < s.want) {
        const long long f = page_at[b] + (lp - s.have);
        if (f < a.n_free) pg = __ldcg(a.free_list + f);
      }
      if (pg >= 0) slot = (long long)pg * a.page_size + (pos - lp * a.page_size);
    }
    a.positions[i] = pos;
    a.slots[i] = slot;
  }
  __threadfence();
}

// ------------------------------------------------------------------ RoPE + append
// Rotate-half pairs (i, i + 64), angle = position * inv_freq[i]: the angle is formed and reduced
// to [-pi, pi] in 64 bits (at position 10^5 a 32-bit product is off by 2^-8 rad), sine and
// cosine of the remainder in 32 bits. A warp has one token (or a share of its heads): lane
// (g, c) of 4 x 8 computes 2 of the 8 pairs of chunk c, gets the rest by shuffle, and then
// moves heads g, g + 4, ... as two 16-byte vectors each. One read and one write of every
// value: bound by HBM at many tokens (8,192 tokens, 64 / 8 heads: 58.4 us, 5.7 TB/s, 88 % of a
// plain copy), by latency at few (then heads are spread over warps; 77 tokens: 3.1 us).
constexpr int kRopeWarps = 8;

struct RopeArgs {
  const void* qkv;
  const int32_t* pos;
  const int64_t* slots;
  const float* inv_freq;
  void *q, *k, *v;
  int tokens, hq, hkv, page_size, shares;      // warps per token
  long long n_slots;
};

template <typename T>
__global__ void __launch_bounds__(kRopeWarps * 32) rope_append_kernel(const __grid_constant__ RopeArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, g = lane >> 3, c = lane & 7;
  const long long w = (long long)blockIdx.x * kRopeWarps + (threadIdx.x >> 5);
  const long long t = w / a.shares;
  const int share = (int)(w - t * a.shares);
  if (t >= a.tokens) return;
  const int pos = __ldcg(a.pos + t);
  const long long slot = __ldcg(a.slots + t);
  float cs[8], sn[8];
  {
    float c2[2], s2[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const double turns = (double)pos * (double)__ldg(a.inv_freq + c * 8 + g * 2 + e) * 0.15915494309189535;
      const float rem = (float)((turns - rint(turns)) * 6.283185307179586);
      sincosf(rem, &s2[e], &c2[e]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int src = ((e >> 1) << 3) | c;
      cs[e] = __shfl_sync(0xffffffffu, c2[e & 1], src);
      sn[e] = __shfl_sync(0xffffffffu, s2[e & 1], src);
    }
  }
  const int heads = a.hq + 2 * a.hkv, rot = a.hq + a.hkv;
  const bool keep = slot >= 0 && slot < a.n_slots;
  const long long page = keep ? slot / a.page_size : 0;
  const int off = keep ? (int)(slot - page * a.page_size) : 0;
  const T* src = static_cast<const T*>(a.qkv) + (size_t)t * heads * 128 + c * 8;
  auto move = [&](int h, const uint4& lo4, const uint4& hi4) {
    T* dst;
    if (h < a.hq) {
      dst = static_cast<T*>(a.q) + ((size_t)t * a.hq + h) * 128;
    } else {
      if (!keep) return;
      const int kh = h < rot ? h - a.hq : h - rot;
      dst = static_cast<T*>(h < rot ? a.k : a.v) +
            (((size_t)page * a.hkv + kh) * a.page_size + off) * 128;
    }
    uint4 ol = lo4, oh = hi4;
    if (h < rot) {
      float x[8], y[8], u[8], v[8];
      unpack8<T>(lo4, x);
      unpack8<T>(hi4, y);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        u[e] = x[e] * cs[e] - y[e] * sn[e];
        v[e] = y[e] * cs[e] + x[e] * sn[e];
      }
      ol = make_uint4(Mma<T>::pack(u[0], u[1]), Mma<T>::pack(u[2], u[3]), Mma<T>::pack(u[4], u[5]),
                      Mma<T>::pack(u[6], u[7]));
      oh = make_uint4(Mma<T>::pack(v[0], v[1]), Mma<T>::pack(v[2], v[3]), Mma<T>::pack(v[4], v[5]),
                      Mma<T>::pack(v[6], v[7]));
    }
    *reinterpret_cast<uint4*>(dst + c * 8) = ol;
    *reinterpret_cast<uint4*>(dst + 64 + c * 8) = oh;
  };
  const int stride = 4 * a.shares;
  for (int h = share * 4 + g; h < heads; h += 4 * stride) {
    uint4 lo4[4], hi4[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (h + k * stride < heads) {
        lo4[k] = ldg_nc_v4(src + (size_t)(h + k * stride) * 128);
        hi4[k] = ldg_nc_v4(src + (size_t)(h + k * stride) * 128 + 64);
      }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (h + k * stride < heads) move(h + k * stride, lo4[k], hi4[k]);
  }
  __threadfence();
}

}  // namespace
}  // namespace dbk

using namespace dbk;

extern "C" int dbk_page_plan(const int32_t* ctx_lens, const int32_t* new_lens,
                             const int32_t* free_pages, int32_t* page_table, int32_t* seq_lens,
                             int32_t* cu_seqlens, int32_t* positions, int64_t* slots,
                             int32_t* used, int batch, int n_free, int page_size,
                             int max_pages_per_seq, int tokens, void* stream) {
  if (!ctx_lens || !new_lens || !page_table || !seq_lens || !cu_seqlens || !used) return DBK_ENULL;
  if (batch < 1 || batch > kPlanMaxBatch || n_free < 0 || page_size < 1 || max_pages_per_seq < 1 ||
      tokens < 0 || (int64_t)batch * max_pages_per_seq > INT_MAX)
    return DBK_ESHAPE;
  if ((n_free > 0 && !free_pages) || (tokens > 0 && (!positions || !slots))) return DBK_ENULL;
  const size_t lens = (size_t)batch * 4;
  const Span outs[] = {{page_table, lens * max_pages_per_seq}, {seq_lens, lens}, {cu_seqlens, lens + 4},
                       {positions, (size_t)tokens * 4}, {slots, (size_t)tokens * 8}, {used, 4}};
  const Span ins[] = {{ctx_lens, lens}, {new_lens, lens}, {free_pages, (size_t)n_free * 4}};
  if (outputs_overlap(outs, ins)) return DBK_ESHAPE;
  DeviceInfo dev;
  if (int rc = current_device_info(&dev)) return rc;
  PlanArgs a{};
  a.ctx = ctx_lens; a.fresh = new_lens; a.free_list = free_pages; a.table = page_table;
  a.seq_lens = seq_lens; a.cu = cu_seqlens; a.positions = positions; a.slots = slots; a.used = used;
  a.batch = batch; a.n_free = n_free; a.page_size = page_size; a.max_pages = max_pages_per_seq;
  a.tokens = tokens;
  const size_t smem = (size_t)2 * batch * sizeof(int);
  const void* kern = reinterpret_cast<const void*>(&page_plan_kernel);
  if (int rc = allow_dynamic_smem(kern, dev, smem)) return rc;
  const int64_t most = tokens > batch ? tokens : batch;
  int64_t grid = (most + kPlanThreads - 1) / kPlanThreads;
  if (grid > dev.num_sms) grid = dev.num_sms;
  return launch_pdl(kern, dim3((unsigned)grid), dim3(kPlanThreads), smem,
                    static_cast<cudaStream_t>(stream), &a);
}

extern "C" int dbk_rope_append(const void* qkv, const int32_t* positions, const int64_t* slots,
                               const float* inv_freq, void* q_out, void* k_cache, void* v_cache,
                               int tokens, int n_q_heads, int n_kv_heads, int head_dim,
                               int num_pages, int page_size, int dtype, void* stream) {
  if (!inv_freq || !k_cache || !v_cache) return DBK_ENULL;
  if (dtype != DBK_F16 && dtype != DBK_BF16) return DBK_EDTYPE;
  if (head_dim != 128 || tokens < 0 || n_q_heads < 1 || n_kv_heads < 1 || n_q_heads > 65536 ||
      n_kv_heads > 65536 || num_pages < 1 || page_size < 1)
    return DBK_ESHAPE;
  if (tokens == 0) return DBK_OK;
  if (!qkv || !positions || !slots || !q_out) return DBK_ENULL;
  if (!aligned16(qkv) || !aligned16(q_out) || !aligned16(k_cache) || !aligned16(v_cache))
    return DBK_EALIGN;
  const size_t cache = cache_bytes(num_pages, n_kv_heads, page_size);
  const Span outs[] = {{q_out, (size_t)tokens * n_q_heads * 256}, {k_cache, cache}, {v_cache, cache}};
  const Span ins[] = {{qkv, (size_t)tokens * (n_q_heads + 2 * n_kv_heads) * 256}, {positions, (size_t)tokens * 4},
                      {slots, (size_t)tokens * 8}, {inv_freq, 256}};
  if (outputs_overlap(outs, ins)) return DBK_ESHAPE;
  DeviceInfo dev;
  if (int rc = current_device_info(&dev)) return rc;
  RopeArgs a{};
  a.qkv = qkv; a.pos = positions; a.slots = slots; a.inv_freq = inv_freq;
  a.q = q_out; a.k = k_cache; a.v = v_cache;
  a.tokens = tokens; a.hq = n_q_heads; a.hkv = n_kv_heads; a.page_size = page_size;
  a.n_slots = (long long)num_pages * page_size;
  // Warps per token: as many as the heads feed (4 heads at a time each) while the tokens alone
  // leave the GPU short of warps.
  const int heads = n_q_heads + 2 * n_kv_heads, most = (heads + 3) / 4;
  int shares = 1;
  while (shares * 2 <= most && (int64_t)tokens * shares * 2 <= (int64_t)dev.num_sms * 16) shares *= 2;
  a.shares = shares;
  const int64_t grid = ((int64_t)tokens * shares + kRopeWarps - 1) / kRopeWarps;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const void* kern = dtype == DBK_F16 ? reinterpret_cast<const void*>(&rope_append_kernel<__half>)
                                      : reinterpret_cast<const void*>(&rope_append_kernel<__nv_bfloat16>);
  return launch_pdl(kern, dim3((unsigned)grid), dim3(kRopeWarps * 32), 0, st, &a);
}
