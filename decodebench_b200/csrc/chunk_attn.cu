// chunk_attn.cu - attention of chunks of new tokens over a paged (or contiguous) KV cache.
//
//   out[t, h] = sum_{j <= p} softmax_j(scale * q[t, h] . K[j, h/G]) V[j, h/G]
//
// for the new token at position p of its sequence (p = seq_len - new + i for the i-th of its
// `new` tokens, whose K and V are in the cache already). head_dim 128, fp16 / bf16.
//
// Work. A tile is 128 rows = (token, head of one KV group): T = 128 / G tokens x G heads, so
// every K/V byte that is brought in serves all G heads. Two tiles (2T tokens) form an item;
// S = Q K^T and O += P V of both run on tcgen05 with M = N = 128, and while the tensor cores
// work on one tile the other tile's softmax runs (one warpgroup per tile, one thread per row,
// running maximum and sum in fp32 registers). TMEM holds S0, S1, O0, O1 (4 x 128 columns);
// P overwrites its own S as 16-bit pairs (high parts in the first 64 columns, low parts behind them)
// and is the PV product's A operand straight from TMEM.
// An item with one tile only gives both warpgroups that tile and every other key block, and
// merges the two halves from TMEM at its end. Beside the two softmax warpgroups a warp brings
// tiles by TMA, one looks over them, one issues the MMAs, one hands out the items.
//
// Weights. Each goes to the tensor cores as the sum of two 16-bit values, so that the result's
// rounding is the only one of its size (root-mean-square error against 64 bits: that of a result
// rounded once, to four digits); as one value it is 1.3 times that, and faster (below: "one part").
//
// What bounds it. A block of an item with two tiles is 2 x 3 x 128^3 products, 3,072 cycles of the
// tensor core, and 2,048 of the exponential unit; it takes ~4,300 (tensor pipe active 71 % of the
// cycles of a prompt of 8,192 tokens; one part: 2,048, ~3,400): the two tiles' chains (S -> softmax ->
// PV -> next S) overlap but for their ends. One prompt of 16,384 tokens, 32 / 8 heads: 2.40 to 2.77 ms
// from call to call, around 1,650 MHz under the power limit (one part: 1.72 to 2.07), 1.19 to 1.37
// PFLOP/s of issued products (a plain square library product: 1.68 in bursts, 1.40 sustained). Few
// rows over a long cache are bound by HBM: 8 requests of one token at 16,384, 64 / 8 heads: 103 us,
// 5.2 TB/s. Short calls pay ~9 us from launch to the first product (cold code, lengths, cuts, first
// tiles) and ~4 for the join; the pages' size makes no difference (24 ragged prompts in pages of
// 16, 32, 64 and 128: 298 to 309 us).
// Measured and not kept: a share of the exponentials by polynomial on the FMA pipe (1/8: +2 %,
// 1/2: +13 %), two issuing threads (+18 %: the tiles fall into step), no row maximum but a bound
// from the weights' sum (+12 %), S loaded from TMEM in two halves (+10 %).
//
// Split. The (item, 128-key block) units of the whole batch form one line, weighted by their
// cost; CTA c of at most one per SM takes the c-th equal part of it, whatever the lengths are
// (they are read on the device: no host sync). A part that begins or ends inside an item
// leaves an fp32 partial with its maximum and sum in the workspace, and a second kernel joins
// the partials in order, so results do not depend on timing.
#include <climits>
#include <type_traits>

#include "common.cuh"
#include "dbk_internal.h"

namespace dbk {
namespace {

constexpr int kRows = 128;                  // rows of a tile (MMA M)
constexpr int kKeys = 128;                  // keys of a block (MMA N of S, K of PV)
constexpr int kHd = 128;                    // head dim
constexpr int kHalf = 128 * 128;            // bytes of 128 rows x 64 16-bit values (one swizzled half)
constexpr int kTile = 2 * kHalf;            // a Q, K or V tile
constexpr int kMaxBatch = 65536;            // a CTA looks over all lengths, a part over its empty sequences
constexpr int kRing = 5;                    // K/V tiles in flight
constexpr int kThreadsCa = 384;             // 2 softmax warpgroups; TMA, MMA, inspecting, item warps
// Registers: launched with 168 a thread (384 x 168 of the SM's 65,536); the third warpgroup keeps
// 72 (fewer and its roles spill), which lets a softmax thread hold its row of S (128 values):
// 256 x 216 + 128 x 72 = 384 x 168.
constexpr int kRegsSoftmax = 216, kRegsOther = 72;
static_assert(256 * kRegsSoftmax + 128 * kRegsOther <= kThreadsCa * 168, "register split");
// Items the item warp is ahead at most. The inspecting warp is up to four items (of one block) ahead of
// the softmax warps that read its note `odd`, so notes are kept for more than five.
constexpr int kItems = 8;
constexpr int kMinBox = 8;                  // rows of the smallest TMA box
constexpr int kOver = 256;                  // an item's fixed cost, in keys
constexpr int kOneTile = 5;                 // cost of a key of a one-tile item, in eighths
constexpr int kSnap = 2;                    // a cut this near an item's end moves to the end
constexpr long long kMinWork = 1024;        // least work of a CTA, in keys
// Neighbouring cuts are at least kMinWork apart and move by less than half of that, so no part
// between two others is empty (the join walks the parts of an item one by one).
static_assert(kMinWork > kOver + (2 * kSnap + 1) * 128, "cuts could meet");
constexpr float kLog2eF = 1.4426950408889634f;

struct ChunkArgs {
  CUtensorMap qmap, kmap, vmap;
  const int32_t* cu;         // [batch + 1] first row of each sequence's new tokens
  const int32_t* lens;       // [batch] tokens in the cache, the new ones included
  const int32_t* pages;      // [batch, max_pages] or nullptr (contiguous)
  const void* v;             // the cache's values
  void* out;
  float* part_o;             // [2 * grid][32][slot_rows][4]: column fours, rows, columns
  float2* part_ml;           // [2 * grid][slot_rows] (maximum in log2 units, sum)
  int4* desc;                // [2 * grid] {first token, tokens, kv head, 0 | 1 goes on | 2 last}
  int batch, tokens, hq, hkv, G, T;
  int cap;                   // tokens a sequence can have in the cache
  int page_size, max_pages, num_pages, box, total_rows, slot_rows;
  unsigned page_mul;         // floor(2^page_shift / (page_size / 8)) + 1; 0 for a contiguous cache
  int page_shift;
  float cs;                  // scale * log2(e)
};

// ------------------------------------------------------------------ the line of work
struct Seq {
  int t0, n, len;            // first row, new tokens, cached tokens
  int items;
  long long per_head;        // cost of one KV head
};

__device__ __forceinline__ long long cost_before(const ChunkArgs& a, const Seq& s, int i) {
  const long long base = max(s.len - s.n, 0) + kOver, w = 2 * a.T;
  return i * base + w * i * (i + 1ll) / 2;
}

__device__ __forceinline__ Seq load_seq(const ChunkArgs& a, int b) {
  Seq s;
  s.t0 = min(max(__ldcg(a.cu + b), 0), a.tokens);
  const int t1 = min(max(__ldcg(a.cu + b + 1), s.t0), a.tokens);
  s.n = t1 - s.t0;
  s.len = min(max(__ldcg(a.lens + b), 0), a.cap);
  s.items = (s.n + 2 * a.T - 1) / (2 * a.T);
  s.per_head = 0;
  if (s.n > 0) {
    const int rem = s.n - (s.items - 1) * 2 * a.T;
    const long long seen = max(s.len, s.n);
    s.per_head = cost_before(a, s, s.items - 1) + kOver + (rem <= a.T ? (seen * kOneTile + 7) / 8 : seen);
  }
  return s;
}

struct Item {
  int tok, ntok;             // first row, rows' tokens
  int pos;                   // position of the first token (negative: sees nothing)
  int b, h;
  int kend;                  // keys that some row sees
  int nblk, b0, b1;          // key blocks of the item, and of this CTA's piece
  bool two;
};

__device__ __forceinline__ void item_shape(const ChunkArgs& a, const Seq& s, int i, Item& it) {
  const int first = i * 2 * a.T;
  it.tok = s.t0 + first;
  it.ntok = min(s.n - first, 2 * a.T);
  it.two = it.ntok > a.T;
  it.pos = s.len - s.n + first;
  it.kend = max(it.pos + it.ntok, 0);
  it.nblk = max(1, (it.kend + kKeys - 1) / kKeys);
}

// First (b, h, item, block) of the part that starts at cost `off` inside sequence b, and the
// sequence it is in. Quotients and the root of the quadratic cost_before come from 32-bit floats and are
// then put right: wide divisions or a search take thousands of cycles before a CTA's start.
__device__ __forceinline__ int4 locate(const ChunkArgs& a, int b, long long off, Seq& s) {
  s = load_seq(a, b);
  int h = min((int)__fdividef((float)off, (float)s.per_head), a.hkv - 1);
  off -= h * s.per_head;
  while (off < 0) { --h; off += s.per_head; }
  while (off >= s.per_head) { ++h; off -= s.per_head; }
  const float base = (float)(max(s.len - s.n, 0) + kOver + a.T), w = (float)a.T;
  int i = (int)((__fsqrt_rn(base * base + 4.f * w * (float)off) - base) * __frcp_rn(2.f * w));
  i = min(max(i, 0), s.items - 1);
  while (i > 0 && cost_before(a, s, i) > off) --i;
  while (i + 1 < s.items && cost_before(a, s, i + 1) <= off) ++i;
  off -= cost_before(a, s, i);
  Item it;
  item_shape(a, s, i, it);
  const int left = (int)min(off, (long long)INT_MAX / 16);
  int blk = it.two ? (left + kKeys / 2) / kKeys : (left * 8 + kOneTile * kKeys / 2) / (kOneTile * kKeys);
  if (blk < kSnap) blk = 0;
  else if (blk + kSnap > it.nblk) {
    blk = 0;
    if (++i == s.items) {
      i = 0;
      if (++h == a.hkv) {
        h = 0;
        if (++b < a.batch) s = load_seq(a, b);   // (it may have no new token: the walk looks further)
      }
    }
  }
  return make_int4(b, h, i, blk);
}

// Key block `blk` has keys that some row of the item does not see.
__device__ __forceinline__ bool uneven(const Item& it, int blk) { return (blk + 1) * kKeys > it.pos + 1; }

// The items of one CTA's part, in order. A whole warp walks.
struct Walk {
  int4 at, end;
  Seq s;
  __device__ __forceinline__ Walk(const ChunkArgs& a, int4 from, int4 to, const Seq& first) : at(from), end(to), s(first) {
    if (at.x < a.batch && s.n == 0) seek(a);
  }
  // To the next sequence with a new token: 32 are looked at together (one after the other, two
  // dependent loads each, a batch of 20,000 empty ones took 2.1 ms; this way 0.17).
  __device__ __forceinline__ void seek(const ChunkArgs& a) {
    int b = at.x + 1;
    for (; b < a.batch; b += 32) {
      const int j = b + (threadIdx.x & 31);
      bool some = false;
      if (j < a.batch) {
        const int t0 = min(max(__ldcg(a.cu + j), 0), a.tokens);
        some = min(__ldcg(a.cu + j + 1), a.tokens) > t0;
      }
      const unsigned int m = __ballot_sync(0xffffffffu, some);
      if (m) { b += __ffs(m) - 1; break; }
    }
    at = make_int4(min(b, a.batch), 0, 0, 0);
    if (b < a.batch) s = load_seq(a, b);
  }
  __device__ __forceinline__ bool next(const ChunkArgs& a, Item& it) {
    if (at.x >= a.batch) return false;
    const int ahead = at.x != end.x ? at.x - end.x : at.y != end.y ? at.y - end.y : at.z - end.z;
    const bool last = ahead == 0;
    if (ahead > 0 || (last && at.w >= end.w)) return false;
    item_shape(a, s, at.z, it);
    it.b = at.x;
    it.h = at.y;
    it.b0 = at.w;
    it.b1 = last ? end.w : it.nblk;
    if (last) { at.w = end.w; return true; }
    at.w = 0;
    if (++at.z == s.items) {
      at.z = 0;
      if (++at.y == a.hkv) seek(a);
    }
    return true;
  }
};

// ------------------------------------------------------------------ tcgen05 / TMA
// Shared-memory matrix descriptors, 128-byte swizzle, as a low word (address and leading offset, in
// units of 16 bytes) over one high word (8-row groups 1024 bytes apart, version, swizzle).
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_kmajor(uint32_t saddr) { return ((saddr >> 4) & 0x3FFF) | (1u << 16); }
// MN-major operand (V: 64 head dims per 128-byte row, one row per key): the second 64 dims lie
// kHalf bytes on (leading offset), the next 8 keys 1024 bytes on (stride offset).
__device__ __forceinline__ uint32_t desc_mnmajor(uint32_t saddr) {
  return ((saddr >> 4) & 0x3FFF) | ((uint32_t)(kHalf >> 4) << 16);
}
__device__ __forceinline__ uint32_t idesc_128x128(bool bf16, bool b_mn) {
  const uint32_t f = bf16 ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | ((b_mn ? 1u : 0u) << 16) | ((128u >> 3) << 17) |
         ((128u >> 4) << 24);
}
// The MMA warp runs as a whole, converged, and each of these is issued by the thread that
// elect.sync chose (`one`). Issued from a branch for one thread instead, with a branch after
// every wait, 128 x 128 x 16 MMAs went out every 94 cycles in a loop with four waits for 16 of
// them; this way every 66 (the tensor core takes 64).
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}
__device__ __forceinline__ void mma_ss(uint32_t one, uint32_t d, uint32_t a_lo, uint32_t b_lo,
                                       uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "mov.b64 x, {%1, %5};\n\tmov.b64 y, {%2, %5};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}"
      ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(acc), "n"(kDescHi), "r"(one) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t one, uint32_t d, uint32_t ta, uint32_t b_lo,
                                       uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "mov.b64 y, {%2, %5};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}"
      ::"r"(d), "r"(ta), "r"(b_lo), "r"(idesc), "r"(acc), "n"(kDescHi), "r"(one) : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t one, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
      ::"r"(smem_u32(bar)), "r"(one) : "memory");
}
// Bounded wait without a branch on its outcome: true if the phase completed within `polls`.
__device__ __forceinline__ bool poll_wait(uint64_t* bar, uint32_t parity, uint32_t polls) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .u32 i;\n\tmov.u32 i, %3;\n\t"
      "DBK_POLL:\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t@p bra DBK_DONE;\n\t"
      "sub.u32 i, i, 1;\n\tsetp.ne.u32 q, i, 0;\n\t@q bra DBK_POLL;\n\t"
      "DBK_DONE:\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity), "r"(polls) : "memory");
  return ok != 0;
}
__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tma_2d(void* dst, const void* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];"
      ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tma_3d(void* dst, const void* map, int x, int y, int z,
                                       uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar)) : "memory");
}

#define DBK_R8(v, o) "=r"(v[o]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3]), \
                     "=r"(v[o + 4]), "=r"(v[o + 5]), "=r"(v[o + 6]), "=r"(v[o + 7])
#define DBK_I8(v, o) "r"(v[o]), "r"(v[o + 1]), "r"(v[o + 2]), "r"(v[o + 3]), \
                     "r"(v[o + 4]), "r"(v[o + 5]), "r"(v[o + 6]), "r"(v[o + 7])
// This warp's 32 lanes x 32 columns.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : DBK_R8(v, 0), DBK_R8(v, 8), DBK_R8(v, 16), DBK_R8(v, 24) : "r"(addr));
}
__device__ __forceinline__ void tmem_ld16u(uint32_t addr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15}, [%16];"
      : DBK_R8(v, 0), DBK_R8(v, 8) : "r"(addr));
}
__device__ __forceinline__ void tmem_st(uint32_t addr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15,%16};"
      ::"r"(addr), DBK_I8(v, 0), DBK_I8(v, 8) : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t addr, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"r"(addr), DBK_I8(v, 0) : "memory");
}
// Waits for this thread's TMEM loads; the values pass through it, so no use can move before it.
#define DBK_RW8(v, o) "+r"(v[o]), "+r"(v[o + 1]), "+r"(v[o + 2]), "+r"(v[o + 3]), \
                      "+r"(v[o + 4]), "+r"(v[o + 5]), "+r"(v[o + 6]), "+r"(v[o + 7])
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : DBK_RW8(v, 0), DBK_RW8(v, 8), DBK_RW8(v, 16), DBK_RW8(v, 24) :: "memory");
}
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : DBK_RW8(v, 0), DBK_RW8(v, 8) :: "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void st_32(void* p, const uint32_t (&v)[8]) {   // one 32-byte sector
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 values in one 64-bit register: one instruction for both (same rounding as single).
using f2 = unsigned long long;
__device__ __forceinline__ f2 f2_make(float a, float b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2_split(f2 v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ f2 f2_fma(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f2 f2_add(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// A weight as the sum of two 16-bit values, a pair of keys at a time: its leading bits (8 in bf16, 11
// in fp16), cut off, and the rest, rounded: 2^-16 of the weight are left, or 2^-22 (in fp16 no
// less than 2^-25 of 1). 2^-24 of the weight is added to the rest, for 0 * Inf is NaN: the low part
// of a weight must not be 0 where a row sees an infinite V.
template <typename T>
__device__ __forceinline__ uint32_t high_parts(float x0, float x1) {
  uint32_t r;
  if constexpr (std::is_same<T, __nv_bfloat16>::value) r = __byte_perm(__float_as_uint(x0), __float_as_uint(x1), 0x7632);
  else asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(x1), "f"(x0));
  return r;
}
template <typename T>
__device__ __forceinline__ uint32_t low_parts(float x0, float x1) {
  constexpr uint32_t kLead = std::is_same<T, __nv_bfloat16>::value ? 0xffff0000u : 0xffffe000u;
  constexpr float kLess = -(1.f - 0x1p-24f);
  const f2 h = f2_make(__uint_as_float(__float_as_uint(x0) & kLead), __uint_as_float(__float_as_uint(x1) & kLead));
  f2_split(f2_fma(h, f2_make(kLess, kLess), f2_make(x0, x1)), x0, x1);
  return Mma<T>::pack(x0, x1);
}
// kGrow: log2 growth of a row's maximum over the one in use that forces a rescale; kBias: log2 of the
// weight at the maximum in use. fp16 has no value between 0 and 2^-24, and l counts what P V then
// lacks (30,000 equal keys 17 nats below a sink whose v is 0, with weights up to 2^8: 14 times the
// half step of a rounded weight off). Here weights reach up to 2^15, so that those down to 2^-25 of the
// largest have all 11 bits and the others are off by 2^-36 of it at most. Sums, O and partials
// scale alike. A rescale at 2^4 instead of 2^8 costs nothing measurable.
template <typename T> constexpr float kGrow = std::is_same<T, __nv_bfloat16>::value ? 8.f : 4.f;
template <typename T> constexpr float kBias = std::is_same<T, __nv_bfloat16>::value ? 0.f : 11.f;

// The whole warp waits, and agrees on the outcome.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, code));
}

struct Shared {
  uint64_t full[kRing], empty[kRing];
  uint64_t ready[kRing];
  uint64_t q_full, q_empty;
  uint64_t s_full[2], p_full[2][2], o_full[2], o_free[2], half_ready;
  uint64_t teardown, drain;
  uint32_t tmem;
  volatile int bail;
  long long wsum[kThreadsCa / 32], before[kThreadsCa / 32];
  long long total;
  int4 cut[2];
  Seq first;                 // the sequence of the first cut
  Item items[kItems];
  uint64_t item_full[kItems], item_empty[kItems];
  int odd[kItems];           // some V value of the item's later tokens is not finite (see add_odd)
  float2 half_ml[kRows];     // the second warpgroup's maximum and sum (one-tile items)
};

// What values of V that are not finite add to one row that sees them: the inspecting warp took those
// of the chunk's later tokens out of the tiles (0 * Inf would reach every row), so each row adds
// its own, from global memory, to what it has written. The weight is positive and the sum is not
// finite whatever it is, so it counts as 1. One thread; at most 2 T keys, whatever the length.
template <typename T>
__device__ __noinline__ void add_odd(const ChunkArgs& a, Item it, int vis, float inv, T* dst, float* pdst) {
  const int j0 = max(it.pos + 1, it.b0 * kKeys), j1 = min(vis, it.b1 * kKeys);
  for (int d = 0; d < kHd; d += 8) {
    float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    bool some = false;
    for (int j = max(j0, 0); j < j1; ++j) {
      int pg = it.b, off = j;
      if (a.pages) {
        pg = __ldcg(a.pages + (size_t)it.b * a.max_pages + j / a.page_size);
        off = j % a.page_size;
        if (pg < 0 || pg >= a.num_pages) continue;
      }
      float y[8];
      unpack8<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(a.v) +
                                                 (((size_t)pg * a.hkv + it.h) * a.page_size + off) * kHd + d), y);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (!isfinite(y[e])) { o[e] += y[e]; some = true; }
    }
    if (!some) continue;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (o[e] == 0.f) continue;
      if (dst) dst[d + e] = Elem<T>::from_f(Elem<T>::to_f(dst[d + e]) + o[e] * inv);
      else pdst[(size_t)((d + e) / 4) * a.slot_rows * 4 + (d + e) % 4] += o[e];
    }
  }
}

static_assert(sizeof(Shared) <= 2048, "shared memory: 227 KB less 7 tiles and the alignment");

// ------------------------------------------------------------------ the kernel
template <typename T, bool kTwo>
__global__ void __launch_bounds__(kThreadsCa, 1)
chunk_attention_kernel(const __grid_constant__ ChunkArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sq = smem;                                  // Q tiles 0 and 1
  uint8_t* ring = smem + 2 * kTile;
  Shared& sh = *reinterpret_cast<Shared*>(ring + kRing * kTile);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < kRing; ++i) { mbar_init(&sh.full[i], 1); mbar_init(&sh.empty[i], 2); mbar_init(&sh.ready[i], 1); }
    mbar_init(&sh.q_full, 1);
    mbar_init(&sh.q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_full[i][0], 4);
      mbar_init(&sh.p_full[i][1], 4);
      mbar_init(&sh.o_full[i], 1);
      mbar_init(&sh.o_free[i], 4);
      sh.cut[i] = make_int4(a.batch, 0, 0, 0);
    }
    for (int i = 0; i < kItems; ++i) { mbar_init(&sh.item_full[i], 1); mbar_init(&sh.item_empty[i], 11); }
    mbar_init(&sh.half_ready, 4);
    mbar_init(&sh.teardown, kThreadsCa / 32);
    mbar_init(&sh.drain, 1);
    fence_barrier_init();
    sh.bail = 0;
    prefetch_tmap(&a.qmap);
    prefetch_tmap(&a.kmap);
    prefetch_tmap(&a.vmap);
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;"
                 ::"r"(smem_u32(&sh.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // Lengths, q and the cache come from earlier kernels: nothing is read before they are done.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");

  // This CTA's two cuts of the line: cost of each sequence, prefix sum, then the thread whose
  // sequences a cut falls in locates it.
  const int chunk = (a.batch + kThreadsCa - 1) / kThreadsCa;
  const int sb0 = min(tid * chunk, a.batch), sb1 = min(sb0 + chunk, a.batch);
  long long mine = 0;
  for (int b = sb0; b < sb1; ++b) mine += load_seq(a, b).per_head * a.hkv;
  long long inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  if (lane == 31) sh.wsum[warp] = inc;
  fence_before();
  __syncthreads();
  fence_after();
  if (tid == 0) {
    long long t = 0;
    for (int w = 0; w < kThreadsCa / 32; ++w) { sh.before[w] = t; t += sh.wsum[w]; }
    sh.total = t;
  }
  __syncthreads();
  const long long W = sh.total;
  const int parts = (int)min((long long)gridDim.x, max(1ll, W / kMinWork));   // (a power of two)
  {
    const long long lo = sh.before[warp] + inc - mine;
    // W / parts to 46 bits, the same in every CTA: cuts agree and ascend.
    double inv = (double)__frcp_rn((float)parts);
    inv = inv * (2.0 - (double)parts * inv);
    const double part = (double)W * inv;
#pragma unroll 1
    for (int e = 0; e < 2; ++e) {
      const int c = blockIdx.x + e;
      if (c >= parts) break;
      long long w = (long long)(part * c) - lo;
      if (mine == 0 || w < 0 || w >= mine) continue;
      for (int b = sb0; b < sb1; ++b) {
        const long long cost = load_seq(a, b).per_head * a.hkv;
        if (w < cost) {
          Seq s;
          sh.cut[e] = locate(a, b, w, s);
          if (e == 0) sh.first = s;
          break;
        }
        w -= cost;
      }
    }
  }
  __syncthreads();
  const uint32_t tmem = sh.tmem;
  // The item warp walks this CTA's part and hands the items out; the other warps take a copy each
  // (walked by every warp, the walk's state spilled, and a spilled register is an L2 access here).
  Item it;
  int taken = 0;
  auto take_item = [&]() -> bool {
    const int k = taken % kItems;
    if (sh.bail || !warp_wait(&sh.item_full[k], (taken / kItems) & 1, kDevTimeoutFull)) { sh.bail = 1; return false; }
    it = sh.items[k];
    ++taken;
    return it.b1 > 0;
  };
  auto give_back = [&]() {                      // the item last taken is not read any more
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.item_empty[(taken - 1) % kItems]);
  };
  auto next_item = [&]() -> bool {
    const bool some = take_item();
    if (some) give_back();
    return some;
  };

  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
  if (warp == 8) {
    // ---------------------------------------------------------- TMA: Q, then K and V tiles
    int n = 0, items = 0;                       // ring tiles issued, items
    const int pieces = kKeys / a.box;
    const uint32_t piece_bytes = (uint32_t)a.box * 256;
    while (next_item()) {
      // Lane p < pieces brings the p-th piece of each block; `row` is its row in the cache (-1: not
      // wanted; no such page: past the end, which reads as zeros). No branches around the page
      // loads: several are in flight.
      const int* pages = a.pages ? a.pages + (size_t)it.b * a.max_pages : nullptr;
      auto row_of = [&](int blk) -> int {
        const int tok = blk * kKeys + lane * a.box;
        const bool wanted = blk < it.b1 && lane < pieces && tok < it.kend;
        // tok / page_size: both multiples of 8, the quotient by a product (exact below 2^28)
        const int lp = wanted ? (int)(((unsigned long long)(unsigned)(tok >> 3) * a.page_mul) >> a.page_shift) : 0;
        int pg = it.b;
        if (pages) pg = __ldcg(pages + lp);
        const int off = tok - lp * a.page_size;
        const int row = pg < 0 || pg >= a.num_pages ? a.total_rows : (pg * a.hkv + it.h) * a.page_size + off;
        return wanted ? row : -1;
      };
      auto issue = [&](const CUtensorMap* map, int blk, int row) -> bool {
        const int st = n % kRing;
        if (!warp_wait(&sh.empty[st], ((n / kRing) & 1) ^ 1, kDevTimeoutEmpty)) { sh.bail = 1; return false; }
        const int have = min(pieces, (it.kend - blk * kKeys + a.box - 1) / a.box);
        if (lane == 0) mbar_arrive_expect_tx(&sh.full[st], (uint32_t)max(have, 0) * piece_bytes);
        __syncwarp();
        if (row >= 0) {
          uint8_t* dst = ring + st * kTile + lane * a.box * 128;
          tma_2d(dst, map, 0, row, &sh.full[st]);
          tma_2d(dst + kHalf, map, 64, row, &sh.full[st]);
        }
        ++n;
        return true;
      };
      const int ahead = it.two ? 1 : 2;
      int r0 = row_of(it.b0), r1 = row_of(it.b0 + 1), r2 = row_of(it.b0 + 2);
      if (!issue(&a.kmap, it.b0, r0)) break;      // the ring has room before the last item's Q is free
      if (items > 0 && !warp_wait(&sh.q_empty, (items - 1) & 1, kDevTimeoutEmpty)) { sh.bail = 1; break; }
      if (lane == 0) {
        const uint32_t qb = (uint32_t)(a.T * a.G) * 256;
        mbar_arrive_expect_tx(&sh.q_full, it.two ? 2 * qb : qb);
        for (int t = 0; t < (it.two ? 2 : 1); ++t)
          for (int hf = 0; hf < 2; ++hf)
            tma_3d(sq + t * kTile + hf * kHalf, &a.qmap, hf * 64, it.h * a.G, it.tok + t * a.T,
                   &sh.q_full);
      }
      __syncwarp();
      ++items;
      if (ahead == 2 && it.b0 + 1 < it.b1 && !issue(&a.kmap, it.b0 + 1, r1)) break;
      for (int j = it.b0; j < it.b1; ++j) {
        const int r3 = row_of(j + 3);
        if (!issue(&a.vmap, j, r0)) break;
        if (j + ahead < it.b1 && !issue(&a.kmap, j + ahead, ahead == 1 ? r1 : r2)) break;
        r0 = r1; r1 = r2; r2 = r3;
      }
    }
    // All copies have landed before the CTA goes (they have, unless a wait gave up).
    for (int k = max(0, n - kRing); k < n; ++k)
      mbar_wait(&sh.full[k % kRing], (k / kRing) & 1, kDevTimeoutDrain);
    if (items > 0) mbar_wait(&sh.q_full, (items - 1) & 1, kDevTimeoutDrain);
  } else if (warp == 9) {
    // ---------------------------------------------------------- MMA issue
    {
      const bool bf = std::is_same<T, __nv_bfloat16>::value;
      const uint32_t id_s = idesc_128x128(bf, false), id_o = idesc_128x128(bf, true);
      const uint32_t dq = desc_kmajor(smem_u32(sq));
      const uint32_t dk = desc_kmajor(smem_u32(ring)), dv = desc_mnmajor(smem_u32(ring));
      int st = 0, ph = 0;                       // ring position
      // Parities of what has been waited for, a bit each: weights and O of slot 0 and 1, Q (one register).
      // A wait for the other parity of a barrier that nobody has arrived at yet passes.
      constexpr uint32_t kP = 1, kO = 4, kQ = 16;
      uint32_t par = 0;
      const uint32_t one = elect_one();
      uint32_t polls = spin_limit();            // 1 once a wait has given up
      int gave_up = 0;
      auto wait = [&](uint64_t* bar, int parity, int code) {
        const bool ok = poll_wait(bar, parity & 1, polls);
        gave_up = ok || gave_up ? gave_up : code;
        polls = ok ? polls : 1;
        fence_after();
      };
      auto failed = [&]() { return __any_sync(0xffffffffu, gave_up != 0); };   // alike in all lanes
      auto advance = [&]() { if (++st == kRing) { st = 0; ph ^= 1; } };
      auto score = [&](int slot, int stage, int qt) {            // S[slot] = Q[qt] K^T
        const uint32_t a0 = dq + qt * (kTile >> 4), b0 = dk + stage * (kTile >> 4);
#pragma unroll
        for (int s = 0; s < 8; ++s) {
          const uint32_t o = (s >> 2) * (kHalf >> 4) + (s & 3) * 2;
          mma_ss(one, tmem + slot * 128, a0 + o, b0 + o, id_s, s != 0);
        }
        mma_commit(one, &sh.s_full[slot]);
      };
      // O[slot] (+)= P[slot] V: the high parts of each half of the keys as soon as they are there,
      // then the low parts. (Addresses formed ahead of the loop would be spilled: the compiler
      // is kept from knowing that `ta` is the same every time.)
      auto weigh = [&](int slot, int stage, bool first) {
        const uint32_t b0 = dv + stage * (kTile >> 4);
        uint32_t ta = tmem + slot * 128;
        asm volatile("" : "+r"(ta));
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          wait(&sh.p_full[slot][hf], (par >> slot) & 1, kDevTimeoutMma);
#pragma unroll
          for (int lo = 0; lo < (kTwo ? 2 : 1); ++lo)
#pragma unroll
            for (int s = 4 * hf; s < 4 * hf + 4; ++s)
              mma_ts(one, ta + 256, ta + lo * 64 + s * 8, b0 + s * (2048 >> 4), id_o,
                     (first && lo == 0 && s == 0) ? 0u : 1u);
        }
        par ^= kP << slot;
      };
      // O[slot] of the item before has been read.
      auto o_free = [&](int slot) { wait(&sh.o_free[slot], ((par >> (2 + slot)) & 1) ^ 1, kDevTimeoutMma); };
      while (!failed() && next_item()) {
        wait(&sh.q_full, (par >> 4) & 1, kDevTimeoutFull);
        par ^= kQ;
        const int nb = it.b1 - it.b0;
        wait(&sh.ready[st], ph, kDevTimeoutFull);
        score(0, st, 0);
        if (it.two) {
          // Ring order: K0 | V0 K1 | V1 K2 | ...; every tile serves both slots.
          score(1, st, 1);
          mma_commit(one, &sh.empty[st]);
          if (nb == 1) mma_commit(one, &sh.q_empty);
          advance();
          for (int j = 0; j < nb && !failed(); ++j) {
            const int vs = st, vp = ph;
            const bool last = j + 1 == nb;
            advance();
            const int ks = st, kp = ph;
            if (j == 0) o_free(0);
            wait(&sh.ready[vs], vp, kDevTimeoutFull);
            weigh(0, vs, j == 0);
            if (last) mma_commit(one, &sh.o_full[0]);
            else {
              wait(&sh.ready[ks], kp, kDevTimeoutFull);
              score(0, ks, 0);
            }
            if (j == 0) o_free(1);
            weigh(1, vs, j == 0);
            mma_commit(one, &sh.empty[vs]);
            if (last) mma_commit(one, &sh.o_full[1]);
            else {
              score(1, ks, 1);
              mma_commit(one, &sh.empty[ks]);
              advance();
              if (j + 2 == nb) mma_commit(one, &sh.q_empty);
            }
          }
          par ^= kO | (kO << 1);
        } else {
          // Ring order: K0 K1 | V0 K2 | V1 K3 | ...; block j belongs to slot j & 1.
          mma_commit(one, &sh.empty[st]);
          advance();
          if (nb > 1) {
            wait(&sh.ready[st], ph, kDevTimeoutFull);
            score(1, st, 0);
            mma_commit(one, &sh.empty[st]);
            advance();
          }
          if (nb <= 2) mma_commit(one, &sh.q_empty);
          for (int j = 0; j < nb && !failed(); ++j) {
            const bool odd = j & 1;
            if (j == 0) o_free(0);
            if (j == 1) o_free(1);
            wait(&sh.ready[st], ph, kDevTimeoutFull);
            if (odd) weigh(1, st, j < 2);
            else weigh(0, st, j < 2);
            mma_commit(one, &sh.empty[st]);
            advance();
            if (j + 2 >= nb) mma_commit(one, &sh.o_full[odd]);
            else {
              wait(&sh.ready[st], ph, kDevTimeoutFull);
              score(odd, st, 0);
              mma_commit(one, &sh.empty[st]);
              advance();
              if (j + 3 == nb) mma_commit(one, &sh.q_empty);
            }
          }
          par ^= nb > 1 ? kO | (kO << 1) : kO;
        }
      }
      if (gave_up) {
        record_error(gave_up);
        sh.bail = 1;
      }
      __syncwarp();
      mma_commit(one, &sh.drain);                    // every MMA issued has finished
      mbar_wait(&sh.drain, 0, kDevTimeoutDrain);
    }
  } else if (warp == 10) {
    // ---------------------------------------------------------- tiles looked over
    // Every tile passes here on its way to the MMA warp, ahead of its use. A weight of 0 does not
    // hide a value that is not finite: 0 * NaN spoils every row. Keys past the item's last
    // visible one may hold anything (a freed page's NaN): their V rows become zeros. Values of the
    // chunk's later tokens that are not finite become zeros too and are noted: the rows that see
    // them add them at the end (add_odd). An exponent of ones, plus one, carries into the sign bit.
    constexpr uint32_t kExp = std::is_same<T, __nv_bfloat16>::value ? 0x7f807f80u : 0x7c007c00u;
    constexpr uint32_t kOne = std::is_same<T, __nv_bfloat16>::value ? 0x00800080u : 0x04000400u;
    int n = 0;
    while (next_item()) {
      const int nb = it.b1 - it.b0;
      if (lane == 0) sh.odd[(taken - 1) % kItems] = 0;   // read after the item's last product
      for (int i = 0; i < 2 * nb; ++i, ++n) {
        const int st = n % kRing;
        if (!warp_wait(&sh.full[st], (n / kRing) & 1, kDevTimeoutFull)) { sh.bail = 1; break; }
        // the tile's key block if it is a V tile, in the ring's orders (see the MMA warp)
        const int j = it.two ? (i & 1 ? i >> 1 : -1) : (i == 2 * nb - 1 ? nb - 1 : (i >= 2 && !(i & 1) ? (i - 2) >> 1 : -1));
        if (j >= 0 && uneven(it, it.b0 + j)) {
          const int blk = it.b0 + j;
          uint8_t* t = ring + st * kTile;
          const int from = min(max(it.kend - blk * kKeys, 0), kKeys);
          for (int o = from * 128 + lane * 16; o < kHalf; o += 512) {
            *reinterpret_cast<uint4*>(t + o) = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(t + kHalf + o) = make_uint4(0, 0, 0, 0);
          }
          uint32_t carry = 0;
          auto look = [&](const uint4& x) {
            carry |= ((x.x & kExp) + kOne) | ((x.y & kExp) + kOne) | ((x.z & kExp) + kOne) | ((x.w & kExp) + kOne);
          };
          const int seen = max(it.pos + 1 - blk * kKeys, 0) * 128 + lane * 16;
#pragma unroll 4
          for (int o = seen; o < from * 128; o += 512) {
            look(*reinterpret_cast<const uint4*>(t + o));
            look(*reinterpret_cast<const uint4*>(t + kHalf + o));
          }
          if (__any_sync(0xffffffffu, (carry & 0x80008000u) != 0)) {
            if (lane == 0) sh.odd[(taken - 1) % kItems] = 1;
#pragma unroll 1
            for (int o = seen; o < from * 128; o += 512)
#pragma unroll 1
              for (int e = 0; e < 8; ++e) {
                uint32_t* x = reinterpret_cast<uint32_t*>(t + (e >> 2) * kHalf + o) + (e & 3);
                *x &= ~(((((*x & kExp) + kOne) & 0x80008000u) >> 15) * 0xffffu);
              }
          }
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&sh.ready[st]);
          mbar_arrive(&sh.empty[st]);            // this warp's half of `empty`
        }
      }
    }
  } else {
    // ---------------------------------------------------------- items
    Walk walk(a, sh.cut[0], sh.cut[1], sh.first);
    bool more = true;
    for (int n = 0; more && !sh.bail; ++n) {
      more = walk.next(a, it);
      if (!more) it.b1 = 0;                     // no more: the last one handed out
      const int k = n % kItems;
      if (!warp_wait(&sh.item_empty[k], ((n / kItems) & 1) ^ 1, kDevTimeoutEmpty)) { sh.bail = 1; break; }
      if (lane == 0) {
        sh.items[k] = it;
        mbar_arrive(&sh.item_full[k]);
      }
      __syncwarp();
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    // ---------------------------------------------------------- softmax, one thread per row
    const int slot = warp >> 2;
    const int r = tid & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lanes + slot * 128, t_o = tmem + lanes + 256;
    const int rt = r / a.G, rg = r - rt * a.G;   // this row's token in the tile, head in the group
    T* out = static_cast<T*>(a.out);
    int ns = 0, no[2] = {0, 0}, nh = 0;
    if (tid < 2) a.desc[2 * blockIdx.x + tid] = make_int4(0, 0, 0, 0);
    named_bar_sync(1, 256);
    while (take_item()) {
      const int nb = it.b1 - it.b0;
      const int tok = it.two && slot == 1 ? a.T + rt : rt;        // token within the item
      const int vis = max(it.pos + tok + 1, 0);                    // keys this row sees
      const int ahead = vis - it.b0 * kKeys;                       // of them from the piece's first key on
      const int step = it.two ? 1 : 2;
      const bool live = r < a.T * a.G && tok < it.ntok;
      const bool rows = __any_sync(0xffffffffu, live);
      float m = -INFINITY, l = 0.f;
      int mine_n = 0;
      bool ok = true;
      for (int j = step == 1 ? 0 : slot; j < nb; j += step, ++mine_n) {
        if (!warp_wait(&sh.s_full[slot], ns & 1, kDevTimeoutMma)) { sh.bail = 1; ok = false; break; }
        ++ns;
        fence_after();
        if (!rows) {                              // no row of this warp is in the item
          __syncwarp();
          if (lane == 0) { mbar_arrive(&sh.p_full[slot][0]); mbar_arrive(&sh.p_full[slot][1]); }
          continue;
        }
        uint32_t s[4][32];
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld32(t_s + q * 32, s[q]);
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_wait_ld(s[q]);
        const int lim = ahead - j * kKeys;                         // keys this row sees of the block
        if (lim < kKeys) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (q * 32 + c >= lim) s[q][c] = 0xff800000u;        // -inf
        }
        __syncwarp();
        // The weights of the first 64 keys are formed, and put in place of their scores, with the
        // maximum of the blocks before while the row's maximum is still being found (the exponential
        // unit is what they wait for). Only if a row's maximum grew by more than kGrow (in log2 units) are
        // they formed again and O is rescaled: weights stay below 2^(kGrow + kBias), in range for
        // 16 bits. Measured and not kept: low parts formed behind all the high ones, while the tensor
        // core works on those, with a barrier of their own (+4 %), or two (+7 %).
        constexpr int kG = kTwo ? 8 : 16;        // pairs stored at a time (16 spill with two parts, 8 with one)
        auto weights = [&](int hf, float nm, f2 (&sum)[2]) {
          const f2 cs2 = f2_make(a.cs, a.cs), nm2 = f2_make(nm, nm);
#pragma unroll
          for (int c0 = 0; c0 < 32; c0 += kG) {
            uint32_t hi[kG], lo[kG];
#pragma unroll
            for (int c = c0; c < c0 + kG; ++c) {
              const int q = hf * 2 + (c >> 4), e = (2 * c) & 31;
              const f2 x = f2_fma(f2_make(__uint_as_float(s[q][e]), __uint_as_float(s[q][e + 1])), cs2, nm2);
              float x0, x1;
              f2_split(x, x0, x1);
              x0 = ex2(x0);
              x1 = ex2(x1);
              sum[c & 1] = f2_add(sum[c & 1], f2_make(x0, x1));
              if (kTwo) {
                hi[c - c0] = high_parts<T>(x0, x1);
                lo[c - c0] = low_parts<T>(x0, x1);
              } else {
                hi[c - c0] = Mma<T>::pack(x0, x1);
              }
            }
            tmem_st(t_s + hf * 32 + c0, hi);
            if (kTwo) tmem_st(t_s + 64 + hf * 32 + c0, lo);
          }
        };
        auto publish = [&](int hf) {
          tmem_wait_st();
          fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.p_full[slot][hf]);
        };
        auto offset = [&]() { return m == -INFINITY ? 0.f : kBias<T> - m; };
        float top;
        {
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < 32; c += 2)
#pragma unroll
            for (int q = 0; q < 4; ++q)
              mx[q] = fmaxf(fmaxf(mx[q], __uint_as_float(s[q][c])), __uint_as_float(s[q][c + 1]));
          top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.cs;
        }
        if (mine_n == 0) m = top;
        f2 sum[2] = {0, 0};
        weights(0, offset(), sum);
        const bool grow = top > m + kGrow<T>;
        if (__any_sync(0xffffffffu, grow)) {
          const float mn = grow ? top : m;
          const float f = grow ? ex2(m - mn) : 1.f;               // m = -inf: 0
          if (mine_n > 0) {
#pragma unroll 1
            for (int q = 0; q < 8; ++q) {
              uint32_t o[16];
              tmem_ld16u(t_o + slot * 128 + q * 16, o);
              tmem_wait_ld(o);
#pragma unroll
              for (int c = 0; c < 16; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * f);
              tmem_st(t_o + slot * 128 + q * 16, o);
            }
          }
          l *= f;
          m = mn;
          sum[0] = sum[1] = 0;
          tmem_wait_st();
          weights(0, offset(), sum);
        }
        publish(0);
        weights(1, offset(), sum);
        publish(1);
        float l0, l1;
        f2_split(f2_add(sum[0], sum[1]), l0, l1);
        l += l0 + l1;
      }
      if (!ok) break;

      // Epilogue: O / l to the output, or O, m, l to the workspace. (The item is read again: its
      // registers are wanted in the loop.)
      it = sh.items[(taken - 1) % kItems];
      const bool joined = !it.two && nb > 1;      // slot 1 holds the odd blocks
      if (it.two || slot == 0 || joined) {
        if (!warp_wait(&sh.o_full[slot], no[slot] & 1, kDevTimeoutMma)) { sh.bail = 1; break; }
        ++no[slot];
        fence_after();
      }
      if (!it.two && slot == 1) {
        if (joined) {
          sh.half_ml[r] = make_float2(m, l);
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.half_ready);
        }
        give_back();
        continue;
      }
      float f0 = 1.f, f1 = 0.f;
      if (joined) {
        if (!warp_wait(&sh.half_ready, nh & 1, kDevTimeoutMma)) { sh.bail = 1; break; }
        ++nh;
        fence_after();
        const float2 o = sh.half_ml[r];
        const float mm = fmaxf(m, o.x);
        const float ref = mm == -INFINITY ? 0.f : mm;
        f0 = ex2(m - ref);
        f1 = ex2(o.x - ref);
        l = l * f0 + o.y * f1;
        m = mm;
      }
      const bool whole = it.b0 == 0 && it.b1 == it.nblk;
      const int sl = 2 * blockIdx.x + (it.b0 > 0 ? 0 : 1);
      if (!whole && tid == 0)
        a.desc[sl] = make_int4(it.tok, it.ntok, it.h, it.b1 == it.nblk ? 2 : 1);
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);   // nothing seen: zeros; NaN stays
      const int prow = slot * kRows + r;
      T* dst = out + ((size_t)(it.tok + tok) * a.hq + it.h * a.G + rg) * kHd;
      float* pdst = a.part_o + (size_t)sl * a.slot_rows * kHd + prow * 4;    // [32 column fours][rows][4]
      const bool wide = (reinterpret_cast<uintptr_t>(a.out) & 31) == 0;
      if (rows) {
#pragma unroll 1
        for (int q = 0; q < 4; ++q) {
          uint32_t o[32];
          tmem_ld32(t_o + slot * 128 + q * 32, o);
          tmem_wait_ld(o);
          if (joined) {
            uint32_t o1[32];
            tmem_ld32(t_o + 128 + q * 32, o1);
            tmem_wait_ld(o1);
#pragma unroll
            for (int c = 0; c < 32; ++c)
              o[c] = __float_as_uint(__uint_as_float(o[c]) * f0 + __uint_as_float(o1[c]) * f1);
          }
          if (live) {
            if (whole) {
#pragma unroll
              for (int c = 0; c < 32; c += 16) {
                uint32_t v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  v[e] = Mma<T>::pack(__uint_as_float(o[c + 2 * e]) * inv, __uint_as_float(o[c + 2 * e + 1]) * inv);
                if (wide) st_32(dst + q * 32 + c, v);
                else {
                  *reinterpret_cast<uint4*>(dst + q * 32 + c) = make_uint4(v[0], v[1], v[2], v[3]);
                  *reinterpret_cast<uint4*>(dst + q * 32 + c + 8) = make_uint4(v[4], v[5], v[6], v[7]);
                }
              }
            } else {
#pragma unroll
              for (int c = 0; c < 32; c += 4)
                *reinterpret_cast<uint4*>(pdst + (size_t)(q * 8 + c / 4) * a.slot_rows * 4) =
                    make_uint4(o[c], o[c + 1], o[c + 2], o[c + 3]);
            }
          }
          __syncwarp();
        }
      }
      if (uneven(it, it.b1 - 1) && sh.odd[(taken - 1) % kItems] != 0) {
        if (live) add_odd<T>(a, it, vis, inv, whole ? dst : nullptr, pdst);
      }
      __syncwarp();
      if (live && !whole) a.part_ml[(size_t)sl * a.slot_rows + prow] = make_float2(m, l);
      fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&sh.o_free[slot]);
        if (joined) mbar_arrive(&sh.o_free[1]);
      }
      give_back();
    }
  }
  // Teardown: every warp arrives once; the MMA warp frees TMEM when all have.
  __syncwarp();
  fence_before();
  if (lane == 0) mbar_arrive(&sh.teardown);
  if (warp == 9) {
    mbar_wait(&sh.teardown, 0, kDevTimeoutDrain);
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// Joins the partials of the items that CTA cuts went through. Block (c, y): rows 32 y .. 32 y + 31 of
// the item whose first piece CTA c left; a row's pieces are weighted by 2^(m - max m) in the
// order of the keys. A lane has a row and a warp NC of its column fours, so that every load is 512
// contiguous bytes; the result turns through shared memory into whole rows. NC = 1 spreads the
// columns over four blocks, for few rows whose pieces are many.
constexpr int kJoinRows = 32;
constexpr int kJoinWarps = 8;
template <typename T, int NC>
__global__ void __launch_bounds__(kJoinWarps * 32) chunk_join_kernel(const __grid_constant__ ChunkArgs a) {
  __shared__ float turn[kJoinRows][kJoinWarps * NC * 4 + 4];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const int c = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int4 d = __ldcg(a.desc + 2 * c + 1);
  const int r0 = blockIdx.y * kJoinRows;
  if (d.w != 1 || r0 >= a.slot_rows || r0 >= (d.y > a.T ? 2 * kRows : kRows)) return;
  int pieces = 1;
  while (c + pieces < (int)gridDim.x) {
    const int f = __ldcg(&a.desc[2 * (c + pieces)].w);
    if (f == 0) break;
    ++pieces;
    if (f == 2) break;
  }
  auto slot_of = [&](int p) { return p == 0 ? 2 * c + 1 : 2 * (c + p); };
  auto token_of = [&](int r) {                     // of row r within the item; -1: no such row
    const int rr = r & (kRows - 1), tok = (r >> 7) * a.T + rr / a.G;
    return r < a.slot_rows && rr < a.T * a.G && tok < d.y ? tok : -1;
  };
  const int r = r0 + lane;
  const bool live = token_of(r) >= 0;
  const float2* ml = a.part_ml + r;
  float m = -INFINITY;
  if (live) {
#pragma unroll 8
    for (int p = 0; p < pieces; ++p) m = fmaxf(m, __ldcg(ml + (size_t)slot_of(p) * a.slot_rows).x);
  }
  const float ref = m == -INFINITY ? 0.f : m;
  constexpr int kCols = kJoinWarps * NC * 4;       // columns of this block
  const int four0 = (blockIdx.z * kJoinWarps + warp) * NC;
  float l = 0.f;
  float4 acc[NC];
#pragma unroll
  for (int q = 0; q < NC; ++q) acc[q] = make_float4(0.f, 0.f, 0.f, 0.f);
  if (live) {
#pragma unroll (NC == 1 ? 8 : 2)
    for (int p = 0; p < pieces; ++p) {
      const float2 s = __ldcg(ml + (size_t)slot_of(p) * a.slot_rows);
      const float w = ex2(s.x - ref);
      l += s.y * w;
      const float4* src = reinterpret_cast<const float4*>(a.part_o) + (size_t)slot_of(p) * 32 * a.slot_rows + r;
#pragma unroll
      for (int q = 0; q < NC; ++q) {
        const float4 o = __ldcg(src + (size_t)(four0 + q) * a.slot_rows);
        acc[q].x += o.x * w; acc[q].y += o.y * w; acc[q].z += o.z * w; acc[q].w += o.w * w;
      }
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
    for (int q = 0; q < NC; ++q)
      *reinterpret_cast<float4*>(&turn[lane][(warp * NC + q) * 4]) =
          make_float4(acc[q].x * inv, acc[q].y * inv, acc[q].z * inv, acc[q].w * inv);
  }
  __syncthreads();
  constexpr int kLanes = kCols / 4;                // lanes of a row's columns
  for (int k = threadIdx.x / kLanes; k < kJoinRows; k += kJoinWarps * 32 / kLanes) {
    const int tok = token_of(r0 + k), e = (threadIdx.x % kLanes) * 4;
    if (tok < 0) continue;
    const int rg = ((r0 + k) & (kRows - 1)) % a.G;
    const float4 o = *reinterpret_cast<const float4*>(&turn[k][e]);
    uint2 v;
    v.x = Mma<T>::pack(o.x, o.y);
    v.y = Mma<T>::pack(o.z, o.w);
    T* dst = static_cast<T*>(a.out) + ((size_t)(d.x + tok) * a.hq + d.z * a.G + rg) * kHd;
    *reinterpret_cast<uint2*>(dst + blockIdx.z * kCols + e) = v;
  }
}

int slot_rows_of(int64_t tokens, int G) { return tokens * G <= kRows ? (int)(tokens * G) : 2 * kRows; }

size_t ws_bytes_of(int sms, int64_t tokens, int G) {
  const size_t rows = (size_t)2 * sms * slot_rows_of(tokens, G);
  return rows * (kHd * sizeof(float) + sizeof(float2)) + (size_t)2 * sms * sizeof(int4) + 256;
}

template <typename T, bool kTwo>
int launch(ChunkArgs& a, const DeviceInfo& dev, cudaStream_t st) {
  const size_t smem = 1024 + (size_t)(2 + kRing) * kTile + sizeof(Shared);
  const void* kern = reinterpret_cast<const void*>(&chunk_attention_kernel<T, kTwo>);
  if (int rc = allow_dynamic_smem(kern, dev, smem)) return rc;
  if (int rc = launch_pdl(kern, dim3(dev.num_sms), dim3(kThreadsCa), smem, st, &a)) return rc;
  const unsigned y = (a.slot_rows + kJoinRows - 1) / kJoinRows;
  const bool few = a.slot_rows <= kRows;
  return launch_pdl(few ? reinterpret_cast<const void*>(&chunk_join_kernel<T, 1>)
                        : reinterpret_cast<const void*>(&chunk_join_kernel<T, 4>),
                    dim3(dev.num_sms, y, few ? 4 : 1), dim3(kJoinWarps * 32), 0, st, &a);
}

}  // namespace

namespace {
// One warp and a barrier that nobody arrives at, by this file's two kinds of wait.
__global__ void chunk_wait_probe_kernel(int branchless) {
  __shared__ uint64_t bar;
  if (threadIdx.x == 0) {
    mbar_init(&bar, 1);
    fence_barrier_init();
  }
  __syncwarp();
  if (!branchless) (void)warp_wait(&bar, 0, kDevTimeoutEmpty);
  else if (!poll_wait(&bar, 0, spin_limit()) && threadIdx.x == 0) record_error(kDevTimeoutMma);
}
}  // namespace

int chunk_test_bounded_wait(int branchless, cudaStream_t stream) {
  chunk_wait_probe_kernel<<<1, 32, 0, stream>>>(branchless);
  return (int)cudaGetLastError();
}

int chunk_take_error(int* code) {
  const int zero = 0;
  cudaError_t e = cudaMemcpyFromSymbol(code, dbk_device_error, sizeof(int));
  if (e == cudaSuccess) e = cudaMemcpyToSymbol(dbk_device_error, &zero, sizeof(int));
  return (int)e;
}
int chunk_set_spin_limit(uint32_t polls) {
  return (int)cudaMemcpyToSymbol(dbk_spin_limit, &polls, sizeof(polls));
}

}  // namespace dbk

using namespace dbk;

extern "C" size_t dbk_chunk_attention_workspace_bytes(int64_t tokens, int n_q_heads,
                                                      int n_kv_heads) {
  if (tokens < 1 || n_kv_heads < 1 || n_q_heads < n_kv_heads || n_q_heads % n_kv_heads) return 0;
  DeviceInfo dev;
  int sms = 148;
  if (current_device_info(&dev) == DBK_OK) sms = dev.num_sms;
  return ws_bytes_of(sms, tokens, n_q_heads / n_kv_heads);
}

extern "C" int dbk_chunk_attention(const void* q, const void* k_cache, const void* v_cache,
                                   const int32_t* cu_seqlens, const int32_t* seq_lens,
                                   const int32_t* page_table, void* out, int tokens, int batch,
                                   int n_q_heads, int n_kv_heads, int head_dim, int num_pages,
                                   int page_size, int max_pages_per_seq, float scale, int dtype,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  if (!k_cache || !v_cache || !cu_seqlens || !seq_lens) return DBK_ENULL;
  const bool two = !(dtype & DBK_WEIGHTS_ONE);
  dtype &= ~DBK_WEIGHTS_ONE;
  if (dtype != DBK_F16 && dtype != DBK_BF16) return DBK_EDTYPE;
  if (head_dim != kHd || tokens < 0 || batch < 1 || n_kv_heads < 1 || n_q_heads < n_kv_heads ||
      n_q_heads % n_kv_heads != 0 || num_pages < 1 || page_size < 1)
    return DBK_ESHAPE;
  const int G = n_q_heads / n_kv_heads;
  if (G > kRows || !(scale > 0.f) || scale > 1e38f || batch > kMaxBatch) return DBK_ESHAPE;
  const int64_t rows = (int64_t)num_pages * n_kv_heads;
  if (rows > INT_MAX || rows * page_size > INT_MAX - kKeys) return DBK_ESHAPE;
  int box = kKeys;
  if (page_table) {
    if (max_pages_per_seq < 1) return DBK_ESHAPE;
    while (box > page_size || page_size % box) box >>= 1;
    if (box < kMinBox) return DBK_ESHAPE;
  } else if (num_pages != batch) {
    return DBK_ESHAPE;
  }
  if (tokens == 0) return DBK_OK;
  if (!q || !out) return DBK_ENULL;
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out)) return DBK_EALIGN;
  const size_t q_bytes = (size_t)tokens * n_q_heads * kHd * 2;
  const size_t cache = cache_bytes(num_pages, n_kv_heads, page_size);
  const Span outs[] = {{out, q_bytes}, {workspace, workspace_bytes}};
  const Span ins[] = {{q, q_bytes}, {k_cache, cache}, {v_cache, cache}, {cu_seqlens, ((size_t)batch + 1) * 4},
                      {seq_lens, (size_t)batch * 4}, {page_table, page_table ? (size_t)batch * max_pages_per_seq * 4 : 0}};
  if (outputs_overlap(outs, ins)) return DBK_ESHAPE;
  DeviceInfo dev;
  int rc = current_device_info(&dev);
  if (rc) return rc;
  if (!workspace || workspace_bytes < ws_bytes_of(dev.num_sms, tokens, G)) return DBK_EWORKSPACE;
  if (!aligned16(workspace)) return DBK_EALIGN;

  ChunkArgs a{};
  a.v = v_cache;
  a.cu = cu_seqlens; a.lens = seq_lens; a.pages = page_table; a.out = out;
  a.batch = batch; a.tokens = tokens; a.hq = n_q_heads; a.hkv = n_kv_heads;
  a.G = G; a.T = kRows / G;
  a.page_size = page_size; a.max_pages = page_table ? max_pages_per_seq : 1;
  a.num_pages = num_pages; a.box = box; a.total_rows = (int)(rows * page_size);
  const int64_t cap = (int64_t)page_size * a.max_pages;
  a.cap = (int)(cap < INT_MAX - 2 * kKeys ? cap : INT_MAX - 2 * kKeys);
  a.slot_rows = slot_rows_of(tokens, G);
  a.cs = scale * kLog2eF;
  if (page_table) {
    const unsigned d = (unsigned)page_size / 8;
    int log = 0;
    while ((1u << log) < d) ++log;
    a.page_shift = 28 + log;
    a.page_mul = (unsigned)((1ull << a.page_shift) / d) + 1;
  }
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const size_t prow = (size_t)2 * dev.num_sms * a.slot_rows;
  a.part_o = reinterpret_cast<float*>(ws);
  ws += prow * kHd * sizeof(float);
  a.desc = reinterpret_cast<int4*>(ws);
  ws += (size_t)2 * dev.num_sms * sizeof(int4);
  a.part_ml = reinterpret_cast<float2*>(ws);
  rc = encode_tmap_heads3d(&a.qmap, q, dtype, tokens, n_q_heads, G, a.T);
  if (rc) return rc;
  const uint64_t cache_rows = (uint64_t)rows * page_size;
  rc = encode_tmap_2d(&a.kmap, k_cache, dtype, kHd, cache_rows, kHd * 2, 64, box, true);
  if (rc) return rc;
  rc = encode_tmap_2d(&a.vmap, v_cache, dtype, kHd, cache_rows, kHd * 2, 64, box, true);
  if (rc) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == DBK_F16) return two ? launch<__half, true>(a, dev, st) : launch<__half, false>(a, dev, st);
  return two ? launch<__nv_bfloat16, true>(a, dev, st) : launch<__nv_bfloat16, false>(a, dev, st);
}
