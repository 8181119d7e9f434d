// Attention of a block of consecutive positions over the 4-bit cache (format in shd_kv4.cuh) on the
// tensor cores (tcgen05).
//
// A tile is 128 (position, head) pairs of one kv head, heads fastest, so that the heads of a group
// share every unpacked row. It walks the rows that any of its positions sees, 64 at a time:
//   S [128 x 64]       = Q [128 x HD] K^T      O [128 x HD] += P [128 x 64] V
// Operands are f16 in two terms. The keys of 32 rows are divided by a power of two of theirs and
// s (c - 7.5) is then exactly two terms (11 + 5 bits); queries, their group sums, weights and the values'
// middles keep 22 bits of theirs, the keys' minima are exact. Three of the
// four term products are formed (the fourth is below 2^-22 of the sum), accumulated in f32 in
// tensor memory. Where the 32 rows' sizes are more than 2^6 apart, each row has a power of two of its own
// and the softmax goes row by row (a large row that weighs nothing would else take the bits of the others).
// Within a row a group 2^-k of the largest loses bits from k = 12 on. What the minima add,
//   sum_g (z_tg + 7.5 s_tg) (sum_(i in g) q_i)    and    sum_t p_t (z_tg + 7.5 s_tg),
// is one more step of 16 along the first product's depth (a row's parameters against the groups' query
// sums) and 16 more columns of the second's width. 32 value rows are divided by a power of two 2^e of
// theirs too, and their weights are 2^(score + e - ref): the running reference follows score + e, so no
// product overflows f16 whatever the scales of the rows, and the softmax's sum takes 2^-e back out.
//
// Warps: 0-7 softmax (two threads share a row, half of its 64 scores each: scores come from tensor
// memory, weights go back to the same columns as the second product's A operand), 8-11 unpack keys and
// 12-15 values into shared memory, 16 issues the MMAs, 17 walks ahead, fetching rows as they are stored
// and noting which queries see them. Scores, keys and values are double-buffered, so
// that S of the next 64 rows and O of the last run while the softmax works; the queries' high terms are
// an A operand in tensor memory too, which spares shared memory most of the first product's reads. A
// value row is unpacked as it lies (the second product's B operand is the wide dimension's major). O
// stays in tensor memory; it is rescaled only when a row's reference has to grow by more than 2^7.75, which
// the f16 range of the weights leaves room for. The tensor core's f32 sums round toward 0, so every
// kPDrain steps the softmax threads add O to a second accumulator, rounding to nearest, and the MMAs
// start afresh: without it the error grows with the length (2.3e-5 of the result at 8700 positions; a
// plain f32 evaluation is 1.9e-6 off).
//
// Work: the 64-row steps of all (tile, kv head) items and kPItem for an item's start and end, laid end to
// end, are cut into equal shares, one persistent CTA an SM; an item that is cut leaves its parts (weighted
// values, reference, sum) in context scratch, and each CTA the place of the cut at its end, and a second
// kernel joins them.
//
// Measured on a B200 (4 H HD FLOP a visible position): 512 positions after 8191, 40 heads over 8, 292 us,
// 303 TFLOP/s, over 100 launches, 302 to 319 us in long runs; 512 from the start, 28 heads over 4, 32.7 us; 2000 under
// a window of 512, 12 heads over 2, masked, 57.3 us. Of these 9, 0.4 and 1.3 us are the price of telling rows of
// unlike size apart. The three term products make the tensor work 3.1 times that. Before that a 64-row step took
// 3040 clocks of the softmax warps (scores to weights 1700, drains 690 on average, the rest waiting for the
// tensor core, which is issued MMAs for 1970 of them), now some 3 % more; an item's queries and results take some
// 11000, which is what bounds short prompts.
#include <cmath>

#include "shd_kv4.cuh"
#include "shd_tcgen05.cuh"

namespace shd {
namespace {

constexpr int kPRows = kKv4Tile;  // (position, head) pairs of a tile
constexpr int kPKV = kKv4Step;    // cache rows of a step
constexpr int kPThreads = 576;
constexpr int kPTiles = 2048;  // tiles a launch (their step counts are in shared memory)
// steps of rows on their way as stored: three, since a step's values are unpacked only when the product
// before the last has let go of their buffer, and the keys of the step after next must not wait for that
// (512 positions after 8191, 40 heads over 8: 296 us where two took 302; short items the same)
constexpr int kPRaw = 3;
// cost of an item's queries and results, in steps: at 4, 6, 8 and 11 the short prompt above takes 34.0, 31.8,
// 32.3 and 32.3 us, the windowed one 61.0, 57.3, 56.2 and 55.6, the long one 284.1, 283.3, 282.8 and 284.5
constexpr int kPItem = kKv4Item;
constexpr int kPDrain = 4;     // steps that the tensor core sums up on its own
// weights are 2^(score' - ref + 6), score' - ref <= 7.75, and with what is rounded of scores up to 2^23 below 2^15.5
constexpr float kRoom = 7.75f, kHead = 6.0f;
// rows of 32 whose sizes lie within 2^6 share a power of two, else each has its own: the weight of the row that adds
// most is then at least 1, which leaves its two f16 terms their 22 bits
constexpr int kSpread = 6;

template <int HD>
struct PromptShape {
  static constexpr int NG = HD / kKv4Group;
  static constexpr int KB = HD / 64;            // 64-channel blocks
  static constexpr uint32_t QL = 0;             // [KB][128 rows][128 B]: low terms of the queries
  static constexpr uint32_t QX = QL + KB * kPRows * 128;       // [128 rows][32 B]: query sums
  static constexpr uint32_t K = QX + kPRows * 32;              // [2 buffers][2 terms][KB][64 rows][128 B]
  static constexpr uint32_t BUF = 2 * KB * kPKV * 128;
  static constexpr uint32_t V = K + 2 * BUF;                   // the same
  static constexpr uint32_t KX = V + 2 * BUF;                  // [2 buffers][64 rows][32 B]: key parameters
  static constexpr uint32_t KXBUF = kPKV * 32;
  static constexpr uint32_t VX = KX + 2 * KXBUF;               // [2 buffers][64 rows / 8][16 columns][16 B]: value middles
  static constexpr uint32_t VXBUF = kPKV * 32;
  static constexpr uint32_t RAW = VX + 2 * VXBUF;              // [kPRaw][keys, values] codes, then parameters, as stored
  static constexpr uint32_t RAWC = kPKV * HD / 2, RAWP = kPKV * 4 * NG, RAWBUF = 2 * (RAWC + RAWP);
  static constexpr uint32_t ROW = RAW + kPRaw * RAWBUF;        // [8][2][64]: a row's position, out of sight from
  static constexpr uint32_t ROWBUF = 2 * kPKV * 4;
  // [8][2][4], of 32 rows: 2^(key e), e, 2^-e, seen by every query; 2^(key e) or 2^-e is 0 where rows have their own
  static constexpr uint32_t OF32 = ROW + 8 * ROWBUF;
  static constexpr uint32_t OWN = OF32 + 8 * 2 * 16;           // [8][2][64], of rows that have their own: 2^(key e), e
  static constexpr uint32_t RED = OWN + 8 * ROWBUF;            // [3][2 halves][128]: maxima of even and odd steps; the query's, then the sums
  static constexpr uint32_t BAR = RED + 6 * kPRows * 4;
  static constexpr uint32_t PRE = BAR + 256;                   // [kPTiles] cost of the tiles before
  // [8 warps][32 rows][32 channels] of queries on their way to their threads: the low terms' place, where it is wide enough
  static constexpr uint32_t TURN = HD == 128 ? QL : PRE + kPTiles * 4, TURNBUF = 32 * 32 * 4;
  static constexpr size_t SMEM = PRE + kPTiles * 4 + (HD == 128 ? 0 : 8 * TURNBUF) + 1024;  // + alignment slack
  static_assert(TURN != QL || 8 * TURNBUF <= QX - QL, "turned queries run over");
  static constexpr int PART = HD + 4;                          // of a row: reference, sum, 2 unused, weighted values
  static constexpr int SC = HD / 4;                            // channels of a row staged together on the way out
  static_assert(8 * 32 * (SC + 4) * 4 <= K - QL, "staged results run over");
};

// Tensor memory columns. Of each 16 columns of scores, 8 take the weights' high terms and 8 the low ones.
constexpr uint32_t kColS = 0, kColO = 128, kColSum = 272, kColQ = 416, kCols = 512;

enum Bar { B_QFULL = 0, B_KFULL = 1, B_KFREE = 3, B_VFULL = 5, B_VFREE = 7, B_SFULL = 9, B_PFULL = 11, B_PDONE = 13, B_EFULL = 15, B_RFULL = 19, B_RFREE = 19 + kPRaw, B_END = 19 + 2 * kPRaw };

// D f32, A and B f16, both K-major
__host__ __device__ constexpr uint32_t idesc_f16_f32(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
constexpr uint32_t kBWide = 1u << 16;  // B has its N dimension contiguous
// Without swizzle, 8-row x 16-byte pieces of 128 bytes: `k` bytes from one 16 B of depth to the next, `n`
// from one row group to the next.
__device__ __forceinline__ uint64_t smem_desc_plain(const void* p, uint32_t k, uint32_t n) {
  return ((uint64_t)(smem_u32(p) & 0x3FFFFu) >> 4) | ((uint64_t)(k >> 4) << 16) | ((uint64_t)(n >> 4) << 32) | (1ull << 46);
}
// 32 B of depth a row, the two pieces of a row group next to each other
__device__ __forceinline__ uint32_t plain16_offset(int r, int half) { return (uint32_t)(r >> 3) * 256u + half * 128u + (r & 7) * 16u; }
// N-contiguous operand with the 128-byte swizzle: rows of depth of 64 N elements, 8-row atoms 1024 bytes
// apart, the next 64 N elements `n` bytes on
__device__ __forceinline__ uint64_t smem_desc_wide128(const void* p, uint32_t n) {
  return ((uint64_t)(smem_u32(p) & 0x3FFFFu) >> 4) | ((uint64_t)(n >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

// Sleeps on the barrier for up to 0.1 ms: many warps wait here, and a poll takes issue slots from the others.
__device__ __forceinline__ bool mbar_try_wait_long(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(100000u)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ void bulk_copy(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
// One thread of a converged warp, the same one each time.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
// D[tmem] (+)= A[tmem] * B[smem]^T
__device__ __forceinline__ void tc_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {  // and waits
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// no use of the loaded values moves above the wait before this
__device__ __forceinline__ void tmem_loaded16(uint32_t (&r)[16]) {
#pragma unroll
  for (int i = 0; i < 16; i += 8)
    asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7]));
}

// Two centred codes times their scales: the product is exact in two f16 terms.
__device__ __forceinline__ void scale_pair(__half2 c, __half2 s, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __hmul2(s, c);
  hi = as_u32(h);
  lo = as_u32(__hfma2(s, c, __hneg2(h)));
}

// A row's parameters and the power of two that it is divided by: 8 s and |z| (values: |z + 7.5 s|) come to at
// most 2^9. It is that of its warp's 32 rows where they are of like size, else the row's own (set gives true): keys
// of 0 fit any size, but a value row of 0 does not, since its weight follows the power of two. Rows that
// no query sees come as zeros and do not count.
template <int NG>
struct RowParams {
  float s[NG], z[NG];
  int e;
  __device__ __forceinline__ bool set(const uint32_t (&w)[NG], bool middle, bool seen) {  // NG scales, NG minima
    float top = 0.0f;
#pragma unroll
    for (int g = 0; g < NG; g += 2) {
      const float2 a = unpack_f16(w[g / 2]), b = unpack_f16(w[NG / 2 + g / 2]);
      s[g] = a.x; s[g + 1] = a.y;
      z[g] = middle ? fmaf(7.5f, a.x, b.x) : b.x;
      z[g + 1] = middle ? fmaf(7.5f, a.y, b.y) : b.y;
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) top = fmaxf(top, fmaxf(8.0f * s[g], fabsf(z[g])));
    const int own = max(ceil_exp2(top), -40) - 9;
    e = __reduce_max_sync(0xffffffffu, own);
    const bool wide = __any_sync(0xffffffffu, (middle ? seen : top > 0.0f) && own < e - kSpread);
    if (wide) e = own;
    return wide;
  }
};

// Score + e row by row, or out of sight, in the scores' place: where rows have their own powers of two, or scores may
// pass 2^23 and a reference that is rounded would be off by more than the weights' room (here the scores are
// rounded as it is). Seldom, and so apart from the walk, whose code this would spread out.
__device__ __noinline__ void own_scores(uint32_t t_s, const float* own, const int* rp, float4 of32, float rowf, int p) {
#pragma unroll 1
  for (int y = 0; y < 32; y += 8) {
    uint32_t w[8];
    tmem_ld8(t_s + y, w);
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const bool in_sight = rp[y + x] <= p && p < rp[64 + y + x];
      const float f = of32.x == 0.0f ? own[y + x] : of32.x, e = of32.z == 0.0f ? own[64 + y + x] : of32.y;
      w[x] = in_sight ? __float_as_uint(fmaf(__uint_as_float(w[x]), rowf * f, e)) : 0xff800000u;
    }
    tmem_st8(t_s + y, w);
  }
  tmem_wait_st();
}
// The weights' sum without 2^e where value rows have their own.
__device__ __noinline__ float own_sum(uint32_t t_s, const float* own, float shift) {
  float part = 0.0f;
#pragma unroll 1
  for (int y = 0; y < 32; y += 8) {
    uint32_t w[8];
    tmem_ld8(t_s + y, w);
#pragma unroll
    for (int x = 0; x < 8; ++x) part = fmaf(exp2_fast(__uint_as_float(w[x]) + shift), exp2_fast(-own[64 + y + x]), part);
  }
  return part;
}

struct PromptArgs {
  Kv4AttnArgs a;
  float* parts;    // [CTA][2][128][PART]
  int4* cuts;      // [CTA]: of the item first cut at the CTA's end, tile, head, parts (0: none) and which of the CTA's two parts is its first
  int tiles;       // of a kv head
  int last;        // newest position written
  uint32_t per_group;  // 2^32 / G, rounded up (0 for G = 1): r / G = high word of the product for r < 2^18
};

// Positions of a tile's first and last row.
__device__ __forceinline__ void tile_positions(const Kv4AttnArgs& a, int tile, int G, int& lo, int& hi) {
  lo = a.pos0 + (int)((int64_t)tile * kPRows / G);
  hi = a.pos0 + min((int)(((int64_t)tile * kPRows + kPRows - 1) / G), a.M - 1);
}
__device__ __forceinline__ int tile_cost(const Kv4AttnArgs& a, int tile, int G) {
  int lo, hi;
  tile_positions(a, tile, G, lo, hi);
  return kv4_tile_cost(a.c, lo, hi, a.window);
}

// Costs of the tiles before each into pre[0 .. tiles), their sum returned; all threads of the block.
__device__ __forceinline__ int plan_tiles(const Kv4AttnArgs& a, int tiles, int G, int* pre, int* scratch) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = blockDim.x, warps = n / 32;
  int sum = 0;
  for (int t0 = 0; t0 < tiles; t0 += n) {
    const int t = t0 + tid;
    const int v = t < tiles ? tile_cost(a, t, G) : 0;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) scratch[warp] = x;
    __syncthreads();
    int base = sum;
    for (int w = 0; w < warps; ++w) {
      if (w < warp) base += scratch[w];
      sum += scratch[w];
    }
    if (t < tiles) pre[t] = base + x - v;
    __syncthreads();
  }
  return sum;
}

// A CTA's next stretch of one item: steps [begin, end) of its `steps` (maybe none), up to cost `next`.
struct Segment {
  int tile, head, begin, end, steps;
  int64_t item, next;
};
__device__ __forceinline__ Segment find_segment(const int* pre, int tiles, int sum, int heads, int64_t t, int64_t t_end) {
  int lo = 0, hi = tiles - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((int64_t)pre[mid] * heads <= t) lo = mid; else hi = mid - 1;
  }
  Segment s;
  s.tile = lo;
  const int cost = (lo + 1 < tiles ? pre[lo + 1] : sum) - pre[lo], in = (int)(t - (int64_t)pre[lo] * heads);
  s.steps = cost - kPItem;
  s.head = in / cost;
  s.item = (int64_t)pre[lo] * heads + (int64_t)s.head * cost;
  s.next = min(s.item + cost, t_end);
  s.begin = max((int)(t - s.item) - kPItem, 0);
  s.end = max((int)(s.next - s.item) - kPItem, s.begin);
  return s;
}
// The first stretch from t on that has steps; false: none before t_end.
__device__ __forceinline__ bool next_segment(Segment& s, const int* pre, int tiles, int sum, int heads, int64_t& t, int64_t t_end) {
  while (t < t_end) {
    s = find_segment(pre, tiles, sum, heads, t, t_end);
    if (s.end > s.begin) return true;
    t = s.next;
  }
  return false;
}

// O's columns: 8 u + 2 n + (g & 1) of block g / 2 is channel 32 g + 4 u + n, the order in which a word of
// stored values unpacks.

template <int HD>
__global__ void __launch_bounds__(kPThreads, 1) kv4_prefill_kernel(const __grid_constant__ PromptArgs pa) {
  using SH = PromptShape<HD>;
  constexpr int NG = SH::NG, KB = SH::KB;
  const Kv4AttnArgs& a = pa.a;
  const Kv4View& c = a.c;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + SH::BAR);
  int* pre = reinterpret_cast<int*>(smem + SH::PRE);
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  __shared__ uint32_t tmem_base;
  __shared__ int abort_word;
  __shared__ int scratch[32];
  volatile int* abort_flag = &abort_word;

  if (tid == 0) {
    abort_word = 0;
    for (int i = 0; i <= B_END; ++i) {
      const bool eight = i == B_QFULL || i == B_PFULL || i == B_PFULL + 1 || (i >= B_RFREE && i < B_RFREE + kPRaw);
      const bool four = i == B_KFULL || i == B_KFULL + 1 || i == B_VFULL || i == B_VFULL + 1 || (i >= B_EFULL && i < B_EFULL + 4);
      mbar_init(bar + i, eight ? 8 : four ? 4 : 1);
    }
    mbar_fence_init();
  }
  if (warp == 16) tmem_alloc(&tmem_base, kCols);
  // the middles' columns past 2 NG are never written again
  for (int i = tid; i < 2 * SH::VXBUF / 16; i += kPThreads)
    *reinterpret_cast<uint4*>(smem + SH::VX + i * 16) = make_uint4(0u, 0u, 0u, 0u);
  fence_proxy_async_smem();
  pdl_trigger();
  pdl_wait();
  const int G = a.H / c.heads;
  const int sum = plan_tiles(a, pa.tiles, G, pre, scratch);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = tmem_base;
  const int64_t T = (int64_t)sum * c.heads, per = (T + gridDim.x - 1) / gridDim.x;
  const int64_t t_begin = blockIdx.x * per, t_end = min(T, t_begin + per);
  const int last = pa.last;

  // Bounded wait of one thread; false: it ran out here or elsewhere, and the CTA gives up.
  auto wait_one = [&](int b, uint32_t parity) -> bool {
    bool ok = mbar_try_wait(bar + b, parity);
    if (ok) return true;
    const uint64_t t0 = globaltimer_ns();  // some 200 clocks: not read for a phase that is complete
    while (true) {
      ok = mbar_try_wait_long(bar + b, parity);
      if (ok || *abort_flag) break;
      if (globaltimer_ns() - t0 > SHD_WAIT_LIMIT_NS) {
        *abort_flag = 1;
        atomicOr(a.err, SHD_DEVERR_TIMEOUT_FULL);
        break;
      }
    }
    return ok;
  };
  auto group_of = [&](int r) -> int { return pa.per_group ? (int)__umulhi((uint32_t)r, pa.per_group) : r; };
  // The same for a whole warp.
  auto wait = [&](int b, uint32_t parity) -> bool { return __all_sync(0xffffffffu, wait_one(b, parity)); };

  if (warp < 8) {
    // ---- softmax ------------------------------------------------------------------------------
    // registers of the block: 256 x 120 + 256 x 72 + 64 x 96 = 576 x 96, as launched
    asm volatile("setmaxnreg.inc.sync.aligned.u32 120;");
    // After a wait that ran out the walk goes on without waiting: the warps meet at their barriers.
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t t_row = tbase + ((uint32_t)((warp & 3) * 32) << 16);
    float* red = reinterpret_cast<float*>(smem + SH::RED);
    int it = 0;
    bool ok = true;
    Segment sg;
    for (int64_t t = t_begin; next_segment(sg, pre, pa.tiles, sum, c.heads, t, t_end); t = sg.next) {
      const int r0 = sg.tile * kPRows, rows = a.M * G;  // at most kPTiles * kPRows
      // queries as two terms of q * 2^k, |q| 2^k < 2^7, channels in the order of the key words; a thread takes
      // its row's half, so that nothing but the exponent crosses threads (with a warp to a row and shuffles
      // the code was five times as long, fetched anew for every item: short prompt 42.9 us, this 40.1)
      const bool live = r0 + row < rows;
      float rowf;
      {
        constexpr int N = HD / 8;
        // as they lie, 8 lanes a row, and by way of shared memory to their threads (a thread reading its own
        // row touches 32 lines a load: 40.1 us of a short prompt, this 39.1)
        float* turn = reinterpret_cast<float*>(smem + SH::TURN + warp * SH::TURNBUF);
        float4 v[N];
        float top = 0.0f, sums[HD / 64];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = r0 + (warp & 3) * 32 + 4 * i + lane / 8, mm = group_of(r);
          const float* src = a.q + (size_t)mm * a.ldq + (size_t)(sg.head * G + r - mm * G) * HD + half * (HD / 2) + 4 * (lane & 7);
#pragma unroll
          for (int g = 0; g < HD / 64; ++g) {
            v[8 * g + i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < rows) v[8 * g + i] = *reinterpret_cast<const float4*>(src + 32 * g);
          }
        }
#pragma unroll
        for (int g = 0; g < HD / 64; ++g) {
#pragma unroll
          for (int i = 0; i < 8; ++i)  // column ^ row: both sides without bank conflicts
            *reinterpret_cast<float4*>(turn + (4 * i + lane / 8) * 32 + 4 * ((lane & 7) ^ ((4 * i + lane / 8) & 7))) = v[8 * g + i];
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) v[8 * g + i] = *reinterpret_cast<const float4*>(turn + lane * 32 + 4 * (i ^ (lane & 7)));
          __syncwarp();
        }
#pragma unroll
        for (int g = 0; g < HD / 64; ++g) {
          float4 t = v[8 * g], y = make_float4(fabsf(t.x), fabsf(t.y), fabsf(t.z), fabsf(t.w));
#pragma unroll
          for (int i = 8 * g + 1; i < 8 * g + 8; ++i) {
            t.x = __fadd_rn(t.x, v[i].x); t.y = __fadd_rn(t.y, v[i].y); t.z = __fadd_rn(t.z, v[i].z); t.w = __fadd_rn(t.w, v[i].w);
            y.x = fmaxf(y.x, fabsf(v[i].x)); y.y = fmaxf(y.y, fabsf(v[i].y)); y.z = fmaxf(y.z, fabsf(v[i].z)); y.w = fmaxf(y.w, fabsf(v[i].w));
          }
          sums[g] = __fadd_rn(__fadd_rn(t.x, t.y), __fadd_rn(t.z, t.w));
          top = fmaxf(top, fmaxf(fmaxf(y.x, y.y), fmaxf(y.z, y.w)));
        }
        red[(4 + half) * kPRows + row] = top;
        named_bar_sync(1, 256);  // also: every warp's queries have left their place
        top = fmaxf(top, red[(4 + (half ^ 1)) * kPRows + row]);
        // at least -121 for a finite query, whose group sums times 7.5 then stay below 2^15; the upper limit keeps 2^-k
        // times a power of two of the keys normal
        const int k = min(7 - ceil_exp2(top), 60);
        const float up = pow2i(k);
        rowf = a.scale * 1.44269504088896341f * pow2i(-k);
#pragma unroll
        for (int x = 0; x < HD / 64; ++x) {
          const int ch = half * (HD / 2) + 32 * x;  // 32 channels: 16 columns
          uint32_t h[16];
#pragma unroll
          for (int y = 0; y < 4; ++y) {  // of 8 channels the pairs (0, 4), (1, 5), (2, 6), (3, 7)
            const float4 f = v[8 * x + 2 * y], g = v[8 * x + 2 * y + 1];
            uint4 lo;
            split_f16(f.x * up, g.x * up, h[4 * y], lo.x);
            split_f16(f.y * up, g.y * up, h[4 * y + 1], lo.y);
            split_f16(f.z * up, g.z * up, h[4 * y + 2], lo.z);
            split_f16(f.w * up, g.w * up, h[4 * y + 3], lo.w);
            *reinterpret_cast<uint4*>(smem + SH::QL + (ch >> 6) * (kPRows * 128) + sw128_offset(row, (ch & 63) + 8 * y)) = lo;
          }
          tmem_st16(t_row + kColQ + ch / 2, h);
          // 7.5 x and 1 x the group's sum, as elements g and NG + g of the high terms' 8 and the low terms'
          uint32_t hi, lo;
          split_f16(sums[x] * up * 7.5f, sums[x] * up, hi, lo);
          uint16_t* to = reinterpret_cast<uint16_t*>(smem + SH::QX + plain16_offset(row, 0)) + ch / 32;
          to[0] = (uint16_t)hi; to[NG] = (uint16_t)(hi >> 16);
          to[64] = (uint16_t)lo; to[64 + NG] = (uint16_t)(lo >> 16);
        }
        if (HD == 64 && half == 0) {
          *reinterpret_cast<uint2*>(smem + SH::QX + plain16_offset(row, 0) + 8) = make_uint2(0u, 0u);
          *reinterpret_cast<uint2*>(smem + SH::QX + plain16_offset(row, 1) + 8) = make_uint2(0u, 0u);
        }
        tmem_wait_st();
      }
      tc_fence_before();
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar + B_QFULL);

      const int p = a.pos0 + (live ? group_of(r0 + row) : a.M - 1);
      // 2^(key e) from which a score of the warp's may pass 2^23: queries are below 2^7, keys 3 x 2^9
      const float large = 0.25f / (__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(rowf))) * (HD / 128.0f));
      float ref = kKv4Never, l = 0.0f;
      bool summed = false;  // the second accumulator holds something
      for (int j = sg.begin; j < sg.end; ++j, ++it) {
        const int b = it & 1;
        ok = ok && wait(B_EFULL + (it & 3), (it >> 2) & 1) && wait(B_SFULL + b, (it >> 1) & 1);
        tc_fence_after();
        const int* rp = reinterpret_cast<const int*>(smem + SH::ROW + (it & 7) * SH::ROWBUF) + 32 * half;
        const float4 of32 = *reinterpret_cast<const float4*>(smem + SH::OF32 + ((it & 7) * 2 + half) * 16);
        const uint32_t t_s = t_row + kColS + b * kPKV + 32 * half;
        // this half's 32 scores: score + e in log2 units is fac * v + add
        const bool wide = of32.x * of32.z == 0.0f || of32.x >= large, masked = of32.w == 0.0f && !wide;
        const float fac = wide ? 1.0f : rowf * of32.x, add = wide ? 0.0f : of32.y;
        const float* own = reinterpret_cast<const float*>(smem + SH::OWN + (it & 7) * SH::ROWBUF) + 32 * half;
        if (wide) own_scores(t_s, own, rp, of32, rowf, p);
        uint32_t v[2][16];
        tmem_ld16(t_s, v[0]);
        tmem_ld16(t_s + 16, v[1]);
        tmem_wait_ld();
        tmem_loaded16(v[0]);
        tmem_loaded16(v[1]);
        auto mask_scores = [&]() {  // fac > 0: a value of -inf weighs 0
#pragma unroll
          for (int y = 0; y < 32; y += 4) {
            const int4 from = *reinterpret_cast<const int4*>(rp + y), until = *reinterpret_cast<const int4*>(rp + 64 + y);
            uint32_t* w = &v[y / 16][y % 16];
            if (!(from.x <= p && p < until.x)) w[0] = 0xff800000u;
            if (!(from.y <= p && p < until.y)) w[1] = 0xff800000u;
            if (!(from.z <= p && p < until.z)) w[2] = 0xff800000u;
            if (!(from.w <= p && p < until.w)) w[3] = 0xff800000u;
          }
        };
        if (masked) mask_scores();
        float t4[4];  // short chains: a dependent instruction takes 8 clocks here
#pragma unroll
        for (int y = 0; y < 4; ++y) t4[y] = __uint_as_float(v[0][y]);
#pragma unroll
        for (int y = 4; y < 32; y += 8)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float e = y + 4 + x < 32 ? __uint_as_float(v[((y + 4 + x) % 32) / 16][(y + 4 + x) % 16]) : -INFINITY;
            t4[x] = fmaxf(t4[x], fmaxf(__uint_as_float(v[(y + x) / 16][(y + x) % 16]), e));
          }
        float top = fmaf(fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3])), fac, add);
        red[(2 * b + half) * kPRows + row] = top;
        // weights as two f16 terms (in the scores' places: high terms of 16 first), and their sum without 2^e
        float part = 0.0f;
        auto weigh = [&]() {
          const float sh = add + (kHead - ref);
          const uint64_t shift = pair(sh, sh), fac2 = pair(fac, fac);
          uint64_t s0 = pair(0.0f, 0.0f), s1 = s0;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t w[16];
#pragma unroll
            for (int y = 0; y < 16; y += 4) {
              const float2 x0 = unpair(fma2(pair(__uint_as_float(v[i][y]), __uint_as_float(v[i][y + 1])), fac2, shift));
              const float2 x1 = unpair(fma2(pair(__uint_as_float(v[i][y + 2]), __uint_as_float(v[i][y + 3])), fac2, shift));
              const uint64_t w0 = pair(exp2_fast(x0.x), exp2_fast(x0.y)), w1 = pair(exp2_fast(x1.x), exp2_fast(x1.y));
              s0 = add2(s0, w0);
              s1 = add2(s1, w1);
              split_pair(w0, w[y / 2], w[8 + y / 2]);
              split_pair(w1, w[y / 2 + 1], w[8 + y / 2 + 1]);
            }
#pragma unroll
            for (int y = 0; y < 16; ++y) v[i][y] = w[y];
          }
          const float2 f = unpair(add2(s0, s1));
          part = f.x + f.y;
        };
        // under the reference as it is, while the other half's maximum is on its way; again, rarely, when
        // the reference has to grow
        if (j > sg.begin) weigh();
        named_bar_sync(4 + (warp & 3), 64);
        top = fmaxf(top, red[(2 * b + (half ^ 1)) * kPRows + row]);
        float al = 1.0f;
        const bool grow = __any_sync(0xffffffffu, top - ref > kRoom);  // alike in both halves
        if (grow) {
          const float now = fmaxf(ref, top);
          al = exp2_fast(ref - now);
          ref = now;
          l *= al;
        }
        if (grow || j == sg.begin) {
          if (j > sg.begin) {
            tmem_ld16(t_s, v[0]);
            tmem_ld16(t_s + 16, v[1]);
            tmem_wait_ld();
            tmem_loaded16(v[0]);
            tmem_loaded16(v[1]);
            if (masked) mask_scores();
          }
          weigh();
        }
        if (of32.z == 0.0f) part = own_sum(t_s, own, kHead - ref);
        l = fmaf(part, of32.z == 0.0f ? 1.0f : of32.z, l);
        tmem_st16(t_s, v[0]);
        tmem_st16(t_s + 16, v[1]);
        // every kPDrain steps the sums so far go to the second accumulator; both follow the reference
        const int step = j - sg.begin;
        const bool drain = step > 0 && step % kPDrain == 0;
        if (step > 0 && (drain || grow)) {
          ok = ok && wait(B_PDONE + (b ^ 1), ((it - 1) >> 1) & 1);
          tc_fence_after();
          const uint64_t al2 = pair(al, al);
          const int end = half ? HD + 16 : HD / 2;
#pragma unroll 1
          for (int i = half * (HD / 2); i < end; i += 16) {
            uint32_t o[16], s[16];
            tmem_ld16(t_row + kColO + i, o);
            if (summed) tmem_ld16(t_row + kColSum + i, s);
            tmem_wait_ld();
            tmem_loaded16(o);
            if (summed) {
              tmem_loaded16(s);
            } else {
#pragma unroll
              for (int y = 0; y < 16; ++y) s[y] = 0u;
            }
#pragma unroll
            for (int y = 0; y < 16; y += 2) {
              uint64_t ov = pair(__uint_as_float(o[y]), __uint_as_float(o[y + 1])), sv = pair(__uint_as_float(s[y]), __uint_as_float(s[y + 1]));
              if (drain) sv = add2(sv, ov);
              const float2 f = unpair(mul2(sv, al2)), h = unpair(mul2(ov, al2));
              s[y] = __float_as_uint(f.x); s[y + 1] = __float_as_uint(f.y);
              o[y] = __float_as_uint(h.x); o[y + 1] = __float_as_uint(h.y);
            }
            if (summed || drain) tmem_st16(t_row + kColSum + i, s);
            if (!drain) tmem_st16(t_row + kColO + i, o);
          }
          summed |= drain;
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar + B_PFULL + b);
      }

      // the rows' results, or their parts: 2 SC columns of a half's at a time through the queries' place
      ok = ok && wait(B_PDONE + ((it - 1) & 1), ((it - 1) >> 1) & 1);
      tc_fence_after();
      red[(4 + half) * kPRows + row] = l;
      named_bar_sync(1, 256);  // also: every warp is past its queries
      l = __fadd_rn(red[4 * kPRows + row], red[5 * kPRows + row]);
      const bool whole = sg.begin == 0 && sg.end == sg.steps;
      const float inv = whole ? __frcp_rn(l == 0.0f ? 1.0f : l) : 1.0f;
      float* parts = pa.parts + ((size_t)blockIdx.x * 2 + (t == t_begin ? 0 : 1)) * kPRows * SH::PART;
      if (!whole && live && half == 0)
        *reinterpret_cast<float2*>(parts + (size_t)row * SH::PART) = make_float2(ref == kKv4Never ? -INFINITY : ref, l);
      // columns of O, both accumulators
      auto load_o = [&](int i, float (&y)[16]) {
        uint32_t o[16], s[16];
        tmem_ld16(t_row + kColO + i, o);
        if (summed) tmem_ld16(t_row + kColSum + i, s);
        tmem_wait_ld();
        tmem_loaded16(o);
        if (summed) tmem_loaded16(s);
#pragma unroll
        for (int n = 0; n < 16; ++n) y[n] = summed ? __uint_as_float(o[n]) + __uint_as_float(s[n]) : __uint_as_float(o[n]);
      };
      float z[4];
      {
        float y[16];
        load_o(HD, y);
#pragma unroll
        for (int n = 0; n < 4; ++n) z[n] = y[n] + y[4 + n];
      }
      constexpr int SC = SH::SC, STRIDE = SC + 4;
      float* stage = reinterpret_cast<float*>(smem + SH::QL) + warp * (32 * STRIDE);
      // HD 128: a half is one block (groups 2 half, + 1), HD 64: half of the one block
      const int g0 = HD == 128 ? 2 * half : 0;
      const float za = (HD == 128 && half) ? z[2] : z[0], zb = (HD == 128 && half) ? z[3] : z[1];
#pragma unroll 1
      for (int q = 0; q < (HD / 2) / SC; ++q) {
        const int col = half * (HD / 2) + q * SC;
#pragma unroll
        for (int x = 0; x < SC / 16; ++x) {
          float y[16];
          load_o(col + 16 * x, y);
#pragma unroll
          for (int u = 0; u < 2; ++u) {  // units of 4 channels of both groups
            const float* f = y + 8 * u;
            *reinterpret_cast<float4*>(stage + lane * STRIDE + 4 * (2 * x + u)) =
                make_float4((f[0] + za) * inv, (f[2] + za) * inv, (f[4] + za) * inv, (f[6] + za) * inv);
            *reinterpret_cast<float4*>(stage + lane * STRIDE + SC / 2 + 4 * (2 * x + u)) =
                make_float4((f[1] + zb) * inv, (f[3] + zb) * inv, (f[5] + zb) * inv, (f[7] + zb) * inv);
          }
        }
        __syncwarp();
        // SC / 2 channels of each group from 4 * (first unit)
        const int unit = (col & 63) / 8;
        constexpr int LPR = SC / 4;
        constexpr int RPI = 32 / LPR, B = 4;
        const int f = lane % LPR, g = g0 + f / (LPR / 2), ch = 32 * g + 4 * unit + 4 * (f % (LPR / 2));
        const int y0 = (warp & 3) * 32;
        if (whole && a.mask) {  // of four rows on their way at a time: one by one, their latency is most of a short item
#pragma unroll 1
          for (int i0 = lane / LPR; i0 < 32; i0 += B * RPI) {
            float4 mk[B];
#pragma unroll
            for (int x = 0; x < B; ++x) {
              const int rr = r0 + y0 + i0 + x * RPI, mm = group_of(rr);
              mk[x] = make_float4(0.f, 0.f, 0.f, 0.f);
              if (rr < rows) mk[x] = *reinterpret_cast<const float4*>(a.mask + mm * a.ldmask + (sg.head * G + rr - mm * G) * HD + ch);
            }
#pragma unroll
            for (int x = 0; x < B; ++x) {
              const int i = i0 + x * RPI, rr = r0 + y0 + i, mm = group_of(rr);
              if (rr >= rows) continue;
              const float4 v = *reinterpret_cast<const float4*>(stage + i * STRIDE + 4 * f);
              const size_t to = (size_t)mm * a.H * HD + (sg.head * G + rr - mm * G) * HD + ch;
              *reinterpret_cast<float4*>(a.out_c + to) =
                  make_float4(__fsub_rn(v.x, mk[x].x), __fsub_rn(v.y, mk[x].y), __fsub_rn(v.z, mk[x].z), __fsub_rn(v.w, mk[x].w));
              *reinterpret_cast<float4*>(a.out_s + to) = mk[x];
            }
          }
        } else {
#pragma unroll 1
          for (int i = lane / LPR; i < 32; i += RPI) {
            const int rr = r0 + y0 + i;
            if (rr >= rows) continue;
            const float4 v = *reinterpret_cast<const float4*>(stage + i * STRIDE + 4 * f);
            if (whole) {
              const int mm = group_of(rr);
              const size_t to = (size_t)mm * a.H * HD + (sg.head * G + rr - mm * G) * HD + ch;
              *reinterpret_cast<float4*>(a.out_c + to) = v;
              *reinterpret_cast<float4*>(a.out_s + to) = make_float4(0.f, 0.f, 0.f, 0.f);
            } else {
              *reinterpret_cast<float4*>(parts + (size_t)(y0 + i) * SH::PART + 4 + ch) = v;
            }
          }
        }
        __syncwarp();
      }
      tc_fence_before();
      named_bar_sync(1, 256);  // the queries' place is free again
    }
  } else if (warp < 16) {
    // ---- unpacking: keys (warps 8-11) or values (12-15), thread -> row th % 64, half th / 64 of its bytes --
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    const bool vals = warp >= 12;
    const int th = tid & 127, r = th & 63, kh = th >> 6;
    int it = 0;
    bool ok = true;
    Segment sg;
    for (int64_t t = t_begin; ok && next_segment(sg, pre, pa.tiles, sum, c.heads, t, t_end); t = sg.next) {
      for (int j = sg.begin; j < sg.end; ++j, ++it) {
        const int b = it & 1;
        const int st = it % kPRaw;
        const uint8_t* raw = smem + SH::RAW + st * SH::RAWBUF + (vals ? SH::RAWC : 0);
        const uint8_t* rawp = smem + SH::RAW + st * SH::RAWBUF + 2 * SH::RAWC + (vals ? SH::RAWP : 0);
        const int* rp = reinterpret_cast<const int*>(smem + SH::ROW + (it & 7) * SH::ROWBUF);
        float* of32 = reinterpret_cast<float*>(smem + SH::OF32 + ((it & 7) * 2 + (warp & 1)) * 16);
        if (!(ok = wait(B_RFULL + st, (it / kPRaw) & 1))) break;
        uint32_t w[NG];
        if constexpr (NG == 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(rawp + r * 16);
          w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        } else {
          const uint2 v = *reinterpret_cast<const uint2*>(rawp + r * 8);
          w[0] = v.x; w[1] = v.y;
        }
        const bool seen = rp[64 + r] != 0;
        if (!seen) {  // no query sees it: its parameters may be anything
#pragma unroll
          for (int g = 0; g < NG; ++g) w[g] = 0u;
        }
        RowParams<NG> q;
        const bool wide = q.set(w, vals, seen);
        float* own = reinterpret_cast<float*>(smem + SH::OWN + (it & 7) * SH::ROWBUF) + (vals ? kPKV : 0);
        const float down = pow2i(-q.e), up9 = down * 512.0f;
        if (vals) {
          if (wide) {
            if (kh == 0) own[r] = (float)q.e;
            __syncwarp();
          }
          if (lane == 0) {
            if (kh == 0) {
              of32[1] = (float)q.e;
              of32[2] = wide ? 0.0f : pow2i(-q.e);
            }
            mbar_arrive(bar + B_EFULL + (it & 3));
          }
        }
        if (it >= 2 && !(ok = wait((vals ? B_VFREE : B_KFREE) + b, ((it - 2) >> 1) & 1))) break;
        if (kh == 0) {
          if (!vals) {
            uint32_t y[4] = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int g = 0; g < NG; g += 2) {
              y[g / 2] = pack_f16(q.s[g] * down, q.s[g + 1] * down);
              y[NG / 2 + g / 2] = pack_f16(q.z[g] * down, q.z[g + 1] * down);
            }
            uint8_t* kx = smem + SH::KX + b * SH::KXBUF;
            *reinterpret_cast<uint4*>(kx + plain16_offset(r, 0)) = make_uint4(y[0], y[1], y[2], y[3]);
            *reinterpret_cast<uint4*>(kx + plain16_offset(r, 1)) = make_uint4(y[0], y[1], y[2], y[3]);
            if (wide) own[r] = pow2i(q.e);
            if (lane == 0) of32[0] = wide ? 0.0f : pow2i(q.e);
          } else {
            // middles: column g the high term, 4 + g the low one
            __half* vx = reinterpret_cast<__half*>(smem + SH::VX + b * SH::VXBUF + (r >> 3) * 256 + (r & 7) * 2);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              const float y = q.z[g] * down;
              const __half h = __float2half_rn(y);
              vx[g * 8] = h;
              vx[(4 + g) * 8] = __float2half_rn(__fsub_rn(y, __half2float(h)));
            }
          }
        }
        uint8_t* to = smem + (vals ? SH::V : SH::K) + b * SH::BUF + (r >> 3) * 1024 + (r & 7) * 128;
        __half2 s2[NG / 2];
#pragma unroll
        for (int g = 0; g < NG; g += 2) s2[g / 2] = __floats2half2_rn(q.s[g] * up9, q.s[g + 1] * up9);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          // a quarter of the row's bytes; of keys neighbouring rows take theirs in another order, so that
          // the reads of 8 lanes fall into different banks (values would then collide where they go)
          const int part = HD == 128 && !vals ? (2 * kh + x) ^ ((r >> 1) & 3) : 2 * kh + x;
          uint32_t cw[NG];
          if constexpr (NG == 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(raw + r * 64 + part * 16);
            cw[0] = v.x; cw[1] = v.y; cw[2] = v.z; cw[3] = v.w;
          } else {
            const uint2 v = *reinterpret_cast<const uint2*>(raw + r * 32 + part * 8);
            cw[0] = v.x; cw[1] = v.y;
          }
#pragma unroll
          for (int i = 0; i < NG; ++i) {
            // keys: word `part` of group i; values: unit 2 part + i / (NG / 2) of groups 2 (i % (NG / 2)), + 1
            const int ublk = i % (NG / 2), unit = 2 * part + i / (NG / 2);
            const int blk = vals ? ublk : i >> 1, chunk = vals ? unit : (i & 1) * 4 + part;
            const __half2 sv = vals ? s2[ublk] : ((i & 1) ? __high2half2(s2[i / 2]) : __low2half2(s2[i / 2]));
            const uint32_t cwi = cw[i], c8 = cwi >> 8;
            uint4 h, l;
            scale_pair(centre_low(cwi), sv, h.x, l.x);
            scale_pair(centre_high(cwi), sv, h.y, l.y);
            scale_pair(centre_low(c8), sv, h.z, l.z);
            scale_pair(centre_high(c8), sv, h.w, l.w);
            uint8_t* y = to + blk * (kPKV * 128) + ((chunk ^ (r & 7)) << 4);
            *reinterpret_cast<uint4*>(y) = h;
            *reinterpret_cast<uint4*>(y + KB * kPKV * 128) = l;
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(bar + (vals ? B_VFULL : B_KFULL) + b);
          mbar_arrive(bar + B_RFREE + st);
        }
      }
    }
  } else if (warp == 17) {
    // ---- fetching: a step's chunks as they are stored, and from and until which position its rows are seen --
    int it = 0;
    bool ok = true;
    Segment sg;
    for (int64_t t = t_begin; ok && next_segment(sg, pre, pa.tiles, sum, c.heads, t, t_end); t = sg.next) {
      int lo, hi;
      tile_positions(a, sg.tile, G, lo, hi);
      const Kv4Spans sp = kv4_spans(c, lo, hi, a.window);
      const size_t base = kv4_base(c, a.slot0, sg.head);
      // the next item's queries into L2: the softmax warps take them with nothing else to do meanwhile
      Segment then;
      int64_t t2 = sg.next;
      if (next_segment(then, pre, pa.tiles, sum, c.heads, t2, t_end)) {
        for (int i = lane; i < kPRows; i += 32) {
          const int r = then.tile * kPRows + i, m = group_of(r);
          const float* q = a.q + (size_t)m * a.ldq + (size_t)(then.head * G + r - m * G) * HD;
          if (m < a.M) {
#pragma unroll
            for (int x = 0; x < HD; x += 32) asm volatile("prefetch.global.L2 [%0];" ::"l"(q + x));
          }
        }
      }
      for (int j = sg.begin; j < sg.end; ++j, ++it) {
        const int st = it % kPRaw;
        if (it >= kPRaw && !(ok = wait(B_RFREE + st, (it / kPRaw - 1) & 1))) break;
        const int x0 = j * (kPKV / kKv4Chunk), chunks = min(kPKV / kKv4Chunk, sp.total - x0);
        int* rp = reinterpret_cast<int*>(smem + SH::ROW + (it & 7) * SH::ROWBUF);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = 32 * h + lane;
          int from = 0x7fffffff, until = 0;
          if (r / kKv4Chunk < chunks) {
            const int row = kv4_span_chunk(sp, x0 + r / kKv4Chunk) * kKv4Chunk + r % kKv4Chunk;
            const int held = kv4_held(c, row, last);
            const int64_t end = a.window > 0 && row >= c.sinks ? (int64_t)held + a.window : 0x7fffffff;
            if ((row < c.sinks || held >= c.sinks) && held <= hi && end > lo) {
              from = held;
              until = (int)min(end, (int64_t)0x7fffffff);
            }
          }
          rp[r] = from;
          rp[64 + r] = until;
          const int full = __all_sync(0xffffffffu, from <= lo && hi < until);
          if (lane == 0) reinterpret_cast<float*>(smem + SH::OF32)[((it & 7) * 2 + h) * 4 + 3] = full ? 1.0f : 0.0f;
        }
        constexpr uint32_t CODE = kKv4Chunk * HD / 2, PAR = kKv4Chunk * 4 * NG;
        __syncwarp();
        if (lane == 0) mbar_arrive_expect_tx(bar + B_RFULL + st, chunks * 2 * (CODE + PAR));
        __syncwarp();
        if (lane < 16 && (lane & 3) < chunks) {
          const size_t row0 = base + (size_t)kv4_span_chunk(sp, x0 + (lane & 3)) * kKv4Chunk;
          const int kind = lane >> 2;  // key codes, value codes, key and value parameters
          uint8_t* raw = smem + SH::RAW + st * SH::RAWBUF;
          if (kind < 2)
            bulk_copy(raw + kind * SH::RAWC + (lane & 3) * CODE, (kind ? c.vc : c.kc) + row0 * (HD / 2), CODE, bar + B_RFULL + st);
          else
            bulk_copy(raw + 2 * SH::RAWC + (kind - 2) * SH::RAWP + (lane & 3) * PAR,
                      reinterpret_cast<const uint8_t*>(kind == 3 ? c.vp : c.kp) + row0 * (4 * NG), PAR, bar + B_RFULL + st);
        }
      }
    }
    if (lane == 0) {
      int4 cut = make_int4(0, 0, 0, 0);
      if (t_end < T && t_begin < t_end) {
        const Segment at = find_segment(pre, pa.tiles, sum, c.heads, t_end, T);
        if (at.begin > 0 && (at.item + kPItem) / per == (int64_t)blockIdx.x)
          cut = make_int4(at.tile, at.head, (int)((at.item + kPItem + at.steps - 1) / per) - (int)blockIdx.x + 1, t_begin >= at.item ? 0 : 1);
      }
      pa.cuts[blockIdx.x] = cut;
    }
    // no copy is in flight when the block ends
    for (int i = max(it - kPRaw, 0); i < it; ++i)
      if (lane == 0 && !mbar_wait_bounded(bar + B_RFULL + i % kPRaw, (i / kPRaw) & 1)) atomicOr(a.err, SHD_DEVERR_TIMEOUT_DRAIN);
  } else {
    // ---- MMAs: the whole warp walks, one elected thread issues --------------------------------------
    // Operands that the compiler knows to be the same in the warp (by way of the shuffles) keep an issue
    // at 10 clocks; from a single thread's registers it takes 45, longer than most of these MMAs.
    constexpr uint32_t ids = idesc_f16_f32(kPRows, kPKV), idv = idesc_f16_f32(kPRows, HD) | kBWide, idx = idesc_f16_f32(kPRows, 16);
    const uint32_t tb = __shfl_sync(0xffffffffu, tbase, 0);
    int it = 0, seg = 0;
    bool ok = true;
    auto scores = [&](int i) -> bool {
      const int b = __shfl_sync(0xffffffffu, i & 1, 0);
      if (!wait(B_KFULL + b, (i >> 1) & 1)) return false;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t d = tb + kColS + b * kPKV;
        const uint8_t* kb = smem + SH::K + b * SH::BUF;
        // small terms first: low high, high low, then the parameters and high high
#pragma unroll
        for (int x = 0; x < KB; ++x) {
          const uint64_t ad = smem_desc_sw128(smem + SH::QL + x * kPRows * 128), bd = smem_desc_sw128(kb + x * kPKV * 128);
#pragma unroll
          for (int k = 0; k < 4; ++k) tc_mma(d, ad + 2 * k, bd + 2 * k, ids, (x > 0 || k > 0) ? 1u : 0u);
        }
#pragma unroll
        for (int x = 0; x < KB; ++x) {
          const uint64_t bd = smem_desc_sw128(kb + (KB + x) * kPKV * 128);
#pragma unroll
          for (int k = 0; k < 4; ++k) tc_mma_ts(d, tb + kColQ + 8 * (4 * x + k), bd + 2 * k, ids, 1u);
        }
        tc_mma(d, smem_desc_plain(smem + SH::QX, 128, 256), smem_desc_plain(smem + SH::KX + b * SH::KXBUF, 128, 256), ids, 1u);
#pragma unroll
        for (int x = 0; x < KB; ++x) {
          const uint64_t bd = smem_desc_sw128(kb + x * kPKV * 128);
#pragma unroll
          for (int k = 0; k < 4; ++k) tc_mma_ts(d, tb + kColQ + 8 * (4 * x + k), bd + 2 * k, ids, 1u);
        }
        tc_commit(bar + B_KFREE + b);
        tc_commit(bar + B_SFULL + b);
      }
      __syncwarp();
      return true;
    };
    Segment sg;
    for (int64_t t = t_begin; ok && next_segment(sg, pre, pa.tiles, sum, c.heads, t, t_end); ++seg, t = sg.next) {
      const int n = sg.end - sg.begin;
      if (!(ok = wait(B_QFULL, seg & 1))) break;
      if (!(ok = scores(it))) break;
      for (int j = 0; j < n; ++j, ++it) {
        const int b = __shfl_sync(0xffffffffu, it & 1, 0);
        const uint32_t more = __shfl_sync(0xffffffffu, j % kPDrain > 0 ? 1u : 0u, 0);
        if (j + 1 < n && !(ok = scores(it + 1))) break;
        if (!(ok = wait(B_VFULL + b, (it >> 1) & 1))) break;
        if (!(ok = wait(B_PFULL + b, (it >> 1) & 1))) break;
        tc_fence_after();
        if (elect_one()) {
          const uint8_t* vb = smem + SH::V + b * SH::BUF;
          const uint32_t pcol = tb + kColS + b * kPKV, o = tb + kColO;
          // low and high weights with both terms of the middles; low high, high low, high high
          const uint64_t xd = smem_desc_plain(smem + SH::VX + b * SH::VXBUF, 256, 128);
#pragma unroll
          for (int k = 0; k < 4; ++k) tc_mma_ts(o + HD, pcol + 8 + 16 * k, xd + 32 * k, idx, k > 0 ? 1u : more);
#pragma unroll
          for (int k = 0; k < 4; ++k) tc_mma_ts(o + HD, pcol + 16 * k, xd + 32 * k, idx, 1u);
#pragma unroll
          for (int p = 0; p < 3; ++p) {
            const uint64_t bd = smem_desc_wide128(vb + (p == 1 ? KB * kPKV * 128 : 0), kPKV * 128);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              tc_mma_ts(o, pcol + (p == 0 ? 8 : 0) + 16 * k, bd + 128 * k, idv, (p > 0 || k > 0) ? 1u : more);
          }
          tc_commit(bar + B_VFREE + b);
          tc_commit(bar + B_PDONE + b);
        }
        __syncwarp();
      }
    }
    // every MMA issued has completed before tensor memory is released (commits follow the thread that issued)
    if (elect_one()) {
      tc_commit(bar + B_END);
      if (!mbar_wait_bounded(bar + B_END, 0)) atomicOr(a.err, SHD_DEVERR_TIMEOUT_DRAIN);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 16) tmem_dealloc(tbase, kCols);
}

// Items that a share boundary cuts, joined in CTA order: block (b, y) takes rows 8 y .. + 7 of the item
// whose first cut is the end of CTA b's share; a warp takes a row. The cuts come from the CTAs, which have
// the tiles planned: planned again in every block, they made this kernel 7 to 11 us of the call.
template <int HD>
__global__ void __launch_bounds__(256) kv4_join_kernel(const __grid_constant__ PromptArgs pa) {
  using SH = PromptShape<HD>;
  constexpr int CPL = HD / 32;  // channels a lane
  const Kv4AttnArgs& a = pa.a;
  pdl_trigger();
  pdl_wait();
  const int4 cut = __ldcg(pa.cuts + blockIdx.x);
  const int parts = cut.z, G = a.H / a.c.heads;
  const int lane = threadIdx.x & 31, row = blockIdx.y * 8 + (threadIdx.x >> 5);
  const int r = cut.x * kPRows + row, mm = pa.per_group ? (int)__umulhi((uint32_t)r, pa.per_group) : r;
  if (parts == 0 || mm >= a.M) return;
  const int in_row = (cut.y * G + r - mm * G) * HD + CPL * lane;
  const size_t at = (size_t)mm * a.H * HD + in_row;
  float mk[CPL];
#pragma unroll
  for (int i = 0; i < CPL; ++i) mk[i] = a.mask ? a.mask[mm * a.ldmask + in_row + i] : 0.0f;
  const size_t step = (size_t)2 * kPRows * SH::PART;
  const float* first = pa.parts + ((size_t)blockIdx.x * 2 + cut.w) * kPRows * SH::PART + (size_t)row * SH::PART;
  const float* next = pa.parts + (size_t)(blockIdx.x + 1) * step + (size_t)row * SH::PART;
  auto part = [&](int w) { return w == 0 ? first : next + (size_t)(w - 1) * step; };
  float M = -INFINITY, L = 0.0f;
  for (int w = lane; w < parts; w += 32) M = fmaxf(M, __ldcg(part(w)));
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  float y[CPL];
#pragma unroll
  for (int i = 0; i < CPL; ++i) y[i] = 0.0f;
#pragma unroll 4
  for (int w = 0; w < parts; ++w) {
    const float* in = part(w);
    const float2 ml = __ldcg(reinterpret_cast<const float2*>(in));
    const float e = ml.x == -INFINITY ? 0.0f : exp2_fast(ml.x - M);
    L = fmaf(ml.y, e, L);
    float v[CPL];
    if constexpr (CPL == 4) {
      const float4 q = __ldcg(reinterpret_cast<const float4*>(in + 4) + lane);
      v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
      const float2 q = __ldcg(reinterpret_cast<const float2*>(in + 4) + lane);
      v[0] = q.x; v[1] = q.y;
    }
#pragma unroll
    for (int i = 0; i < CPL; ++i) y[i] = fmaf(v[i], e, y[i]);
  }
  const float D = L == 0.0f ? 1.0f : L;
#pragma unroll
  for (int i = 0; i < CPL; ++i) y[i] = __fsub_rn(__fdiv_rn(y[i], D), mk[i]);
  if constexpr (CPL == 4) {
    *reinterpret_cast<float4*>(a.out_c + at) = make_float4(y[0], y[1], y[2], y[3]);
    *reinterpret_cast<float4*>(a.out_s + at) = make_float4(mk[0], mk[1], mk[2], mk[3]);
  } else {
    *reinterpret_cast<float2*>(a.out_c + at) = make_float2(y[0], y[1]);
    *reinterpret_cast<float2*>(a.out_s + at) = make_float2(mk[0], mk[1]);
  }
}

template <int HD>
int launch_prefill_t(shd_ctx* ctx, const Kv4AttnArgs& a0) {
  using SH = PromptShape<HD>;
  static unsigned attr_devices = 0;
  if (!(attr_devices & (1u << (ctx->device & 31)))) {
    SHD_CHECK_CUDA(ctx, cudaFuncSetAttribute(kv4_prefill_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SH::SMEM));
    attr_devices |= 1u << (ctx->device & 31);
  }
  const int ctas = ctx->num_sms;
  const size_t need = (size_t)ctas * 2 * kPRows * PromptShape<128>::PART;
  if (!ctx->d_kv4_parts) SHD_CHECK_CUDA(ctx, cudaMalloc(&ctx->d_kv4_parts, need * 4 + ctas * sizeof(int4)));
  const int G = a0.H / a0.c.heads;
  // launches of whole positions, of at most kPTiles tiles and a plan that fits
  const int step = kv4_launch_positions(a0.c, a0.M, G, a0.pos0 + a0.M - 1, kPTiles);
  SHD_REQUIRE(ctx, step > 0, "shd_kv4_attn_prefill: too many heads");
  for (int m = 0; m < a0.M; m += step) {
    PromptArgs pa{};
    pa.a = a0;
    const size_t width = (size_t)a0.H * HD;
    pa.a.M = std::min(step, a0.M - m);
    pa.a.pos0 += m;
    pa.a.q += (size_t)m * a0.ldq;
    if (a0.mask) pa.a.mask += m * a0.ldmask;
    pa.a.out_c += m * width;
    pa.a.out_s += m * width;
    pa.last = a0.pos0 + a0.M - 1;
    pa.per_group = G == 1 ? 0u : (uint32_t)(((1ull << 32) + G - 1) / G);
    pa.parts = ctx->d_kv4_parts;
    pa.cuts = reinterpret_cast<int4*>(ctx->d_kv4_parts + need);
    pa.tiles = (int)(((int64_t)pa.a.M * G + kPRows - 1) / kPRows);
    SHD_CHECK_CUDA(ctx, launch_pdl(kv4_prefill_kernel<HD>, dim3(ctas), dim3(kPThreads), SH::SMEM, ctx->stream, pa));
    SHD_CHECK_CUDA(ctx, launch_pdl(kv4_join_kernel<HD>, dim3(ctas - 1, kPRows / 8), dim3(256), 0, ctx->stream, pa));
    ctx->launches += 2;
  }
  return SHD_OK;
}

}  // namespace

int launch_kv4_prefill(shd_ctx* ctx, const Kv4AttnArgs& a) {
  return a.c.head_dim == 128 ? launch_prefill_t<128>(ctx, a) : launch_prefill_t<64>(ctx, a);
}

}  // namespace shd
