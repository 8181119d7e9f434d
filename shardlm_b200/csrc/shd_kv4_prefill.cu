// Attention of a block of consecutive positions over the 4-bit cache (format in shd_kv4.cuh) on the
// tensor cores (tcgen05).
//
// A tile is 128 (position, head) pairs of one kv head, heads fastest, so that the heads of a group
// share every unpacked row. It walks the rows that any of its positions sees, 64 at a time:
//   S [128 x 64]       = Q [128 x HD] K^T      O [128 x HD] += P [128 x 64] V
// Operands are f16 in two terms. A key row is divided by a power of two of its own and s (c - 7.5) is
// then exactly two terms (11 + 5 bits); queries, weights and minima keep 22 bits of theirs. Three of the
// four term products are formed (the fourth is below 2^-22 of the sum), accumulated in f32 in
// tensor memory. What the minima add,
//   sum_g (z_tg + 7.5 s_tg) (sum_(i in g) q_i)    and    sum_t p_t (z_tg + 7.5 s_tg),
// is one more step of 16 along the first product's depth (a row's parameters against the groups' query
// sums) and 16 more columns of the second's width. A value row is divided by a power of two 2^e of
// its own too, and its weight is 2^(score + e - ref): the running reference follows score + e, so no
// product overflows f16 whatever the scales of the rows, and the softmax's sum takes 2^-e back out.
//
// Warps: 0-3 softmax (a thread owns a row: its 64 scores come from tensor memory, its weights go back
// to the same columns as the second product's A operand), 4-7 unpack keys and values into shared
// memory, 8 issues the MMAs. Scores, keys and values are double-buffered, so that S of the next 64 rows
// and O of the last run while the softmax works; the queries' high terms are an A operand in tensor
// memory too, which spares shared memory most of the first product's reads. O stays in tensor memory; it
// is rescaled only when a row's reference has to grow by more than 2^8, which the f16 range of the
// weights leaves room for. The tensor core's f32 sums round toward 0, so every kPDrain steps the softmax
// threads add O to a second accumulator, rounding to nearest, and the MMAs start afresh: without it the
// error grows with the length (2.3e-5 of the result at 8700 positions; the exact values need 1e-6).
// The roles' inner loops stay rolled at 16 columns: unrolled, four of five cycles went to instruction
// fetches (four kinds of warps run different code).
//
// Work: the 64-row steps of all (tile, kv head) items, laid end to end, are cut into equal shares, one
// persistent CTA an SM; an item that is cut leaves its parts (weighted values, reference, sum) in
// context scratch and a second kernel joins them.
#include <cmath>

#include "shd_kv4.cuh"
#include "shd_tcgen05.cuh"

namespace shd {
namespace {

constexpr int kPRows = 128;    // (position, head) pairs of a tile
constexpr int kPKV = 64;       // cache rows of a step
constexpr int kPThreads = 288;
constexpr int kPTiles = 2048;  // tiles a launch (their step counts are in shared memory)
constexpr int kPDrain = 4;     // steps that the tensor core sums up on its own
constexpr float kRoom = 8.0f, kHead = 6.0f;  // weights are 2^(score' - ref + 6), score' - ref <= 8

template <int HD>
struct PromptShape {
  static constexpr int NG = HD / kKv4Group;
  static constexpr int KB = HD / 64;            // 64-channel blocks of the first product's depth
  static constexpr int NV = HD + 16;            // width of the second product
  static constexpr uint32_t QL = 0;             // [KB][128 rows][128 B]: low terms of the queries
  static constexpr uint32_t K = QL + KB * kPRows * 128;        // [2 buffers][2 terms][KB][64 rows][128 B]
  static constexpr uint32_t KBUF = 2 * KB * kPKV * 128;
  static constexpr uint32_t V = K + 2 * KBUF;                  // [2 buffers][2 terms][NV rows][128 B]
  static constexpr uint32_t VBUF = 2 * NV * 128;
  static constexpr uint32_t QX = V + 2 * VBUF;                 // [128 rows][32 B]: query sums
  static constexpr uint32_t KX = QX + kPRows * 32;             // [2 buffers][64 rows][32 B]: parameters
  static constexpr uint32_t KXBUF = kPKV * 32;
  static constexpr uint32_t RAW = KX + 2 * KXBUF;              // [2 buffers] keys, values, their parameters as stored
  static constexpr uint32_t RAWC = kPKV * HD / 2, RAWP = kPKV * 4 * NG;
  static constexpr uint32_t RAWBUF = 2 * (RAWC + RAWP);
  static constexpr uint32_t KS = RAW + 2 * RAWBUF;             // [64 rows][NG] f16: scaled key scales
  static constexpr uint32_t VS = KS + kPKV * NG * 2;           // [NG][64 rows] f16: scaled value scales
  static constexpr uint32_t VM = VS + kPKV * NG * 2;           // [2 terms][NG][64 rows] f16: scaled middles
  static constexpr uint32_t ROW = VM + 2 * kPKV * NG * 2;      // [4][5][64]: key scale, e, 2^-e, position, out of sight from
  static constexpr uint32_t ROWBUF = 5 * kPKV * 4;
  static constexpr uint32_t FULL = ROW + 4 * ROWBUF;           // [4][2]: every query sees all of 32 rows
  static constexpr uint32_t BAR = FULL + 32;
  static constexpr uint32_t PRE = BAR + 128;                   // [kPTiles] steps of the tiles before
  static constexpr size_t SMEM = PRE + kPTiles * 4 + 1024;     // + alignment slack
  static constexpr int PART = HD + 4;                          // of a row: reference, sum, 2 unused, weighted values
};

// Tensor memory columns. Of each 16 columns of scores, 8 take the weights' high terms and 8 the low ones.
constexpr uint32_t kColS = 0, kColO = 128, kColSum = 272, kColQ = 416, kCols = 512;

enum Bar { B_QFULL = 0, B_KFULL = 1, B_KFREE = 3, B_VFULL = 5, B_VFREE = 7, B_SFULL = 9, B_PFULL = 11, B_PDONE = 13, B_END = 15 };

// D f32, A and B f16, both K-major
__host__ __device__ constexpr uint32_t idesc_f16_f32(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// 16 columns (32 B a row) without swizzle: 8-row x 16-byte pieces of 128 bytes, the two of a row group
// next to each other
__device__ __forceinline__ uint64_t smem_desc_plain16(const void* p) {
  return ((uint64_t)(smem_u32(p) & 0x3FFFFu) >> 4) | ((uint64_t)(128 >> 4) << 16) | ((uint64_t)(256 >> 4) << 32) | (1ull << 46);
}
__device__ __forceinline__ uint32_t plain16_offset(int r, int half) { return (uint32_t)(r >> 3) * 256u + half * 128u + (r & 7) * 16u; }

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
__device__ __forceinline__ void tmem_st4(uint32_t taddr, const uint4& r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w)
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

// A row's parameters and the power of two that it is divided by: 8 s and |z| (values: |z + 7.5 s|) come
// to at most 2^9.
template <int NG>
struct RowParams {
  float s[NG], z[NG];
  int e;
  __device__ __forceinline__ void set(const uint32_t (&w)[NG], bool middle) {  // NG scales, NG minima
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
    e = max(ceil_exp2(top), -40) - 9;
  }
};

struct PromptArgs {
  Kv4AttnArgs a;
  float* parts;    // [CTA][2][128][PART]
  int tiles;       // of a kv head
  int last;        // newest position written
};

// Positions of a tile's first and last row.
__device__ __forceinline__ void tile_positions(const Kv4AttnArgs& a, int tile, int G, int& lo, int& hi) {
  lo = a.pos0 + (int)((int64_t)tile * kPRows / G);
  hi = a.pos0 + min((int)(((int64_t)tile * kPRows + kPRows - 1) / G), a.M - 1);
}
__device__ __forceinline__ int tile_steps(const Kv4AttnArgs& a, int tile, int G) {
  int lo, hi;
  tile_positions(a, tile, G, lo, hi);
  return (kv4_spans(a.c, lo, hi, a.window).total * kKv4Chunk + kPKV - 1) / kPKV;
}

// Steps of the tiles before each into pre[0 .. tiles), their sum returned; all threads of the block.
__device__ __forceinline__ int plan_tiles(const Kv4AttnArgs& a, int tiles, int G, int* pre, int* scratch) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = blockDim.x, warps = n / 32;
  int sum = 0;
  for (int t0 = 0; t0 < tiles; t0 += n) {
    const int t = t0 + tid;
    const int v = t < tiles ? tile_steps(a, t, G) : 0;
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

// A CTA's next stretch of one item.
struct Segment {
  int tile, head, begin, end, steps;  // steps [begin, end) of the item's `steps`
};
__device__ __forceinline__ Segment find_segment(const int* pre, int tiles, int sum, int heads, int64_t t, int64_t t_end) {
  int lo = 0, hi = tiles - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((int64_t)pre[mid] * heads <= t) lo = mid; else hi = mid - 1;
  }
  Segment s;
  s.tile = lo;
  s.steps = (lo + 1 < tiles ? pre[lo + 1] : sum) - pre[lo];
  const int64_t in = t - (int64_t)pre[lo] * heads;
  s.head = (int)(in / s.steps);
  s.begin = (int)(in - (int64_t)s.head * s.steps);
  s.end = (int)min((int64_t)s.steps, s.begin + (t_end - t));
  return s;
}

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
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  __shared__ uint32_t tmem_base;
  __shared__ int abort_word;
  __shared__ int scratch[16];
  volatile int* abort_flag = &abort_word;

  if (tid == 0) {
    abort_word = 0;
    for (int i = 0; i <= B_END; ++i) {
      const bool four = i == B_QFULL || i == B_KFULL || i == B_KFULL + 1 || i == B_VFULL || i == B_VFULL + 1 || i == B_PFULL || i == B_PFULL + 1;
      mbar_init(bar + i, four ? 4 : 1);
    }
    mbar_fence_init();
  }
  if (warp == 8) tmem_alloc(&tmem_base, kCols);
  // the columns of V past the minima are never written again
  for (int i = tid; i < 4 * 16 * 128 / 16; i += kPThreads)
    *reinterpret_cast<uint4*>(smem + SH::V + (i / 128) * (SH::NV * 128) + HD * 128 + (i % 128) * 16) = make_uint4(0u, 0u, 0u, 0u);
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
    bool ok = false;
    const uint64_t t0 = globaltimer_ns();
    while (true) {
#pragma unroll 1
      for (int i = 0; i < 64 && !ok; ++i) ok = mbar_try_wait(bar + b, parity);
      if (ok || *abort_flag) break;
      if (globaltimer_ns() - t0 > SHD_WAIT_LIMIT_NS) {
        *abort_flag = 1;
        atomicOr(a.err, SHD_DEVERR_TIMEOUT_FULL);
        break;
      }
    }
    return ok;
  };
  // The same for a whole warp.
  auto wait = [&](int b, uint32_t parity) -> bool { return __all_sync(0xffffffffu, wait_one(b, parity)); };

  if (warp < 4) {
    // ---- softmax ------------------------------------------------------------------------------
    const int row = tid;
    const uint32_t t_row = tbase + ((uint32_t)(warp * 32) << 16);
    int it = 0;
    bool ok = true;
    for (int64_t t = t_begin; ok && t < t_end;) {
      const Segment sg = find_segment(pre, pa.tiles, sum, c.heads, t, t_end);
      const int64_t r = (int64_t)sg.tile * kPRows + row;
      const bool live = r < (int64_t)a.M * G;
      const int m = live ? (int)(r / G) : a.M - 1, hq = sg.head * G + (live ? (int)(r % G) : 0);
      const int p = a.pos0 + m;
      // the row's queries as two terms of q * 2^k, |q| 2^k < 2^7, channels in the order of the key words
      float rowf;
      {
        const float* q = a.q + (size_t)m * a.ldq + (size_t)hq * HD;
        float top = 0.0f, qs[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          qs[g] = 0.0f;
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 v = *reinterpret_cast<const float4*>(q + 32 * g + i);
            top = fmaxf(fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y))), fmaxf(fabsf(v.z), fabsf(v.w)));
            qs[g] = __fadd_rn(qs[g], __fadd_rn(__fadd_rn(v.x, v.y), __fadd_rn(v.z, v.w)));
          }
        }
        const int k = max(min(7 - ceil_exp2(top), 100), -100);
        const float up = live ? pow2i(k) : 0.0f;
        rowf = a.scale * 1.44269504088896341f * pow2i(-k);
#pragma unroll 2
        for (int x = 0; x < HD / 8; ++x) {
          const float4 u = *reinterpret_cast<const float4*>(q + 8 * x), v = *reinterpret_cast<const float4*>(q + 8 * x + 4);
          uint4 hi, lo;
          split_f16(u.x * up, v.x * up, hi.x, lo.x);
          split_f16(u.y * up, v.y * up, hi.y, lo.y);
          split_f16(u.z * up, v.z * up, hi.z, lo.z);
          split_f16(u.w * up, v.w * up, hi.w, lo.w);
          tmem_st4(t_row + kColQ + 4 * x, hi);
          *reinterpret_cast<uint4*>(smem + SH::QL + (x >> 3) * (kPRows * 128) + sw128_offset(row, (x & 7) * 8)) = lo;
        }
        uint32_t h[4], l[4];  // 7.5 x and 1 x the groups' sums
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = l[i] = 0u;
#pragma unroll
        for (int g = 0; g < NG; g += 2) {
          split_f16(qs[g] * up * 7.5f, qs[g + 1] * up * 7.5f, h[g / 2], l[g / 2]);
          split_f16(qs[g] * up, qs[g + 1] * up, h[NG / 2 + g / 2], l[NG / 2 + g / 2]);
        }
        *reinterpret_cast<uint4*>(smem + SH::QX + plain16_offset(row, 0)) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(smem + SH::QX + plain16_offset(row, 1)) = make_uint4(l[0], l[1], l[2], l[3]);
      }
      tmem_wait_st();
      tc_fence_before();
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar + B_QFULL);

      const uint64_t rowf2 = pair(rowf, rowf);
      float ref = kKv4Never;
      uint64_t l2 = pair(0.0f, 0.0f);
      bool summed = false;  // the second accumulator holds something
      for (int j = sg.begin; j < sg.end; ++j, ++it) {
        const int b = it & 1;
        if (!(ok = wait(B_SFULL + b, (it >> 1) & 1))) break;
        tc_fence_after();
        const float* rp = reinterpret_cast<const float*>(smem + SH::ROW + (it & 3) * SH::ROWBUF);
        const int* full = reinterpret_cast<const int*>(smem + SH::FULL) + (it & 3) * 2;
        const bool masked = !(full[0] && full[1]);
        const uint32_t t_s = t_row + kColS + b * kPKV;
        // score + e in log2 units, back to the same columns, and the row's maximum
        float top = -INFINITY;
#pragma unroll 1
        for (int i = 0; i < kPKV; i += 16) {
          uint32_t v[16];
          tmem_ld16(t_s + i, v);
          tmem_wait_ld();
          tmem_loaded16(v);
          float x[16];
#pragma unroll
          for (int y = 0; y < 16; y += 4) {
            const ulonglong2 kf = *reinterpret_cast<const ulonglong2*>(rp + i + y), ve = *reinterpret_cast<const ulonglong2*>(rp + 64 + i + y);
            const float2 x0 = unpair(fma2(mul2(pair(__uint_as_float(v[y]), __uint_as_float(v[y + 1])), rowf2), kf.x, ve.x));
            const float2 x1 = unpair(fma2(mul2(pair(__uint_as_float(v[y + 2]), __uint_as_float(v[y + 3])), rowf2), kf.y, ve.y));
            x[y] = x0.x; x[y + 1] = x0.y; x[y + 2] = x1.x; x[y + 3] = x1.y;
          }
          if (masked) {
            const int* at = reinterpret_cast<const int*>(rp + 3 * kPKV) + i;
#pragma unroll
            for (int y = 0; y < 16; ++y)
              if (!(at[y] <= p && p < at[kPKV + y])) x[y] = -INFINITY;
          }
#pragma unroll
          for (int y = 0; y < 16; y += 2) top = fmaxf(top, fmaxf(x[y], x[y + 1]));
#pragma unroll
          for (int y = 0; y < 16; ++y) v[y] = __float_as_uint(x[y]);
          tmem_st16(t_s + i, v);
        }
        float al = 1.0f;
        const bool grow = __any_sync(0xffffffffu, top > ref + kRoom);
        if (grow) {
          const float now = fmaxf(ref, top);
          al = exp2_fast(ref - now);
          ref = now;
          l2 = mul2(l2, pair(al, al));
        }
        tmem_wait_st();
        // weights as two f16 terms, over the scores; their sum without the rows' powers of two
        const uint64_t shift = pair(kHead - ref, kHead - ref);
#pragma unroll 1
        for (int i = 0; i < kPKV; i += 16) {
          uint32_t v[16], w[16];
          tmem_ld16(t_s + i, v);
          tmem_wait_ld();
          tmem_loaded16(v);
#pragma unroll
          for (int y = 0; y < 16; y += 4) {
            const ulonglong2 ie = *reinterpret_cast<const ulonglong2*>(rp + 128 + i + y);
            const float2 x0 = unpair(add2(pair(__uint_as_float(v[y]), __uint_as_float(v[y + 1])), shift));
            const float2 x1 = unpair(add2(pair(__uint_as_float(v[y + 2]), __uint_as_float(v[y + 3])), shift));
            const uint64_t w0 = pair(exp2_fast(x0.x), exp2_fast(x0.y)), w1 = pair(exp2_fast(x1.x), exp2_fast(x1.y));
            l2 = fma2(w0, ie.x, l2);
            l2 = fma2(w1, ie.y, l2);
            split_pair(w0, w[y / 2], w[8 + y / 2]);
            split_pair(w1, w[y / 2 + 1], w[8 + y / 2 + 1]);
          }
          tmem_st16(t_s + i, w);
        }
        // every kPDrain steps the sums so far go to the second accumulator; both follow the reference
        const int step = j - sg.begin;
        const bool drain = step > 0 && step % kPDrain == 0;
        if (step > 0 && (drain || grow)) {
          if (!(ok = wait(B_PDONE + (b ^ 1), ((it - 1) >> 1) & 1))) break;
          tc_fence_after();
          const uint64_t al2 = pair(al, al);
#pragma unroll 1
          for (int i = 0; i < SH::NV; i += 16) {
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
              const float2 so = unpair(mul2(sv, al2)), oo = unpair(mul2(ov, al2));
              s[y] = __float_as_uint(so.x); s[y + 1] = __float_as_uint(so.y);
              o[y] = __float_as_uint(oo.x); o[y + 1] = __float_as_uint(oo.y);
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
      if (!ok) break;

      // the row's result, or its part
      if (!(ok = wait(B_PDONE + ((it - 1) & 1), ((it - 1) >> 1) & 1))) break;
      tc_fence_after();
      const float2 lv = unpair(l2);
      const float l = lv.x + lv.y, D = l == 0.0f ? 1.0f : l;
      float z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      const bool whole = sg.begin == 0 && sg.end == sg.steps;
      float* part = pa.parts + (((size_t)blockIdx.x * 2 + (t == t_begin ? 0 : 1)) * kPRows + row) * SH::PART;
      const size_t out_at = (size_t)m * a.H * HD + (size_t)hq * HD;
#pragma unroll 1
      for (int x = SH::NV / 16 - 1; x >= 0; --x) {  // the minima's columns first
        const int i = 16 * x;
        uint32_t o[16], s[16];
        tmem_ld16(t_row + kColO + i, o);
        if (summed) tmem_ld16(t_row + kColSum + i, s);
        tmem_wait_ld();
        tmem_loaded16(o);
        float y[16];
#pragma unroll
        for (int n = 0; n < 16; ++n) y[n] = __uint_as_float(o[n]);
        if (summed) {
          tmem_loaded16(s);
#pragma unroll
          for (int n = 0; n < 16; ++n) y[n] += __uint_as_float(s[n]);
        }
        if (i == HD) {
#pragma unroll
          for (int n = 0; n < 4; ++n) z[n] = y[n];
          continue;
        }
        if (!live) continue;
        const int g = i / 32;
        const float zg = g == 0 ? z[0] : g == 1 ? z[1] : g == 2 ? z[2] : z[3];
#pragma unroll
        for (int n = 0; n < 16; n += 4) {
          const float4 f = make_float4(y[n] + zg, y[n + 1] + zg, y[n + 2] + zg, y[n + 3] + zg);
          if (whole) {
            const float4 mk = a.mask ? *reinterpret_cast<const float4*>(a.mask + out_at + i + n) : make_float4(0.f, 0.f, 0.f, 0.f);
            *reinterpret_cast<float4*>(a.out_c + out_at + i + n) =
                make_float4(__fsub_rn(__fdiv_rn(f.x, D), mk.x), __fsub_rn(__fdiv_rn(f.y, D), mk.y),
                            __fsub_rn(__fdiv_rn(f.z, D), mk.z), __fsub_rn(__fdiv_rn(f.w, D), mk.w));
            *reinterpret_cast<float4*>(a.out_s + out_at + i + n) = mk;
          } else {
            *reinterpret_cast<float4*>(part + 4 + i + n) = f;
          }
        }
      }
      if (!whole && live) *reinterpret_cast<float2*>(part) = make_float2(ref == kKv4Never ? -INFINITY : ref, l);
      tc_fence_before();
      t += sg.end - sg.begin;
    }
  } else if (warp < 8) {
    // ---- unpacking ----------------------------------------------------------------------------
    const int th = tid - 128, w4 = warp - 4;
    // a walk over the CTA's steps
    struct Walk {
      int64_t t;
      Segment sg;
      Kv4Spans sp;
      size_t base;
      int lo, hi, j;
    };
    auto enter = [&](Walk& w) {
      if (w.t >= t_end) return;
      w.sg = find_segment(pre, pa.tiles, sum, c.heads, w.t, t_end);
      tile_positions(a, w.sg.tile, G, w.lo, w.hi);
      w.sp = kv4_spans(c, w.lo, w.hi, a.window);
      w.base = kv4_base(c, a.slot0, w.sg.head);
      w.j = w.sg.begin;
    };
    auto advance = [&](Walk& w) {
      ++w.t;
      if (++w.j == w.sg.end) enter(w);
    };
    // asynchronous copies of a step's rows as they are stored: warp w4 copies its w4-th chunk
    constexpr int CPR = HD / 32, NC = kKv4Chunk * CPR, NP = kKv4Chunk * 4 * NG / 16;
    auto fetch = [&](const Walk& w, int buf) {
      const int x = w.j * (kPKV / kKv4Chunk) + w4;
      if (w.t < t_end && x < w.sp.total) {
        const size_t row0 = w.base + (size_t)kv4_span_chunk(w.sp, x) * kKv4Chunk;
        uint8_t* raw = smem + SH::RAW + buf * SH::RAWBUF;
#pragma unroll
        for (int i = 0; i < NC / 32; ++i) {
          const int y = lane + 32 * i, r = w4 * kKv4Chunk + y / CPR, q = y % CPR;
          const uint32_t at = (uint32_t)(r * CPR + (HD == 128 ? q ^ ((r >> 1) & 3) : q)) * 16;
          cp_async16(raw + at, c.kc + row0 * (HD / 2) + y * 16, 16);
          cp_async16(raw + SH::RAWC + at, c.vc + row0 * (HD / 2) + y * 16, 16);
        }
        if (lane < 2 * NP) {
          const bool v = lane >= NP;
          const int y = v ? lane - NP : lane;
          cp_async16(raw + 2 * SH::RAWC + (v ? SH::RAWP : 0) + w4 * (kKv4Chunk * 4 * NG) + y * 16,
                     reinterpret_cast<const uint8_t*>(v ? c.vp : c.kp) + row0 * (4 * NG) + y * 16, 16);
        }
      }
      cp_async_commit();
    };
    bool ok = true;
    Walk at{}, ahead{};
    at.t = ahead.t = t_begin;
    enter(at);
    enter(ahead);
    if (t_begin < t_end) {
      fetch(ahead, 0);
      advance(ahead);
    }
    for (int it = 0; at.t < t_end; ++it) {
      const int b = it & 1;
      const uint8_t* raw = smem + SH::RAW + b * SH::RAWBUF;
      cp_async_wait<0>();
      named_bar_sync(1, 128);  // this step's rows have landed, and nobody reads the last step's
      fetch(ahead, b ^ 1);
      advance(ahead);
      // after a wait that ran out the walk goes on without waiting: the four warps meet at their barriers
      ok = ok && (it < 2 || wait(B_KFREE + b, ((it - 2) >> 1) & 1));
      // one row a thread: keys 0-63, values 64-127
      {
        const int r = th & 63;
        const bool vals = th >= 64;
        // whether any query of the tile sees the row: at positions [from, until)
        int from = 0x7fffffff, until = 0;
        const int x = at.j * (kPKV / kKv4Chunk) + r / kKv4Chunk;
        if (x < at.sp.total) {
          const int row = kv4_span_chunk(at.sp, x) * kKv4Chunk + r % kKv4Chunk;
          const int held = kv4_held(c, row, last);
          const int64_t end = a.window > 0 && row >= c.sinks ? (int64_t)held + a.window : 0x7fffffff;
          if ((row < c.sinks || held >= c.sinks) && held <= at.hi && end > at.lo) {
            from = held;
            until = (int)min(end, (int64_t)0x7fffffff);
          }
        }
        uint32_t w[NG];
        const uint8_t* src = raw + 2 * SH::RAWC + (vals ? SH::RAWP : 0) + r * (4 * NG);
        if constexpr (NG == 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(src);
          w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        } else {
          const uint2 v = *reinterpret_cast<const uint2*>(src);
          w[0] = v.x; w[1] = v.y;
        }
        if (until == 0) {
#pragma unroll
          for (int g = 0; g < NG; ++g) w[g] = 0u;
        }
        RowParams<NG> q;
        q.set(w, vals);
        const float down = pow2i(-q.e), up9 = down * 512.0f;
        float* rp = reinterpret_cast<float*>(smem + SH::ROW + (it & 3) * SH::ROWBUF);
        if (!vals) {
          uint32_t s[NG / 2], y[4] = {0u, 0u, 0u, 0u};
#pragma unroll
          for (int g = 0; g < NG; g += 2) {
            s[g / 2] = pack_f16(q.s[g] * up9, q.s[g + 1] * up9);
            y[g / 2] = pack_f16(q.s[g] * down, q.s[g + 1] * down);
            y[NG / 2 + g / 2] = pack_f16(q.z[g] * down, q.z[g + 1] * down);
          }
          if constexpr (NG == 4)
            *reinterpret_cast<uint2*>(smem + SH::KS + r * 8) = make_uint2(s[0], s[1]);
          else
            *reinterpret_cast<uint32_t*>(smem + SH::KS + r * 4) = s[0];
          uint8_t* kx = smem + SH::KX + b * SH::KXBUF;
          *reinterpret_cast<uint4*>(kx + plain16_offset(r, 0)) = make_uint4(y[0], y[1], y[2], y[3]);
          *reinterpret_cast<uint4*>(kx + plain16_offset(r, 1)) = make_uint4(y[0], y[1], y[2], y[3]);
          rp[r] = pow2i(q.e);
          reinterpret_cast<int*>(rp)[192 + r] = from;
          reinterpret_cast<int*>(rp)[256 + r] = until;
          const int full = __all_sync(0xffffffffu, from <= at.lo && at.hi < until);
          if (lane == 0) reinterpret_cast<int*>(smem + SH::FULL)[(it & 3) * 2 + w4] = full;
        } else {
          rp[64 + r] = (float)q.e;
          rp[128 + r] = pow2i(-q.e);
          __half *vs = reinterpret_cast<__half*>(smem + SH::VS), *vm = reinterpret_cast<__half*>(smem + SH::VM);
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            vs[g * kPKV + r] = __float2half_rn(q.s[g] * up9);
            const float y = q.z[g] * down;
            const __half h = __float2half_rn(y);
            vm[g * kPKV + r] = h;
            vm[(NG + g) * kPKV + r] = __float2half_rn(__fsub_rn(y, __half2float(h)));
          }
        }
      }
      named_bar_sync(1, 128);
      // keys: thread -> row th % 64, words 2 (th / 64), + 1 of every group
      {
        const int r = th & 63, kh = th >> 6;
        uint8_t* kb = smem + SH::K + b * SH::KBUF;
        uint32_t s[NG / 2];
        if constexpr (NG == 4) {
          const uint2 v = *reinterpret_cast<const uint2*>(smem + SH::KS + r * 8);
          s[0] = v.x; s[1] = v.y;
        } else {
          s[0] = *reinterpret_cast<const uint32_t*>(smem + SH::KS + r * 4);
        }
#pragma unroll 1
        for (int x = 0; x < 2; ++x) {
          const int u = 2 * kh + x;
          uint32_t kw[NG];
          if constexpr (NG == 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(raw + r * 64 + ((u ^ ((r >> 1) & 3)) << 4));
            kw[0] = v.x; kw[1] = v.y; kw[2] = v.z; kw[3] = v.w;
          } else {
            const uint2 v = *reinterpret_cast<const uint2*>(raw + r * 32 + u * 8);
            kw[0] = v.x; kw[1] = v.y;
          }
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const __half2 sv = (g & 1) ? __high2half2(as_half2(s[g / 2])) : __low2half2(as_half2(s[g / 2]));
            const uint32_t w = kw[g], w8 = w >> 8;
            uint4 h, l;
            scale_pair(centre_low(w), sv, h.x, l.x);
            scale_pair(centre_high(w), sv, h.y, l.y);
            scale_pair(centre_low(w8), sv, h.z, l.z);
            scale_pair(centre_high(w8), sv, h.w, l.w);
            uint8_t* to = kb + (g >> 1) * (kPKV * 128) + sw128_offset(r, (g & 1) * 32 + u * 8);
            *reinterpret_cast<uint4*>(to) = h;
            *reinterpret_cast<uint4*>(to + KB * kPKV * 128) = l;
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar + B_KFULL + b);
      ok = ok && (it < 2 || wait(B_VFREE + b, ((it - 2) >> 1) & 1));
      // values, transposed: thread -> rows 2 lane, + 1, units 2 w4, + 1
      {
        uint8_t* vb = smem + SH::V + b * SH::VBUF;
        const uint32_t col = (uint32_t)(lane >> 2), in = (uint32_t)(lane & 3) * 4;
        const uint8_t* rv = raw + SH::RAWC;
#pragma unroll 1
        for (int x = 0; x < 2; ++x) {
          const int u = 2 * w4 + x;
          uint32_t va[NG / 2], vc[NG / 2];
          if constexpr (NG == 4) {
            const uint8_t* y = rv + lane * 128 + ((w4 ^ (lane & 3)) << 4) + x * 8;
            const uint2 y0 = *reinterpret_cast<const uint2*>(y), y1 = *reinterpret_cast<const uint2*>(y + 64);
            va[0] = y0.x; va[1] = y0.y; vc[0] = y1.x; vc[1] = y1.y;
          } else {
            va[0] = *reinterpret_cast<const uint32_t*>(rv + lane * 64 + u * 4);
            vc[0] = *reinterpret_cast<const uint32_t*>(rv + lane * 64 + 32 + u * 4);
          }
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const __half2 sv = *reinterpret_cast<const __half2*>(smem + SH::VS + g * (kPKV * 2) + lane * 4);
            const uint32_t w = __byte_perm(va[g / 2], vc[g / 2], (g & 1) ? 0x7632 : 0x5410), w8 = w >> 8;
            uint32_t h[4], l[4];
            scale_pair(centre_low(w), sv, h[0], l[0]);
            scale_pair(centre_high(w), sv, h[1], l[1]);
            scale_pair(centre_low(w8), sv, h[2], l[2]);
            scale_pair(centre_high(w8), sv, h[3], l[3]);
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              const int ch = 32 * g + 4 * u + n;  // its row in the swizzled tile; (ch & 7) = 4 x + n
              uint8_t* to = vb + (uint32_t)(ch >> 3) * 1024u + (uint32_t)(4 * x + n) * 128u + ((col ^ (uint32_t)(4 * x + n)) << 4) + in;
              *reinterpret_cast<uint32_t*>(to) = h[n];
              *reinterpret_cast<uint32_t*>(to + SH::NV * 128) = l[n];
            }
          }
        }
        if (w4 < NG) {  // the middles of group w4
          uint8_t* to = vb + (HD >> 3) * 1024 + w4 * 128 + ((col ^ (uint32_t)w4) << 4) + in;
          *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(smem + SH::VM + w4 * (kPKV * 2) + lane * 4);
          *reinterpret_cast<uint32_t*>(to + SH::NV * 128) = *reinterpret_cast<const uint32_t*>(smem + SH::VM + (NG + w4) * (kPKV * 2) + lane * 4);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar + B_VFULL + b);
      advance(at);
    }
    cp_async_wait<0>();
  } else if (lane == 0) {
    // ---- MMAs -----------------------------------------------------------------------------------
    constexpr uint32_t ids = idesc_f16_f32(kPRows, kPKV), idv = idesc_f16_f32(kPRows, SH::NV);
    int it = 0, seg = 0;
    bool ok = true;
    auto scores = [&](int i) -> bool {
      const int b = i & 1;
      if (!wait_one(B_KFULL + b, (i >> 1) & 1)) return false;
      tc_fence_after();
      const uint32_t d = tbase + kColS + b * kPKV;
      const uint8_t* kb = smem + SH::K + b * SH::KBUF;
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
        for (int k = 0; k < 4; ++k) tc_mma_ts(d, tbase + kColQ + 8 * (4 * x + k), bd + 2 * k, ids, 1u);
      }
      tc_mma(d, smem_desc_plain16(smem + SH::QX), smem_desc_plain16(smem + SH::KX + b * SH::KXBUF), ids, 1u);
#pragma unroll
      for (int x = 0; x < KB; ++x) {
        const uint64_t bd = smem_desc_sw128(kb + x * kPKV * 128);
#pragma unroll
        for (int k = 0; k < 4; ++k) tc_mma_ts(d, tbase + kColQ + 8 * (4 * x + k), bd + 2 * k, ids, 1u);
      }
      tc_commit(bar + B_KFREE + b);
      tc_commit(bar + B_SFULL + b);
      return true;
    };
    for (int64_t t = t_begin; ok && t < t_end; ++seg) {
      const Segment sg = find_segment(pre, pa.tiles, sum, c.heads, t, t_end);
      const int n = sg.end - sg.begin;
      if (!(ok = wait_one(B_QFULL, seg & 1))) break;
      if (!(ok = scores(it))) break;
      for (int j = 0; j < n; ++j, ++it) {
        const int b = it & 1;
        if (j + 1 < n && !(ok = scores(it + 1))) break;
        if (!(ok = wait_one(B_VFULL + b, (it >> 1) & 1))) break;
        if (!(ok = wait_one(B_PFULL + b, (it >> 1) & 1))) break;
        tc_fence_after();
        const uint8_t* vb = smem + SH::V + b * SH::VBUF;
        const uint32_t pcol = tbase + kColS + b * kPKV;
#pragma unroll
        for (int p = 0; p < 3; ++p) {  // low high, high low, high high
          const uint64_t bd = smem_desc_sw128(vb + (p == 1 ? SH::NV * 128 : 0));
#pragma unroll
          for (int k = 0; k < 4; ++k)
            tc_mma_ts(tbase + kColO, pcol + (p == 0 ? 8 : 0) + 16 * k, bd + 2 * k, idv, (j % kPDrain > 0 || p > 0 || k > 0) ? 1u : 0u);
        }
        tc_commit(bar + B_VFREE + b);
        tc_commit(bar + B_PDONE + b);
      }
      if (!ok) break;
      t += n;
    }
    // every MMA issued has completed before tensor memory is released
    tc_commit(bar + B_END);
    if (!mbar_wait_bounded(bar + B_END, 0)) atomicOr(a.err, SHD_DEVERR_TIMEOUT_DRAIN);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_dealloc(tbase, kCols);
}

// Items that a share boundary cuts, joined in CTA order: block (b, y) takes rows 8 y .. + 7 of the item
// whose first cut is boundary b + 1; a warp takes a row.
template <int HD>
__global__ void __launch_bounds__(256) kv4_join_kernel(const __grid_constant__ PromptArgs pa, int ctas) {
  using SH = PromptShape<HD>;
  const Kv4AttnArgs& a = pa.a;
  __shared__ int pre[kPTiles];
  __shared__ int scratch[16];
  pdl_trigger();
  pdl_wait();
  const int G = a.H / a.c.heads;
  const int sum = plan_tiles(a, pa.tiles, G, pre, scratch);
  const int64_t T = (int64_t)sum * a.c.heads, per = (T + ctas - 1) / ctas, t = (blockIdx.x + 1) * per;
  if (t >= T) return;
  const Segment sg = find_segment(pre, pa.tiles, sum, a.c.heads, t, T);
  const int64_t item = t - sg.begin;
  if (sg.begin == 0 || item / per != (int64_t)blockIdx.x) return;  // not cut here, or not for the first time
  const int w0 = (int)(item / per), parts = (int)((item + sg.steps - 1) / per) - w0 + 1;
  const int lane = threadIdx.x & 31, row = blockIdx.y * 8 + (threadIdx.x >> 5);
  const int64_t r = (int64_t)sg.tile * kPRows + row;
  if (r >= (int64_t)a.M * G) return;
  const size_t step = (size_t)2 * kPRows * SH::PART;
  const float* first = pa.parts + ((size_t)w0 * 2 + (w0 * per >= item ? 0 : 1)) * kPRows * SH::PART + (size_t)row * SH::PART;
  const float* next = pa.parts + (size_t)(w0 + 1) * step + (size_t)row * SH::PART;
  auto part = [&](int w) { return w == 0 ? first : next + (size_t)(w - 1) * step; };
  float M = -INFINITY, L = 0.0f;
  for (int w = lane; w < parts; w += 32) M = fmaxf(M, __ldcg(part(w)));
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  constexpr int CPL = HD / 32;  // channels a lane
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
  const size_t at = (size_t)(r / G) * a.H * HD + (size_t)(sg.head * G + r % G) * HD + CPL * lane;
#pragma unroll
  for (int i = 0; i < CPL; ++i) {
    const float mk = a.mask ? a.mask[at + i] : 0.0f;
    a.out_c[at + i] = __fsub_rn(__fdiv_rn(y[i], D), mk);
    a.out_s[at + i] = mk;
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
  if (!ctx->d_kv4_parts) SHD_CHECK_CUDA(ctx, cudaMalloc(&ctx->d_kv4_parts, need * 4));
  const int G = a0.H / a0.c.heads;
  // launches of at most kPTiles tiles: whole positions
  const int step = (int)std::min<int64_t>(a0.M, (int64_t)kPTiles * kPRows / G);
  SHD_REQUIRE(ctx, step > 0, "shd_kv4_attn_prefill: too many heads");
  for (int m = 0; m < a0.M; m += step) {
    PromptArgs pa{};
    pa.a = a0;
    const size_t width = (size_t)a0.H * HD;
    pa.a.M = std::min(step, a0.M - m);
    pa.a.pos0 += m;
    pa.a.q += (size_t)m * a0.ldq;
    if (a0.mask) pa.a.mask += m * width;
    pa.a.out_c += m * width;
    pa.a.out_s += m * width;
    pa.last = a0.pos0 + a0.M - 1;
    pa.parts = ctx->d_kv4_parts;
    pa.tiles = (int)(((int64_t)pa.a.M * G + kPRows - 1) / kPRows);
    SHD_CHECK_CUDA(ctx, launch_pdl(kv4_prefill_kernel<HD>, dim3(ctas), dim3(kPThreads), SH::SMEM, ctx->stream, pa));
    SHD_CHECK_CUDA(ctx, launch_pdl(kv4_join_kernel<HD>, dim3(ctas - 1, kPRows / 8), dim3(256), 0, ctx->stream, pa, ctas));
    ctx->launches += 2;
  }
  return SHD_OK;
}

}  // namespace

int launch_kv4_prefill(shd_ctx* ctx, const Kv4AttnArgs& a) {
  return a.c.head_dim == 128 ? launch_prefill_t<128>(ctx, a) : launch_prefill_t<64>(ctx, a);
}

}  // namespace shd
