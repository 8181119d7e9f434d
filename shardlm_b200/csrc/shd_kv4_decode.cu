// Single-token attention over the 4-bit cache (format in shd_kv4.cuh), grouped by kv head.
//
// With k = s c + z and v = s c + z per group g of 32 channels,
//   q . k_t  = sum_g s_tg (sum_(i in g) q_i (c_ti - 7.5)) + sum_g (z_tg + 7.5 s_tg) (sum_(i in g) q_i)
//   o        = sum_t p_t v_t = sum_t (p_t s_tg) (c_t - 7.5) + sum_t p_t (z_tg + 7.5 s_tg)
// so the codes themselves are tensor-core operands: a code is at most 4 bits and is exact in f16 as
// the subnormal c * 2^-24 (its bits under a mask, one instruction for two codes; the nibble above it
// is c * 2^-20), centred to (c - 7.5) * 2^-9, also exact, by one more: weights add up to 1 over many rows
// whose values cancel, and sums of codes that are all positive would lose what cancels (measured
// against 64 bits at 131000 positions: 5e-4 of the result). The other operand is split into two f16 terms
// (22 bits, or 2^-37 of the largest beside them): the queries and their group sums, scaled by powers of two
// of their head, and the weights p_t s_tg, scaled by a running power of two of their head that follows
// the largest weight times its row's largest scale, so that a row which weighs nothing has no say however
// large its values are. A group whose scales are 2^-k of the row's largest loses bits from k = 15 on.
// Sums are f32. Rows of the first product's A are the 8 heads' high terms and the 8 heads' low terms;
// the second takes the two terms one after the other:
//   S [8 + 8 heads x 8 rows]      += Q [16 x 16 channels] K^T   per group, then scaled by s
//   O^T [16 channels x 8 heads]   += V^T [16 x 16 rows] W       per group
// The accumulator of S has the layout of the B operand of the second product, so weights never
// leave their thread. A lane's row order within 8 rows (sigma) is t, t + 4: with it every shared-memory
// read below is free of bank conflicts.
//
// Work: an item is (query row, kv head, up to 8 query heads) with its visible 16-row chunks (kv4_spans).
// When the items are few, each is cut evenly into as many parts as give every CTA at most one (one sequence
// at 554 positions: 11.4 us where equal shares took 14.7); else the
// chunks of all items, with kDItem for an item's start and end, are laid end to end and cut into equal
// shares, whatever the lengths. In a CTA the 8 warps take chunks in turn, each with its own ring
// of asynchronous copies and its own online softmax, and are combined in warp order. An item that is cut
// leaves partial results; the CTA that arrives last joins them in CTA order, so results do not depend on
// timing.
//
// Measured on a B200: one sequence at 131001 positions, 28 heads over 4, 42.1 us (2.0 TB/s of cache); 64
// ragged ones under a window of 2048 and 4 sinks, 40 heads over 8, 73.1 us (2.3 TB/s); 8 at 1041 to 1280
// positions 15.1 us; one at 554 positions 10.2 us. No pipe is full in the long ones (of the windowed batch's
// time on the SMs the integer pipe is busy 38 %, tensor 23 %, issue slots 56 %, memory 27 %): a chunk of 16
// rows is some 500 instructions of a warp in dependent steps, and the registers hold four warps a scheduler.
// It takes 196 clocks of an SM, where its 215 integer and conversion instructions alone take 107. Short ones
// are bound by the chain of launch, plan, first rows from memory, combine and join, one after the other.
#include <cmath>

#include "shd_kv4.cuh"

namespace shd {
namespace {

constexpr int kDWarps = 8;
constexpr int kDThreads = 32 * kDWarps;
constexpr int kDStages = 4;       // chunks of a warp's ring
constexpr int kDRows = 512;       // query rows of one launch (their chunk counts are in shared memory)
// what an item costs a CTA besides its chunks, in chunks: at 12, 18 and 24 the windowed batch above takes 82.5,
// 72.8 and 72.4 us
constexpr int kDItem = 18;
constexpr int kDJoin = 12;        // parts that are joined at once, and in groups of how many where there are more
constexpr int kDGroup = 10;
constexpr int kDGroupMax = 32;    // (the larger of kDJoin, kDGroup and the groups of all CTAs)
constexpr int kDCounters = 1 << 15;  // items' counters, then the groups'
constexpr int kDSizes = 8;        // sizes of a part that are tried, kDWarps chunks apart
// stands for the exponent of scales that are all 0 (such a row adds its minima only, in f32): low enough that the row
// has no say where another has, and 2^-kFlat sums of 2^17 rows of any minima stay in f32
constexpr float kFlat = -60.0f;

template <int HD>
struct DecodeShape {
  static constexpr int NG = HD / kKv4Group;
  static constexpr int CODE = kKv4Chunk * HD / 2;      // bytes of a chunk's codes (K or V)
  static constexpr int PAR = kKv4Chunk * 4 * NG;       // bytes of a chunk's parameters
  static constexpr int STAGE = 2 * (CODE + PAR);
  static constexpr int PART = HD + 4;                  // of one head: running max, sum, 2 unused, weighted V
  static constexpr int LEFT = 8 * HD + 16;             // of a cut item: weighted V of 8 heads, maxima, sums
  // a chunk's parameters in f32: [keys, values][scale, middle][half of the chunk][tig][group][row sigma(2 tig),
  // sigma(2 tig + 1)], then of each row 13 less the exponent of its largest value scale: [half of the chunk][tig][the two rows]
  static constexpr int ROWS = 4 * kKv4Chunk * NG * 4 + kKv4Chunk * 4;
  static constexpr int RING = kDWarps * (kDStages * STAGE + ROWS);
  static constexpr int JOIN = kDWarps * 8 * PART * 4;  // per warp and head, over the rings
  static constexpr size_t SMEM = (RING > JOIN ? RING : JOIN) + kDRows * 16 + 64 * 4 + 16 * 4 + 256;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// the same with nothing to add to
__device__ __forceinline__ void mma_f16_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                            uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma_f16_k8_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5}, {%6}, {%7, %7, %7, %7};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(b0), "f"(0.0f));
}

// Asynchronous copies of a chunk: this lane's source addresses for row 0 of the (slot, head) and its
// places within a stage.
template <int HD>
struct Feed {
  using S = DecodeShape<HD>;
  static constexpr int CPR = HD / 32;         // 16-byte pieces of a row of codes
  static constexpr int NC = kKv4Chunk * CPR;  // pieces of a chunk's codes: 64 or 32
  static constexpr int NP = S::PAR / 16;      // pieces of a chunk's parameters: 16 or 8
  const uint8_t *k, *v, *p;
  uint32_t dk[NC / 32], dv[NC / 32], dp;

  __device__ __forceinline__ void places(int lane) {
#pragma unroll
    for (int i = 0; i < NC / 32; ++i) {
      const int x = lane + 32 * i, r = x / CPR, q = x % CPR;
      // keys: row sigma(n) of each 8 stored as n-th, so that a quad's 8 neighbours are contiguous
      const int n = (r & 8) | ((r & 4) ? 2 * (r & 3) + 1 : 2 * (r & 3));
      dk[i] = (n * CPR + q) * 16;
      // values: rows 2, 3 (mod 4) with their halves exchanged
      dv[i] = S::CODE + (r * CPR + (HD == 128 ? q ^ (r & 2) : q)) * 16;
    }
    dp = 2 * S::CODE + min(lane, 2 * NP - 1) * 16;
  }
  __device__ __forceinline__ void source(const Kv4View& c, size_t base, int lane) {
    k = c.kc + base * (HD / 2) + lane * 16;
    v = c.vc + base * (HD / 2) + lane * 16;
    p = reinterpret_cast<const uint8_t*>(lane < NP ? c.kp : c.vp) + base * (4 * S::NG) + (lane & (NP - 1)) * 16;
  }
  __device__ __forceinline__ void chunk(int i, uint32_t st, int lane) const {
#pragma unroll
    for (int j = 0; j < NC / 32; ++j) {
      copy(st + dk[j], k + (size_t)i * S::CODE + j * 512);
      copy(st + dv[j], v + (size_t)i * S::CODE + j * 512);
    }
    if (lane < 2 * NP) copy(st + dp, p + (size_t)i * S::PAR);
  }
  static __device__ __forceinline__ void copy(uint32_t dst, const uint8_t* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  }
};

// f32 pairs (rows sigma(2 tig), sigma(2 tig + 1)) of NG groups
template <int NG>
__device__ __forceinline__ void load_pairs(const float* p, uint64_t (&v)[NG]) {
#pragma unroll
  for (int g = 0; g < NG; g += 2) {
    const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(p + 2 * g);
    v[g] = x.x;
    v[g + 1] = x.y;
  }
}

// What a query sees, by row: rows below the sinks hold their own position; the others hold position
// r + up while r <= edge, r + down past it.
struct Seen {
  int p, sinks, lowest, edge, up, down;
  __device__ __forceinline__ bool row(int r) const {
    const int t = r <= edge ? r + up : r + down;
    return r < sinks ? r <= p : (t >= lowest && t <= p);
  }
};

__device__ __forceinline__ Seen make_seen(const Kv4View& c, int p, int window) {
  Seen s;
  s.p = p;
  s.sinks = c.sinks;
  const int64_t far = (int64_t)p - window + 1;
  s.lowest = window > 0 && far > c.sinks ? (int)far : c.sinks;
  if (p < c.capacity) {
    s.edge = c.capacity;
    s.up = s.down = 0;
  } else {
    s.edge = kv4_row(c, p);
    s.up = p - s.edge;
    s.down = s.up - (c.capacity - c.sinks);
  }
  return s;
}

// y += e * v; a part with weight 0 may hold anything
__device__ __forceinline__ void add_part4(float4& y, const float4& v, float e) {
  if (e == 0.0f) return;
  y.x = fmaf(e, v.x, y.x);
  y.y = fmaf(e, v.y, y.y);
  y.z = fmaf(e, v.z, y.z);
  y.w = fmaf(e, v.w, y.w);
}
__device__ __forceinline__ void add_part(float4& y, const float* p, float e) {
  add_part4(y, *reinterpret_cast<const float4*>(p), e);
}

// (y / L - mask, mask); a row that sees nothing (L = 0) gives 0
__device__ __forceinline__ void store_shares(const Kv4AttnArgs& a, int m, int col, const float4& y, float L) {
  const size_t at = (size_t)m * a.H * a.c.head_dim + col;
  const float4 mk = a.mask ? *reinterpret_cast<const float4*>(a.mask + m * a.ldmask + col) : make_float4(0.f, 0.f, 0.f, 0.f);
  const float D = L == 0.0f ? 1.0f : L;
  *reinterpret_cast<float4*>(a.out_c + at) =
      make_float4(__fsub_rn(__fdiv_rn(y.x, D), mk.x), __fsub_rn(__fdiv_rn(y.y, D), mk.y),
                  __fsub_rn(__fdiv_rn(y.z, D), mk.z), __fsub_rn(__fdiv_rn(y.w, D), mk.w));
  *reinterpret_cast<float4*>(a.out_s + at) = mk;
}

template <int HD>
__global__ void __launch_bounds__(kDThreads, 2) kv4_decode_kernel(const Kv4AttnArgs a, float* ws, int* counters) {
  using SH = DecodeShape<HD>;
  constexpr int NG = SH::NG, PART = SH::PART;
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr size_t kBody = SH::RING > SH::JOIN ? SH::RING : SH::JOIN;
  int64_t* pre = reinterpret_cast<int64_t*>(smem + kBody);              // costs (or parts) of the rows before
  int2* rows = reinterpret_cast<int2*>(smem + kBody + kDRows * 8);      // (position or -1, slot)
  float* wgt = reinterpret_cast<float*>(smem + kBody + kDRows * 16);    // [warp][head] combine weights
  float* total = wgt + 64;                                              // [head] max, [head] sum
  int* flag = reinterpret_cast<int*>(total + 16);
  int64_t* scan = reinterpret_cast<int64_t*>(total + 32);               // [8] warp sums
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, tig = lane & 3;
  const Kv4View& c = a.c;
  Feed<HD> feed;
  feed.places(lane);
  pdl_trigger();
  pdl_wait();

  // chunk counts of the rows (a row that sees nothing counts one, for its output), and sums of costs or
  // parts over the rows before each: up to 32 rows in every warp's registers, more by way of shared memory
  const int G = a.H / c.heads, nsub = (G + 7) / 8, HS = c.heads * nsub;
  const bool few = a.M <= 32;
  auto row_of = [&](int m, int& p, int& sl) -> int {
    p = a.pos[m];
    sl = a.slot[m];
    const bool ok = p >= 0 && sl >= 0 && sl < c.slots && kv4_in_reach(c, p, a.window, 0);
    if (p >= 0 && !ok && blockIdx.x == 0) atomicOr(a.err, SHD_DEVERR_ARG);
    if (!ok) p = -1;
    return max(kv4_spans(c, p, p, a.window).total, 1);
  };
  int my_p = -1, my_slot = 0;            // of row `lane`, where the rows are few
  int64_t my_pre = 0, sum = 0;
  int size = 0;                          // of a part, in chunks; 0: equal shares of all chunks
  if (few) {
    const int n = lane < a.M ? row_of(lane, my_p, my_slot) : 0;
    auto prefix = [&](int64_t v) {
      int64_t x = lane < a.M ? v : 0;
      const int64_t own = x;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      my_pre = x - own;
      sum = __shfl_sync(0xffffffffu, x, 31);
    };
    prefix((int64_t)n + kDItem);
    if (a.M * HS <= (int)gridDim.x) {
      // the least size, in steps of kDWarps, that gives every CTA at most one part: lane y tries the y-th
      const int64_t chunks = (sum - (int64_t)a.M * kDItem) * HS;
      const uint32_t first = (uint32_t)(((chunks + gridDim.x - 1) / gridDim.x + kDWarps - 1) / kDWarps) * kDWarps;
      const uint32_t mine = first + kDWarps * lane;
      uint32_t all = 0;
      for (int m = 0; m < a.M; ++m) all += ((uint32_t)__shfl_sync(0xffffffffu, n, m) + mine - 1) / mine;
      const uint32_t fit = __ballot_sync(0xffffffffu, (uint64_t)all * HS <= gridDim.x) & ((1u << kDSizes) - 1u);
      if (fit) {
        size = (int)first + kDWarps * (__ffs(fit) - 1);
        prefix((n + size - 1) / size);
      }
    }
  } else {
    for (int m0 = 0; m0 < a.M; m0 += kDThreads) {
      const int m = m0 + tid;
      int64_t n = 0;
      if (m < a.M) {
        int p, sl;
        n = row_of(m, p, sl) + kDItem;
        rows[m] = make_int2(p, sl);
      }
      int64_t x = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (lane == 31) scan[warp] = x;
      __syncthreads();
      int64_t base = sum;
#pragma unroll
      for (int w = 0; w < kDWarps; ++w) {
        if (w < warp) base += scan[w];
        sum += scan[w];
      }
      if (m < a.M) pre[m] = base + x - n;
      __syncthreads();
    }
  }
  const int64_t T = sum * HS;
  const int64_t per = size ? 1 : (T + gridDim.x - 1) / gridDim.x;
  const int64_t t_begin = blockIdx.x * per, t_end = min(T, t_begin + per);

  for (int64_t t = t_begin; t < t_end;) {
    // the item that t falls into: its parts, or kDItem for its start and end, then its chunks
    int m, p, sl, cost;
    int64_t row_t;
    if (few) {
      m = 31 - __clz(__ballot_sync(0xffffffffu, lane < a.M && my_pre * HS <= t));
      p = __shfl_sync(0xffffffffu, my_p, m);
      sl = __shfl_sync(0xffffffffu, my_slot, m);
      const int64_t here = __shfl_sync(0xffffffffu, my_pre, m), next = __shfl_sync(0xffffffffu, my_pre, (m + 1) & 31);
      row_t = here * HS;
      cost = (int)((m + 1 < a.M ? next : sum) - here);
    } else {
      int lo = 0, hi = a.M - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (pre[mid] * HS <= t) lo = mid; else hi = mid - 1;
      }
      m = lo;
      p = rows[m].x;
      sl = rows[m].y;
      row_t = pre[m] * HS;
      cost = (int)((m + 1 < a.M ? pre[m + 1] : sum) - pre[m]);
    }
    const uint64_t in_row = (uint64_t)(t - row_t);
    const int hs = in_row >> 32 ? (int)(in_row / (uint64_t)cost) : (int)((uint32_t)in_row / (uint32_t)cost);
    const int64_t item_t = row_t + (int64_t)hs * cost;
    const int64_t done = min(t_end, item_t + cost);
    const Kv4Spans sp = kv4_spans(c, p, p, a.window);
    int n, c0, c1, w0, parts;  // chunks, this CTA's of them, first CTA of the item and how many
    if (size) {
      const int part = (int)(t - item_t);
      n = max(sp.total, 1);
      c0 = (int)((int64_t)n * part / cost);
      c1 = (int)((int64_t)n * (part + 1) / cost);
      w0 = (int)item_t;
      parts = cost;
    } else {
      n = cost - kDItem;
      c0 = max((int)(t - item_t) - kDItem, 0);
      c1 = (int)(done - item_t) - kDItem;
      if (c1 <= c0) {  // none of its chunks
        t = done;
        continue;
      }
      w0 = (int)((item_t + kDItem) / per);
      parts = (int)((item_t + cost - 1) / per) - w0 + 1;
    }
    const int kvh = hs / nsub, h0 = kvh * G + (hs % nsub) * 8, nh = min(8, kvh * G + G - h0);
    const Seen seen = make_seen(c, p, a.window);
    const size_t base = p >= 0 ? kv4_base(c, sl, kvh) : 0;

    // this warp's chunks: c0 + warp, + 8, ..
    const int first = c0 + warp, stop = p >= 0 ? min(c1, sp.total) : 0;
    const int mine = first < stop ? (stop - first + kDWarps - 1) / kDWarps : 0;
    uint8_t* ring = smem + warp * (kDStages * SH::STAGE + SH::ROWS);
    const uint32_t ring_at = smem_u32(ring);
    float* rows_f32 = reinterpret_cast<float*>(ring + kDStages * SH::STAGE);
    feed.source(c, base, lane);
#pragma unroll
    for (int i = 0; i < kDStages - 1; ++i) {
      if (i < mine) feed.chunk(kv4_span_chunk(sp, first + i * kDWarps), ring_at + i * SH::STAGE, lane);
      cp_async_commit();
    }

    // queries of head gid: two f16 terms of q * 2^k, in the order of the masked code words
    uint32_t qh[NG][4], ql[NG][4], zh, zl;
    float factor, zfactor;
    {
      const float* q = a.q + (size_t)m * a.ldq + (size_t)(h0 + min(gid, nh - 1)) * HD + 8 * tig;
      float x[NG][8], qs[NG], top = 0.0f, ztop = 0.0f;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const float4 u = *reinterpret_cast<const float4*>(q + 32 * g), v = *reinterpret_cast<const float4*>(q + 32 * g + 4);
        x[g][0] = u.x; x[g][1] = u.y; x[g][2] = u.z; x[g][3] = u.w;
        x[g][4] = v.x; x[g][5] = v.y; x[g][6] = v.z; x[g][7] = v.w;
        qs[g] = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          top = fmaxf(top, fabsf(x[g][i]));
          qs[g] = __fadd_rn(qs[g], x[g][i]);
        }
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // |q| 2^k <= 2^13, k at least -115 for a finite query; the limit keeps 2^(9 - k) normal
      const int k = min(13 - ceil_exp2(top), 100);
      const float up = pow2i(k);
      const float sc = a.scale * 1.44269504088896341f;
      factor = sc * pow2i(9 - k);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        qs[g] = __fadd_rn(qs[g], __shfl_xor_sync(0xffffffffu, qs[g], 1));
        qs[g] = __fadd_rn(qs[g], __shfl_xor_sync(0xffffffffu, qs[g], 2));
        ztop = fmaxf(ztop, fabsf(qs[g]));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          split_f16(x[g][i] * up, x[g][i + 4] * up, qh[g][i], ql[g][i]);  // channel pairs (i, i + 4)
        }
      }
      // the query sums against a row's parameters (scales, then minima): word tig of the row
      const int kz = min(12 - ceil_exp2(ztop), 100);  // 7.5 |sum| 2^kz < 2^15
      zfactor = sc * pow2i(-kz);
      const float zup = pow2i(kz) * (tig < NG / 2 ? 7.5f : (tig < NG ? 1.0f : 0.0f));
      float za = qs[0], zb = qs[1];
      if constexpr (NG == 4) {
        if (tig & 1) { za = qs[2]; zb = qs[3]; }
      }
      split_f16(za * zup, zb * zup, zh, zl);
    }

    float o[HD / 16][4];  // [2 g + e]: channels 32 g + 4 gid + 2 e (+ 1: third and fourth), heads 2 tig, + 1
#pragma unroll
    for (int i = 0; i < HD / 16; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
    uint64_t oz[NG];  // head gid's minima, even and odd rows
#pragma unroll
    for (int g = 0; g < NG; ++g) oz[g] = pair(0.0f, 0.0f);
    // weights are 2^(score - mx), mx the running maximum of score + e - 13, e the exponent of the row's largest
    // value scale: weight times scale is at most 2^13, and at least 2^12 for the row that adds most
    float mx = kKv4Never, l = 0.0f;

#pragma unroll 1
    for (int i = 0; i < mine; ++i) {
      cp_async_wait<kDStages - 2>();
      __syncwarp();
      const int at = i % kDStages;
      {
        const int nx = i + kDStages - 1;
        if (nx < mine) feed.chunk(kv4_span_chunk(sp, first + nx * kDWarps), ring_at + (nx % kDStages) * SH::STAGE, lane);
        cp_async_commit();
      }
      const uint8_t* st = ring + at * SH::STAGE;
      // lanes 0-15: the rows' key parameters, 16-31: their value parameters, in f32 for the 8 heads' lanes; a
      // row out of sight has them 0, whatever its memory holds
      uint32_t sight;
      {
        const int r = lane & 15, kind = lane >> 4;
        const bool ok = seen.row(kv4_span_chunk(sp, first + i * kDWarps) * kKv4Chunk + r);
        sight = __ballot_sync(0xffffffffu, ok);
        uint8_t* from = ring + at * SH::STAGE + 2 * SH::CODE + kind * SH::PAR + r * (4 * NG);
        uint32_t w[NG];
        if constexpr (NG == 4) {
          const uint4 x = *reinterpret_cast<const uint4*>(from);
          w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
        } else {
          const uint2 x = *reinterpret_cast<const uint2*>(from);
          w[0] = x.x; w[1] = x.y;
        }
        if (!ok) {
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            w[g] = 0u;
            *reinterpret_cast<uint32_t*>(from + 4 * g) = 0u;
          }
        }
        float* out = rows_f32 + kind * (2 * kKv4Chunk * NG) + (((r >> 3) * 4 + (r & 3)) * NG) * 2 + ((r >> 2) & 1);
        float top = 0.0f;
#pragma unroll
        for (int g = 0; g < NG / 2; ++g) {
          const float2 v = unpack_f16(w[g]), z = unpack_f16(w[NG / 2 + g]);
          out[4 * g] = v.x;
          out[4 * g + 2] = v.y;
          out[kKv4Chunk * NG + 4 * g] = fmaf(7.5f, v.x, z.x);
          out[kKv4Chunk * NG + 4 * g + 2] = fmaf(7.5f, v.y, z.y);
          top = fmaxf(top, fmaxf(v.x, v.y));
        }
        // 13 less the exponent e with top < 2^e, as f32: 2^23 + n has n in its low bits
        if (kind)
          rows_f32[4 * kKv4Chunk * NG + ((r >> 3) * 4 + (r & 3)) * 2 + ((r >> 2) & 1)] =
              fminf((8388608.0f + 126.0f + 13.0f) - __uint_as_float(0x4b000000u | (__float_as_uint(top) >> 23)), 13.0f - kFlat);
      }
      __syncwarp();

      // scores (log2 units) of head gid with row 8 j + tig (and + 4): s[2 j (+ 1)]
      float s[4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint8_t* kp = st + 2 * SH::CODE;
        uint32_t kw[NG];
        if constexpr (NG == 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(st + (8 * j + gid) * (HD / 2) + 16 * tig);
          kw[0] = v.x; kw[1] = v.y; kw[2] = v.z; kw[3] = v.w;
        } else {
          const uint2 v = *reinterpret_cast<const uint2*>(st + (8 * j + gid) * (HD / 2) + 8 * tig);
          kw[0] = v.x; kw[1] = v.y;
        }
        uint64_t sc[NG];
        load_pairs<NG>(rows_f32 + (j * 4 + tig) * NG * 2, sc);
        // the minima's part: all parameters of row sigma(gid) times (7.5 and 1) x the groups' query sums
        float z[4];
        const int zr = 8 * j + (gid >> 1) + 4 * (gid & 1);
        mma_f16_k8_new(z, zh, zl, *reinterpret_cast<const uint32_t*>(kp + zr * (4 * NG) + 4 * (NG == 4 ? tig : (tig & 1))));
        uint64_t d = pair(0.0f, 0.0f);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          float acc[4];
          const uint32_t w = kw[g], w8 = w >> 8;
          mma_f16_new(acc, qh[g][0], ql[g][0], qh[g][1], ql[g][1], as_u32(centre_low(w)), as_u32(centre_high(w)));
          mma_f16(acc, qh[g][2], ql[g][2], qh[g][3], ql[g][3], as_u32(centre_low(w8)), as_u32(centre_high(w8)));
          d = fma2(sc[g], add2(pair(acc[0], acc[1]), pair(acc[2], acc[3])), d);
        }
        const float2 y = unpair(fma2(d, pair(factor, factor), mul2(add2(pair(z[0], z[1]), pair(z[2], z[3])), pair(zfactor, zfactor))));
        s[2 * j] = y.x;
        s[2 * j + 1] = y.y;
      }
      if ((sight & 0xffffu) != 0xffffu) {
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if (!(sight >> (4 * x + tig) & 1u)) s[x] = -INFINITY;
      }
      // score + e - 13, and below back to the score from its difference to mx: the difference has no rounding, so that
      // scores of any size leave the weights in range
      const uint64_t* less = reinterpret_cast<const uint64_t*>(rows_f32 + 4 * kKv4Chunk * NG + 2 * tig);
      const uint64_t less0 = less[0], less1 = less[4], minus = pair(-1.0f, -1.0f);
      const uint64_t sum0 = fma2(less0, minus, pair(s[0], s[1])), sum1 = fma2(less1, minus, pair(s[2], s[3]));
      const float2 t0 = unpair(sum0), t1 = unpair(sum1);
      float tm = fmaxf(fmaxf(t0.x, t0.y), fmaxf(t1.x, t1.y));
      tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, 1));
      tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, 2));

      // rescale when a head's maximum grows
      if (__any_sync(0xffffffffu, tm > mx)) {
        const float now = fmaxf(mx, tm);
        const float al = exp2_fast(mx - now);
        mx = now;
        l *= al;
#pragma unroll
        for (int g = 0; g < NG; ++g) oz[g] = mul2(oz[g], pair(al, al));
        const float al0 = __shfl_sync(0xffffffffu, al, 8 * tig), al1 = __shfl_sync(0xffffffffu, al, 8 * tig + 4);
#pragma unroll
        for (int x = 0; x < HD / 16; ++x) {
          o[x][0] *= al0; o[x][1] *= al1; o[x][2] *= al0; o[x][3] *= al1;
        }
      }

      // weights: plain for the sum and the minima, times scale and as two f16 terms for the codes
      float w[4];
      {
        const uint64_t low = pair(-mx, -mx);
        const float2 x0 = unpair(add2(add2(sum0, low), less0)), x1 = unpair(add2(add2(sum1, low), less1));
        w[0] = exp2_fast(x0.x);
        w[1] = exp2_fast(x0.y);
        w[2] = exp2_fast(x1.x);
        w[3] = exp2_fast(x1.y);
        l += w[0];
        l += w[1];
        l += w[2];
        l += w[3];
      }
      uint32_t wh[NG][2], wl[NG][2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint64_t ww = pair(w[2 * j], w[2 * j + 1]);
        const float* v = rows_f32 + 2 * kKv4Chunk * NG + (j * 4 + tig) * NG * 2;
        uint64_t sc[NG], mid[NG];
        load_pairs<NG>(v, sc);
        load_pairs<NG>(v + kKv4Chunk * NG, mid);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          oz[g] = fma2(ww, mid[g], oz[g]);
          split_pair(mul2(ww, sc[g]), wh[g][j], wl[g][j]);
        }
      }
      // value codes of unit gid, rows in the same order
      uint32_t vw[4][NG / 2];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int r = 8 * (x >> 1) + 4 * (x & 1) + tig;
        const uint8_t* v = st + SH::CODE + r * (HD / 2);
        if constexpr (NG == 4) {
          const uint2 y = *reinterpret_cast<const uint2*>(v + 16 * ((gid >> 1) ^ (r & 2)) + 8 * (gid & 1));
          vw[x][0] = y.x; vw[x][1] = y.y;
        } else {
          vw[x][0] = *reinterpret_cast<const uint32_t*>(v + 4 * gid);
        }
      }
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint32_t t0 = __byte_perm(vw[0][g / 2], vw[1][g / 2], (g & 1) ? 0x7632 : 0x5410);
        const uint32_t t1 = __byte_perm(vw[2][g / 2], vw[3][g / 2], (g & 1) ? 0x7632 : 0x5410);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t u0 = e ? t0 >> 8 : t0, u1 = e ? t1 >> 8 : t1;
          const uint32_t a0 = as_u32(centre_low(u0)), a1 = as_u32(centre_high(u0));
          const uint32_t a2 = as_u32(centre_low(u1)), a3 = as_u32(centre_high(u1));
          mma_f16(o[2 * g + e], a0, a1, a2, a3, wh[g][0], wh[g][1]);
          mma_f16(o[2 * g + e], a0, a1, a2, a3, wl[g][0], wl[g][1]);
        }
      }
    }
    cp_async_wait<0>();

    // warp results: head gid's max and sum, every head's weighted values
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    __syncthreads();  // every ring is done with
    float* part = reinterpret_cast<float*>(smem);
    float ozf[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const float2 y = unpair(oz[g]);
      ozf[g] = y.x + y.y;
      ozf[g] += __shfl_xor_sync(0xffffffffu, ozf[g], 1);
      ozf[g] += __shfl_xor_sync(0xffffffffu, ozf[g], 2);
      const float za = __shfl_sync(0xffffffffu, ozf[g], 8 * tig), zb = __shfl_sync(0xffffffffu, ozf[g], 8 * tig + 4);
      float* pa = part + (warp * 8 + 2 * tig) * PART + 4 + 32 * g + 4 * gid;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        pa[2 * e] = fmaf(o[2 * g + e][0], 512.0f, za);  // codes were (c - 7.5) 2^-9
        pa[2 * e + 1] = fmaf(o[2 * g + e][2], 512.0f, za);
        pa[PART + 2 * e] = fmaf(o[2 * g + e][1], 512.0f, zb);
        pa[PART + 2 * e + 1] = fmaf(o[2 * g + e][3], 512.0f, zb);
      }
    }
    if (tig == 0) {
      part[(warp * 8 + gid) * PART] = mx == kKv4Never ? -INFINITY : mx;
      part[(warp * 8 + gid) * PART + 1] = l;
    }
    __syncthreads();
    if (tid < 8) {
      float M = -INFINITY, L = 0.0f;
      for (int w = 0; w < kDWarps; ++w) M = fmaxf(M, part[(w * 8 + tid) * PART]);
      for (int w = 0; w < kDWarps; ++w) {
        const float mw = part[(w * 8 + tid) * PART];
        const float e = mw == -INFINITY ? 0.0f : exp2_fast(mw - M);
        wgt[w * 8 + tid] = e;
        L = fmaf(part[(w * 8 + tid) * PART + 1], e, L);
      }
      total[tid] = M;
      total[8 + tid] = L;
    }
    __syncthreads();
    const bool whole = c0 == 0 && c1 == n;
    float* out = ws + ((size_t)blockIdx.x * 2 + (t == t_begin ? 0 : 1)) * SH::LEFT;
    for (int x = tid; x < nh * (HD / 4); x += kDThreads) {
      const int h = x / (HD / 4), d = x % (HD / 4) * 4;
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kDWarps; ++w) add_part(y, part + (w * 8 + h) * PART + 4 + d, wgt[w * 8 + h]);
      if (whole) {
        store_shares(a, m, (h0 + h) * HD + d, y, total[8 + h]);
      } else {
        *reinterpret_cast<float4*>(out + h * HD + d) = y;
        if (d == 0) {
          out[8 * HD + h] = total[h];
          out[8 * HD + 8 + h] = total[8 + h];
        }
      }
    }
    if (!whole) {
      // The last CTA of the item to arrive joins the parts in CTA order; of many parts the last of each
      // group of `group` CTAs first joins its group's (one SM takes in 64 bytes a clock).
      const int mine_at = (int)blockIdx.x - w0;
      const int group = parts > kDJoin ? kDGroup : parts, g0 = mine_at / group * group, members = min(group, parts - g0);
      auto arrive = [&](int* counter, int n) -> bool {
        __syncthreads();
        if (tid == 0) {
          __threadfence();  // of the whole block's stores, which the barrier has ordered before
          const int last = atomicAdd(counter, 1) == n - 1;
          if (last) *counter = 0;
          *flag = last;
        }
        __syncthreads();
        const bool last = *flag != 0;
        if (last) __threadfence();
        return last;
      };
      // a part's place: in its CTA the item is the first unless it begins there
      auto place_at = [&](int i) -> int { return (w0 + i) * 2 + ((int64_t)(w0 + i) * per >= item_t ? 0 : 1); };
      auto place = [&](int i) -> float* { return ws + (size_t)place_at(i) * SH::LEFT; };
      // parts g0, g0 + step, .. : n of them, into the first one's place or out
      auto join = [&](int i0, int step, int n, bool last) {
        float* sm = reinterpret_cast<float*>(smem);  // [part][8] maxima, then weights; sums
        float* sl = sm + 8 * kDGroupMax;
        float* first_part = place(i0);
        const float* next_parts = n > 1 ? place(i0 + step) : first_part;
        const size_t far = (size_t)step * 2 * SH::LEFT;
        for (int x = tid; x < n * 8; x += kDThreads) {
          const int w = x / 8, h = x % 8;
          const float* in = w == 0 ? first_part : next_parts + (w - 1) * far;
          sm[x] = h < nh ? __ldcg(in + 8 * HD + h) : -INFINITY;
          sl[x] = h < nh ? __ldcg(in + 8 * HD + 8 + h) : 0.0f;
        }
        __syncthreads();
        {
          const int h = warp;
          float M = -INFINITY, L = 0.0f;
          for (int w = lane; w < n; w += 32) M = fmaxf(M, sm[w * 8 + h]);
#pragma unroll
          for (int x = 16; x >= 1; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
          for (int w = lane; w < n; w += 32) {
            const float mw = sm[w * 8 + h], e = mw == -INFINITY ? 0.0f : exp2_fast(mw - M);
            L = fmaf(sl[w * 8 + h], e, L);
            sm[w * 8 + h] = e;
          }
#pragma unroll
          for (int x = 16; x >= 1; x >>= 1) L += __shfl_xor_sync(0xffffffffu, L, x);
          if (lane == 0) {
            total[h] = M;
            total[8 + h] = L;
          }
        }
        __syncthreads();
        for (int x = tid; x < nh * (HD / 4); x += kDThreads) {
          const int h = x / (HD / 4), d = x % (HD / 4) * 4;
          float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
          add_part4(y, __ldcg(reinterpret_cast<const float4*>(first_part + h * HD + d)), sm[h]);
#pragma unroll 8
          for (int w = 1; w < n; ++w)
            add_part4(y, __ldcg(reinterpret_cast<const float4*>(next_parts + (w - 1) * far + h * HD + d)), sm[w * 8 + h]);
          if (last) {
            store_shares(a, m, (h0 + h) * HD + d, y, total[8 + h]);
          } else {
            *reinterpret_cast<float4*>(first_part + h * HD + d) = y;
            if (d == 0) {
              first_part[8 * HD + h] = total[h];
              first_part[8 * HD + 8 + h] = total[8 + h];
            }
          }
        }
      };
      int* counter = counters + (size_t)m * HS + hs;
      if (group == parts) {
        if (arrive(counter, parts)) join(0, 1, parts, true);
      } else if (arrive(counters + kDCounters + place_at(g0), members)) {
        join(g0, 1, members, false);
        __syncthreads();
        const int groups = (parts + group - 1) / group;
        if (arrive(counter, groups)) join(0, group, groups, true);
      }
    }
    __syncthreads();  // the shared memory is used again
    t = done;
  }
}

template <int HD>
int launch_decode_t(shd_ctx* ctx, const Kv4AttnArgs& a0) {
  using SH = DecodeShape<HD>;
  static unsigned attr_devices = 0;
  if (!(attr_devices & (1u << (ctx->device & 31)))) {
    SHD_CHECK_CUDA(ctx, cudaFuncSetAttribute(kv4_decode_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SH::SMEM));
    attr_devices |= 1u << (ctx->device & 31);
  }
  const int HS = a0.c.heads * ((a0.H / a0.c.heads + 7) / 8);
  SHD_REQUIRE(ctx, HS <= kDCounters, "shd_kv4_attn_decode: too many heads");
  const int step = std::min(kDRows, kDCounters / HS);
  const int grid = kv4_decode_ctas(ctx->num_sms);
  SHD_REQUIRE(ctx, kDCounters + 2 * grid <= ctx->n_counters && grid <= kDGroup * kDGroupMax, "shd_kv4_attn_decode: unknown GPU size");
  for (int m = 0; m < a0.M; m += step) {
    Kv4AttnArgs a = a0;
    const size_t width = (size_t)a.H * HD;
    a.M = std::min(step, a0.M - m);
    a.q += (size_t)m * a.ldq;
    a.slot += m;
    a.pos += m;
    if (a.mask) a.mask += m * a.ldmask;
    a.out_c += m * width;
    a.out_s += m * width;
    SHD_CHECK_CUDA(ctx, launch_pdl(kv4_decode_kernel<HD>, dim3(grid), dim3(kDThreads), SH::SMEM, ctx->stream, a,
                                   ctx->d_kv4, ctx->d_counters));
    ctx->launches++;
  }
  return SHD_OK;
}

}  // namespace

int launch_kv4_decode(shd_ctx* ctx, const Kv4AttnArgs& a) {
  return a.c.head_dim == 128 ? launch_decode_t<128>(ctx, a) : launch_decode_t<64>(ctx, a);
}

}  // namespace shd
