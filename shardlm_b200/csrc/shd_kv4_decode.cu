// Single-token attention over the 4-bit cache (format in shd_kv4.cuh), grouped by kv head.
//
// With k = s c + z and v = s c + z per group g of 32 channels,
//   q . k_t  = sum_g s_tg (sum_(i in g) q_i (c_ti - 7.5)) + sum_g (z_tg + 7.5 s_tg) (sum_(i in g) q_i)
//   o        = sum_t p_t v_t = sum_t (p_t s_tg) (c_t - 7.5) + sum_t p_t (z_tg + 7.5 s_tg)
// so the codes themselves are tensor-core operands: a code is at most 4 bits and is exact in f16 as
// the subnormal c * 2^-24 (its bits under a mask, one instruction for two codes; the nibble above it
// is c * 2^-20), centred to (c - 7.5) * 2^-9, also exact, by one more: weights add up to 1 over many rows
// whose values cancel, and sums of codes that are all positive would lose what cancels (measured
// against 64 bits at 131000 positions: 5e-4 of the result). The other operand is split into two f16 terms (22 bits): the queries, scaled by a power
// of two of their head, and the weights p_t s_tg, scaled by a running power of two of the scales.
// Sums are f32. Rows of the first product's A are the 8 heads' high terms and the 8 heads' low terms;
// the second takes the two terms one after the other:
//   S [8 + 8 heads x 8 rows]      += Q [16 x 16 channels] K^T   per group, then scaled by s
//   O^T [16 channels x 8 heads]   += V^T [16 x 16 rows] W       per group
// The accumulator of S has the layout of the B operand of the second product, so weights never
// leave their thread. A lane's row order within 8 rows (sigma) is t, t + 4: with it every shared-memory
// read below is free of bank conflicts.
//
// Work: an item is (query row, kv head, up to 8 query heads); its visible 16-row chunks (kv4_spans)
// are laid end to end with those of every other item and cut into equal shares, one a CTA, whatever
// the lengths. In a CTA the 8 warps take chunks in turn, each with its own ring of asynchronous copies
// and its own online softmax, and are combined in warp order. An item that is cut leaves partial
// results; the CTA that arrives last joins them in CTA order, so results do not depend on timing.
#include <cmath>

#include "shd_kv4.cuh"

namespace shd {
namespace {

constexpr int kDWarps = 8;
constexpr int kDThreads = 32 * kDWarps;
constexpr int kDStages = 4;
constexpr int kDRows = 1024;      // query rows of one launch (their chunk counts are in shared memory)
constexpr int kDMinShare = 16;    // fewest chunks worth a CTA

template <int HD>
struct DecodeShape {
  static constexpr int NG = HD / kKv4Group;
  static constexpr int CODE = kKv4Chunk * HD / 2;      // bytes of a chunk's codes (K or V)
  static constexpr int PAR = kKv4Chunk * 4 * NG;       // bytes of a chunk's parameters
  static constexpr int STAGE = 2 * (CODE + PAR);
  static constexpr int PART = HD + 4;                  // of one head: running max, sum, 2 unused, weighted V
  static constexpr int LEFT = 8 * HD + 16;             // of a cut item: weighted V of 8 heads, maxima, sums
  static constexpr int RING = kDWarps * kDStages * STAGE;
  static constexpr int JOIN = kDWarps * 8 * PART * 4;  // per warp and head, over the rings
  static constexpr size_t SMEM = (RING > JOIN ? RING : JOIN) + kDRows * 8 + 8 * 8 * 4 * 2 + 256;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_f16(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
// two values as two f16 terms each
__device__ __forceinline__ void split_f16(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack_f16(a, b);
  const float2 h = unpack_f16(hi);
  lo = pack_f16(__fsub_rn(a, h.x), __fsub_rn(b, h.y));
}

// two codes under a mask, c * 2^-24 (up = 2^15) or c * 2^-20 (up = 2^11), as (c - 7.5) * 2^-9
__device__ __forceinline__ uint32_t centre(uint32_t codes, __half2 up) {
  const __half2 y = __hfma2(*reinterpret_cast<const __half2*>(&codes), up, __floats2half2_rn(-7.5f / 512, -7.5f / 512));
  return *reinterpret_cast<const uint32_t*>(&y);
}

// 2^e as f32, -126 <= e <= 127
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }

// Exponent that scales |x| <= 2^e: biased exponent arithmetic, 0 and denormals as the least, inf and
// NaN as the greatest (the scaled value is then not finite either).
__device__ __forceinline__ int ceil_exp2(float x) { return (int)((__float_as_uint(x) >> 23) & 255u) - 126; }

template <int HD>
__device__ __forceinline__ void issue_chunk(const Kv4View& c, size_t row0, uint8_t* st, int lane) {
  using S = DecodeShape<HD>;
  constexpr int CPR = HD / 32;           // 16-byte pieces of a row of codes
  constexpr int NC = kKv4Chunk * CPR;    // pieces of a chunk's codes: 64 or 32
  const uint8_t* kc = c.kc + row0 * (HD / 2);
  const uint8_t* vc = c.vc + row0 * (HD / 2);
#pragma unroll
  for (int i = 0; i < NC / 32; ++i) {
    const int p = lane + 32 * i, r = p / CPR, q = p % CPR;
    // keys: row sigma(n) of each 8 stored as n-th, so that a quad's 8 neighbours are contiguous
    const int n = (r & 8) | ((r & 4) ? 2 * (r & 3) + 1 : 2 * (r & 3));
    cp_async16(st + (n * CPR + q) * 16, kc + p * 16, 16);
    // values: rows 2, 3 (mod 4) with their halves exchanged
    const int x = HD == 128 ? q ^ (r & 2) : q;
    cp_async16(st + S::CODE + (r * CPR + x) * 16, vc + p * 16, 16);
  }
  constexpr int NP = S::PAR / 16;  // 16 or 8
  if (lane < 2 * NP) {
    const bool v = lane >= NP;
    const int p = v ? lane - NP : lane;
    cp_async16(st + 2 * S::CODE + (v ? S::PAR : 0) + p * 16,
               reinterpret_cast<const uint8_t*>(v ? c.vp : c.kp) + row0 * (4 * S::NG) + p * 16, 16);
  }
}

// NG scales and NG minima of a row
template <int NG>
__device__ __forceinline__ void load_params(const uint8_t* p, uint32_t (&s)[NG / 2], uint32_t (&z)[NG / 2]) {
  if constexpr (NG == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    s[0] = v.x; s[1] = v.y; z[0] = v.z; z[1] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    s[0] = v.x; z[0] = v.y;
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
  // every row of the 16 from r0
  __device__ __forceinline__ bool chunk(int r0) const {
    const bool below = r0 + kKv4Chunk - 1 <= edge;
    const int t = below ? r0 + up : r0 + down;
    return r0 >= sinks && (below || r0 > edge) && t >= lowest && t + kKv4Chunk - 1 <= p;
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
__device__ __forceinline__ void store_shares(const Kv4AttnArgs& a, size_t at, const float4& y, float L) {
  const float4 mk = a.mask ? *reinterpret_cast<const float4*>(a.mask + at) : make_float4(0.f, 0.f, 0.f, 0.f);
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
  int64_t* pre = reinterpret_cast<int64_t*>(smem + kBody);              // chunks of the rows before
  float* wgt = reinterpret_cast<float*>(smem + kBody + kDRows * 8);     // [warp][head] combine weights
  float* total = wgt + 64;                                              // [head] max, [head] sum
  int* flag = reinterpret_cast<int*>(total + 16);
  int64_t* scan = reinterpret_cast<int64_t*>(total + 32);               // [8] warp sums
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, tig = lane & 3;
  const Kv4View& c = a.c;
  const __half2 low_up = __floats2half2_rn(32768.0f, 32768.0f), high_up = __floats2half2_rn(2048.0f, 2048.0f);
  pdl_trigger();
  pdl_wait();

  // chunk counts of the rows, summed up to each (a row that sees nothing counts one, for its output)
  const int G = a.H / c.heads, nsub = (G + 7) / 8, HS = c.heads * nsub;
  int64_t sum = 0;
  for (int m0 = 0; m0 < a.M; m0 += kDThreads) {
    const int m = m0 + tid;
    int64_t n = 0;
    if (m < a.M) {
      const int p = a.pos[m], sl = a.slot[m];
      const bool ok = p >= 0 && sl >= 0 && sl < c.slots && kv4_in_reach(c, p, a.window, 0);
      if (p >= 0 && !ok && blockIdx.x == 0) atomicOr(a.err, SHD_DEVERR_ARG);
      n = ok ? max(kv4_spans(c, p, p, a.window).total, 1) : 1;
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
    for (int w = 0; w < kDWarps; ++w) {
      if (w < warp) base += scan[w];
      sum += scan[w];
    }
    if (m < a.M) pre[m] = base + x - n;
    __syncthreads();
  }
  const int64_t T = sum * HS;
  const int64_t per = max((T + gridDim.x - 1) / gridDim.x, (int64_t)kDMinShare);
  const int64_t t_begin = blockIdx.x * per, t_end = min(T, t_begin + per);

  for (int64_t t = t_begin; t < t_end;) {
    // the item that chunk t belongs to
    int lo = 0, hi = a.M - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (pre[mid] * HS <= t) lo = mid; else hi = mid - 1;
    }
    const int m = lo;
    const int64_t row_t = pre[m] * HS;
    const int n = (int)((m + 1 < a.M ? pre[m + 1] : sum) - pre[m]);
    const int hs = (int)((t - row_t) / n);
    const int64_t item_t = row_t + (int64_t)hs * n;
    const int c0 = (int)(t - item_t), c1 = (int)min((int64_t)n, t_end - item_t);
    const int kvh = hs / nsub, h0 = kvh * G + (hs % nsub) * 8, nh = min(8, kvh * G + G - h0);
    int p = a.pos[m], sl = a.slot[m];
    if (!(p >= 0 && sl >= 0 && sl < c.slots && kv4_in_reach(c, p, a.window, 0))) p = -1;
    const Kv4Spans sp = kv4_spans(c, p, p, a.window);
    const Seen seen = make_seen(c, p, a.window);
    const size_t base = p >= 0 ? kv4_base(c, sl, kvh) : 0;

    // this warp's chunks: c0 + warp, + 8, ..
    const int first = c0 + warp;
    const int mine = p >= 0 && first < min(c1, sp.total) ? (min(c1, sp.total) - first + kDWarps - 1) / kDWarps : 0;
    uint8_t* ring = smem + warp * (kDStages * SH::STAGE);
#pragma unroll
    for (int i = 0; i < kDStages - 1; ++i) {
      if (i < mine) issue_chunk<HD>(c, base + (size_t)kv4_span_chunk(sp, first + i * kDWarps) * kKv4Chunk, ring + i * SH::STAGE, lane);
      cp_async_commit();
    }

    // queries of head gid: two f16 terms of q * 2^k, in the order of the masked code words
    uint32_t qh[NG][4], ql[NG][4];
    float qs[NG], factor;
    {
      const float* q = a.q + (size_t)m * a.ldq + (size_t)(h0 + min(gid, nh - 1)) * HD + 8 * tig;
      float x[NG][8], top = 0.0f;
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
      // |q| 2^k <= 2^13; the limits keep 2^k and 2^(9 - k) normal
      const int k = max(min(13 - ceil_exp2(top), 100), -100);
      const float up = pow2i(k);
      const float sc = a.scale * 1.44269504088896341f;
      factor = sc * pow2i(9 - k);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        qs[g] = __fadd_rn(qs[g], __shfl_xor_sync(0xffffffffu, qs[g], 1));
        qs[g] = __fadd_rn(qs[g], __shfl_xor_sync(0xffffffffu, qs[g], 2)) * sc;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          split_f16(x[g][i] * up, x[g][i + 4] * up, qh[g][i], ql[g][i]);  // channel pairs (i, i + 4)
        }
      }
    }

    float o[HD / 16][4];  // [2 g + e]: channels 32 g + 4 gid + 2 e (+ 1: third and fourth), heads 2 tig, + 1
#pragma unroll
    for (int i = 0; i < HD / 16; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
    float oz[NG], mx = -INFINITY, l = 0.0f;
#pragma unroll
    for (int g = 0; g < NG; ++g) oz[g] = 0.0f;
    // the weights are scaled by 2^(13 - ev); every value scale so far is <= evf = 2^ev, or 0
    int ev = -100;
    float evf = 0.0f;

    for (int i = 0; i < mine; ++i) {
      cp_async_wait<kDStages - 2>();
      __syncwarp();
      {
        const int nx = i + kDStages - 1;
        if (nx < mine)
          issue_chunk<HD>(c, base + (size_t)kv4_span_chunk(sp, first + nx * kDWarps) * kKv4Chunk,
                          ring + (nx % kDStages) * SH::STAGE, lane);
        cp_async_commit();
      }
      const uint8_t* st = ring + (i % kDStages) * SH::STAGE;
      const int r0 = kv4_span_chunk(sp, first + i * kDWarps) * kKv4Chunk;

      // scores of head gid with rows 8 j + tig and 8 j + tig + 4 (log2 units)
      float s[2][2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t kw[NG];
        if constexpr (NG == 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(st + (8 * j + gid) * (HD / 2) + 16 * tig);
          kw[0] = v.x; kw[1] = v.y; kw[2] = v.z; kw[3] = v.w;
        } else {
          const uint2 v = *reinterpret_cast<const uint2*>(st + (8 * j + gid) * (HD / 2) + 8 * tig);
          kw[0] = v.x; kw[1] = v.y;
        }
        const uint8_t* kp = st + 2 * SH::CODE;
        uint32_t s0[NG / 2], z0[NG / 2], s1[NG / 2], z1[NG / 2];
        load_params<NG>(kp + (8 * j + tig) * (4 * NG), s0, z0);
        load_params<NG>(kp + (8 * j + tig + 4) * (4 * NG), s1, z1);
        float d0 = 0.0f, d1 = 0.0f, e0 = 0.0f, e1 = 0.0f;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          const uint32_t w = kw[g], w8 = w >> 8;
          mma_f16(acc, qh[g][0], ql[g][0], qh[g][1], ql[g][1], centre(w & 0x000f000fu, low_up), centre(w & 0x00f000f0u, high_up));
          mma_f16(acc, qh[g][2], ql[g][2], qh[g][3], ql[g][3], centre(w8 & 0x000f000fu, low_up), centre(w8 & 0x00f000f0u, high_up));
          const float2 sa = unpack_f16(s0[g / 2]), sb = unpack_f16(s1[g / 2]);
          const float2 za = unpack_f16(z0[g / 2]), zb = unpack_f16(z1[g / 2]);
          const float s_a = (g & 1) ? sa.y : sa.x, s_b = (g & 1) ? sb.y : sb.x;
          d0 = fmaf(s_a, acc[0] + acc[2], d0);
          d1 = fmaf(s_b, acc[1] + acc[3], d1);
          e0 = fmaf(fmaf(7.5f, s_a, (g & 1) ? za.y : za.x), qs[g], e0);
          e1 = fmaf(fmaf(7.5f, s_b, (g & 1) ? zb.y : zb.x), qs[g], e1);
        }
        s[j][0] = fmaf(d0, factor, e0);
        s[j][1] = fmaf(d1, factor, e1);
      }

      // value parameters of the same rows; rows out of sight weigh 0 and their parameters are not used
      uint32_t vs[4][NG / 2], vz[4][NG / 2];
#pragma unroll
      for (int x = 0; x < 4; ++x)
        load_params<NG>(st + 2 * SH::CODE + SH::PAR + (8 * (x >> 1) + 4 * (x & 1) + tig) * (4 * NG), vs[x], vz[x]);
      if (!seen.chunk(r0)) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          if (!seen.row(r0 + 8 * (x >> 1) + 4 * (x & 1) + tig)) {
            s[x >> 1][x & 1] = -INFINITY;
#pragma unroll
            for (int g = 0; g < NG / 2; ++g) vs[x][g] = vz[x][g] = 0u;
          }
        }
      }

      // running maximum of the head and running bound of the value scales: rescale when either grows
      float tm = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
      tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, 1));
      tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, 2));
      __half2 hm = *reinterpret_cast<const __half2*>(&vs[0][0]);
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int g = 0; g < NG / 2; ++g) hm = __hmax2(hm, *reinterpret_cast<const __half2*>(&vs[x][g]));
      float vm = fmaxf(__low2float(hm), __high2float(hm));
      vm = fmaxf(vm, __shfl_xor_sync(0xffffffffu, vm, 1));
      vm = fmaxf(vm, __shfl_xor_sync(0xffffffffu, vm, 2));
      if (__any_sync(0xffffffffu, tm > mx || vm > evf)) {
        const float mn = fmaxf(mx, tm);
        const float al = mx == -INFINITY ? 0.0f : exp2_fast(mx - mn);
        mx = mn;
        l *= al;
#pragma unroll
        for (int g = 0; g < NG; ++g) oz[g] *= al;
        float down = 1.0f;
        if (vm > evf) {  // the same in every lane
          const int e = ceil_exp2(vm) + 1;
          down = evf == 0.0f ? 0.0f : pow2i(ev - e);
          ev = e;
          evf = pow2i(e);
        }
        const float al0 = __shfl_sync(0xffffffffu, al, 8 * tig) * down, al1 = __shfl_sync(0xffffffffu, al, 8 * tig + 4) * down;
#pragma unroll
        for (int x = 0; x < HD / 16; ++x) {
          o[x][0] *= al0; o[x][1] *= al1; o[x][2] *= al0; o[x][3] *= al1;
        }
      }

      // weights: plain for the sum and the minima, times scale and as two f16 terms for the codes
      float w[4];
      const float wup = pow2i(13 - ev);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float sx = s[x >> 1][x & 1];
        w[x] = sx == -INFINITY ? 0.0f : exp2_fast(sx - mx);
        l += w[x];
      }
      uint32_t wh[NG][2], wl[NG][2];
#pragma unroll
      for (int g = 0; g < NG / 2; ++g) {
        float2 sv[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          sv[x] = unpack_f16(vs[x][g]);
          const float2 zv = unpack_f16(vz[x][g]);
          oz[2 * g] = fmaf(w[x], fmaf(7.5f, sv[x].x, zv.x), oz[2 * g]);
          oz[2 * g + 1] = fmaf(w[x], fmaf(7.5f, sv[x].y, zv.y), oz[2 * g + 1]);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float wa = w[2 * j] * wup, wb = w[2 * j + 1] * wup;
          split_f16(wa * sv[2 * j].x, wb * sv[2 * j + 1].x, wh[2 * g][j], wl[2 * g][j]);
          split_f16(wa * sv[2 * j].y, wb * sv[2 * j + 1].y, wh[2 * g + 1][j], wl[2 * g + 1][j]);
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
          const uint32_t a0 = centre(u0 & 0x000f000fu, low_up), a1 = centre(u0 & 0x00f000f0u, high_up);
          const uint32_t a2 = centre(u1 & 0x000f000fu, low_up), a3 = centre(u1 & 0x00f000f0u, high_up);
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
    const float f0 = evf * 0.0625f;  // 2^(ev - 13) * 2^9
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      oz[g] += __shfl_xor_sync(0xffffffffu, oz[g], 1);
      oz[g] += __shfl_xor_sync(0xffffffffu, oz[g], 2);
      const float za = __shfl_sync(0xffffffffu, oz[g], 8 * tig), zb = __shfl_sync(0xffffffffu, oz[g], 8 * tig + 4);
      float* pa = part + (warp * 8 + 2 * tig) * PART + 4 + 32 * g + 4 * gid;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        pa[2 * e] = fmaf(o[2 * g + e][0], f0, za);
        pa[2 * e + 1] = fmaf(o[2 * g + e][2], f0, za);
        pa[PART + 2 * e] = fmaf(o[2 * g + e][1], f0, zb);
        pa[PART + 2 * e + 1] = fmaf(o[2 * g + e][3], f0, zb);
      }
    }
    if (tig == 0) {
      part[(warp * 8 + gid) * PART] = mx;
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
        store_shares(a, (size_t)m * a.H * HD + (size_t)(h0 + h) * HD + d, y, total[8 + h]);
      } else {
        *reinterpret_cast<float4*>(out + h * HD + d) = y;
        if (d == 0) {
          out[8 * HD + h] = total[h];
          out[8 * HD + 8 + h] = total[8 + h];
        }
      }
    }
    if (!whole) {
      // the last CTA of the item joins the parts in CTA order
      const int w0 = (int)(item_t / per), parts = (int)((item_t + n - 1) / per) - w0 + 1;
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        int* counter = counters + (size_t)m * HS + hs;
        const int last = atomicAdd(counter, 1) == parts - 1;
        if (last) *counter = 0;
        *flag = last;
      }
      __syncthreads();
      if (*flag) {
        __threadfence();
        // of part w: in its CTA the item is the first unless it begins there
        const float* first_part = ws + ((size_t)w0 * 2 + ((int64_t)w0 * per >= item_t ? 0 : 1)) * SH::LEFT;
        const float* next_parts = ws + (size_t)(w0 + 1) * 2 * SH::LEFT;
        float* sm = reinterpret_cast<float*>(smem);  // [part][8] maxima, then weights
        float* sl = sm + 8 * gridDim.x;
        for (int x = tid; x < parts * 8; x += kDThreads) {
          const int w = x / 8, h = x % 8;
          const float* in = w == 0 ? first_part : next_parts + (size_t)(w - 1) * 2 * SH::LEFT;
          sm[x] = h < nh ? __ldcg(in + 8 * HD + h) : -INFINITY;
          sl[x] = h < nh ? __ldcg(in + 8 * HD + 8 + h) : 0.0f;
        }
        __syncthreads();
        if (warp < 8) {
          const int h = warp;
          float M = -INFINITY, L = 0.0f;
          for (int w = lane; w < parts; w += 32) M = fmaxf(M, sm[w * 8 + h]);
#pragma unroll
          for (int x = 16; x >= 1; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
          for (int w = lane; w < parts; w += 32) {
            const float mw = sm[w * 8 + h], e = mw == -INFINITY ? 0.0f : exp2_fast(mw - M);
            L = fmaf(sl[w * 8 + h], e, L);
            sm[w * 8 + h] = e;
          }
#pragma unroll
          for (int x = 16; x >= 1; x >>= 1) L += __shfl_xor_sync(0xffffffffu, L, x);
          if (lane == 0) total[8 + h] = L;
        }
        __syncthreads();
        for (int x = tid; x < nh * (HD / 4); x += kDThreads) {
          const int h = x / (HD / 4), d = x % (HD / 4) * 4;
          float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
          add_part4(y, __ldcg(reinterpret_cast<const float4*>(first_part + h * HD + d)), sm[h]);
#pragma unroll 8
          for (int w = 1; w < parts; ++w)
            add_part4(y, __ldcg(reinterpret_cast<const float4*>(next_parts + (size_t)(w - 1) * 2 * SH::LEFT + h * HD + d)), sm[w * 8 + h]);
          store_shares(a, (size_t)m * a.H * HD + (size_t)(h0 + h) * HD + d, y, total[8 + h]);
        }
      }
    }
    __syncthreads();  // the shared memory is used again
    t += c1 - c0;
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
  SHD_REQUIRE(ctx, HS <= ctx->n_counters, "shd_kv4_attn_decode: too many heads");
  const int step = std::min(kDRows, ctx->n_counters / HS);
  const int grid = kv4_decode_ctas(ctx->num_sms);
  for (int m = 0; m < a0.M; m += step) {
    Kv4AttnArgs a = a0;
    const size_t width = (size_t)a.H * HD;
    a.M = std::min(step, a0.M - m);
    a.q += (size_t)m * a.ldq;
    a.slot += m;
    a.pos += m;
    if (a.mask) a.mask += m * width;
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
