// The 4-bit key/value cache: format, addressing and visibility shared by its kernels (shd_kv4.cu,
// shd_kv4_decode.cu, shd_kv4_prefill.cu).
//
// A row is one position of one kv head: head_dim channels in groups of 32, a group being 32 codes
// c in 0..15 with a scale s and a minimum z in f16 and standing for s * c + z. Stored orders, chosen
// so that one thread's share of a tensor-core fragment is contiguous:
//   keys    32-bit word (t, g), t = 0..3 of group g, holds channels 32 g + 8 t .. + 7 and is word
//           t * NG + g of the row: thread t of a quad reads its words of all NG groups at once
//   values  16-bit half word (u, g), u = 0..7, holds channels 32 g + 4 u .. + 3 and is half word
//           u * NG + g of the row
//   params  [2][NG] f16 a row: the NG scales, then the NG minima
// nibble n of a word is its n-th channel, lowest first.
#pragma once

#include <cuda_fp16.h>

#include <algorithm>

#include "shd_common.cuh"

namespace shd {

constexpr int kKv4Group = 32;
constexpr int kKv4Chunk = 16;  // rows the kernels take together; capacity is a multiple of it

struct Kv4View {
  uint8_t* kc;   // [slots][heads][capacity][HD / 2]
  __half* kp;    // [slots][heads][capacity][2][HD / 32]
  uint8_t* vc;
  __half* vp;
  int slots, heads, capacity, head_dim, sinks;
};

// Row of the cache that holds position p >= 0: itself up to the capacity, then a ring over the rows
// behind the sinks.
__host__ __device__ __forceinline__ int kv4_row(const Kv4View& c, int p) {
  return p < c.capacity ? p : c.sinks + (p - c.sinks) % (c.capacity - c.sinks);
}

// First row of (slot, head): 64-bit, a long cache passes 2^31 bytes.
__host__ __device__ __forceinline__ size_t kv4_base(const Kv4View& c, int slot, int head) {
  return ((size_t)slot * c.heads + head) * (size_t)c.capacity;
}

// Whether queries at positions up to `last` can be served with the newest position being `last`:
// past the capacity only what the ring still holds for the oldest query may be visible.
__host__ __device__ __forceinline__ bool kv4_in_reach(const Kv4View& c, int last, int window, int extra) {
  return last < c.capacity || (window > 0 && (int64_t)window + extra <= (int64_t)c.capacity - c.sinks);
}

// The rows that queries at positions [lo, hi] see as up to three intervals of 16-row chunks in
// increasing order (the sinks; the ring's two parts, or the one run of positions). Every visible row is
// in exactly one of them. Call only where kv4_in_reach holds.
struct Kv4Spans {
  int begin[3], end[3];
  int total;
};

__host__ __device__ __forceinline__ Kv4Spans kv4_spans(const Kv4View& c, int lo, int hi, int window) {
  Kv4Spans s;
#pragma unroll
  for (int i = 0; i < 3; ++i) s.begin[i] = s.end[i] = 0;
  s.total = 0;
  if (hi < 0) return s;
  const int64_t far = (int64_t)lo - window + 1;
  if (window <= 0 || far <= c.sinks) {
    // everything from position 0: the sequence is within the capacity
    s.end[0] = ((hi < c.capacity ? hi + 1 : c.capacity) + kKv4Chunk - 1) / kKv4Chunk;
  } else {
    s.end[0] = (c.sinks + kKv4Chunk - 1) / kKv4Chunk;
    const int first = kv4_row(c, (int)far), last = kv4_row(c, hi);
    const bool wrapped = first > last;  // the ring's end lies between the two
    const int b1 = wrapped ? c.sinks : first, e1 = last + 1;
    s.begin[1] = max(b1 / kKv4Chunk, s.end[0]);
    s.end[1] = max((e1 + kKv4Chunk - 1) / kKv4Chunk, s.begin[1]);
    if (wrapped) {
      s.begin[2] = max(first / kKv4Chunk, s.end[1]);
      s.end[2] = max(c.capacity / kKv4Chunk, s.begin[2]);
    }
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) s.total += s.end[i] - s.begin[i];
  return s;
}

// i-th chunk of the spans, 0 <= i < total.
__host__ __device__ __forceinline__ int kv4_span_chunk(const Kv4Spans& s, int i) {
  const int n0 = s.end[0] - s.begin[0], n1 = s.end[1] - s.begin[1];
  if (i < n0) return s.begin[0] + i;
  if (i < n0 + n1) return s.begin[1] + (i - n0);
  return s.begin[2] + (i - n0 - n1);
}

// Position held by row r when `last` is the newest position written (negative, or below the sinks for
// a row behind them: none).
__host__ __device__ __forceinline__ int kv4_held(const Kv4View& c, int r, int last) {
  if (r < c.sinks || last < c.capacity) return r;
  const int ring = c.capacity - c.sinks;
  int back = (last - r) % ring;
  return last - back;
}

// A block of positions (shd_kv4_prefill.cu) is planned in tiles of kKv4Tile (position, head) pairs of a kv head, whose
// cost is that of the steps of kKv4Step cache rows they walk and kKv4Item more.
constexpr int kKv4Tile = 128, kKv4Step = 64, kKv4Item = 8;

__host__ __device__ __forceinline__ int kv4_tile_cost(const Kv4View& c, int lo, int hi, int window) {
  return (kv4_spans(c, lo, hi, window).total * kKv4Chunk + kKv4Step - 1) / kKv4Step + kKv4Item;
}
// Positions of one launch, of at most `tiles` tiles and M positions: plans are kept in 31 bits, the sum of the tiles'
// costs and one tile's cost over all kv heads. 0: not even one position fits.
inline int kv4_launch_positions(const Kv4View& c, int M, int G, int last, int tiles) {
  const int64_t rows = last < c.capacity ? (int64_t)last + 1 : c.capacity;
  const int64_t cost = (rows + kKv4Chunk - 1 + kKv4Step - 1) / kKv4Step + kKv4Item;  // no tile's is above
  if (cost * c.heads > 0x7fffffff) return 0;
  return (int)std::min<int64_t>(M, std::min<int64_t>(tiles, 0x7fffffff / cost) * kKv4Tile / G);
}

#ifdef __CUDACC__
// ------------------------------------------------------------------------------------------------
// Arithmetic of the attention kernels
// ------------------------------------------------------------------------------------------------
constexpr float kKv4Never = -3.0e38f;  // running maximum before any row

// the hardware's 2^x, to some 2^-22 of it and 0 below 2^-126: the rounding of an ordinary score moves a weight by more
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^e as f32, -126 <= e <= 127
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }
// an e with |x| < 2^e <= 2 |x|: 0 and denormals as the least, inf and NaN as the greatest
__device__ __forceinline__ int ceil_exp2(float x) { return (int)((__float_as_uint(x) >> 23) & 255u) - 126; }

__device__ __forceinline__ __half2 as_half2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }
__device__ __forceinline__ uint32_t as_u32(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) { return as_u32(__floats2half2_rn(lo, hi)); }
__device__ __forceinline__ float2 unpack_f16(uint32_t v) { return __half22float2(as_half2(v)); }

// two f32 operations in one instruction
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
  return v;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// a pair of values as two f16 terms each
__device__ __forceinline__ void split_pair(uint64_t y, uint32_t& hi, uint32_t& lo) {
  const float2 f = unpair(y);
  hi = pack_f16(f.x, f.y);
  const float2 h = unpack_f16(hi);
  const float2 r = unpair(fma2(pair(h.x, h.y), pair(-1.0f, -1.0f), y));
  lo = pack_f16(r.x, r.y);
}
__device__ __forceinline__ void split_f16(float a, float b, uint32_t& hi, uint32_t& lo) { split_pair(pair(a, b), hi, lo); }

// two codes under a mask, c * 2^-24 (low nibbles of a half word: up = 2^15) or c * 2^-20 (the next: up =
// 2^11), as (c - 7.5) * 2^-9, exactly
__device__ __forceinline__ __half2 centre(uint32_t codes, __half2 up) {
  return __hfma2(as_half2(codes), up, __floats2half2_rn(-7.5f / 512, -7.5f / 512));
}
__device__ __forceinline__ __half2 centre_low(uint32_t w) { return centre(w & 0x000f000fu, __floats2half2_rn(32768.0f, 32768.0f)); }
__device__ __forceinline__ __half2 centre_high(uint32_t w) { return centre(w & 0x00f000f0u, __floats2half2_rn(2048.0f, 2048.0f)); }
#endif

// Attention over the cache: rows of several sequences (slot, pos) or consecutive positions of one.
struct Kv4AttnArgs {
  Kv4View c;
  const float* q;  // reconstructed queries [M][ldq], H heads
  int ldq, H, M;
  const int32_t *slot, *pos;  // [M] device; null: row m is position pos0 + m of slot0
  int slot0, pos0;
  int window;   // 0: every earlier position
  float scale;  // 1 / sqrt(head_dim)
  const float* mask;       // [M][ldmask], H * head_dim used, nullable
  int64_t ldmask;          // 0: one row for all
  float *out_c, *out_s;    // [M][H * head_dim]
  int* err;
};

// Rows of K and V into the cache and back (shd_kv4.cu; arguments as at the C entries, checked there).
struct Kv4WriteArgs {
  Kv4View c;
  const float *kc, *ks, *vc, *vs;  // shares [M][ld]; the server's null: the client's hold the values
  int ld;
  const int32_t *slot, *pos;  // null: row m is position pos0 + m of slot0
  int slot0, pos0, M;
  float *k_val, *v_val;  // [M][heads * head_dim], nullable
  int* err;
};
int launch_kv4_write(shd_ctx* ctx, const Kv4WriteArgs& a);
int launch_kv4_read(shd_ctx* ctx, const Kv4View& c, int slot, int pos0, int n, float* k_out, float* v_out);

// Single-token attention (shd_kv4_decode.cu): CTAs of a launch, and the context scratch they leave the
// parts of cut items in, two a CTA.
inline int kv4_decode_ctas(int num_sms) { return 2 * num_sms; }
inline size_t kv4_scratch_floats(int num_sms) { return (size_t)kv4_decode_ctas(num_sms) * 2 * (8 * 128 + 16); }
int launch_kv4_decode(shd_ctx* ctx, const Kv4AttnArgs& a);
// Blocks of positions (shd_kv4_prefill.cu).
int launch_kv4_prefill(shd_ctx* ctx, const Kv4AttnArgs& a);

}  // namespace shd
