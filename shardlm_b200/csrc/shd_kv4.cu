// The 4-bit key/value cache: quantising rows as they are written, reading them back, and the entry
// points of the attention over it (format and addressing in shd_kv4.cuh). The reference keeps its
// reconstructed cache in f32 (crates/v2/server/src/routes/secure_inference.rs:2452-2471); a row of
// this one takes 5/32 of that.
#include <cmath>

#include "shd_kv4.cuh"

namespace shd {
namespace {

constexpr int kWriteThreads = 256;

// One group's scale and minimum from its least and greatest value; every step is one operation
// rounded as it says, so that a plain evaluation of the format gives the same bits.
__device__ __forceinline__ void group_params(float lo, float hi, __half& s, __half& z) {
  z = __float2half_rn(lo);
  s = __float2half_rn(__fmul_rn(fmaxf(__fsub_rn(hi, __half2float(z)), 0.0f), 1.0f / 15.0f));
}

// Four channels a thread, so a group is 8 neighbouring lanes and its least and greatest value three
// shuffles each. Bound by memory: 4096 rows of 8 heads of 128 with shares and values out, 106 MB, in 19.2 us,
// 5.5 TB/s (a plain copy measures 6.5). Few rows cost a launch: 333 rows of 2 heads of 64, 2.6 us.
__global__ void __launch_bounds__(kWriteThreads) kv4_write_kernel(const Kv4WriteArgs a) {
  pdl_trigger();
  pdl_wait();
  const int hd = a.c.head_dim, lanes = hd / 4, ng = hd / kKv4Group;
  // (row, head) of this thread; below 2^31 by the launch's limit
  const uint32_t unit = blockIdx.x * (kWriteThreads / lanes) + threadIdx.x / lanes;
  const int l = threadIdx.x % lanes;
  const bool live = unit < (uint32_t)a.M * (uint32_t)a.c.heads;
  const int m = live ? (int)(unit / (uint32_t)a.c.heads) : 0, h = live ? (int)(unit - (uint32_t)m * a.c.heads) : 0;
  int slot = a.slot0, pos = a.pos0 + m;
  if (a.pos) {
    slot = live ? a.slot[m] : 0;
    pos = live ? a.pos[m] : -1;
  }
  const bool bad = slot < 0 || slot >= a.c.slots;
  const bool store = live && pos >= 0 && !bad;
  if (live && pos >= 0 && bad && l == 0) atomicOr(a.err, SHD_DEVERR_ARG);
  const size_t src = (size_t)m * a.ld + (size_t)h * hd + 4 * l;
  const size_t dst = ((size_t)m * a.c.heads + h) * hd + 4 * l;
  const size_t row = store ? kv4_base(a.c, slot, h) + kv4_row(a.c, pos) : 0;
  bool odd = false;
  float4 in[2][2];  // [K, V][client, server], all requested before any is used
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    const float* pc = kv ? a.vc : a.kc;
    const float* ps = kv ? a.vs : a.ks;
    in[kv][0] = store ? __ldcs(reinterpret_cast<const float4*>(pc + src)) : make_float4(0.f, 0.f, 0.f, 0.f);
    in[kv][1] = store && ps ? __ldcs(reinterpret_cast<const float4*>(ps + src)) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const bool shared = a.ks != nullptr;
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    float x[4] = {in[kv][0].x, in[kv][0].y, in[kv][0].z, in[kv][0].w};
    if (shared) {
      x[0] = __fadd_rn(x[0], in[kv][1].x); x[1] = __fadd_rn(x[1], in[kv][1].y);
      x[2] = __fadd_rn(x[2], in[kv][1].z); x[3] = __fadd_rn(x[3], in[kv][1].w);
    }
    // values that f16 parameters cannot hold: clamped, NaN as 0, and reported
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      odd |= !(fabsf(x[i]) <= 65504.0f);
      x[i] = isnan(x[i]) ? 0.0f : fminf(fmaxf(x[i], -65504.0f), 65504.0f);
    }
    float lo = fminf(fminf(x[0], x[1]), fminf(x[2], x[3])), hi = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
#pragma unroll
    for (int o = 4; o >= 1; o >>= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    __half s, z;
    group_params(lo, hi, s, z);
    const float sf = __half2float(s), zf = __half2float(z);
    const float r = sf > 0.0f ? __fdiv_rn(1.0f, sf) : 0.0f;
    uint32_t code = 0;
    float val[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float c = fminf(fmaxf(rintf(__fmul_rn(__fsub_rn(x[i], zf), r)), 0.0f), 15.0f);
      code |= (uint32_t)c << (4 * i);
      val[i] = __fmaf_rn(sf, c, zf);
    }
    if (store) {
      const int g = l / 8, u = l % 8;  // group, four-channel unit of it
      uint16_t* codes = reinterpret_cast<uint16_t*>((kv ? a.c.vc : a.c.kc) + row * (hd / 2));
      codes[kv ? u * ng + g : 2 * ((u >> 1) * ng + g) + (u & 1)] = (uint16_t)code;
      if (u == 0) {
        __half* p = (kv ? a.c.vp : a.c.kp) + row * (2 * ng);
        p[g] = s;
        p[ng + g] = z;
      }
    }
    float* out = kv ? a.v_val : a.k_val;
    if (live && out)
      __stcs(reinterpret_cast<float4*>(out + dst), store ? make_float4(val[0], val[1], val[2], val[3]) : make_float4(0.f, 0.f, 0.f, 0.f));
  }
  if (odd) atomicOr(a.err, SHD_DEVERR_NONFINITE);
}

// 8 threads a row (slot, head): thread u reads 2 NG bytes of the keys' codes (words of NG / 2 groups) and
// unit u of the values, and writes both. A value unit's NG pieces of 4 channels go out 128 bytes at a time;
// of the keys neighbouring threads exchange halves, so that theirs do too. Bound by memory: 32768 rows of 8
// heads of 128, 310 MB, in 48.7 us, 6.4 TB/s.
template <int NG>
__global__ void __launch_bounds__(kWriteThreads) kv4_read_kernel(const Kv4View c, int slot, int pos0, uint32_t units,
                                                                 float* k_out, float* v_out) {
  constexpr int HD = NG * kKv4Group;
  pdl_trigger();
  pdl_wait();
  const uint32_t unit = blockIdx.x * (kWriteThreads / 8) + threadIdx.x / 8;  // (row, head)
  const int u = threadIdx.x % 8;
  const bool live = unit < units;
  const uint32_t m = live ? unit / (uint32_t)c.heads : 0, h = live ? unit - m * c.heads : 0;
  const size_t row = kv4_base(c, slot, (int)h) + kv4_row(c, pos0 + (int)m);
  const size_t dst = ((size_t)m * c.heads + h) * HD;
  uint32_t kw[NG / 2], vw[NG / 2];
  uint32_t kp[NG], vp[NG];  // NG scales, NG minima, two a word
  if constexpr (NG == 4) {
    const uint2 x = __ldcs(reinterpret_cast<const uint2*>(c.kc + row * 64) + u), y = __ldcs(reinterpret_cast<const uint2*>(c.vc + row * 64) + u);
    const uint4 p = __ldg(reinterpret_cast<const uint4*>(c.kp + row * 8)), q = __ldg(reinterpret_cast<const uint4*>(c.vp + row * 8));
    kw[0] = x.x; kw[1] = x.y; vw[0] = y.x; vw[1] = y.y;
    kp[0] = p.x; kp[1] = p.y; kp[2] = p.z; kp[3] = p.w;
    vp[0] = q.x; vp[1] = q.y; vp[2] = q.z; vp[3] = q.w;
  } else {
    kw[0] = __ldcs(reinterpret_cast<const uint32_t*>(c.kc + row * 32) + u);
    vw[0] = __ldcs(reinterpret_cast<const uint32_t*>(c.vc + row * 32) + u);
    const uint2 p = __ldg(reinterpret_cast<const uint2*>(c.kp + row * 4)), q = __ldg(reinterpret_cast<const uint2*>(c.vp + row * 4));
    kp[0] = p.x; kp[1] = p.y; vp[0] = q.x; vp[1] = q.y;
  }
  if (k_out) {
    // word t of group g is number t NG + g: this thread's are 2 u, 2 u + 1 (HD 64: u)
#pragma unroll
    for (int i = 0; i < NG / 2; ++i) {
      const int w = u * (NG / 2) + i, t = w / NG, g = w % NG;
      const float2 s2 = unpack_f16(NG == 4 && g >= 2 ? kp[1] : kp[0]), z2 = unpack_f16(NG == 4 ? (g >= 2 ? kp[3] : kp[2]) : kp[1]);
      const float s = (g & 1) ? s2.y : s2.x, z = (g & 1) ? z2.y : z2.x;
      float y[8];
#pragma unroll
      for (int n = 0; n < 8; ++n) y[n] = __fmaf_rn(s, (float)((kw[i] >> (4 * n)) & 15u), z);
      // words t, t + 1 (t even) of the group are NG / 2 threads apart (HD 64: 2): the first keeps the low
      // halves of both, and with them 16 neighbouring bytes of each
      constexpr int FAR = 2;  // NG == 4: u + 2 holds t + 1 of the same groups; NG == 2: u + 2 as well
      const bool odd = t & 1;
      float4 mine, other;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const float send = odd ? y[n] : y[4 + n];
        const float got = __shfl_xor_sync(0xffffffffu, send, FAR);
        (&mine.x)[n] = odd ? got : y[n];       // of word t (even)
        (&other.x)[n] = odd ? y[4 + n] : got;  // of word t + 1
      }
      if (live) {
        float* to = k_out + dst + 32 * g + 8 * (t & ~1) + (odd ? 4 : 0);
        __stcs(reinterpret_cast<float4*>(to), mine);
        __stcs(reinterpret_cast<float4*>(to + 8), other);
      }
    }
  }
  if (v_out && live) {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const uint32_t w = (vw[g / 2] >> (16 * (g & 1))) & 0xffffu;
      const float2 s2 = unpack_f16(vp[g / 2]), z2 = unpack_f16(vp[NG / 2 + g / 2]);
      const float s = (g & 1) ? s2.y : s2.x, z = (g & 1) ? z2.y : z2.x;
      float4 y;
      y.x = __fmaf_rn(s, (float)(w & 15u), z);
      y.y = __fmaf_rn(s, (float)((w >> 4) & 15u), z);
      y.z = __fmaf_rn(s, (float)((w >> 8) & 15u), z);
      y.w = __fmaf_rn(s, (float)(w >> 12), z);
      __stcs(reinterpret_cast<float4*>(v_out + dst + 32 * g + 4 * u), y);
    }
  }
}

int check_cache(shd_ctx* ctx, const char* fn, const shd_kv4_cache* cache, Kv4View& c) {
  const std::string f(fn);
  SHD_REQUIRE(ctx, cache && cache->k_codes && cache->k_params && cache->v_codes && cache->v_params, f + ": null cache");
  SHD_REQUIRE(ctx, cache->head_dim == 64 || cache->head_dim == 128, f + ": head_dim must be 64 or 128");
  SHD_REQUIRE(ctx, cache->slots > 0 && cache->n_kv_heads > 0 && (int64_t)cache->n_kv_heads * cache->head_dim <= 0x7fffffff, f + ": bad cache shape");
  SHD_REQUIRE(ctx, cache->capacity > 0 && cache->capacity % kKv4Chunk == 0, f + ": capacity must be a multiple of 16");
  SHD_REQUIRE(ctx, cache->sinks >= 0 && cache->sinks < cache->capacity, f + ": sinks must be below the capacity");
  SHD_REQUIRE(ctx, shd_aligned16(cache->k_codes) && shd_aligned16(cache->k_params) && shd_aligned16(cache->v_codes) &&
                       shd_aligned16(cache->v_params), f + ": cache tensors must be 16-byte aligned");
  c.kc = cache->k_codes;
  c.kp = reinterpret_cast<__half*>(cache->k_params);
  c.vc = cache->v_codes;
  c.vp = reinterpret_cast<__half*>(cache->v_params);
  c.slots = cache->slots;
  c.heads = cache->n_kv_heads;
  c.capacity = cache->capacity;
  c.head_dim = cache->head_dim;
  c.sinks = cache->sinks;
  return SHD_OK;
}

int check_attn(shd_ctx* ctx, const char* fn, const shd_kv4_cache* cache, const float* q, int ldq, int H, int M,
               int window, const float* mask, float* out_c, float* out_s, Kv4AttnArgs& a) {
  const std::string f(fn);
  const int rc = check_cache(ctx, fn, cache, a.c);
  if (rc) return rc;
  SHD_REQUIRE(ctx, q && out_c && out_s, f + ": null pointer");
  SHD_REQUIRE(ctx, H > 0 && H % a.c.heads == 0, f + ": num_heads must be a multiple of num_kv_heads");
  SHD_REQUIRE(ctx, M > 0 && window >= 0, f + ": bad shape");
  SHD_REQUIRE(ctx, ldq >= (int64_t)H * a.c.head_dim && ldq % 4 == 0, f + ": query rows must be 16-byte aligned");
  SHD_REQUIRE(ctx, shd_aligned16(q) && shd_aligned16(out_c) && shd_aligned16(out_s) && shd_aligned16(mask),
              f + ": tensors must be 16-byte aligned");
  a.q = q;
  a.ldq = ldq;
  a.H = H;
  a.M = M;
  a.window = window;
  a.scale = 1.0f / sqrtf((float)a.c.head_dim);
  a.mask = mask;
  a.ldmask = (int64_t)H * a.c.head_dim;
  a.out_c = out_c;
  a.out_s = out_s;
  a.err = ctx->d_err;
  return SHD_OK;
}

}  // namespace

int launch_kv4_write(shd_ctx* ctx, const Kv4WriteArgs& a) {
  SHD_REQUIRE(ctx, (int64_t)a.M * a.c.heads <= 0x7fffffff, "shd_kv4_write: too many rows");
  const int per_block = kWriteThreads / (a.c.head_dim / 4);
  const int64_t blocks = ((int64_t)a.M * a.c.heads + per_block - 1) / per_block;
  SHD_CHECK_CUDA(ctx, launch_pdl(kv4_write_kernel, dim3((unsigned)blocks), dim3(kWriteThreads), 0, ctx->stream, a));
  ctx->launches++;
  return SHD_OK;
}

int launch_kv4_read(shd_ctx* ctx, const Kv4View& c, int slot, int pos0, int n, float* k_out, float* v_out) {
  SHD_REQUIRE(ctx, (int64_t)n * c.heads <= 0x7fffffff, "shd_kv4_read: too many rows");
  const uint32_t units = (uint32_t)n * (uint32_t)c.heads, blocks = units / (kWriteThreads / 8) + (units % (kWriteThreads / 8) ? 1 : 0);
  SHD_CHECK_CUDA(ctx, launch_pdl(c.head_dim == 128 ? kv4_read_kernel<4> : kv4_read_kernel<2>, dim3(blocks),
                                 dim3(kWriteThreads), 0, ctx->stream, c, slot, pos0, units, k_out, v_out));
  ctx->launches++;
  return SHD_OK;
}

}  // namespace shd

using namespace shd;

extern "C" int shd_kv4_write(shd_ctx* ctx, const shd_kv4_cache* cache, const float* kc, const float* ks, const float* vc,
                             const float* vs, int ld, const int32_t* slot, const int32_t* pos, int slot0, int pos0,
                             int M, float* k_val, float* v_val) {
  if (!ctx) return SHD_ERR_ARG;
  Kv4WriteArgs a{};
  const int rc = check_cache(ctx, "shd_kv4_write", cache, a.c);
  if (rc) return rc;
  SHD_REQUIRE(ctx, kc && vc && (ks == nullptr) == (vs == nullptr), "shd_kv4_write: null pointer");
  SHD_REQUIRE(ctx, (slot == nullptr) == (pos == nullptr), "shd_kv4_write: slot and pos are given together");
  SHD_REQUIRE(ctx, M > 0 && ld >= (int64_t)a.c.heads * a.c.head_dim && ld % 4 == 0, "shd_kv4_write: bad shape");
  SHD_REQUIRE(ctx, shd_aligned16(kc) && shd_aligned16(ks) && shd_aligned16(vc) && shd_aligned16(vs) &&
                       shd_aligned16(k_val) && shd_aligned16(v_val), "shd_kv4_write: tensors must be 16-byte aligned");
  if (!pos) {
    SHD_REQUIRE(ctx, slot0 >= 0 && slot0 < a.c.slots, "shd_kv4_write: slot outside the cache");
    SHD_REQUIRE(ctx, pos0 >= 0 && (int64_t)pos0 + M <= 0x7fffffff, "shd_kv4_write: bad position");
    // past the capacity the rows of one call must not meet in the ring
    SHD_REQUIRE(ctx, (int64_t)pos0 + M <= a.c.capacity || M <= a.c.capacity - a.c.sinks,
                "shd_kv4_write: more rows than the ring holds");
  }
  SHD_CHECK_CUDA(ctx, cudaSetDevice(ctx->device));
  a.kc = kc; a.ks = ks; a.vc = vc; a.vs = vs; a.ld = ld;
  a.slot = slot; a.pos = pos; a.slot0 = slot0; a.pos0 = pos0; a.M = M;
  a.k_val = k_val; a.v_val = v_val;
  a.err = ctx->d_err;
  return launch_kv4_write(ctx, a);
}

extern "C" int shd_kv4_read(shd_ctx* ctx, const shd_kv4_cache* cache, int slot, int pos0, int n, float* k_out,
                            float* v_out) {
  if (!ctx) return SHD_ERR_ARG;
  Kv4View c{};
  const int rc = check_cache(ctx, "shd_kv4_read", cache, c);
  if (rc) return rc;
  SHD_REQUIRE(ctx, k_out || v_out, "shd_kv4_read: null pointer");
  SHD_REQUIRE(ctx, slot >= 0 && slot < c.slots, "shd_kv4_read: slot outside the cache");
  SHD_REQUIRE(ctx, pos0 >= 0 && n > 0 && (int64_t)pos0 + n <= 0x7fffffff, "shd_kv4_read: bad position");
  SHD_REQUIRE(ctx, (int64_t)pos0 + n <= c.capacity || n <= c.capacity - c.sinks, "shd_kv4_read: more rows than the ring holds");
  SHD_REQUIRE(ctx, shd_aligned16(k_out) && shd_aligned16(v_out), "shd_kv4_read: tensors must be 16-byte aligned");
  SHD_CHECK_CUDA(ctx, cudaSetDevice(ctx->device));
  return launch_kv4_read(ctx, c, slot, pos0, n, k_out, v_out);
}

extern "C" int shd_kv4_attn_decode(shd_ctx* ctx, const shd_kv4_cache* cache, const float* q, int ldq, int H,
                                   const int32_t* slot, const int32_t* pos, int M, int window, const float* mask,
                                   float* out_c, float* out_s) {
  if (!ctx) return SHD_ERR_ARG;
  Kv4AttnArgs a{};
  const int rc = check_attn(ctx, "shd_kv4_attn_decode", cache, q, ldq, H, M, window, mask, out_c, out_s, a);
  if (rc) return rc;
  SHD_REQUIRE(ctx, slot && pos, "shd_kv4_attn_decode: null pointer");
  SHD_CHECK_CUDA(ctx, cudaSetDevice(ctx->device));
  a.slot = slot;
  a.pos = pos;
  return launch_kv4_decode(ctx, a);
}

extern "C" int shd_kv4_attn_prefill(shd_ctx* ctx, const shd_kv4_cache* cache, const float* q, int ldq, int H, int slot,
                                    int pos0, int M, int window, const float* mask, float* out_c, float* out_s) {
  if (!ctx) return SHD_ERR_ARG;
  Kv4AttnArgs a{};
  const int rc = check_attn(ctx, "shd_kv4_attn_prefill", cache, q, ldq, H, M, window, mask, out_c, out_s, a);
  if (rc) return rc;
  SHD_REQUIRE(ctx, slot >= 0 && slot < a.c.slots, "shd_kv4_attn_prefill: slot outside the cache");
  SHD_REQUIRE(ctx, pos0 >= 0 && (int64_t)pos0 + M <= 0x7fffffff, "shd_kv4_attn_prefill: bad position");
  SHD_REQUIRE(ctx, kv4_in_reach(a.c, pos0 + M - 1, window, M - 1),
              "shd_kv4_attn_prefill: the window reaches positions that the cache no longer holds");
  SHD_CHECK_CUDA(ctx, cudaSetDevice(ctx->device));
  a.slot0 = slot;
  a.pos0 = pos0;
  return launch_kv4_prefill(ctx, a);
}
