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

struct WriteArgs {
  Kv4View c;
  const float *kc, *ks, *vc, *vs;  // shares [M][ld]; the server's null: the client's hold the values
  int ld;
  const int32_t *slot, *pos;  // null: row m is position pos0 + m of slot0
  int slot0, pos0, M;
  float *k_val, *v_val;  // [M][heads * head_dim], nullable
  int* err;
};

// Four channels a thread, so a group is 8 neighbouring lanes and its least and greatest value three
// shuffles each.
__global__ void __launch_bounds__(kWriteThreads) kv4_write_kernel(const WriteArgs a) {
  pdl_trigger();
  pdl_wait();
  const int hd = a.c.head_dim, lanes = hd / 4, ng = hd / kKv4Group;
  const int64_t unit = ((int64_t)blockIdx.x * kWriteThreads + threadIdx.x) / lanes;  // (row, head)
  const int l = threadIdx.x % lanes;
  const bool live = unit < (int64_t)a.M * a.c.heads;
  const int m = live ? (int)(unit / a.c.heads) : 0, h = live ? (int)(unit % a.c.heads) : 0;
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
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    const float* pc = kv ? a.vc : a.kc;
    const float* ps = kv ? a.vs : a.ks;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    if (store) {
      const float4 c4 = *reinterpret_cast<const float4*>(pc + src);
      x[0] = c4.x; x[1] = c4.y; x[2] = c4.z; x[3] = c4.w;
      if (ps) {
        const float4 s4 = *reinterpret_cast<const float4*>(ps + src);
        x[0] = __fadd_rn(x[0], s4.x); x[1] = __fadd_rn(x[1], s4.y);
        x[2] = __fadd_rn(x[2], s4.z); x[3] = __fadd_rn(x[3], s4.w);
      }
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
    if (live && out) *reinterpret_cast<float4*>(out + dst) = store ? make_float4(val[0], val[1], val[2], val[3])
                                                                   : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  if (odd) atomicOr(a.err, SHD_DEVERR_NONFINITE);
}

// Four channels a thread (one half word), [n][heads * head_dim] f32 out.
__global__ void __launch_bounds__(kWriteThreads) kv4_read_kernel(const Kv4View c, int slot, int pos0, int n,
                                                                 float* k_out, float* v_out) {
  pdl_trigger();
  pdl_wait();
  const int hd = c.head_dim, lanes = hd / 4, ng = hd / kKv4Group;
  const int64_t unit = ((int64_t)blockIdx.x * kWriteThreads + threadIdx.x) / lanes;
  if (unit >= (int64_t)n * c.heads) return;
  const int l = threadIdx.x % lanes, g = l / 8, u = l % 8;
  const int m = (int)(unit / c.heads), h = (int)(unit % c.heads);
  const size_t row = kv4_base(c, slot, h) + kv4_row(c, pos0 + m);
  const size_t dst = ((size_t)m * c.heads + h) * hd + 4 * l;
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    float* out = kv ? v_out : k_out;
    if (!out) continue;
    const uint16_t* codes = reinterpret_cast<const uint16_t*>((kv ? c.vc : c.kc) + row * (hd / 2));
    const __half* p = (kv ? c.vp : c.kp) + row * (2 * ng);
    const uint32_t w = codes[kv ? u * ng + g : 2 * ((u >> 1) * ng + g) + (u & 1)];
    const float s = __half2float(p[g]), z = __half2float(p[ng + g]);
    float4 y;
    y.x = __fmaf_rn(s, (float)(w & 15u), z);
    y.y = __fmaf_rn(s, (float)((w >> 4) & 15u), z);
    y.z = __fmaf_rn(s, (float)((w >> 8) & 15u), z);
    y.w = __fmaf_rn(s, (float)((w >> 12) & 15u), z);
    *reinterpret_cast<float4*>(out + dst) = y;
  }
}

// Attention of one (query row, head) a warp, one position at a time: lane l holds head_dim / 32
// channels, scores are summed over the warp, the softmax is online.
__global__ void __launch_bounds__(256) kv4_attn_kernel(const Kv4AttnArgs a) {
  const Kv4View& c = a.c;
  const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (item >= (int64_t)a.M * a.H) return;
  const int lane = threadIdx.x & 31, hd = c.head_dim, ng = hd / kKv4Group;
  const int m = (int)(item / a.H), hq = (int)(item % a.H), h = hq / (a.H / c.heads);
  int slot = a.slot0, pos = a.pos0 + m, last = a.pos0 + a.M - 1;
  if (a.pos) {
    slot = a.slot[m];
    pos = last = a.pos[m];
    if (pos >= 0 && (slot < 0 || slot >= c.slots || !kv4_in_reach(c, pos, a.window, 0))) {
      if (lane == 0) atomicOr(a.err, SHD_DEVERR_ARG);
      pos = -1;
    }
  }
  const size_t base = pos >= 0 ? kv4_base(c, slot, h) : 0;
  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, mx = -INFINITY, sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = lane + 32 * i < hd ? a.q[(size_t)m * a.ldq + (size_t)hq * hd + lane + 32 * i] : 0.0f;
  const Kv4Spans sp = kv4_spans(c, pos, last, a.window);
  for (int i = 0; pos >= 0 && i < sp.total; ++i) {
    const int r0 = kv4_span_chunk(sp, i) * kKv4Chunk;
    for (int r = r0; r < r0 + kKv4Chunk; ++r) {
      const int t = kv4_held(c, r, last);
      if (!kv4_sees(c, pos, r, t, a.window)) continue;
      const uint16_t* kc = reinterpret_cast<const uint16_t*>(c.kc + (base + r) * (hd / 2));
      const uint16_t* vc = reinterpret_cast<const uint16_t*>(c.vc + (base + r) * (hd / 2));
      const __half *kp = c.kp + (base + r) * (2 * ng), *vp = c.vp + (base + r) * (2 * ng);
      float dot = 0.0f, v[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        v[g] = 0.0f;
        if (g >= ng) continue;
        const int u = lane / 4, n = lane % 4;  // channel 32 g + lane
        const uint32_t kw = kc[2 * ((u >> 1) * ng + g) + (u & 1)], vw = vc[u * ng + g];
        dot = fmaf(q[g], fmaf(__half2float(kp[g]), (float)((kw >> (4 * n)) & 15u), __half2float(kp[ng + g])), dot);
        v[g] = fmaf(__half2float(vp[g]), (float)((vw >> (4 * n)) & 15u), __half2float(vp[ng + g]));
      }
#pragma unroll
      for (int s = 16; s >= 1; s >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, s);
      dot *= a.scale;
      const float mn = fmaxf(mx, dot), al = mx == -INFINITY ? 0.0f : expf(mx - mn), w = expf(dot - mn);
      mx = mn;
      sum = fmaf(sum, al, w);
#pragma unroll
      for (int g = 0; g < 4; ++g) o[g] = fmaf(w, v[g], o[g] * al);
    }
  }
  const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    if (g >= ng) continue;
    const size_t at = (size_t)m * a.H * hd + (size_t)hq * hd + 32 * g + lane;
    const float mk = a.mask ? a.mask[at] : 0.0f;
    a.out_c[at] = __fsub_rn(o[g] * inv, mk);
    a.out_s[at] = mk;
  }
}

int check_cache(shd_ctx* ctx, const char* fn, const shd_kv4_cache* cache, Kv4View& c) {
  const std::string f(fn);
  SHD_REQUIRE(ctx, cache && cache->k_codes && cache->k_params && cache->v_codes && cache->v_params, f + ": null cache");
  SHD_REQUIRE(ctx, cache->head_dim == 64 || cache->head_dim == 128, f + ": head_dim must be 64 or 128");
  SHD_REQUIRE(ctx, cache->slots > 0 && cache->n_kv_heads > 0, f + ": bad cache shape");
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
  SHD_REQUIRE(ctx, ldq >= H * a.c.head_dim && ldq % 4 == 0, f + ": query rows must be 16-byte aligned");
  SHD_REQUIRE(ctx, shd_aligned16(q) && shd_aligned16(out_c) && shd_aligned16(out_s) && shd_aligned16(mask),
              f + ": tensors must be 16-byte aligned");
  a.q = q;
  a.ldq = ldq;
  a.H = H;
  a.M = M;
  a.window = window;
  a.scale = 1.0f / sqrtf((float)a.c.head_dim);
  a.mask = mask;
  a.out_c = out_c;
  a.out_s = out_s;
  a.err = ctx->d_err;
  return SHD_OK;
}

int launch_attn(shd_ctx* ctx, const Kv4AttnArgs& a) {
  const int64_t blocks = ((int64_t)a.M * a.H + 7) / 8;
  SHD_REQUIRE(ctx, blocks <= 0x7fffffff, "kv4 attention: too many rows");
  kv4_attn_kernel<<<(unsigned)blocks, 256, 0, ctx->stream>>>(a);
  SHD_CHECK_LAUNCH(ctx, "kv4_attn_kernel");
  return SHD_OK;
}

}  // namespace
}  // namespace shd

using namespace shd;

extern "C" int shd_kv4_write(shd_ctx* ctx, const shd_kv4_cache* cache, const float* kc, const float* ks, const float* vc,
                             const float* vs, int ld, const int32_t* slot, const int32_t* pos, int slot0, int pos0,
                             int M, float* k_val, float* v_val) {
  if (!ctx) return SHD_ERR_ARG;
  WriteArgs a{};
  const int rc = check_cache(ctx, "shd_kv4_write", cache, a.c);
  if (rc) return rc;
  SHD_REQUIRE(ctx, kc && vc && (ks == nullptr) == (vs == nullptr), "shd_kv4_write: null pointer");
  SHD_REQUIRE(ctx, (slot == nullptr) == (pos == nullptr), "shd_kv4_write: slot and pos are given together");
  SHD_REQUIRE(ctx, M > 0 && ld >= a.c.heads * a.c.head_dim && ld % 4 == 0, "shd_kv4_write: bad shape");
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
  const int64_t threads = (int64_t)M * a.c.heads * (a.c.head_dim / 4);
  const int64_t blocks = (threads + kWriteThreads - 1) / kWriteThreads;
  SHD_REQUIRE(ctx, blocks <= 0x7fffffff, "shd_kv4_write: too many rows");
  SHD_CHECK_CUDA(ctx, launch_pdl(kv4_write_kernel, dim3((unsigned)blocks), dim3(kWriteThreads), 0, ctx->stream, a));
  ctx->launches++;
  return SHD_OK;
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
  const int64_t blocks = ((int64_t)n * c.heads * (c.head_dim / 4) + kWriteThreads - 1) / kWriteThreads;
  SHD_REQUIRE(ctx, blocks <= 0x7fffffff, "shd_kv4_read: too many rows");
  SHD_CHECK_CUDA(ctx, launch_pdl(kv4_read_kernel, dim3((unsigned)blocks), dim3(kWriteThreads), 0, ctx->stream, c, slot,
                                 pos0, n, k_out, v_out));
  ctx->launches++;
  return SHD_OK;
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
