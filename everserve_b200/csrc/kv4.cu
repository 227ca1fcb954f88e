// Writes and reads of the paged cache held in 4 bits (format: kv4.cuh), and the copy of pages.
#include "api.h"
#include "common.cuh"
#include "kv4.cuh"
#include "launch.h"

namespace es {
namespace kv4 {

constexpr int kThreads = 256;

struct WriteParams {
  const __nv_bfloat16* qkv;  // [T, (hq + 2 hkv) * D] rows of qkv_stride
  int64_t qkv_stride;
  const __nv_bfloat16* bias;  // nullable
  const int64_t* positions;
  const float* cos_sin;  // [max_pos, D]
  int64_t max_pos;
  const int64_t* slots;
  __nv_bfloat16* q_out;  // [T, hq, D]
  uint8_t* cache;
  int64_t s_block;  // bytes between blocks
  int64_t num_slots;
  int T, hq, hkv;
  int share;  // log2 of the warps that share a token
  int* status;
};

// A quantised run of 8 channels as its word. A code is rint((x - zero) / scale) of the correctly rounded
// quotient; the product with `inv`, the scale's rounded reciprocal, is within 15 * 2^-22 of it, so it gives the
// same code unless it falls next to a half: then (1 word in 3000) the quotients are taken. The rounding is an
// addition of 1.5 * 2^23, whose low bits are the code.
ES_DEVICE uint32_t pack_word(const float* x, float scale, float zero, float inv) {
  constexpr float kMagic = 12582912.f;
  uint32_t w = 0;
  bool near = scale > 0.f && scale < 1e-30f;  // (a reciprocal that overflows)
  const uint64_t z2 = ptx::pair_f32(-zero, -zero), m2 = ptx::pair_f32(kMagic, kMagic), n2 = ptx::pair_f32(-kMagic, -kMagic);
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float2 d = ptx::unpair_f32(ptx::add_f32x2(ptx::pair_f32(x[i], x[i + 1]), z2));
    const float q0 = fminf(fmaxf(d.x * inv, 0.f), 15.f), q1 = fminf(fmaxf(d.y * inv, 0.f), 15.f);
    const uint64_t r2 = ptx::add_f32x2(ptx::pair_f32(q0, q1), m2);
    const float2 r = ptx::unpair_f32(r2), c = ptx::unpair_f32(ptx::add_f32x2(r2, n2));
    near |= fabsf(q0 - c.x) > 0.49998f || fabsf(q1 - c.y) > 0.49998f;
    w += (__float_as_uint(r.x) - __float_as_uint(kMagic)) << (2 * i);
    w += (__float_as_uint(r.y) - __float_as_uint(kMagic)) << (2 * i + 16);
  }
  if (near) {
    w = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float c = rintf(__fdiv_rn(x[i] - zero, scale));
      w |= (uint32_t)fminf(fmaxf(c, 0.f), 15.f) << (4 * (i / 2) + 16 * (i % 2));
    }
  }
  return w;
}

// RoPE (rotate-half) on q and k, q written in bf16, k and v quantised into their slots.
//
// D / 16 neighbouring lanes hold one head of one token: lane l its channels 8 l.. and D / 2 + 8 l..,
// which are the two halves RoPE pairs, the two groups of a head in two groups, and (at D = 128) the two
// words of one 8-byte piece of the row. A group's minimum and maximum are shuffles among these lanes.
// The rotation rounds each product (no fused multiply-add), so a code does not depend on contraction.
//
// Bound by memory on paper (177 MB for 8190 rows of 48 heads: 27 us at the copy's rate), by instructions and
// latency in fact: 43 us. A warp takes a token's heads, 32 / (D / 16) at a time, so the angles are read once;
// 32 warps a SM (with four heads' loads at once and half the warps: 49 us; with IEEE quotients for every code: 60).
// With few tokens several warps share one.
template <int D, int NG, int BS>
__global__ void __launch_bounds__(kThreads, 4) write_kernel(WriteParams p) {
  using R = Rec<D, NG, BS>;
  constexpr int L = D / 16, H4 = 32 / L;  // lanes of a head, heads of a warp at a time
  const int warp = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int t = warp >> p.share, part = warp & ((1 << p.share) - 1);
  if (t >= p.T) return;
  const int l = lane % L, H = p.hq + 2 * p.hkv, step = H4 << p.share;
  pdl_wait();
  pdl_launch();
  int64_t pos = p.positions[t];
  const int64_t slot = p.slots[t];
  bool bad = slot >= p.num_slots;
  if (pos < 0 || pos >= p.max_pos) bad = true, pos = 0;  // no table row: q is rotated as position 0
  if (bad && lane == 0 && p.status) atomicExch(p.status, (int)kBadShape);
  const bool kept = slot >= 0 && !bad;
  float c[8], s[8];
  {
    const float4* cs = reinterpret_cast<const float4*>(p.cos_sin + pos * D + 8 * l);
    const float4* sn = reinterpret_cast<const float4*>(p.cos_sin + pos * D + D / 2 + 8 * l);
    const float4 c0 = cs[0], c1 = cs[1], s0 = sn[0], s1 = sn[1];
    c[0] = c0.x, c[1] = c0.y, c[2] = c0.z, c[3] = c0.w, c[4] = c1.x, c[5] = c1.y, c[6] = c1.z, c[7] = c1.w;
    s[0] = s0.x, s[1] = s0.y, s[2] = s0.z, s[3] = s0.w, s[4] = s1.x, s[5] = s1.y, s[6] = s1.z, s[7] = s1.w;
  }
  const __nv_bfloat16* src = p.qkv + t * p.qkv_stride + 8 * l;
  uint8_t* block = p.cache + (kept ? slot / BS : 0) * p.s_block;
  const int off = (int)((kept ? slot : 0) % BS);
  for (int base = part * H4; base < H; base += step) {
    const int h = min(base + lane / L, H - 1);
    const bool live = base + lane / L < H;
    float a[8], b[8];
    unpack8(__ldcs(reinterpret_cast<const uint4*>(src + h * D)), a);
    unpack8(__ldcs(reinterpret_cast<const uint4*>(src + h * D + D / 2)), b);
    if (p.bias != nullptr) {
      float x[8];
      unpack8(*reinterpret_cast<const uint4*>(p.bias + h * D + 8 * l), x);
#pragma unroll
      for (int i = 0; i < 8; i++) a[i] += x[i];
      unpack8(*reinterpret_cast<const uint4*>(p.bias + h * D + D / 2 + 8 * l), x);
#pragma unroll
      for (int i = 0; i < 8; i++) b[i] += x[i];
    }
    if (h < p.hq + p.hkv) {
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float x = a[i], y = b[i];
        a[i] = __fsub_rn(__fmul_rn(x, c[i]), __fmul_rn(y, s[i]));
        b[i] = __fadd_rn(__fmul_rn(y, c[i]), __fmul_rn(x, s[i]));
      }
    }
    if (h < p.hq && live) {
      uint4* q = reinterpret_cast<uint4*>(p.q_out + ((int64_t)t * p.hq + h) * D);
      q[l] = pack8(a);
      q[L + l] = pack8(b);
    }
    if (base + H4 <= p.hq || !kept) continue;  // query heads alone, or a padding row (the whole warp)
    // the groups' ranges (every lane shuffles; a query head's are not used)
    float mn[2], mx[2], bad[2];  // bad: 0, or NaN where the group holds a value that is not finite
#pragma unroll
    for (int g = 0; g < 2; g++) {
      const float* x = g ? b : a;
      mn[g] = mx[g] = x[0];
#pragma unroll
      for (int i = 1; i < 8; i++) {
        mn[g] = fminf(mn[g], x[i]);
        mx[g] = fmaxf(mx[g], x[i]);
      }
      uint64_t sum = ptx::pair_f32(0.f, 0.f);  // (scaled: it cannot overflow)
#pragma unroll
      for (int i = 0; i < 4; i++)
        sum = ptx::fma_f32x2(ptx::pair_f32(x[2 * i], x[2 * i + 1]), ptx::pair_f32(0x1p-20f, 0x1p-20f), sum);
      const float2 both = ptx::unpair_f32(sum);
      bad[g] = (both.x + both.y) - (both.x + both.y);
    }
    if (NG == 1) {
      mn[0] = fminf(mn[0], mn[1]);
      mx[0] = fmaxf(mx[0], mx[1]);
      bad[0] += bad[1];
    }
#pragma unroll
    for (int g = 0; g < NG; g++) {
#pragma unroll
      for (int o = 1; o < L; o <<= 1) {
        mn[g] = fminf(mn[g], __shfl_xor_sync(0xffffffffu, mn[g], o));
        mx[g] = fmaxf(mx[g], __shfl_xor_sync(0xffffffffu, mx[g], o));
        bad[g] += __shfl_xor_sync(0xffffffffu, bad[g], o);
      }
    }
    if (!live || h < p.hq) continue;
    const int side = h >= p.hq + p.hkv;  // 0: K, 1: V
    uint8_t* rec = block + (h - p.hq - side * p.hkv) * R::kBytes;
    uint32_t pair = 0;  // lane l < NG stores the l-th group's
    float sc[NG], z[NG], inv[NG];
#pragma unroll
    for (int g = 0; g < NG; g++) {
      // a group holding a value that is not finite gets a NaN scale: all of it reads as NaN
      const __nv_bfloat16 sb = f2bf(__fadd_rn(__fmul_rn(mx[g] - mn[g], 1.0f / 15.0f), bad[g]));
      const __nv_bfloat16 zb = f2bf(mn[g]);
      sc[g] = bf2f(sb);
      z[g] = bf2f(zb);
      inv[g] = sc[g] > 0.f ? __frcp_rn(sc[g]) : 0.f;
      if (g == l) pair = (uint32_t)__bfloat16_as_ushort(sb) | ((uint32_t)__bfloat16_as_ushort(zb) << 16);
    }
    const uint32_t wa = pack_word(a, sc[0], z[0], inv[0]);
    const uint32_t wb = pack_word(b, sc[NG - 1], z[NG - 1], inv[NG - 1]);
    uint8_t* row = rec + side * R::kV + off * R::kRow;
    if (D == 128) {
      *reinterpret_cast<uint2*>(row + 8 * l) = make_uint2(wa, wb);
    } else {
      *reinterpret_cast<uint32_t*>(row + 4 * l) = wa;
      *reinterpret_cast<uint32_t*>(row + R::kRow / 2 + 4 * l) = wb;
    }
    if (l < NG) *reinterpret_cast<uint32_t*>(rec + R::kKMeta + side * BS * R::kMeta + off * R::kMeta + 4 * l) = pair;
  }
}

struct ReadParams {
  const uint8_t* cache;
  int64_t s_block, num_slots;
  const int64_t* slots;
  __nv_bfloat16 *k, *v;  // [n, hkv, D]
  uint32_t items, hkv;   // n * hkv
  int* status;
};

// The values of rows, in bf16: the lanes of write_kernel, the other way round. (scale * code has 12
// significant bits, so the fused multiply-add rounds the exact value once.) 8190 rows of 8 heads: 9 us, 43 MB.
template <int D, int NG, int BS>
__global__ void __launch_bounds__(kThreads) read_kernel(ReadParams p) {
  using R = Rec<D, NG, BS>;
  constexpr int L = D / 16;
  pdl_wait();
  pdl_launch();
  const uint32_t item = blockIdx.x * (kThreads / L) + threadIdx.x / L;  // (token, kv head)
  if (item >= p.items) return;
  const int l = threadIdx.x % L;
  const uint32_t t = item / p.hkv;
  const int64_t slot = p.slots[t];
  const bool in = slot >= 0 && slot < p.num_slots;  // a negative slot reads as zeros
  if (slot >= p.num_slots && l == 0 && p.status) atomicExch(p.status, (int)kBadShape);
  uint2 w[2];
  uint32_t pa[2], pb[2];
  if (in) {
    const uint8_t* rec = p.cache + slot / BS * p.s_block + (item - t * p.hkv) * R::kBytes;
    const int off = (int)(slot % BS);
#pragma unroll
    for (int side = 0; side < 2; side++) {
      const uint8_t* codes = rec + side * R::kV + off * R::kRow;
      const uint32_t* pair = reinterpret_cast<const uint32_t*>(rec + R::kKMeta + side * BS * R::kMeta + off * R::kMeta);
      if (D == 128) {
        w[side] = *reinterpret_cast<const uint2*>(codes + 8 * l);
      } else {
        w[side].x = *reinterpret_cast<const uint32_t*>(codes + 4 * l);
        w[side].y = *reinterpret_cast<const uint32_t*>(codes + R::kRow / 2 + 4 * l);
      }
      pa[side] = pair[0], pb[side] = pair[NG - 1];
    }
  }
#pragma unroll
  for (int side = 0; side < 2; side++) {
    float a[8], b[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int bit = 4 * (i / 2) + 16 * (i % 2);
      a[i] = in ? fmaf((float)((w[side].x >> bit) & 15u), pair_scale(pa[side]), pair_zero(pa[side])) : 0.f;
      b[i] = in ? fmaf((float)((w[side].y >> bit) & 15u), pair_scale(pb[side]), pair_zero(pb[side])) : 0.f;
    }
    uint4* dst = reinterpret_cast<uint4*>((side ? p.v : p.k) + (int64_t)item * D);
    dst[l] = pack8(a);
    dst[L + l] = pack8(b);
  }
}

// ---- pages ---------------------------------------------------------------------------------------

constexpr int kMaxLayers = 256;  // layer addresses carried as kernel arguments (2 KB of the 4 KB)
constexpr int kCopyVecs = 1024;  // 16-byte vectors one CTA copies at most

struct CopyParams {
  const int64_t* pairs;  // [n, 2]: source page, destination page
  int64_t n, units;      // units = layers * n * chunks
  int64_t stride;        // bytes between pages
  int64_t num_pages;
  int vecs, chunks, per;  // 16-byte vectors of a page; CTAs a page is cut into; vectors of each
  int* status;
  uint8_t* base[kMaxLayers];
};

// One CTA per (layer, pair, chunk of the page), which has all its loads on the way before its first store:
// 1023 pages in 32 layers, 1.2 GB read and written, in 180 us, 6.7 TB/s (the copy's own rate).
__global__ void __launch_bounds__(kThreads) copy_kernel(const __grid_constant__ CopyParams p) {
  pdl_wait();
  pdl_launch();
  const int64_t u = blockIdx.x;
  const int chunk = (int)(u % p.chunks);
  const int64_t pair = u / p.chunks % p.n;
  const int layer = (int)(u / p.chunks / p.n);
  const int64_t from = p.pairs[2 * pair], to = p.pairs[2 * pair + 1];
  if (from < 0 || to < 0) return;  // padding
  if (from >= p.num_pages || to >= p.num_pages) {
    if (threadIdx.x == 0 && p.status) atomicExch(p.status, (int)kBadShape);
    return;
  }
  const int v0 = chunk * p.per, v1 = min(p.vecs, v0 + p.per);
  const uint4* src = reinterpret_cast<const uint4*>(p.base[layer] + from * p.stride);
  uint4* dst = reinterpret_cast<uint4*>(p.base[layer] + to * p.stride);
  uint4 r[kCopyVecs / kThreads];
#pragma unroll
  for (int i = 0; i < kCopyVecs / kThreads; i++) {
    const int v = v0 + i * kThreads + threadIdx.x;
    if (v < v1) r[i] = src[v];
  }
#pragma unroll
  for (int i = 0; i < kCopyVecs / kThreads; i++) {
    const int v = v0 + i * kThreads + threadIdx.x;
    if (v < v1) dst[v] = r[i];
  }
}

}  // namespace kv4

cudaError_t launch_rope_kv4(const Kv4WriteArgs& a, cudaStream_t stream) {
  kv4::WriteParams p{};
  p.qkv = static_cast<const __nv_bfloat16*>(a.qkv);
  p.qkv_stride = a.qkv_stride;
  p.bias = static_cast<const __nv_bfloat16*>(a.bias);
  p.positions = a.positions;
  p.cos_sin = a.cos_sin;
  p.max_pos = a.max_pos;
  p.slots = a.slots;
  p.q_out = static_cast<__nv_bfloat16*>(a.q_out);
  p.cache = static_cast<uint8_t*>(a.c.base);
  p.s_block = a.c.s_block;
  p.num_slots = a.c.num_blocks * a.c.block_size;
  p.hq = a.hq;
  p.hkv = a.c.hkv;
  p.T = (int)a.T;
  p.status = a.status;
  if (a.T == 0) return cudaSuccess;
  if (a.T > INT32_MAX / 64 || (int64_t)(a.hq + 2 * a.c.hkv) * a.c.d > INT32_MAX) return cudaErrorInvalidValue;
  return kv4::pick(a.c.d, a.c.groups, a.c.block_size, [&](auto d, auto ng, auto bs) {
    // as many warps to a token (a power of two) as its heads fill, while the tokens alone do not fill the SMs
    const int fill = (a.hq + 2 * a.c.hkv + 32 / (d / 16) - 1) / (32 / (d / 16));
    while (p.share < 5 && (1 << p.share) < fill && (a.T << p.share) < 2048) p.share++;
    const int64_t grid = ((a.T << p.share) + kv4::kThreads / 32 - 1) / (kv4::kThreads / 32);
    return launch_ex(kv4::write_kernel<d, ng, bs>, dim3((unsigned)grid), dim3(kv4::kThreads), 0, stream, 0, p);
  });
}

cudaError_t launch_kv4_read(const Kv4ReadArgs& a, cudaStream_t stream) {
  kv4::ReadParams p{};
  p.cache = static_cast<const uint8_t*>(a.c.base);
  p.s_block = a.c.s_block;
  p.num_slots = a.c.num_blocks * a.c.block_size;
  p.slots = a.slots;
  p.k = static_cast<__nv_bfloat16*>(a.k);
  p.v = static_cast<__nv_bfloat16*>(a.v);
  p.hkv = a.c.hkv;
  p.status = a.status;
  if (a.n == 0) return cudaSuccess;
  if (a.n * a.c.hkv > INT32_MAX) return cudaErrorInvalidValue;
  p.items = (uint32_t)(a.n * a.c.hkv);
  return kv4::pick(a.c.d, a.c.groups, a.c.block_size, [&](auto d, auto ng, auto bs) {
    const int64_t grid = ((int64_t)p.items + kv4::kThreads / (d / 16) - 1) / (kv4::kThreads / (d / 16));
    return launch_ex(kv4::read_kernel<d, ng, bs>, dim3((unsigned)grid), dim3(kv4::kThreads), 0, stream, 0, p);
  });
}

cudaError_t launch_copy_pages(const CopyPagesArgs& a, cudaStream_t stream) {
  if (a.page_bytes <= 0 || a.page_bytes % 16 != 0 || a.stride % 16 != 0 || a.page_bytes / 16 > INT32_MAX)
    return cudaErrorInvalidValue;
  if (a.n == 0 || a.layers == 0) return cudaSuccess;
  for (int l0 = 0; l0 < a.layers; l0 += kv4::kMaxLayers) {
    const int nl = a.layers - l0 < kv4::kMaxLayers ? a.layers - l0 : kv4::kMaxLayers;
    kv4::CopyParams p{};
    p.pairs = a.pairs;
    p.n = a.n;
    p.stride = a.stride;
    p.num_pages = a.num_pages;
    p.vecs = (int)(a.page_bytes / 16);
    p.chunks = (p.vecs + kv4::kCopyVecs - 1) / kv4::kCopyVecs;
    p.per = (p.vecs + p.chunks - 1) / p.chunks;
    p.units = (int64_t)nl * a.n * p.chunks;
    p.status = a.status;
    for (int l = 0; l < nl; l++) {
      p.base[l] = static_cast<uint8_t*>(a.caches[l0 + l]);
      if (reinterpret_cast<uintptr_t>(p.base[l]) % 16 != 0) return cudaErrorInvalidValue;
    }
    if (p.units > INT32_MAX) return cudaErrorInvalidValue;
    const cudaError_t e =
        launch_ex(kv4::copy_kernel, dim3((unsigned)p.units), dim3(kv4::kThreads), 0, stream, 0, p);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace es
