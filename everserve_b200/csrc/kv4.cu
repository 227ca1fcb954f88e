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
  int64_t items;  // T * (hq + 2 hkv)
  int hq, hkv;
  int* status;
};

// A quantised run of 8 channels as its word.
ES_DEVICE uint32_t pack_word(const float* x, float scale, float zero) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    // the plain quotient, not a product with a reciprocal: a code is then what the formula says
    const float c = scale > 0.f ? rintf(__fdiv_rn(x[i] - zero, scale)) : 0.f;
    const uint32_t code = (uint32_t)fminf(fmaxf(c, 0.f), 15.f);
    w |= code << (4 * (i / 2) + 16 * (i % 2));
  }
  return w;
}

// RoPE (rotate-half) on q and k, q written in bf16, k and v quantised into their slots.
//
// D / 16 neighbouring lanes hold one head of one token: lane l its channels 8 l.. and D / 2 + 8 l..,
// which are the two halves RoPE pairs, the two groups of a head in two groups, and (at D = 128) the two
// words of one 8-byte piece of the row. A group's minimum and maximum are shuffles among these lanes.
// The rotation rounds each product (no fused multiply-add), so a code does not depend on contraction.
template <int D, int NG, int BS>
__global__ void __launch_bounds__(kThreads) write_kernel(WriteParams p) {
  using R = Rec<D, NG, BS>;
  constexpr int L = D / 16;
  pdl_wait();
  pdl_launch();
  const int64_t item0 = (int64_t)blockIdx.x * (kThreads / L) + threadIdx.x / L;
  const bool live = item0 < p.items;
  const int64_t item = live ? item0 : p.items - 1;
  const int l = threadIdx.x % L;
  const int H = p.hq + 2 * p.hkv;
  const int64_t t = item / H;
  const int h = (int)(item % H);
  const __nv_bfloat16* src = p.qkv + t * p.qkv_stride + (int64_t)h * D;
  float a[8], b[8];
  unpack8(*reinterpret_cast<const uint4*>(src + 8 * l), a);
  unpack8(*reinterpret_cast<const uint4*>(src + D / 2 + 8 * l), b);
  if (p.bias != nullptr) {
    float c[8];
    unpack8(*reinterpret_cast<const uint4*>(p.bias + (int64_t)h * D + 8 * l), c);
#pragma unroll
    for (int i = 0; i < 8; i++) a[i] += c[i];
    unpack8(*reinterpret_cast<const uint4*>(p.bias + (int64_t)h * D + D / 2 + 8 * l), c);
#pragma unroll
    for (int i = 0; i < 8; i++) b[i] += c[i];
  }
  if (h < p.hq + p.hkv) {
    int64_t pos = p.positions[t];
    if (pos < 0 || pos >= p.max_pos) {  // no table row: reported, and rotated as position 0
      if (live && l == 0 && p.status) atomicExch(p.status, (int)kBadShape);
      pos = 0;
    }
    const float4* cs = reinterpret_cast<const float4*>(p.cos_sin + pos * D + 8 * l);
    const float4* sn = reinterpret_cast<const float4*>(p.cos_sin + pos * D + D / 2 + 8 * l);
    const float4 c0 = cs[0], c1 = cs[1], s0 = sn[0], s1 = sn[1];
    const float c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
    const float s[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float x = a[i], y = b[i];
      a[i] = __fsub_rn(__fmul_rn(x, c[i]), __fmul_rn(y, s[i]));
      b[i] = __fadd_rn(__fmul_rn(y, c[i]), __fmul_rn(x, s[i]));
    }
  }
  // the groups' ranges (every lane shuffles; a query head's are not used)
  float mn[2], mx[2], bad[2];  // bad: 0, or NaN where the group holds a value that is not finite
#pragma unroll
  for (int g = 0; g < 2; g++) {
    const float* x = g ? b : a;
    mn[g] = mx[g] = x[0];
    bad[g] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      mn[g] = fminf(mn[g], x[i]);
      mx[g] = fmaxf(mx[g], x[i]);
      bad[g] += x[i] - x[i];
    }
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
  if (!live) return;
  if (h < p.hq) {
    uint4* q = reinterpret_cast<uint4*>(p.q_out + (t * p.hq + h) * D);
    q[l] = pack8(a);
    q[L + l] = pack8(b);
    return;
  }
  const int64_t slot = p.slots[t];
  if (slot < 0) return;  // a padding row
  if (slot >= p.num_slots) {
    if (l == 0 && p.status) atomicExch(p.status, (int)kBadShape);
    return;
  }
  const int side = h >= p.hq + p.hkv;  // 0: K, 1: V
  const int kvh = h - p.hq - side * p.hkv;
  uint8_t* rec = p.cache + (slot / BS) * p.s_block + (int64_t)kvh * R::kBytes;
  const int off = (int)(slot % BS);
  uint32_t pair = 0;  // lane l < NG stores the l-th group's
  float s[NG], z[NG];
#pragma unroll
  for (int g = 0; g < NG; g++) {
    // a group holding a value that is not finite gets a NaN scale: all of it reads as NaN
    const __nv_bfloat16 sb = f2bf(__fadd_rn(__fmul_rn(mx[g] - mn[g], 1.0f / 15.0f), bad[g]));
    const __nv_bfloat16 zb = f2bf(mn[g]);
    s[g] = bf2f(sb);
    z[g] = bf2f(zb);
    if (g == l) pair = (uint32_t)__bfloat16_as_ushort(sb) | ((uint32_t)__bfloat16_as_ushort(zb) << 16);
  }
  const uint32_t wa = pack_word(a, s[0], z[0]), wb = pack_word(b, s[NG - 1], z[NG - 1]);
  uint8_t* row = rec + side * R::kV + off * R::kRow;
  if (D == 128) {
    *reinterpret_cast<uint2*>(row + 8 * l) = make_uint2(wa, wb);
  } else {
    *reinterpret_cast<uint32_t*>(row + 4 * l) = wa;
    *reinterpret_cast<uint32_t*>(row + R::kRow / 2 + 4 * l) = wb;
  }
  if (l < NG) *reinterpret_cast<uint32_t*>(rec + R::kKMeta + side * BS * R::kMeta + off * R::kMeta + 4 * l) = pair;
}

struct ReadParams {
  const uint8_t* cache;
  int64_t s_block, num_slots;
  const int64_t* slots;
  __nv_bfloat16 *k, *v;  // [n, hkv, D]
  int64_t items;         // n * hkv * 2
  int hkv;
  int* status;
};

// The values of rows, in bf16: the lanes of write_kernel, the other way round. (scale * code has 12
// significant bits, so the fused multiply-add rounds the exact value once.)
template <int D, int NG, int BS>
__global__ void __launch_bounds__(kThreads) read_kernel(ReadParams p) {
  using R = Rec<D, NG, BS>;
  constexpr int L = D / 16;
  pdl_wait();
  pdl_launch();
  const int64_t item = (int64_t)blockIdx.x * (kThreads / L) + threadIdx.x / L;
  if (item >= p.items) return;
  const int l = threadIdx.x % L;
  const int side = (int)(item & 1);
  const int64_t row = item >> 1;  // token * hkv + kv head
  const int64_t slot = p.slots[row / p.hkv];
  float a[8], b[8];
#pragma unroll
  for (int i = 0; i < 8; i++) a[i] = b[i] = 0.f;  // a negative slot reads as zeros
  if (slot >= p.num_slots) {
    if (l == 0 && p.status) atomicExch(p.status, (int)kBadShape);
  } else if (slot >= 0) {
    const uint8_t* rec = p.cache + (slot / BS) * p.s_block + (row % p.hkv) * R::kBytes;
    const int off = (int)(slot % BS);
    const uint8_t* codes = rec + side * R::kV + off * R::kRow;
    const uint32_t* pair = reinterpret_cast<const uint32_t*>(rec + R::kKMeta + side * BS * R::kMeta + off * R::kMeta);
    uint2 w;
    if (D == 128) {
      w = *reinterpret_cast<const uint2*>(codes + 8 * l);
    } else {
      w.x = *reinterpret_cast<const uint32_t*>(codes + 4 * l);
      w.y = *reinterpret_cast<const uint32_t*>(codes + R::kRow / 2 + 4 * l);
    }
    const uint32_t pa = pair[0], pb = pair[NG - 1];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int bit = 4 * (i / 2) + 16 * (i % 2);
      a[i] = fmaf((float)((w.x >> bit) & 15u), pair_scale(pa), pair_zero(pa));
      b[i] = fmaf((float)((w.y >> bit) & 15u), pair_scale(pb), pair_zero(pb));
    }
  }
  uint4* dst = reinterpret_cast<uint4*>((side ? p.v : p.k) + row * D);
  dst[l] = pack8(a);
  dst[L + l] = pack8(b);
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

// One CTA per (layer, pair, chunk of the page).
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
  p.items = a.T * (a.hq + 2 * a.c.hkv);
  p.status = a.status;
  if (p.items == 0) return cudaSuccess;
  return kv4::pick(a.c.d, a.c.groups, a.c.block_size, [&](auto d, auto ng, auto bs) {
    const int64_t grid = (p.items + kv4::kThreads / (d / 16) - 1) / (kv4::kThreads / (d / 16));
    if (grid > INT32_MAX) return cudaErrorInvalidValue;
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
  p.items = a.n * a.c.hkv * 2;
  p.status = a.status;
  if (p.items == 0) return cudaSuccess;
  return kv4::pick(a.c.d, a.c.groups, a.c.block_size, [&](auto d, auto ng, auto bs) {
    const int64_t grid = (p.items + kv4::kThreads / (d / 16) - 1) / (kv4::kThreads / (d / 16));
    if (grid > INT32_MAX) return cudaErrorInvalidValue;
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
