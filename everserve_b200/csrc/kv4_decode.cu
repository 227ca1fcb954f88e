// Decode attention over the paged cache held in 4 bits: one query row per sequence.
//
// With codes c (0..15) and a (scale, zero) per key t and group g of channels,
//   q . k_t   = sum_g scale_tg * (sum_{d in g} q_d c_td) + zero_tg * (sum_{d in g} q_d)
//   sum_t P_t v_t = sum_t (P_t scale_tg) c_td + sum_t P_t zero_tg         (channel d of group g),
// so the products run on the codes alone, and scales and zeros meet scores and probabilities. A code
// becomes an f16 operand by masking: the bits 0..3 (or 4..7) of a half are the subnormal number
// c * 2^-24 (c * 2^-20), which the tensor core takes exactly; the factor 16 between the two is in the
// query (K) and in the epilogue (V). That is 5 integer operations for 8 codes, where converting them
// would take 12 or more: at 4 bits a key the conversion, not the memory, would bound the kernel.
//
// S^T = K . q^T and O^T = V^T . P^T on mma.sync m16n8k16 (f16, fp32 sums): 16 keys by 8 query heads
// of one kv head, so a group of 8 heads fills the tile. A query row is scaled to at most 2^10 by a power
// of two, which keeps its bf16 values exact in f16 down to 2^-24. P_t scale_tg is rounded to f16 (11
// bits) under a power of two that follows the largest scale seen; scores, sums, the zeros' part and
// the output stay in fp32.
//
// A CTA takes one (sequence, kv head, split of the history), a warp every fourth run of 16 keys. The
// running maximum moves only when a score passes it by 2^6 (a vote per run; the first run sets it),
// so most runs shuffle nothing. The warps merge in shared memory, the splits in a second kernel.
// How a history is cut depends on its length alone: a sequence's result does not depend on the batch.
#include "api.h"
#include "common.cuh"
#include "kv4.cuh"
#include "launch.h"

namespace es {
namespace kv4 {

constexpr int kDecWarps = 4;
constexpr int kDecThreads = kDecWarps * 32;
constexpr float kLog2eF = 1.4426950408889634f;
constexpr float kSlack = 6.f;       // log2 of how far a score may pass the running maximum
constexpr float kPBits = 7.f;       // P * scale enters f16 as at most 2^(6 + 2 + 7) = 2^15

constexpr int kPart = 256;  // keys of a split

struct DecodeParams {
  const __nv_bfloat16* q;
  int64_t q_stride;
  const uint8_t* cache;
  int64_t s_block;
  int64_t num_blocks;
  const int* block_tables;
  int64_t bt_stride;
  int bt_cols;
  const int* ctx_lens;
  __nv_bfloat16* out;
  float* part_o;
  float* part_ml;
  int* status;
  int hq, hkv, head_tiles, max_splits;
  float scale_log2;
};

// Splits of a history of n keys.
__host__ __device__ __forceinline__ int splits_of(int n) { return n <= kPart ? 1 : (n + kPart - 1) / kPart; }

ES_DEVICE void mma_f16_16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// transpose of an 8 x 8 matrix of 16-bit values held two a lane
ES_DEVICE uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
ES_DEVICE uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// 2^e as a float, e in [-126, 127]
ES_DEVICE float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// floor(log2 x) of a positive normal number, clamped to [-90, 90]
ES_DEVICE int exponent(float x) { return min(90, max(-90, (int)((__float_as_uint(x) >> 23) & 255u) - 127)); }

// What a lane (gid = lane / 4, tig = lane % 4) holds of a run of 16 keys.
template <int D, int NG>
struct Run {
  uint32_t k[2][D / 32];        // K words of keys gid and gid + 8
  uint32_t v[4][D / 64];        // V words of keys 2 tig, 2 tig + 1, 2 tig + 8, 2 tig + 9
  uint32_t kp[2][NG], vp[2][NG];  // (scale, zero) pairs of keys gid and gid + 8
};

template <int D, int NG, int BS>
ES_DEVICE void load_run(Run<D, NG>& r, const uint8_t* rec, int sub, int gid, int tig) {
  using R = Rec<D, NG, BS>;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int row = sub * 16 + gid + 8 * i;
    const uint8_t* kp = rec + row * R::kRow + tig * (D / 8);
    if (D == 128) {
      const uint4 w = __ldcs(reinterpret_cast<const uint4*>(kp));
      r.k[i][0] = w.x, r.k[i][1] = w.y, r.k[i][D / 32 - 2] = w.z, r.k[i][D / 32 - 1] = w.w;
    } else {
      const uint2 w = __ldcs(reinterpret_cast<const uint2*>(kp));
      r.k[i][0] = w.x, r.k[i][1] = w.y;
    }
    const uint8_t* mp = rec + R::kKMeta + row * R::kMeta;
    if (NG == 2) {
      const uint2 a = __ldcs(reinterpret_cast<const uint2*>(mp));
      const uint2 b = __ldcs(reinterpret_cast<const uint2*>(mp + BS * R::kMeta));
      r.kp[i][0] = a.x, r.kp[i][NG - 1] = a.y, r.vp[i][0] = b.x, r.vp[i][NG - 1] = b.y;
    } else {
      r.kp[i][0] = __ldcs(reinterpret_cast<const uint32_t*>(mp));
      r.vp[i][0] = __ldcs(reinterpret_cast<const uint32_t*>(mp + BS * R::kMeta));
    }
  }
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int row = sub * 16 + 2 * tig + (j & 1) + 8 * (j >> 1);
    const uint8_t* vp = rec + R::kV + row * R::kRow + gid * (D / 16);
    if (D == 128) {
      const uint2 w = __ldcs(reinterpret_cast<const uint2*>(vp));
      r.v[j][0] = w.x, r.v[j][D / 64 - 1] = w.y;
    } else {
      r.v[j][0] = __ldcs(reinterpret_cast<const uint32_t*>(vp));
    }
  }
}

template <int D, int NG, int BS>
__global__ void __launch_bounds__(kDecThreads) decode_kernel(DecodeParams p) {
  using R = Rec<D, NG, BS>;
  constexpr int KW = D / 32;  // K words a lane holds of a key
  constexpr int VW = D / 64;  // V words
  constexpr int MT = D / 16;  // 16-channel tiles of the output
  __shared__ float red_o[kDecWarps][8][D + 4];
  __shared__ float red_ml[kDecWarps][8][2];

  const int split = blockIdx.x, b = blockIdx.y;
  const int kvh = blockIdx.z / p.head_tiles, ht = blockIdx.z % p.head_tiles;
  const int G = p.hq / p.hkv;
  const int heads = min(8, G - ht * 8);            // query heads of this tile
  const int head0 = kvh * G + ht * 8;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int gid = lane >> 2, tig = lane & 3;

  pdl_wait();
  pdl_launch();
  const int ctx = min(p.ctx_lens[b], p.bt_cols * BS);
  const int ns = min(p.max_splits, splits_of(ctx));
  if (ctx <= 0) {
    if (split == 0)  // an empty history: the output is zero
      for (int i = tid; i < heads * D; i += kDecThreads) p.out[((int64_t)b * p.hq + head0) * D + i] = f2bf(0.f);
    return;
  }
  const int plen = ((ctx + ns - 1) / ns + BS - 1) / BS * BS;  // equal splits, to a block
  const int s0 = split * plen, s1 = min(ctx, s0 + plen);
  if (split >= ns) return;

  // the query: B fragments of S^T (head gid; k = the channels of this lane's K words), scaled to <= 2^10
  uint32_t qb[KW][4];
  float xs[2], sq[2][NG];  // of heads 2 tig and 2 tig + 1: the scores' factor, and scale * sum q by group
  {
    float qv[KW][8];
    float qmax = 0.f, sum[NG];
#pragma unroll
    for (int g = 0; g < NG; g++) sum[g] = 0.f;
    const __nv_bfloat16* qr = p.q + (int64_t)b * p.q_stride + (int64_t)(head0 + min(gid, heads - 1)) * D;
#pragma unroll
    for (int w = 0; w < KW; w++) {
      const int pos = tig * KW + w;  // stored word of the row, and the channels it holds
      const int nat = D == 128 ? (pos >> 1) + 8 * (pos & 1) : pos;
      unpack8(*reinterpret_cast<const uint4*>(qr + 8 * nat), qv[w]);
#pragma unroll
      for (int i = 0; i < 8; i++) {
        if (gid >= heads) qv[w][i] = 0.f;
        qmax = fmaxf(qmax, fabsf(qv[w][i]));
        sum[NG == 2 ? (w & 1) : 0] += qv[w][i];
      }
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      qmax = fmaxf(qmax, __shfl_xor_sync(0xffffffffu, qmax, o));
#pragma unroll
      for (int g = 0; g < NG; g++) sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], o);
    }
    const int e = exponent(qmax);
    const float f = pow2i(9 - e), f16th = f * 0.0625f;
#pragma unroll
    for (int w = 0; w < KW; w++) {
      qb[w][0] = pack_f16x2(qv[w][0] * f, qv[w][1] * f);
      qb[w][1] = pack_f16x2(qv[w][2] * f16th, qv[w][3] * f16th);
      qb[w][2] = pack_f16x2(qv[w][4] * f, qv[w][5] * f);
      qb[w][3] = pack_f16x2(qv[w][6] * f16th, qv[w][7] * f16th);
    }
    const float x = p.scale_log2 * pow2i(24 - 9 + e);
#pragma unroll
    for (int i = 0; i < 2; i++) {
      xs[i] = __shfl_sync(0xffffffffu, x, (2 * tig + i) * 4);
#pragma unroll
      for (int g = 0; g < NG; g++) sq[i][g] = p.scale_log2 * __shfl_sync(0xffffffffu, sum[g], (2 * tig + i) * 4);
    }
  }

  float o[MT][4];
#pragma unroll
  for (int i = 0; i < MT; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // l, zs: this lane's keys alone
  float zs[2][NG];
#pragma unroll
  for (int g = 0; g < NG; g++) zs[0][g] = zs[1][g] = 0.f;
  int ve = -90;                // V scales enter f16 times 2^(kPBits - ve)
  float vlim = 0.f;            // and are at most this

  const int* bt = p.block_tables + (int64_t)b * p.bt_stride;
  const uint8_t* head_base = p.cache + (int64_t)kvh * R::kBytes;
  auto record = [&](int key) -> const uint8_t* {
    int64_t blk = bt[key / BS];
    if (blk < 0 || blk >= p.num_blocks) {  // not a block of this cache: reported, block 0 read instead
      if (lane == 0 && p.status) atomicExch(p.status, (int)kBadShape);
      blk = 0;
    }
    return head_base + blk * p.s_block;
  };

  Run<D, NG> nxt;
  int key0 = s0 + warp * 16;
  if (key0 < s1) load_run<D, NG, BS>(nxt, record(key0), (key0 % BS) / 16, gid, tig);
  for (; key0 < s1; key0 += kDecWarps * 16) {
    Run<D, NG> r = nxt;
    const int ahead = key0 + kDecWarps * 16;
    if (ahead < s1) load_run<D, NG, BS>(nxt, record(ahead), (ahead % BS) / 16, gid, tig);

    // S^T = K . q^T on the codes
    float acc[NG][4];
#pragma unroll
    for (int g = 0; g < NG; g++) acc[g][0] = acc[g][1] = acc[g][2] = acc[g][3] = 0.f;
#pragma unroll
    for (int w = 0; w < KW; w++) {
      float* d = acc[NG == 2 ? (w & 1) : 0];
      uint32_t wa = r.k[0][w], wb = r.k[1][w];
      const uint32_t a0[4] = {wa & 0x000F000Fu, wb & 0x000F000Fu, wa & 0x00F000F0u, wb & 0x00F000F0u};
      mma_f16_16816(d, a0, qb[w][0], qb[w][1]);
      wa >>= 8, wb >>= 8;
      const uint32_t a1[4] = {wa & 0x000F000Fu, wb & 0x000F000Fu, wa & 0x00F000F0u, wb & 0x00F000F0u};
      mma_f16_16816(d, a1, qb[w][2], qb[w][3]);
    }
    // scores in the log2 domain: x[key i][head j]; keys past the history's end count for nothing, and
    // whatever their slots hold (NaN too) is taken out of the products
    float x[2][2], sv[2][NG], zv[2][NG];
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const bool in = key0 + gid + 8 * i < s1;
      float t0 = 0.f, t1 = 0.f, u0 = 0.f, u1 = 0.f;
#pragma unroll
      for (int g = 0; g < NG; g++) {
        const float s = pair_scale(r.kp[i][g]), z = pair_zero(r.kp[i][g]);
        t0 = fmaf(s, acc[g][2 * i], t0);
        t1 = fmaf(s, acc[g][2 * i + 1], t1);
        u0 = fmaf(z, sq[0][g], u0);
        u1 = fmaf(z, sq[1][g], u1);
        sv[i][g] = in ? pair_scale(r.vp[i][g]) : 0.f;
        zv[i][g] = in ? pair_zero(r.vp[i][g]) : 0.f;
      }
      x[i][0] = in ? fmaf(t0, xs[0], u0) : -INFINITY;
      x[i][1] = in ? fmaf(t1, xs[1], u1) : -INFINITY;
    }
    float smax = fmaxf(sv[0][0], sv[1][0]);
    if (NG == 2) smax = fmaxf(smax, fmaxf(sv[0][NG - 1], sv[1][NG - 1]));
    const bool up = fmaxf(x[0][0], x[1][0]) > m[0] + kSlack || fmaxf(x[0][1], x[1][1]) > m[1] + kSlack || smax > vlim;
    if (__any_sync(0xffffffffu, up)) {
      float mt[2] = {fmaxf(x[0][0], x[1][0]), fmaxf(x[0][1], x[1][1])};
#pragma unroll
      for (int s = 4; s < 32; s <<= 1) {
        mt[0] = fmaxf(mt[0], __shfl_xor_sync(0xffffffffu, mt[0], s));
        mt[1] = fmaxf(mt[1], __shfl_xor_sync(0xffffffffu, mt[1], s));
        smax = fmaxf(smax, __shfl_xor_sync(0xffffffffu, smax, s));
      }
      float c[2];
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const float mn = fmaxf(m[j], mt[j]);
        c[j] = m[j] == -INFINITY ? 0.f : ex2(m[j] - mn);
        m[j] = mn;
        l[j] *= c[j];
#pragma unroll
        for (int g = 0; g < NG; g++) zs[j][g] *= c[j];
      }
      if (smax > vlim) {
        const int e = exponent(smax) + 1;
        const float f = pow2i(max(-126, ve - e));
        c[0] *= f, c[1] *= f;
        ve = e;
        vlim = pow2i(e + 2);
      }
#pragma unroll
      for (int i = 0; i < MT; i++) o[i][0] *= c[0], o[i][1] *= c[1], o[i][2] *= c[0], o[i][3] *= c[1];
    }
    // P, its sums, and P * scale as the B fragments of O^T (keys along k): transposed in registers
    float pr[2][2];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int j = 0; j < 2; j++) {
        pr[i][j] = ex2(x[i][j] - m[j]);
        l[j] += pr[i][j];
#pragma unroll
        for (int g = 0; g < NG; g++) zs[j][g] = fmaf(pr[i][j], zv[i][g], zs[j][g]);
      }
    uint32_t pb[NG][2];
    const float vf = pow2i((int)kPBits - ve);
#pragma unroll
    for (int g = 0; g < NG; g++)
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const float s = sv[i][g] * vf;
        pb[g][i] = transpose8(pack_f16x2(pr[i][0] * s, pr[i][1] * s));
      }
    // O^T += V^T . P^T on the codes: rows gid and gid + 8 of tile (w, j) are channels 2 j and 2 j + 1 of
    // word w, the keys of a register's halves 2 tig and 2 tig + 1
#pragma unroll
    for (int w = 0; w < VW; w++) {
      const int g = NG == 2 ? w : 0;
      uint32_t e0 = __byte_perm(r.v[0][w], r.v[1][w], 0x5410), d0 = __byte_perm(r.v[0][w], r.v[1][w], 0x7632);
      uint32_t e1 = __byte_perm(r.v[2][w], r.v[3][w], 0x5410), d1 = __byte_perm(r.v[2][w], r.v[3][w], 0x7632);
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const uint32_t a0[4] = {e0 & 0x000F000Fu, d0 & 0x000F000Fu, e1 & 0x000F000Fu, d1 & 0x000F000Fu};
        mma_f16_16816(o[w * 4 + 2 * h], a0, pb[g][0], pb[g][1]);
        const uint32_t a1[4] = {e0 & 0x00F000F0u, d0 & 0x00F000F0u, e1 & 0x00F000F0u, d1 & 0x00F000F0u};
        mma_f16_16816(o[w * 4 + 2 * h + 1], a1, pb[g][0], pb[g][1]);
        e0 >>= 8, d0 >>= 8, e1 >>= 8, d1 >>= 8;
      }
    }
  }

  // the lanes' sums, the codes' factor, the zeros' part; then the warps
#pragma unroll
  for (int s = 4; s < 32; s <<= 1) {
#pragma unroll
    for (int j = 0; j < 2; j++) {
      l[j] += __shfl_xor_sync(0xffffffffu, l[j], s);
#pragma unroll
      for (int g = 0; g < NG; g++) zs[j][g] += __shfl_xor_sync(0xffffffffu, zs[j][g], s);
    }
  }
  const float of = pow2i(24 - (int)kPBits + ve);
#pragma unroll
  for (int w = 0; w < VW; w++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float f = (j & 1) ? of * 0.0625f : of;
      const int g = NG == 2 ? w : 0;
      const int ch = (w * 8 + gid) * 8 + 2 * j;
      const float* a = o[w * 4 + j];
      *reinterpret_cast<float2*>(&red_o[warp][2 * tig][ch]) = make_float2(fmaf(a[0], f, zs[0][g]), fmaf(a[2], f, zs[0][g]));
      *reinterpret_cast<float2*>(&red_o[warp][2 * tig + 1][ch]) = make_float2(fmaf(a[1], f, zs[1][g]), fmaf(a[3], f, zs[1][g]));
    }
  if (gid == 0) {
#pragma unroll
    for (int j = 0; j < 2; j++) red_ml[warp][2 * tig + j][0] = m[j], red_ml[warp][2 * tig + j][1] = l[j];
  }
  __syncthreads();
  for (int i = tid; i < heads * (D / 8); i += kDecThreads) {
    const int h = i / (D / 8), c8 = i % (D / 8) * 8;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < kDecWarps; w++) mm = fmaxf(mm, red_ml[w][h][0]);
    float ll = 0.f, acc[8];
#pragma unroll
    for (int e = 0; e < 8; e++) acc[e] = 0.f;
#pragma unroll
    for (int w = 0; w < kDecWarps; w++) {
      if (s0 + w * 16 >= s1) continue;  // a warp with no key
      const float mw = red_ml[w][h][0];
      const float f = mw == mm ? 1.f : ex2(mw - mm);
      ll = fmaf(red_ml[w][h][1], f, ll);
#pragma unroll
      for (int e = 0; e < 8; e++) acc[e] = fmaf(red_o[w][h][c8 + e], f, acc[e]);
    }
    const int64_t row = (int64_t)b * p.hq + head0 + h;
    if (ns == 1) {
      const float inv = 1.f / ll;
#pragma unroll
      for (int e = 0; e < 8; e++) acc[e] *= inv;
      *reinterpret_cast<uint4*>(p.out + row * D + c8) = pack8(acc);
    } else {
      float* po = p.part_o + (row * p.max_splits + split) * D + c8;
      *reinterpret_cast<float4*>(po) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      *reinterpret_cast<float4*>(po + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
      if (c8 == 0) {
        float* ml = p.part_ml + (row * p.max_splits + split) * 2;
        ml[0] = mm, ml[1] = ll;
      }
    }
  }
}

// out = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i over a row's splits, in an order of its own: warp w
// takes every fourth split, then the warps add in order. One CTA per (sequence, query head).
template <int D>
__global__ void __launch_bounds__(128) merge_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml,
                                                    const int* __restrict__ ctx_lens, __nv_bfloat16* __restrict__ out,
                                                    int hq, int max_splits, int max_keys) {
  constexpr int E = D / 32;
  __shared__ float so[4][D], sl[4];
  __shared__ float smx[4];
  pdl_wait();
  pdl_launch();
  const int ns = min(max_splits, splits_of(min(ctx_lens[blockIdx.y], max_keys)));
  if (ns <= 1) return;  // written by the split itself
  const int64_t row = (int64_t)blockIdx.y * hq + blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float* ml = part_ml + row * max_splits * 2;
  float mx = -INFINITY;
  for (int i = threadIdx.x; i < ns; i += 128) mx = fmaxf(mx, ml[2 * i]);
  mx = warp_max(mx);
  if (lane == 0) smx[warp] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(smx[0], smx[1]), fmaxf(smx[2], smx[3]));
  float acc[E], l = 0.f;
#pragma unroll
  for (int e = 0; e < E; e++) acc[e] = 0.f;
  for (int i = warp; i < ns; i += 4) {
    const float mi = ml[2 * i];
    const float f = mi == mx ? 1.f : ex2(mi - mx);
    l = fmaf(ml[2 * i + 1], f, l);
    const float* po = part_o + (row * max_splits + i) * D;
#pragma unroll
    for (int e = 0; e < E; e++) acc[e] = fmaf(po[e * 32 + lane], f, acc[e]);
  }
#pragma unroll
  for (int e = 0; e < E; e++) so[warp][e * 32 + lane] = acc[e];
  if (lane == 0) sl[warp] = l;
  __syncthreads();
  if (threadIdx.x < D) {
    const int c = threadIdx.x;
    const float lt = ((sl[0] + sl[1]) + sl[2]) + sl[3];
    const float t = ((so[0][c] + so[1][c]) + so[2][c]) + so[3][c];
    out[row * D + c] = f2bf(t / lt);
  }
}

template <int D, int NG, int BS>
cudaError_t launch_decode(const DecodeParams& p, int B, cudaStream_t stream) {
  cudaError_t e = launch_ex(decode_kernel<D, NG, BS>, dim3(p.max_splits, B, p.hkv * p.head_tiles), dim3(kDecThreads), 0,
                            stream, 0, p);
  if (e != cudaSuccess || p.max_splits == 1) return e;
  return launch_ex(merge_kernel<D>, dim3(p.hq, B), dim3(128), 0, stream, 0, (const float*)p.part_o,
                   (const float*)p.part_ml, p.ctx_lens, p.out, p.hq, p.max_splits, p.bt_cols * BS);
}

}  // namespace kv4

int64_t kv4_max_splits(int64_t max_len) { return kv4::splits_of((int)(max_len < INT32_MAX ? max_len : INT32_MAX)); }

cudaError_t launch_kv4_decode(const Kv4DecodeArgs& a, cudaStream_t stream) {
  if (a.B == 0) return cudaSuccess;
  if (a.c.hkv <= 0 || a.hq % a.c.hkv != 0 || a.B > 65535 || a.max_splits < 1) return cudaErrorInvalidValue;
  if (a.bt_cols * a.c.block_size > INT32_MAX) return cudaErrorInvalidValue;
  kv4::DecodeParams p{};
  p.q = static_cast<const __nv_bfloat16*>(a.q);
  p.q_stride = a.q_stride;
  p.cache = static_cast<const uint8_t*>(a.c.base);
  p.s_block = a.c.s_block;
  p.num_blocks = a.c.num_blocks;
  p.block_tables = a.block_tables;
  p.bt_stride = a.bt_stride;
  p.bt_cols = (int)a.bt_cols;
  p.ctx_lens = a.ctx_lens;
  p.out = static_cast<__nv_bfloat16*>(a.out);
  p.part_o = a.part_o;
  p.part_ml = a.part_ml;
  p.status = a.status;
  p.hq = a.hq;
  p.hkv = a.c.hkv;
  p.head_tiles = (a.hq / a.c.hkv + 7) / 8;
  p.max_splits = a.max_splits;
  p.scale_log2 = a.scale * kv4::kLog2eF;
  if ((int64_t)p.hkv * p.head_tiles > 65535 || p.hq > 65535) return cudaErrorInvalidValue;
  return kv4::pick(a.c.d, a.c.groups, a.c.block_size, [&](auto d, auto ng, auto bs) {
    return kv4::launch_decode<d, ng, bs>(p, a.B, stream);
  });
}

}  // namespace es
